// Checked wrappers over linear attention with one decay per head (include/ext/glm53f_lin.h), in the manner of kernel.hpp:
// every launch first checks on the host that each buffer holds the geometry it is given and that the states written overlap
// neither each other nor one that another request reads, then makes one call into the C ABI. (That `out` lies apart from q, k
// and v is the caller's, as there.) check() never touches the GPU. The batch metadata is kernel.hpp's BatchMeta
// (its conv offsets are not used), so that one set of requests serves layers of both kinds. Header only.
#ifndef GLM53F_LIN_HOST_LIN_HPP
#define GLM53F_LIN_HOST_LIN_HPP

#include "ext/glm53f_lin.h"
#include "kernel.hpp"

namespace glm53f_lin {

using glm53f_kda::BatchMeta;
using glm53f_kda::Buf;
using glm53f_kda::DeviceBuffer;
using glm53f_kda::Error;
using glm53f_kda::launched;
using glm53f_kda::Request;
using glm53f_kda::RowView;
using glm53f_kda::state_bytes;
using glm53f_kda::StateOut;
using glm53f_kda::StateType;
using glm53f_kda::Stream;
using glm53f_kda::to_i32;

/// The heads of a layer: `heads` value heads of value_dim, qk_heads heads of q and k of key_dim, 64 or 128 each.
struct Shape {
    size_t heads = 0, qk_heads = 0, key_dim = 128, value_dim = 128;
    size_t state_len() const { return heads * value_dim * key_dim; }
    size_t qk_width() const { return qk_heads * key_dim; }
    size_t v_width() const { return heads * value_dim; }
    Error check() const {
        if (heads < 1 || heads > 65535 || qk_heads < 1 || heads % qk_heads != 0 || (key_dim != 64 && key_dim != 128) ||
            (value_dim != 64 && value_dim != 128))
            return Error::invalid("heads " + std::to_string(heads) + " / " + std::to_string(qk_heads) + " of " +
                                  std::to_string(key_dim) + " keys and " + std::to_string(value_dim) + " values");
        return Error::ok();
    }
};

/// Device workspace of the chunked form for any call of up to `batch` requests of up to `max_rows` rows (empty where none
/// of them needs one). A smaller batch may need more than a larger one, hence the bound and not the larger one's need.
struct Workspace {
    DeviceBuffer storage;

    static int64_t bytes_for(const Shape& s, size_t batch, size_t max_rows) {
        if (s.heads > 65535 || batch > 65535 || max_rows > (size_t)std::numeric_limits<int32_t>::max()) return -1;
        return glm53f_lin_prefill_workspace_bytes((int32_t)s.heads, (int32_t)s.key_dim, (int32_t)s.value_dim, (int32_t)batch,
                                                  (int32_t)max_rows);
    }
    static size_t bound(const Shape& s, size_t batch, size_t max_rows) {
        const size_t most = (max_rows + 255) / 256;
        return most < 2 ? 0 : std::min<size_t>(1535, s.heads * batch * most) * s.key_dim * s.value_dim * 4;
    }
    static Error create(const Shape& s, size_t batch, size_t max_rows, Workspace* out) {
        KDA_TRY(s.check());
        if (bytes_for(s, batch, max_rows) < 0)
            return Error::invalid("workspace for " + std::to_string(batch) + " requests of " + std::to_string(max_rows) + " rows");
        return DeviceBuffer::alloc(bound(s, batch, max_rows), &out->storage);
    }
};

/// One layer, a batch of requests: recurrent (launch_chain: decode steps, short windows) or chunked (launch_prefill:
/// prompts, verify windows).
struct Attention {
    Shape shape;
    RowView q, k, v;
    Buf log_decay;   // f32 [heads], at most 0
    float scale = 1.0f;
    Buf state;
    StateOut state_out;
    RowView out;

    Error check(const BatchMeta& meta, StateType st, void** state_out_ptr) const {
        KDA_TRY(shape.check());
        int32_t batch;
        KDA_TRY(meta.batch(&batch));
        if (batch > 65535) return Error::invalid("more than 65535 requests");
        const size_t total = meta.total_rows(), es = state_bytes(st);
        KDA_TRY(q.check("q", 2, 0, total, 0, (int64_t)shape.qk_width()));
        KDA_TRY(k.check("k", 2, 0, total, 0, (int64_t)shape.qk_width()));
        KDA_TRY(v.check("v", 2, 0, total, 0, (int64_t)shape.v_width()));
        KDA_TRY(out.check("out", 2, 0, total, 0, (int64_t)shape.v_width()));
        if (q.stride < shape.qk_width() || k.stride < shape.qk_width() || v.stride < shape.v_width() || out.stride < shape.v_width())
            return Error::invalid("rows overlap");
        if (log_decay.bytes < shape.heads * 4) return Error::invalid("one decay per head");
        auto off = [](const Request& r) { return r.state_offset; };
        for (const Request& r : meta.requests())
            if (r.state_offset % 8) return Error::invalid("state offsets are multiples of 8 elements");
        // (windows that only read their states may stand behind the same one)
        KDA_TRY(meta.check_regions("state", state, es, 0, shape.state_len(), state_out.kind != StateOut::Skip, off));
        *state_out_ptr = nullptr;
        if (state_out.kind == StateOut::InPlace) {
            *state_out_ptr = state.p;
        } else if (state_out.kind == StateOut::To) {
            if (state_out.offset != 0) return Error::invalid("a batch writes its states at the requests' offsets");
            KDA_TRY(meta.check_regions("state_out", state_out.buf, es, 0, shape.state_len(), true, off));
            if (glm53f_kda::same(state_out.buf, state)) return Error::invalid("state_out is the state buffer: use InPlace");
            KDA_TRY(check_apart(meta, es));
            *state_out_ptr = state_out.buf.p;
        }
        return Error::ok();
    }

    Error launch_chain(const BatchMeta& meta, StateType st, const Stream& stream) const {
        void* so = nullptr;
        KDA_TRY(check(meta, st, &so));
        if (!meta.on_device()) return Error::invalid("batch metadata has no device arrays");
        int32_t batch;
        KDA_TRY(meta.batch(&batch));
        const int code = st == StateType::F32
            ? glm53f_lin_chain_batch(h(), qk(), dk(), dv(), batch, meta.cu_rows(), row(q), st_of(q), row(k), st_of(k), row(v),
                                     st_of(v), log_decay.ptr<float>(), scale, state.ptr<float>(), static_cast<float*>(so),
                                     meta.state_off(), row(out), st_of(out), stream.raw())
            : glm53f_lin_chain_batch_bf16state(h(), qk(), dk(), dv(), batch, meta.cu_rows(), row(q), st_of(q), row(k), st_of(k),
                                               row(v), st_of(v), log_decay.ptr<float>(), scale, state.ptr<uint16_t>(),
                                               static_cast<uint16_t*>(so), meta.state_off(), row(out), st_of(out), stream.raw());
        return launched(code, "glm53f_lin_chain_batch");
    }

    /// `ws` NULL where the sizes need none.
    Error launch_prefill(const BatchMeta& meta, StateType st, const Workspace* ws, const Stream& stream) const {
        void* so = nullptr;
        KDA_TRY(check(meta, st, &so));
        int32_t batch, most;
        KDA_TRY(meta.batch(&batch));
        KDA_TRY(to_i32(meta.max_rows(), "rows", &most));
        const int64_t need = Workspace::bytes_for(shape, (size_t)batch, meta.max_rows());
        const int64_t have = ws != nullptr ? (int64_t)ws->storage.bytes() : 0;
        if (need > have) return Error::invalid("the chunked form needs " + std::to_string(need) + " bytes of workspace, not " + std::to_string(have));
        if (!meta.on_device()) return Error::invalid("batch metadata has no device arrays");
        void* w = have > 0 ? ws->storage.ptr<unsigned char>() : nullptr;
        const int code = st == StateType::F32
            ? glm53f_lin_prefill_batch(h(), qk(), dk(), dv(), batch, meta.cu_rows(), most, row(q), st_of(q), row(k), st_of(k), row(v),
                                       st_of(v), log_decay.ptr<float>(), scale, state.ptr<float>(), static_cast<float*>(so),
                                       meta.state_off(), row(out), st_of(out), w, have, stream.raw())
            : glm53f_lin_prefill_batch_bf16state(h(), qk(), dk(), dv(), batch, meta.cu_rows(), most, row(q), st_of(q), row(k),
                                                 st_of(k), row(v), st_of(v), log_decay.ptr<float>(), scale, state.ptr<uint16_t>(),
                                                 static_cast<uint16_t*>(so), meta.state_off(), row(out), st_of(out), w, have,
                                                 stream.raw());
        return launched(code, "glm53f_lin_prefill_batch");
    }

  private:
    /// The states that go to state_out lie apart from every state that is read, whatever the two buffers share.
    Error check_apart(const BatchMeta& meta, size_t es) const {
        const uintptr_t bytes = shape.state_len() * es;
        std::vector<uintptr_t> read;
        for (const Request& r : meta.requests()) read.push_back((uintptr_t)state.p + r.state_offset * es);
        std::sort(read.begin(), read.end());
        for (const Request& r : meta.requests()) {
            const uintptr_t at = (uintptr_t)state_out.buf.p + r.state_offset * es;
            const auto next = std::upper_bound(read.begin(), read.end(), at);
            if ((next != read.begin() && at - next[-1] < bytes) || (next != read.end() && *next - at < bytes))
                return Error::invalid("state_out overlaps a state that is read");
        }
        return Error::ok();
    }
    int32_t h() const { return (int32_t)shape.heads; }
    int32_t qk() const { return (int32_t)shape.qk_heads; }
    int32_t dk() const { return (int32_t)shape.key_dim; }
    int32_t dv() const { return (int32_t)shape.value_dim; }
    static uint16_t* row(const RowView& r) { return r.buf.ptr<uint16_t>(r.offset); }
    static int64_t st_of(const RowView& r) { return (int64_t)r.stride; }
};

/// The commit of a verify round over all layers, in place: request r keeps keep[r] rows (`keep` NULL: the metadata's, else
/// device int32 per request, for instance glm53f_spec::Verification's). Layer l's rows lie l * row_layer_stride further, its
/// states l * state_layer_stride; log_decay f32 [layers][heads].
inline Error advance_batch(const Shape& shape, size_t layers, const BatchMeta& meta, const int32_t* keep, const RowView& k,
                           const RowView& v, size_t row_layer_stride, Buf log_decay, Buf state, size_t state_layer_stride,
                           StateType st, const Stream& stream, bool dry_run = false) {
    KDA_TRY(shape.check());
    int32_t batch, l32;
    KDA_TRY(meta.batch(&batch));
    KDA_TRY(to_i32(layers, "layers", &l32));
    if (layers < 1 || layers * shape.heads > 0x3fffffff || batch > 65535) return Error::invalid("advance_batch: no layers, or too many");
    if (k.stride < shape.qk_width() || v.stride < shape.v_width()) return Error::invalid("rows overlap");
    for (size_t l : {(size_t)0, layers - 1}) {
        KDA_TRY(RowView(k.buf, k.offset + l * row_layer_stride, k.stride).check("k", 2, 0, meta.total_rows(), 0, (int64_t)shape.qk_width()));
        KDA_TRY(RowView(v.buf, v.offset + l * row_layer_stride, v.stride).check("v", 2, 0, meta.total_rows(), 0, (int64_t)shape.v_width()));
    }
    if (log_decay.bytes < layers * shape.heads * 4) return Error::invalid("one decay per layer and head");
    size_t max_off = 0;
    for (const Request& r : meta.requests()) {
        if (r.state_offset % 8) return Error::invalid("state offsets are multiples of 8 elements");
        max_off = std::max(max_off, r.state_offset);
    }
    if (layers > 1 && (state_layer_stride % 8 || state_layer_stride < max_off + shape.state_len()))
        return Error::invalid("advance_batch: layers' states overlap");
    KDA_TRY(meta.check_regions("state", state, state_bytes(st), (layers - 1) * state_layer_stride, shape.state_len(), true,
                               [](const Request& r) { return r.state_offset; }));
    if (dry_run) return Error::ok();
    if (!meta.on_device()) return Error::invalid("batch metadata has no device arrays");
    const int32_t h = (int32_t)shape.heads, qk = (int32_t)shape.qk_heads, dk = (int32_t)shape.key_dim, dv = (int32_t)shape.value_dim;
    const int64_t row_l = (int64_t)row_layer_stride, state_l = (int64_t)state_layer_stride;
    const int32_t* kept = keep != nullptr ? keep : meta.keep_dev();
    const uint16_t *kp = k.buf.ptr<uint16_t>(k.offset), *vp = v.buf.ptr<uint16_t>(v.offset);
    const int code = st == StateType::F32
        ? glm53f_lin_advance_batch(h, qk, dk, dv, l32, batch, meta.cu_rows(), kept, kp, (int64_t)k.stride, row_l, vp,
                                   (int64_t)v.stride, row_l, log_decay.ptr<float>(), state.ptr<float>(), state.ptr<float>(),
                                   state_l, meta.state_off(), stream.raw())
        : glm53f_lin_advance_batch_bf16state(h, qk, dk, dv, l32, batch, meta.cu_rows(), kept, kp, (int64_t)k.stride, row_l, vp,
                                             (int64_t)v.stride, row_l, log_decay.ptr<float>(), state.ptr<uint16_t>(),
                                             state.ptr<uint16_t>(), state_l, meta.state_off(), stream.raw());
    return launched(code, "glm53f_lin_advance_batch");
}

}  // namespace glm53f_lin

#endif  // GLM53F_LIN_HOST_LIN_HPP
