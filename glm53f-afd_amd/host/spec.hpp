// Checked wrappers over the two ends of a speculative round (include/ext/glm53f_spec.h), in the manner of kernel.hpp: the
// extents are checked on the host, then one call into the C ABI; check() never touches the GPU. The windows are a BatchMeta's
// requests. Header only.
#ifndef GLM53F_SPEC_HOST_SPEC_HPP
#define GLM53F_SPEC_HOST_SPEC_HPP

#include "ext/glm53f_spec.h"
#include "kernel.hpp"

namespace glm53f_spec {

using glm53f_kda::BatchMeta;
using glm53f_kda::Buf;
using glm53f_kda::DeviceBuffer;
using glm53f_kda::Error;
using glm53f_kda::launched;
using glm53f_kda::RowView;
using glm53f_kda::Stream;
using glm53f_kda::to_i32;

/// Device workspace of both for up to `rows` rows and requests of `vocab` entries.
struct Workspace {
    DeviceBuffer storage;
    static int64_t bytes_for(size_t rows, size_t batch, size_t vocab) {
        if (rows > 65535 || batch > 65535 || vocab > (size_t(1) << 30)) return -1;
        const int64_t p = glm53f_spec_probs_workspace_bytes((int32_t)rows, (int32_t)vocab);
        const int64_t a = glm53f_spec_accept_workspace_bytes((int32_t)batch, (int32_t)vocab);
        return p < 0 || a < 0 ? -1 : std::max(p, a);
    }
    static Error create(size_t rows, size_t batch, size_t vocab, Workspace* out) {
        const int64_t bytes = bytes_for(rows, batch, vocab);
        if (bytes < 0) return Error::invalid("workspace for " + std::to_string(rows) + " rows of " + std::to_string(vocab));
        return DeviceBuffer::alloc((size_t)bytes, &out->storage);
    }
};

/// probs = softmax(logits / temperature), rows of `vocab` entries.
struct Probabilities {
    size_t rows = 0, vocab = 0;
    RowView logits;          // bf16, or f32 with logits_f32
    bool logits_f32 = false;
    Buf temperature;         // f32 [rows]; empty: 1
    RowView probs;           // f32; may be the logits' own rows where those are f32

    Error check(const Workspace& ws) const {
        if (vocab < 1 || vocab > (size_t(1) << 30) || rows > 65535) return Error::invalid("rows or vocabulary out of range");
        KDA_TRY(logits.check("logits", logits_f32 ? 4 : 2, 0, rows, 0, (int64_t)vocab));
        KDA_TRY(probs.check("probs", 4, 0, rows, 0, (int64_t)vocab));
        if (logits.stride < vocab || probs.stride < vocab) return Error::invalid("rows overlap");
        if (temperature.p != nullptr && temperature.bytes < rows * 4) return Error::invalid("one temperature per row");
        if (Workspace::bytes_for(rows, 0, vocab) > (int64_t)ws.storage.bytes()) return Error::invalid("workspace too small");
        return Error::ok();
    }
    Error launch(const Workspace& ws, const Stream& stream) const {
        KDA_TRY(check(ws));
        const void* x = logits_f32 ? (const void*)logits.buf.ptr<float>(logits.offset) : (const void*)logits.buf.ptr<uint16_t>(logits.offset);
        return launched(glm53f_spec_probs((int32_t)rows, (int32_t)vocab, x, logits_f32 ? 1 : 0, (int64_t)logits.stride,
                                          temperature.ptr<float>(), probs.buf.ptr<float>(probs.offset), (int64_t)probs.stride,
                                          ws.storage.ptr<unsigned char>(), (int64_t)ws.storage.bytes(), stream.raw()),
                        "glm53f_spec_probs");
    }
};

/// The verification of the drafted tokens of every request's window: keep and next per request, on the device.
struct Verification {
    size_t vocab = 0;
    Buf tokens;              // int32 [all rows]
    RowView target, draft;   // f32 rows; draft without a buffer: certain drafts
    Buf uniform;             // f32 [all rows]
    Buf keep, next;          // int32 [requests]

    Error check(const BatchMeta& meta, const Workspace& ws) const {
        int32_t batch;
        KDA_TRY(meta.batch(&batch));
        if (vocab < 1 || vocab > (size_t(1) << 30) || batch > 65535) return Error::invalid("requests or vocabulary out of range");
        const size_t total = meta.total_rows();
        if (tokens.bytes < total * 4 || uniform.bytes < total * 4) return Error::invalid("one token and one random number per row");
        if (keep.bytes < (size_t)batch * 4 || next.bytes < (size_t)batch * 4) return Error::invalid("one result per request");
        KDA_TRY(target.check("target", 4, 0, total, 0, (int64_t)vocab));
        if (target.stride < vocab) return Error::invalid("rows overlap");
        if (draft.buf.p != nullptr) {
            KDA_TRY(draft.check("draft", 4, 0, total, 0, (int64_t)vocab));
            if (draft.stride < vocab) return Error::invalid("rows overlap");
        }
        if (Workspace::bytes_for(0, (size_t)batch, vocab) > (int64_t)ws.storage.bytes()) return Error::invalid("workspace too small");
        return Error::ok();
    }
    Error launch(const BatchMeta& meta, const Workspace& ws, const Stream& stream) const {
        KDA_TRY(check(meta, ws));
        if (!meta.on_device()) return Error::invalid("batch metadata has no device arrays");
        int32_t batch;
        KDA_TRY(meta.batch(&batch));
        const float* q = draft.buf.p != nullptr ? draft.buf.ptr<float>(draft.offset) : nullptr;
        return launched(glm53f_spec_accept(batch, (int32_t)vocab, meta.cu_rows(), tokens.ptr<int32_t>(),
                                           target.buf.ptr<float>(target.offset), (int64_t)target.stride, q, (int64_t)draft.stride,
                                           uniform.ptr<float>(), keep.ptr<int32_t>(), next.ptr<int32_t>(),
                                           ws.storage.ptr<unsigned char>(), (int64_t)ws.storage.bytes(), stream.raw()),
                        "glm53f_spec_accept");
    }
};

}  // namespace glm53f_spec

#endif  // GLM53F_SPEC_HOST_SPEC_HPP
