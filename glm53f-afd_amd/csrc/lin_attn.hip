// Linear attention with one decay per head (gfx950): S <- exp(g) S + v k^T, o = scale S q.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ext/glm53f_lin.h"
#include "kda_common.h"

namespace lin {
namespace {

using kda::bf16_t;
using kda::kInvalid;

constexpr int THREADS = 256;

typedef long long ll;

// N consecutive bf16 values, in one access where the address is aligned to all of them.
template <int N, bool VEC>
__device__ __forceinline__ void load_row(const bf16_t* p, bf16_t (&e)[N]) {
    if constexpr (VEC && N >= 8) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const kda::u32x4_t x = *reinterpret_cast<const kda::u32x4_t*>(p + i);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                e[i + 2 * c] = (bf16_t)x[c];
                e[i + 2 * c + 1] = (bf16_t)(x[c] >> 16);
            }
        }
    } else if constexpr (VEC && N == 4) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        e[0] = (bf16_t)x.x, e[1] = (bf16_t)(x.x >> 16), e[2] = (bf16_t)x.y, e[3] = (bf16_t)(x.y >> 16);
    } else if constexpr (VEC && N == 2) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(p);
        e[0] = (bf16_t)x, e[1] = (bf16_t)(x >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = p[i];
    }
}

template <int N, bool VEC>
__device__ __forceinline__ void store_row(bf16_t* p, const float (&x)[N]) {
    if constexpr (VEC && N >= 2) {
        uint32_t w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) w[i] = kda::f2bf2(x[2 * i], x[2 * i + 1]);
        if constexpr (N >= 8) {
#pragma unroll
            for (int i = 0; i < N / 2; i += 4) *reinterpret_cast<uint4*>(p + 2 * i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if constexpr (N == 4) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = kda::f2bf(x[i]);
    }
}

// The sum over the LPR lanes (8, 16 or 32) that share a value row; every one of them gets it.
template <int LPR>
__device__ __forceinline__ float lane_sum(float x) {
    if constexpr (LPR == 32) x += __shfl_xor(x, 16, 64);
    if constexpr (LPR >= 16) x += kda::lane_xor16<8>(x);
    x += kda::lane_xor16<4>(x);
    x += kda::lane_xor16<2>(x);
    x += kda::lane_xor16<1>(x);
    return x;
}

template <typename S>
struct ChainArgs {
    int heads, group, dv;                         // group: value heads that share a head of q and k
    const int32_t* cu_rows;
    const int32_t* keep;                          // NULL: all rows of the request
    int most;                                     // rows of a request beyond this are left out
    const bf16_t* q;
    ll q_stride;
    const bf16_t* k;
    ll k_stride, k_layer;
    const bf16_t* v;
    ll v_stride, v_layer;
    const float* log_decay;
    float scale;
    const S* state_in;
    S* state_out;
    ll state_layer;
    const int64_t* state_off;
    bf16_t* out;
    ll out_stride;
};

// The recurrence row by row: decode steps, short windows, and without the read-out (READ false) the commit of a window's
// accepted rows. Bound by the states: each is read once and written once per call. Workgroup ((layer, head, part), b) holds
// NROW value rows of a state in registers across the rows: LPR lanes share a value row (16 bytes of it each), and a lane
// holds ST consecutive value rows, so that its values and its outputs are one access each. Value rows do not meet, so the
// cut changes no bit; small batches take the finer one to reach more CUs. The product of two bf16 values is exact in f32,
// so the update has one rounding of the decayed state and one of the sum.
template <typename S, int DK, int NROW, bool READ, bool VEC>
__global__ void __launch_bounds__(THREADS) chain_kernel(const ChainArgs<S> a) {
    constexpr int KPL = kda::StateGeo<S>::KPL, LPR = DK / KPL, GROUPS = THREADS / LPR, ST = NROW / GROUPS;
    static_assert(ST >= 1, "a lane holds a value row at least");
    const int parts = a.dv / NROW, b = blockIdx.y;
    const int part = blockIdx.x % parts, lh = blockIdx.x / parts, h = lh % a.heads, layer = lh / a.heads;
    const int row0 = a.cu_rows[b];
    int rows = min(a.cu_rows[b + 1] - row0, a.most);
    if (a.keep) rows = min(rows, a.keep[b]);
    rows = max(rows, 0);
    if (rows == 0 && (a.state_out == nullptr || a.state_out == a.state_in)) return;

    const int key0 = (threadIdx.x % LPR) * KPL, val0 = part * NROW + (threadIdx.x / LPR) * ST;
    const ll at = layer * a.state_layer + a.state_off[b] + ((ll)h * a.dv + val0) * DK + key0;
    const ll hk = h / a.group;
    const bf16_t* k = a.k + layer * a.k_layer + row0 * a.k_stride + hk * DK + key0;
    const bf16_t* q = READ ? a.q + row0 * a.q_stride + hk * DK + key0 : nullptr;
    const bf16_t* v = a.v + layer * a.v_layer + row0 * a.v_stride + (ll)h * a.dv + val0;

    bf16_t kn[KPL], qn[KPL], vn[ST];              // the next row's pieces
    if (rows > 0) {
        load_row<KPL, VEC>(k, kn);
        if constexpr (READ) load_row<KPL, VEC>(q, qn);
        load_row<ST, VEC>(v, vn);
    }
    const float fade = expf(a.log_decay[lh]);
    uint4 raw[ST];
#pragma unroll
    for (int j = 0; j < ST; ++j) raw[j] = kda::ld128(a.state_in + at + j * DK);
    float s[ST][KPL];
#pragma unroll
    for (int j = 0; j < ST; ++j) kda::unpack<S>(raw[j], s[j]);

    for (int t = 0; t < rows; ++t) {
        float kk[KPL], qq[KPL], vv[ST];
#pragma unroll
        for (int c = 0; c < KPL; ++c) kk[c] = kda::bf2f(kn[c]);
        if constexpr (READ) {
#pragma unroll
            for (int c = 0; c < KPL; ++c) qq[c] = kda::bf2f(qn[c]) * a.scale;
        }
#pragma unroll
        for (int j = 0; j < ST; ++j) vv[j] = kda::bf2f(vn[j]);
        if (t + 1 < rows) {
            load_row<KPL, VEC>(k + (t + 1) * a.k_stride, kn);
            if constexpr (READ) load_row<KPL, VEC>(q + (t + 1) * a.q_stride, qn);
            load_row<ST, VEC>(v + (t + 1) * a.v_stride, vn);
        }
        float o[ST];
#pragma unroll
        for (int j = 0; j < ST; ++j) {
            o[j] = 0.0f;
#pragma unroll
            for (int c = 0; c < KPL; ++c) {
                s[j][c] = __builtin_fmaf(vv[j], kk[c], fade * s[j][c]);
                if constexpr (READ) o[j] = __builtin_fmaf(s[j][c], qq[c], o[j]);
            }
            if constexpr (READ) o[j] = lane_sum<LPR>(o[j]);
        }
        if constexpr (READ) {
            if (threadIdx.x % LPR == 0)
                store_row<ST, VEC>(a.out + (row0 + (ll)t) * a.out_stride + (ll)h * a.dv + val0, o);
        }
    }
    if (a.state_out == nullptr) return;
#pragma unroll
    for (int j = 0; j < ST; ++j) kda::st128(a.state_out + at + j * DK, kda::pack<S>(s[j]));
}

inline int launched() { return (int)hipGetLastError(); }
inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool good_shape(int heads, int qk_heads, int dk, int dv, int batch) {
    return heads >= 1 && heads <= 65535 && qk_heads >= 1 && heads % qk_heads == 0 && (dk == 64 || dk == 128) &&
           (dv == 64 || dv == 128) && batch >= 1 && batch <= 65535;
}

// 16-byte accesses of a row buffer: its base and every row.
inline bool fast_rows(const void* p, ll stride) { return aligned(p, 16) && stride % 8 == 0; }

template <typename S, int DK, int NROW, bool READ>
int launch_chain(const ChainArgs<S>& a, int layers, int batch, bool vec, hipStream_t stream) {
    const dim3 grid((unsigned)((ll)layers * a.heads * (a.dv / NROW)), (unsigned)batch);
    if (vec)
        chain_kernel<S, DK, NROW, READ, true><<<grid, THREADS, 0, stream>>>(a);
    else
        chain_kernel<S, DK, NROW, READ, false><<<grid, THREADS, 0, stream>>>(a);
    return launched();
}

template <typename S, bool READ>
int launch_chain(const ChainArgs<S>& a, int dk, int layers, int batch, hipStream_t stream) {
    const bool vec = fast_rows(a.k, a.k_stride) && a.k_layer % 8 == 0 && fast_rows(a.v, a.v_stride) && a.v_layer % 8 == 0 &&
                     (!READ || (fast_rows(a.q, a.q_stride) && fast_rows(a.out, a.out_stride)));
    const bool fine = (ll)layers * a.heads * batch * (a.dv / 64) < 512;   // fewer than two workgroups per CU
    if (dk == 64)
        return fine ? launch_chain<S, 64, 32, READ>(a, layers, batch, vec, stream)
                    : launch_chain<S, 64, 64, READ>(a, layers, batch, vec, stream);
    return fine ? launch_chain<S, 128, 32, READ>(a, layers, batch, vec, stream)
                : launch_chain<S, 128, 64, READ>(a, layers, batch, vec, stream);
}

// What the chain and the prefill check alike.
template <typename S>
bool good_call(int heads, int qk_heads, int dk, int dv, int batch, const ChainArgs<S>& a) {
    if (!good_shape(heads, qk_heads, dk, dv, batch)) return false;
    if (!a.cu_rows || !a.state_off || !a.log_decay || !a.q || !a.k || !a.v || !a.out || !a.state_in) return false;
    if (!aligned(a.q, 2) || !aligned(a.k, 2) || !aligned(a.v, 2) || !aligned(a.out, 2) || !aligned(a.state_in, 16) ||
        !aligned(a.state_out, 16) || !aligned(a.state_off, 8) || !aligned(a.cu_rows, 4) || !aligned(a.log_decay, 4))
        return false;
    return a.q_stride >= (ll)qk_heads * dk && a.k_stride >= (ll)qk_heads * dk && a.v_stride >= (ll)heads * dv &&
           a.out_stride >= (ll)heads * dv;
}

template <typename S>
int chain(int heads, int qk_heads, int dk, int dv, int batch, int most, ChainArgs<S> a, hipStream_t stream) {
    if (!good_call(heads, qk_heads, dk, dv, batch, a)) return kInvalid;
    a.heads = heads, a.group = heads / qk_heads, a.dv = dv, a.keep = nullptr, a.most = most;
    a.k_layer = a.v_layer = a.state_layer = 0;
    return launch_chain<S, true>(a, dk, 1, batch, stream);
}

template <typename S>
int advance(int heads, int qk_heads, int dk, int dv, int layers, int batch, const int32_t* cu_rows, const int32_t* keep,
            const bf16_t* k, ll k_stride, ll k_layer, const bf16_t* v, ll v_stride, ll v_layer, const float* log_decay,
            const S* state_in, S* state_out, ll state_layer, const int64_t* state_off, hipStream_t stream) {
    if (!good_shape(heads, qk_heads, dk, dv, batch) || layers < 1 || (ll)layers * heads > 0x3fffffff) return kInvalid;
    if (!cu_rows || !keep || !k || !v || !log_decay || !state_in || !state_out || !state_off) return kInvalid;
    if (!aligned(k, 2) || !aligned(v, 2) || !aligned(state_in, 16) || !aligned(state_out, 16) || !aligned(state_off, 8) ||
        !aligned(cu_rows, 4) || !aligned(keep, 4) || !aligned(log_decay, 4))
        return kInvalid;
    if (k_stride < (ll)qk_heads * dk || v_stride < (ll)heads * dv) return kInvalid;
    if (layers > 1 && (k_layer < 0 || v_layer < 0 || state_layer < 1 || state_layer % 8)) return kInvalid;
    if (layers == 1) k_layer = v_layer = state_layer = 0;
    const ChainArgs<S> a{heads, heads / qk_heads, dv, cu_rows, keep, 0x7fffffff, nullptr, 0, k, k_stride, k_layer, v, v_stride,
                         v_layer, log_decay, 0.0f, state_in, state_out, state_layer, state_off, nullptr, 0};
    return launch_chain<S, false>(a, dk, layers, batch, stream);
}

}  // namespace
}  // namespace lin

using lin::ChainArgs;

#define LIN_ROWS(S) ChainArgs<S>{0, 0, 0, cu_rows, nullptr, 0, q, q_stride, k, k_stride, 0, v, v_stride, 0, log_decay, scale, \
                                 state_in, state_out, 0, state_off, out, out_stride}

extern "C" int32_t glm53f_lin_chain_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim, int32_t batch,
        const int32_t* cu_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride, const uint16_t* v,
        int64_t v_stride, const float* log_decay, float scale, const float* state_in, float* state_out,
        const int64_t* state_off, uint16_t* out, int64_t out_stride, ihipStream_t* stream) {
    return lin::chain<float>(heads, qk_heads, key_dim, value_dim, batch, 0x7fffffff, LIN_ROWS(float), stream);
}

extern "C" int32_t glm53f_lin_chain_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t batch, const int32_t* cu_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
        const uint16_t* v, int64_t v_stride, const float* log_decay, float scale, const uint16_t* state_in,
        uint16_t* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride, ihipStream_t* stream) {
    return lin::chain<uint16_t>(heads, qk_heads, key_dim, value_dim, batch, 0x7fffffff, LIN_ROWS(uint16_t), stream);
}

extern "C" int32_t glm53f_lin_advance_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t layers, int32_t batch, const int32_t* cu_rows, const int32_t* keep, const uint16_t* k, int64_t k_stride,
        int64_t k_layer_stride, const uint16_t* v, int64_t v_stride, int64_t v_layer_stride, const float* log_decay,
        const float* state_in, float* state_out, int64_t state_layer_stride, const int64_t* state_off,
        ihipStream_t* stream) {
    return lin::advance<float>(heads, qk_heads, key_dim, value_dim, layers, batch, cu_rows, keep, k, k_stride, k_layer_stride,
                               v, v_stride, v_layer_stride, log_decay, state_in, state_out, state_layer_stride, state_off,
                               stream);
}

extern "C" int32_t glm53f_lin_advance_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t layers, int32_t batch, const int32_t* cu_rows, const int32_t* keep, const uint16_t* k, int64_t k_stride,
        int64_t k_layer_stride, const uint16_t* v, int64_t v_stride, int64_t v_layer_stride, const float* log_decay,
        const uint16_t* state_in, uint16_t* state_out, int64_t state_layer_stride, const int64_t* state_off,
        ihipStream_t* stream) {
    return lin::advance<uint16_t>(heads, qk_heads, key_dim, value_dim, layers, batch, cu_rows, keep, k, k_stride,
                                  k_layer_stride, v, v_stride, v_layer_stride, log_decay, state_in, state_out,
                                  state_layer_stride, state_off, stream);
}

extern "C" int64_t glm53f_lin_prefill_workspace_bytes(int32_t heads, int32_t key_dim, int32_t value_dim, int32_t batch,
                                                      int32_t max_rows) {
    if (!lin::good_shape(heads, 1, key_dim, value_dim, batch) || max_rows < 0) return -1;
    return 0;
}

extern "C" int32_t glm53f_lin_prefill_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t batch, const int32_t* cu_rows, int32_t max_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k,
        int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* log_decay, float scale, const float* state_in,
        float* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride, void* workspace,
        int64_t workspace_bytes, ihipStream_t* stream) {
    (void)workspace, (void)workspace_bytes;
    if (max_rows < 0) return kda::kInvalid;
    return lin::chain<float>(heads, qk_heads, key_dim, value_dim, batch, max_rows, LIN_ROWS(float), stream);
}

extern "C" int32_t glm53f_lin_prefill_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t batch, const int32_t* cu_rows, int32_t max_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k,
        int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* log_decay, float scale,
        const uint16_t* state_in, uint16_t* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride,
        void* workspace, int64_t workspace_bytes, ihipStream_t* stream) {
    (void)workspace, (void)workspace_bytes;
    if (max_rows < 0) return kda::kInvalid;
    return lin::chain<uint16_t>(heads, qk_heads, key_dim, value_dim, batch, max_rows, LIN_ROWS(uint16_t), stream);
}
