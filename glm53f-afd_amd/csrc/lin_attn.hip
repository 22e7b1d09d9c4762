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
    int rows = a.cu_rows[b + 1] - row0;
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

// ---------------------------------------------------------------------------------------------------------------
// The chunked form. Over a chunk of n <= 32 rows that starts from state S (rows i, j from 0):
//
//     o_i = scale ( e^{g (i+1)} S q_i + sum_{j <= i} e^{g (i-j)} (q_i . k_j) v_j ),
//     S  <- e^{g n} S + sum_i (e^{g (n-1-i)} v_i) k_i^T
//
// and every sum is a product on the matrix cores (16 x 16 x 32, bf16 operands, f32 sums). q, k and v are bf16 already;
// what is not becomes two or three bf16 terms, so that the products keep the accuracy of f32: the decayed values three (all
// their 24 bits, in three truncations), the scores and the state two each for the read-out, whose outputs are bf16 (2^-17
// of their terms). No power of e^g above 1 is formed, so no decay is too fast.
//
// A workgroup is one head of one request over one segment of its rows; wave w holds the state's value rows 32 w .. 32 w + 31
// in accumulators, s[t][x]: keys 16 t + 4 (lane / 16) + e, value row 32 w + 2 (lane % 16) + x. That order is free, and
// this one makes a lane's loads of v (two neighbouring columns of eight rows) the operand of the products as it is,
// without LDS, its state tiles two operands of the read-out, and its outputs eight consecutive values. q and k pass through
// LDS once per chunk for all waves: as rows for the scores (keys in the order that the state's accumulators have), and k
// transposed for the state, from the same registers.
//
// Few requests leave most CUs idle for a long prompt, so the rows are cut into segments: segment_kernel (SUMS) forms what
// each segment adds to a state, starts_kernel runs over them to the state at every segment's start, and the outputs of
// all segments are computed from there at once. k and v are then read twice, the second time from the caches as far as
// they hold them.

constexpr int C = 32;                             // rows per chunk: one product's depth

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename S>
struct PrefillArgs {
    int heads, group, most;
    const int32_t* cu_rows;
    const bf16_t* q;
    ll q_stride;
    const bf16_t* k;
    ll k_stride;
    const bf16_t* v;
    ll v_stride;
    const float* log_decay;
    float scale;
    const S* state_in;
    S* state_out;
    const int64_t* state_off;
    bf16_t* out;
    ll out_stride;
    float* work;                                  // [batch][heads][segs] states in the waves' order, NULL: one segment
    int segs, seg_rows;                           // seg_rows: a multiple of C
};

// e^{g n}; 1 for n = 0 also where nothing is remembered (g = -inf).
__device__ __forceinline__ float fade_of(float g, int n) { return n == 0 ? 1.0f : expf(g * (float)n); }

__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }

__device__ __forceinline__ bf16x8 operand(const uint32_t (&w)[4]) {
    const kda::u32x4_t x = {w[0], w[1], w[2], w[3]};
    return __builtin_bit_cast(bf16x8, x);
}
__device__ __forceinline__ bf16x8 operand(const bf16_t* lds) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const kda::u32x4_t*>(lds));
}

__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight f32 values as hi + lo: hi their upper halves, lo the rest rounded to bf16.
__device__ __forceinline__ void two_terms(const float (&x)[8], bf16x8& hi, bf16x8& lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(x[2 * i]), b = __float_as_uint(x[2 * i + 1]);
        h[i] = high_halves(a, b);
        l[i] = kda::f2bf2(x[2 * i] - __uint_as_float(a & 0xffff0000u), x[2 * i + 1] - __uint_as_float(b & 0xffff0000u));
    }
    hi = operand(h), lo = operand(l);
}

// Two neighbouring elements of a row; FAST: in one access (the rows are 4-byte aligned).
template <bool FAST>
__device__ __forceinline__ uint32_t load_pair(const bf16_t* p) {
    if constexpr (FAST) return *reinterpret_cast<const uint32_t*>(p);
    return p[0] | ((uint32_t)p[1] << 16);
}

// A wave's part of a state in memory ([value][key]) and its accumulators.
template <typename S, int DK>
__device__ __forceinline__ void load_state(const S* p, f32x4 (&s)[DK / 16][2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            const S* at = p + (32 * wave + 2 * (lane & 15) + x) * DK + 16 * t + 4 * (lane >> 4);
            if constexpr (sizeof(S) == 4) {
                s[t][x] = *reinterpret_cast<const f32x4*>(at);
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(at);
                s[t][x] = f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                                __uint_as_float(w.y & 0xffff0000u)};
            }
        }
}
template <typename S, int DK>
__device__ __forceinline__ void store_state(S* p, const f32x4 (&s)[DK / 16][2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int t = 0; t < DK / 16; ++t) {
            S* at = p + (32 * wave + 2 * (lane & 15) + x) * DK + 16 * t + 4 * (lane >> 4);
            const f32x4 v = s[t][x];
            if constexpr (sizeof(S) == 4)
                *reinterpret_cast<f32x4*>(at) = v;
            else
                *reinterpret_cast<uint2*>(at) = make_uint2(kda::f2bf2(v[0], v[1]), kda::f2bf2(v[2], v[3]));
        }
}

// The same part in the workspace: a lane's accumulators 16 bytes each, a wave's instruction 1 KiB.
template <int DK, int NW>
__device__ __forceinline__ float* work_at(float* work, ll index) {
    return work + index * (32 * NW * DK) + (threadIdx.x >> 6) * (32 * DK) + (threadIdx.x & 63) * 4;
}

// SUMS: what the segment adds to a state, into the workspace; otherwise its outputs, and behind a request's last row
// the state. FAST: q, k and v rows are 4-byte aligned and out rows 16-byte aligned.
template <typename S, int DK, int NW, bool FAST, bool SUMS>
__global__ void __launch_bounds__(64 * NW, NW / 2) segment_kernel(const PrefillArgs<S> a) {
    constexpr int T = 64 * NW, KT = DK / 16, PITCH = DK + 8, DV = 32 * NW;
    constexpr int TERMS = 3;
    constexpr int ITEMS = SUMS ? (2 * DK + T - 1) / T : 4 * DK / T;   // (eight rows, two columns) of k, then of q, per thread
    __shared__ __align__(16) bf16_t ks[SUMS ? 1 : C * PITCH], qs[SUMS ? 1 : C * PITCH], kt[DK * C], ph[SUMS ? 1 : C * C],
        pl[SUMS ? 1 : C * C];
    const int h = blockIdx.x % a.heads, seg = blockIdx.x / a.heads, b = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, grp = lane >> 4;
    const int first = a.cu_rows[b], rows = max(min(a.cu_rows[b + 1] - first, a.most), 0);
    const int begin = seg * a.seg_rows;
    if (begin >= rows && (seg > 0 || SUMS)) return;
    const bool last = rows - begin <= a.seg_rows;  // the request's last segment
    if (SUMS && last) return;                     // nothing starts behind it
    const int n = min(rows - begin, a.seg_rows);  // 0: a request without rows
    const ll state_at = a.state_off[b] + (ll)h * (DV * DK);
    if (n == 0 && (a.state_out == nullptr || a.state_out == a.state_in)) return;
    const float g = a.log_decay[h];
    const ll row0 = (ll)first + begin, hk = h / a.group;

    // what this thread moves of k and q: rows 8 oct .., columns 2 c2 and 2 c2 + 1
    const bf16_t* src[ITEMS];
    ll step[ITEMS];
    int oct[ITEMS], c2[ITEMS];
    bool is_k[ITEMS], on[ITEMS];
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
        const int id = it * T + threadIdx.x;
        is_k[it] = SUMS || id < 2 * DK;
        on[it] = !SUMS || id < 2 * DK;
        oct[it] = (id / (DK / 2)) & 3;
        c2[it] = id % (DK / 2);
        step[it] = is_k[it] ? a.k_stride : a.q_stride;
        src[it] = (is_k[it] ? a.k : a.q) + (row0 + 8 * oct[it]) * step[it] + hk * DK + 2 * c2[it];
    }
    const bf16_t* vsrc = a.v + (row0 + 8 * grp) * a.v_stride + (ll)h * DV + 32 * wave + 2 * col;

    uint32_t raw[ITEMS][8], vraw[8];
    auto load = [&](int c) {
        const int live = n - c * C;               // rows of the request that the chunk holds; the others are zeros
#pragma unroll
        for (int it = 0; it < ITEMS; ++it)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                raw[it][e] = on[it] && 8 * oct[it] + e < live ? load_pair<FAST>(src[it] + (c * C + e) * step[it]) : 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) vraw[e] = 8 * grp + e < live ? load_pair<FAST>(vsrc + (c * C + e) * a.v_stride) : 0u;
    };

    f32x4 s[KT][2];
    if constexpr (SUMS) {
#pragma unroll
        for (int t = 0; t < KT; ++t) s[t][0] = s[t][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    } else if (a.work) {
        const float* w = work_at<DK, NW>(a.work, ((ll)b * a.heads + h) * a.segs + seg);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) s[t][x] = *reinterpret_cast<const f32x4*>(w + (2 * t + x) * 256);
    } else {
        load_state<S, DK>(a.state_in + state_at, s);
    }

    // the decays of a whole chunk that this lane uses
    float in_tail[8], to_row[2], between[4];
    const int tiles_i[3] = {0, 1, 1}, tiles_j[3] = {0, 0, 1};         // the score tiles on and below the diagonal
    if (n > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) in_tail[e] = fade_of(g, C - 1 - (8 * grp + e));
        if constexpr (!SUMS) {
#pragma unroll
            for (int i = 0; i < 2; ++i) to_row[i] = fade_of(g, 16 * i + col + 1);
            for (int i = threadIdx.x; i < C * C / 2; i += T)
                reinterpret_cast<uint32_t*>(ph)[i] = reinterpret_cast<uint32_t*>(pl)[i] = 0u;   // the tile above the diagonal
        }
        load(0);
    }
    const float whole = fade_of(g, C);
    (void)between;

    for (int c = 0; c * C < n; ++c) {
        const int live = min(n - c * C, C);
        // q and k to LDS
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            if (!on[it]) continue;
            if constexpr (!SUMS) {
                // a row's keys in the order 0-3, 16-19, 4-7, 20-23, .. of every 32: what a lane's two state tiles hold
                const int piece = (c2[it] & 15) >> 1, at = (c2[it] & ~15) + ((piece & 3) * 2 + (piece >> 2)) * 2 + (c2[it] & 1);
                uint32_t* dst = reinterpret_cast<uint32_t*>((is_k[it] ? ks : qs) + 8 * oct[it] * PITCH) + at;
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[e * (PITCH / 2)] = raw[it][e];
            }
            if (is_k[it]) {
                bf16_t* dst = kt + 2 * c2[it] * C + 8 * (oct[it] ^ (c2[it] & 3));
                uint32_t w[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) w[m] = low_halves(raw[it][2 * m], raw[it][2 * m + 1]);
                *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
                for (int m = 0; m < 4; ++m) w[m] = high_halves(raw[it][2 * m], raw[it][2 * m + 1]);
                *reinterpret_cast<uint4*>(dst + C) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        // v as operands: itself, and decayed to the chunk's end in terms
        uint32_t vp[2][4], vd[TERMS][2][4];
        {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = live == C ? in_tail[e] : fade_of(g, max(live - 1 - (8 * grp + e), 0));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                vp[0][m] = low_halves(vraw[2 * m], vraw[2 * m + 1]);
                vp[1][m] = high_halves(vraw[2 * m], vraw[2 * m + 1]);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    uint32_t part[TERMS][2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint32_t r = vraw[2 * m + y];
                        float z = f[2 * m + y] * __uint_as_float(x ? r & 0xffff0000u : r << 16);
#pragma unroll
                        for (int i = 0; i < TERMS; ++i) {
                            part[i][y] = __float_as_uint(z);
                            z -= __uint_as_float(part[i][y] & 0xffff0000u);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) vd[i][x][m] = high_halves(part[i][0], part[i][1]);
                }
            }
        }
        __syncthreads();
        if ((c + 1) * C < n) load(c + 1);

        if constexpr (!SUMS) {
            // scores: tile (i, j) with key rows as the first operand, so that a lane holds four consecutive j of a row i
#pragma unroll
            for (int tt = 0; tt < 3; ++tt) {
                if (tt % NW != wave) continue;
                const int ti = tiles_i[tt], tj = tiles_j[tt];
                f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < DK / 32; ++u)
                    p = product(operand(ks + (16 * tj + col) * PITCH + 32 * u + 8 * grp), operand(qs + (16 * ti + col) * PITCH + 32 * u + 8 * grp), p);
                const int i = 16 * ti + col, j = 16 * tj + 4 * grp;
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    float y[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int gap = i - (j + 2 * m + e);
                        y[e] = gap < 0 ? 0.0f : p[2 * m + e] * fade_of(g, gap);
                    }
                    const uint32_t r0 = __float_as_uint(y[0]), r1 = __float_as_uint(y[1]);
                    hi[m] = high_halves(r0, r1);
                    lo[m] = kda::f2bf2(y[0] - __uint_as_float(r0 & 0xffff0000u), y[1] - __uint_as_float(r1 & 0xffff0000u));
                }
                const int at = i * C + 8 * ((j >> 3) ^ ((i >> 1) & 3)) + (j & 7);
                *reinterpret_cast<uint2*>(ph + at) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(pl + at) = make_uint2(lo[0], lo[1]);
            }
            // what the chunk's start gives to its rows
            f32x4 o[2][2] = {};
#pragma unroll
            for (int u = 0; u < DK / 32; ++u) {
                bf16x8 qf[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) qf[i] = operand(qs + (16 * i + col) * PITCH + 32 * u + 8 * grp);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float z[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = s[2 * u][x][e], z[4 + e] = s[2 * u + 1][x][e];
                    bf16x8 hi, lo;
                    two_terms(z, hi, lo);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        o[x][i] = product(hi, qf[i], o[x][i]);
                        o[x][i] = product(lo, qf[i], o[x][i]);
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (16 * i + col) * C + 8 * (grp ^ ((col >> 1) & 3));
                const bf16x8 hi = operand(ph + at), lo = operand(pl + at);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[x][i][e] *= to_row[i];
                    o[x][i] = product(operand(vp[x]), hi, o[x][i]);
                    o[x][i] = product(operand(vp[x]), lo, o[x][i]);
                }
                if (16 * i + col < live) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[2 * e] = o[0][i][e] * a.scale, y[2 * e + 1] = o[1][i][e] * a.scale;
                    store_row<8, FAST>(a.out + (row0 + c * C + 16 * i + col) * a.out_stride + (ll)h * DV + 32 * wave + 8 * grp, y);
                }
            }
        }
        // the state behind the chunk
        const float by = live == C ? whole : fade_of(g, live);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const bf16x8 kf = operand(kt + (16 * t + col) * C + 8 * (grp ^ ((col >> 1) & 3)));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t][x][e] *= by;
#pragma unroll
                for (int i = 0; i < TERMS; ++i) s[t][x] = product(kf, operand(vd[i][x]), s[t][x]);
            }
        }
        __syncthreads();
    }

    if constexpr (SUMS) {
        float* w = work_at<DK, NW>(a.work, ((ll)b * a.heads + h) * a.segs + seg + 1);
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) *reinterpret_cast<f32x4*>(w + (2 * t + x) * 256) = s[t][x];
    } else if (last && a.state_out) {
        store_state<S, DK>(a.state_out + state_at, s);
    }
}

// The state at every segment's start: the one the request came with, and behind each segment what it adds.
template <typename S, int DK, int NW>
__global__ void __launch_bounds__(64 * NW) starts_kernel(const PrefillArgs<S> a) {
    const int h = blockIdx.x, b = blockIdx.y, t = blockIdx.z / 2, x = blockIdx.z % 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rows = max(min(a.cu_rows[b + 1] - a.cu_rows[b], a.most), 0);
    const float by = fade_of(a.log_decay[h], a.seg_rows);
    const S* p = a.state_in + a.state_off[b] + (ll)h * (32 * NW * DK) + (32 * wave + 2 * (lane & 15) + x) * DK + 16 * t + 4 * (lane >> 4);
    f32x4 s;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(S) == 4) s[e] = p[e];
        else s[e] = kda::bf2f(p[e]);
    }
    float* w = work_at<DK, NW>(a.work, ((ll)b * a.heads + h) * a.segs) + (2 * t + x) * 256;
    *reinterpret_cast<f32x4*>(w) = s;
    for (int seg = 1; seg * a.seg_rows < rows; ++seg) {
        w += 32 * NW * DK;
        const f32x4 d = *reinterpret_cast<const f32x4*>(w);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(by, s[e], d[e]);
        *reinterpret_cast<f32x4*>(w) = s;
    }
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
int chain(int heads, int qk_heads, int dk, int dv, int batch, ChainArgs<S> a, hipStream_t stream) {
    if (!good_call(heads, qk_heads, dk, dv, batch, a)) return kInvalid;
    a.heads = heads, a.group = heads / qk_heads, a.dv = dv, a.keep = nullptr;
    a.k_layer = a.v_layer = a.state_layer = 0;
    return launch_chain<S, true>(a, dk, 1, batch, stream);
}

// Segments of a call: enough workgroups for two on every CU and again as many, so that requests of unequal length even
// out; a segment is 256 rows at least, since one costs a state's round through memory. Sizes alone decide.
struct Cut {
    int segs, seg_rows;
};
Cut cut(int heads, int batch, int max_rows) {
    const ll groups = (ll)heads * batch;
    ll segs = (1024 + groups - 1) / groups;
    const ll most = ((ll)max_rows + 255) / 256;
    if (segs > most) segs = most;
    if (groups >= 512 || segs < 1) segs = 1;
    ll rows = ((ll)max_rows + segs - 1) / segs;
    rows = (rows + C - 1) / C * C;
    if (rows < C) rows = C;
    if (segs == 1) return {1, (int)(rows > 0x7fffffff ? 0x7fffffe0 : rows)};
    return {(int)(((ll)max_rows + rows - 1) / rows), (int)rows};
}

template <typename S, int DK, int NW, bool FAST>
int launch_prefill(const PrefillArgs<S>& a, int batch, hipStream_t stream) {
    const dim3 grid((unsigned)((ll)a.heads * a.segs), (unsigned)batch);
    if (a.segs > 1) {
        segment_kernel<S, DK, NW, FAST, true><<<grid, 64 * NW, 0, stream>>>(a);
        starts_kernel<S, DK, NW><<<dim3((unsigned)a.heads, (unsigned)batch, 2 * (DK / 16)), 64 * NW, 0, stream>>>(a);
    }
    segment_kernel<S, DK, NW, FAST, false><<<grid, 64 * NW, 0, stream>>>(a);
    return launched();
}

inline bool pair_rows(const void* p, ll stride) { return aligned(p, 4) && stride % 2 == 0; }

template <typename S>
int prefill(int heads, int qk_heads, int dk, int dv, int batch, int max_rows, const ChainArgs<S>& r, void* workspace,
            ll workspace_bytes, hipStream_t stream) {
    if (max_rows < 0 || !good_call(heads, qk_heads, dk, dv, batch, r)) return kInvalid;
    const Cut c = cut(heads, batch, max_rows);
    if (c.segs > 1 && (!workspace || !aligned(workspace, 16) ||
                       workspace_bytes < glm53f_lin_prefill_workspace_bytes(heads, dk, dv, batch, max_rows)))
        return kInvalid;
    const PrefillArgs<S> a{heads, heads / qk_heads, max_rows, r.cu_rows, r.q, r.q_stride, r.k, r.k_stride, r.v, r.v_stride,
                           r.log_decay, r.scale, r.state_in, r.state_out, r.state_off, r.out, r.out_stride,
                           c.segs > 1 ? static_cast<float*>(workspace) : nullptr, c.segs, c.seg_rows};
    const bool fast = pair_rows(r.q, r.q_stride) && pair_rows(r.k, r.k_stride) && pair_rows(r.v, r.v_stride) &&
                      fast_rows(r.out, r.out_stride);
    if (dk == 64) {
        if (dv == 64)
            return fast ? launch_prefill<S, 64, 2, true>(a, batch, stream) : launch_prefill<S, 64, 2, false>(a, batch, stream);
        return fast ? launch_prefill<S, 64, 4, true>(a, batch, stream) : launch_prefill<S, 64, 4, false>(a, batch, stream);
    }
    if (dv == 64)
        return fast ? launch_prefill<S, 128, 2, true>(a, batch, stream) : launch_prefill<S, 128, 2, false>(a, batch, stream);
    return fast ? launch_prefill<S, 128, 4, true>(a, batch, stream) : launch_prefill<S, 128, 4, false>(a, batch, stream);
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
    const ChainArgs<S> a{heads, heads / qk_heads, dv, cu_rows, keep, nullptr, 0, k, k_stride, k_layer, v, v_stride,
                         v_layer, log_decay, 0.0f, state_in, state_out, state_layer, state_off, nullptr, 0};
    return launch_chain<S, false>(a, dk, layers, batch, stream);
}

}  // namespace
}  // namespace lin

using lin::ChainArgs;

#define LIN_ROWS(S) ChainArgs<S>{0, 0, 0, cu_rows, nullptr, q, q_stride, k, k_stride, 0, v, v_stride, 0, log_decay, scale, \
                                 state_in, state_out, 0, state_off, out, out_stride}

extern "C" int32_t glm53f_lin_chain_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim, int32_t batch,
        const int32_t* cu_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride, const uint16_t* v,
        int64_t v_stride, const float* log_decay, float scale, const float* state_in, float* state_out,
        const int64_t* state_off, uint16_t* out, int64_t out_stride, ihipStream_t* stream) {
    return lin::chain<float>(heads, qk_heads, key_dim, value_dim, batch, LIN_ROWS(float), stream);
}

extern "C" int32_t glm53f_lin_chain_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t batch, const int32_t* cu_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride,
        const uint16_t* v, int64_t v_stride, const float* log_decay, float scale, const uint16_t* state_in,
        uint16_t* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride, ihipStream_t* stream) {
    return lin::chain<uint16_t>(heads, qk_heads, key_dim, value_dim, batch, LIN_ROWS(uint16_t), stream);
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
    const lin::Cut c = lin::cut(heads, batch, max_rows);
    return c.segs > 1 ? (int64_t)heads * batch * c.segs * key_dim * value_dim * (int64_t)sizeof(float) : 0;
}

extern "C" int32_t glm53f_lin_prefill_batch(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t batch, const int32_t* cu_rows, int32_t max_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k,
        int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* log_decay, float scale, const float* state_in,
        float* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride, void* workspace,
        int64_t workspace_bytes, ihipStream_t* stream) {
    return lin::prefill<float>(heads, qk_heads, key_dim, value_dim, batch, max_rows, LIN_ROWS(float), workspace, workspace_bytes, stream);
}

extern "C" int32_t glm53f_lin_prefill_batch_bf16state(int32_t heads, int32_t qk_heads, int32_t key_dim, int32_t value_dim,
        int32_t batch, const int32_t* cu_rows, int32_t max_rows, const uint16_t* q, int64_t q_stride, const uint16_t* k,
        int64_t k_stride, const uint16_t* v, int64_t v_stride, const float* log_decay, float scale,
        const uint16_t* state_in, uint16_t* state_out, const int64_t* state_off, uint16_t* out, int64_t out_stride,
        void* workspace, int64_t workspace_bytes, ihipStream_t* stream) {
    return lin::prefill<uint16_t>(heads, qk_heads, key_dim, value_dim, batch, max_rows, LIN_ROWS(uint16_t), workspace, workspace_bytes, stream);
}
