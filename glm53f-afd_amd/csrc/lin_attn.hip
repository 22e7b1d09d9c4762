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

// N consecutive bf16 values of a row, whatever its address: global memory takes vectors at any element.
template <int N>
__device__ __forceinline__ void load_row(const bf16_t* p, bf16_t (&e)[N]) {
    if constexpr (N == 1) {
        e[0] = p[0];
    } else {
        constexpr int V = N > 8 ? 8 : N;
        typedef uint32_t vec __attribute__((ext_vector_type(V / 2), aligned(2)));
#pragma unroll
        for (int i = 0; i < N; i += V) {
            const vec x = *reinterpret_cast<const vec*>(p + i);
#pragma unroll
            for (int c = 0; c < V / 2; ++c) {
                e[i + 2 * c] = (bf16_t)x[c];
                e[i + 2 * c + 1] = (bf16_t)(x[c] >> 16);
            }
        }
    }
}

template <int N>
__device__ __forceinline__ void store_row(bf16_t* p, const float (&x)[N]) {
    if constexpr (N == 1) {
        p[0] = kda::f2bf(x[0]);
    } else {
        constexpr int V = N > 8 ? 8 : N;
        typedef uint32_t vec __attribute__((ext_vector_type(V / 2), aligned(2)));
#pragma unroll
        for (int i = 0; i < N; i += V) {
            vec w;
#pragma unroll
            for (int c = 0; c < V / 2; ++c) w[c] = kda::f2bf2(x[i + 2 * c], x[i + 2 * c + 1]);
            *reinterpret_cast<vec*>(p + i) = w;
        }
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
// cut changes no bit; small batches take the finer one to reach more CUs (one state of 64 heads: 3.6 us, a launch and one
// chain of loads). The product of two bf16 values is exact in f32, so the update has one rounding of the decayed state and
// one of the sum. Sixteen bf16 states of 64 heads, one row each: 13.1 us, 5.1 TB/s of states; the commit of 48 windows of up to
// sixteen rows 33 us, 6.1 TB/s.
template <typename S, int DK, int NROW, bool READ>
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
        load_row<KPL>(k, kn);
        if constexpr (READ) load_row<KPL>(q, qn);
        load_row<ST>(v, vn);
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
            load_row<KPL>(k + (t + 1) * a.k_stride, kn);
            if constexpr (READ) load_row<KPL>(q + (t + 1) * a.q_stride, qn);
            load_row<ST>(v + (t + 1) * a.v_stride, vn);
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
                store_row<ST>(a.out + (row0 + (ll)t) * a.out_stride + (ll)h * a.dv + val0, o);
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
// what is not (the decayed values, the scores, the state) becomes three bf16 terms, all its 24 bits in three truncations, so
// that the products keep the accuracy of f32. Two terms for the scores and the state would be 4 to 11 % faster (8192 rows of 64
// heads 197 us against 214, nine ragged prompts 93 and 97, six of up to 700 rows of 16 heads with 64 values 44 and 49) and 2^-17 of
// the terms off, more than the rounding of an output whose terms cancel. No power of e^g above 1 is formed, so no decay is too fast.
//
// A workgroup is one head of one request over one segment of its rows; wave w holds the state's value rows 32 w .. 32 w + 31
// in accumulators, 32 keys x 32 values of it per lane and four tiles. The rows of q, k and v go from memory straight to LDS,
// a chunk ahead, and are read from there in both directions: whole 16-byte pieces of sixteen rows (scores, read-out), and
// transposed, four rows of a column per lane (what the state adds, and the values of the read-out). The order of keys in the
// state's tiles and of values over the lanes is free; it is the one that makes a lane's two state tiles eight consecutive keys
// of one value row, so that they are an operand of the read-out as they stand, and its outputs eight consecutive values.
//
// Few requests leave most CUs idle for a long prompt, so the rows are cut into segments: segment_kernel (SUMS) forms what
// each segment adds to a state, starts_kernel runs over them to the state at every segment's start, and the outputs of
// all segments are computed from there at once. k and v are then read twice, the second time from the caches as far as
// they hold them.
//
// Measured on 8192 rows of 64 heads of 128 (k and v 268 MB, with q and the outputs 537 MB): 214 to 225 us from one
// machine to another (under the profiler, which leaves lower clocks and colder caches: what the segments add 64, the starts 14, the
// outputs 189). With k and v twice and eight segments' states written and read twice that moves 940 MB, 184 us at the card's copy
// rate; the products and the splitting into terms do not all hide behind it. The windows of 48 requests of up
// to sixteen rows (bf16 states, only read) 23 us, 4.4 TB/s of states; with f32 states 102 us with their commit.

constexpr int C = 32;                             // rows per chunk: one product's depth

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));   // at any element's address

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

// A value that is the same in all lanes, held once for the wave.
__device__ __forceinline__ float uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }

__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302); }

__device__ __forceinline__ bf16x8 operand(const uint32_t (&w)[4]) {
    const kda::u32x4_t x = {w[0], w[1], w[2], w[3]};
    return __builtin_bit_cast(bf16x8, x);
}
__device__ __forceinline__ bf16x8 operand(const bf16_t* lds) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const kda::u32x4_t*>(lds));
}

// Two of a transposed read: the sixteen lanes of a group name four rows of sixteen values, four lanes of 8 bytes a row, and
// each gets one column of the four rows.
__device__ __forceinline__ void column(const bf16_t* lds, uint32_t* w) {
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)lds);
    w[0] = (uint16_t)x[0] | (uint32_t)(uint16_t)x[1] << 16;
    w[1] = (uint16_t)x[2] | (uint32_t)(uint16_t)x[3] << 16;
}

__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// N f32 values as three bf16 terms whose sum they are: the upper half of each (8 of its 24 bits), of what remains, and the
// last 8 bits; two values to a word.
constexpr int TERMS = 3;
template <int N>
__device__ __forceinline__ void in_terms(const float (&x)[N], uint32_t (&w)[TERMS][N / 2]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int m = 0; m < TERMS; ++m) {
            const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
            w[m][i] = high_halves(ua, ub);
            if (m + 1 < TERMS) a -= __uint_as_float(ua & 0xffff0000u), b -= __uint_as_float(ub & 0xffff0000u);
        }
    }
}

// The scores' tiles on and below the diagonal, (0, 0), (1, 0) and (1, 1), of one term: where piece `piece` (eight columns) of a
// row stands. Rows of tile 0 have two pieces, of tile 1 four; sixteen rows at one piece meet every bank once.
constexpr int SCORES = 3 * 256;

// Where the 16-byte pieces of an LDS row stand: at piece ^ turn(row). Chosen for the two ways of reading: sixteen rows at one
// piece (a group of lanes that LDS serves at a time then meets every bank once), and four consecutive rows at four consecutive
// pieces. PIECES: of a row, 16, 8 or 4.
template <int PIECES>
__device__ __forceinline__ int turn(int row) {
    const int low = ((row >> 2 & 1) << 1) ^ ((row >> 3 & 1) * 3);
    if constexpr (PIECES == 16) return (row & 3) << 2 | low;
    if constexpr (PIECES == 8) return (row >> 1 & 1) << 2 | low;
    return low;
}

__device__ __forceinline__ int score_at(int row, int piece) {
    return row < 16 ? row * 16 + 8 * (piece ^ (row >> 3)) : 256 + (row - 16) * 32 + 8 * (piece ^ turn<4>(row));
}

// 16 bytes per lane from global memory to LDS without a register in between: to lds + 16 lane (lds the same in all lanes). Written
// out because the compiler, which cannot tell the buffers apart, has every read of one wait for the loads of the other;
// who reads waits himself, before a barrier.
__device__ __forceinline__ void to_lds(const bf16_t* src, bf16_t* lds) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) bf16_t*)lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(at) : "memory");
}

// Key and value of element e of a lane's tile (t, x) of its wave's state: eight consecutive keys from tiles t, t + 1 (t even).
__device__ __forceinline__ int key_of(int t, int grp) { return 32 * (t / 2) + 8 * grp + 4 * (t & 1); }
__device__ __forceinline__ int value_of(int x, int wave, int col) { return 32 * wave + 8 * (col >> 2) + 4 * x + (col & 3); }

// A wave's part of a state in memory ([value][key]) and its accumulators.
template <typename S, int DK>
__device__ __forceinline__ f32x4 load_tile(const S* p, int t, int x) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const S* at = p + value_of(x, wave, lane & 15) * DK + key_of(t, lane >> 4);
    if constexpr (sizeof(S) == 4) return *reinterpret_cast<const f32x4*>(at);
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    return f32x4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                 __uint_as_float(w.y & 0xffff0000u)};
}
template <typename S, int DK>
__device__ __forceinline__ void store_tile(S* p, int t, int x, f32x4 v) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    S* at = p + value_of(x, wave, lane & 15) * DK + key_of(t, lane >> 4);
    if constexpr (sizeof(S) == 4)
        *reinterpret_cast<f32x4*>(at) = v;
    else
        *reinterpret_cast<uint2*>(at) = make_uint2(kda::f2bf2(v[0], v[1]), kda::f2bf2(v[2], v[3]));
}

// The same part in the workspace: a lane's accumulators 16 bytes each, a wave's instruction 1 KiB.
template <int DK, int NW>
__device__ __forceinline__ float* work_at(float* work, ll index) {
    return work + index * (32 * NW * DK) + (threadIdx.x >> 6) * (32 * DK) + (threadIdx.x & 63) * 4;
}

__device__ __forceinline__ bool finite(f32x4 a, f32x4 b) {
    return ((a[0] + a[1]) + (a[2] + a[3]) + ((b[0] + b[1]) + (b[2] + b[3]))) * 0.0f == 0.0f;
}

// A segment's outputs once more, of one wave's values and row by row: where v has held an infinity or a NaN. The products of
// a chunk cannot keep it from the rows before it, whose zero scores times it are NaN. Sixteen values at a time, four lanes each.
template <typename S, int DK, int NW>
__device__ void outputs_by_rows(const PrefillArgs<S>& a, const S* state, const float* start, ll row0, int n, int h, float g) {
    constexpr int KEYS = DK / 4, DV = 32 * NW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, key0 = (lane & 3) * KEYS;
    const float fade = expf(g);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        const int r = 16 * half + (lane >> 2), col = 4 * (r >> 3) + (r & 3), x = r >> 2 & 1;   // value r of the wave's: tile x, column col
        float s[KEYS];
#pragma unroll
        for (int i = 0; i < KEYS; i += 4) {
            const int key = key0 + i, t = 2 * (key / 32) + (key >> 2 & 1), grp = key % 32 / 8;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (start) s[i + e] = start[wave * (32 * DK) + (2 * t + x) * 256 + (16 * grp + col) * 4 + e];
                else if constexpr (sizeof(S) == 4) s[i + e] = state[(32 * wave + r) * DK + key + e];
                else s[i + e] = kda::bf2f(state[(32 * wave + r) * DK + key + e]);
            }
        }
        const bf16_t* k = a.k + row0 * a.k_stride + (h / a.group) * DK + key0;
        const bf16_t* q = a.q + row0 * a.q_stride + (h / a.group) * DK + key0;
        const bf16_t* v = a.v + row0 * a.v_stride + (ll)h * DV + 32 * wave + r;
        bf16_t* out = a.out + row0 * a.out_stride + (ll)h * DV + 32 * wave + r;
#pragma unroll 1
        for (int t = 0; t < n; ++t, k += a.k_stride, q += a.q_stride, v += a.v_stride, out += a.out_stride) {
            const float y = kda::bf2f(*v);
            float o = 0.0f;
#pragma unroll
            for (int i = 0; i < KEYS; i += 8) {
                bf16_t ks[8], qs[8];
                load_row<8>(k + i, ks);
                load_row<8>(q + i, qs);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    s[i + e] = __builtin_fmaf(y, kda::bf2f(ks[e]), fade * s[i + e]);
                    o = __builtin_fmaf(s[i + e], kda::bf2f(qs[e]) * a.scale, o);
                }
            }
            o += kda::lane_xor16<2>(o);
            o += kda::lane_xor16<1>(o);
            if ((lane & 3) == 0) *out = kda::f2bf(o);
        }
    }
}

// SUMS: what the segment adds to a state, into the workspace; otherwise its outputs, and behind a request's last row
// the state. FAST: the rows of q, k and v are 16-byte aligned and go straight to LDS; otherwise through registers.
//
// Waves per SIMD: three where the rows go straight to LDS, for the sums two and no more, though the registers would let
// five in: a CU then takes another segment when one of its own ends, which evens out unequal lengths (nine ragged prompts 99 us,
// with three 102, with five 114; equal ones alike). The outputs' three take 166 of the 168 registers that this leaves them,
// without a spill: the places in LDS are formed anew from three of them in every chunk.
//
// ONCE: windows of one chunk whose states are only read. Nothing is double then, no state is kept behind the product that reads
// it, and a bf16 state is its operand as it lies in memory, so that more workgroups share a CU's loads (48 windows of up to
// sixteen rows of 64 heads, bf16 states: 23 us against 34).
constexpr int least_waves(bool fast, int nw, bool sums, bool once) { return once ? (nw == 4 ? 4 : 2) : fast && nw == 4 && !sums ? 3 : 2; }
constexpr int most_waves(bool fast, int nw, bool sums, bool once) { return fast && nw == 4 && !once ? (sums ? 2 : 3) : 8; }
template <typename S, int DK, int NW, bool FAST, bool SUMS, bool ONCE>
__global__ void __launch_bounds__(64 * NW)
__attribute__((amdgpu_waves_per_eu(least_waves(FAST, NW, SUMS, ONCE), most_waves(FAST, NW, SUMS, ONCE))))
segment_kernel(const PrefillArgs<S> a) {
    constexpr int T = 64 * NW, KT = DK / 16, DV = 32 * NW;
    constexpr int KP = DK / 8, VP = DV / 8;                          // pieces of a row
    constexpr int QN = SUMS ? 0 : C * KP / T, KN = C * KP / T, VN = C * VP / T, N = QN + KN + VN;   // pieces per thread and chunk
    static_assert(C * KP % T == 0 && C * VP % T == 0, "whole pieces");
    constexpr int SET = (SUMS ? 1 : 2) * C * DK + C * DV;            // a chunk's rows in LDS: k, v, q
    constexpr int SETS = ONCE ? 1 : 2;
    constexpr bool RAW = ONCE && sizeof(S) == 2;                     // the state's operands as they lie in memory
    __shared__ __align__(16) bf16_t lds[SETS * SET + (SUMS ? 0 : TERMS * SCORES)];
    bf16_t* scores = lds + SETS * SET;
    const int h = blockIdx.x % a.heads, seg = blockIdx.x / a.heads, b = blockIdx.y;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), col = lane & 15, grp = lane >> 4;
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

    // Piece i of this thread: LDS slot t + T i of k's rows, then v's, then q's; row slot / pieces of a row. Whole chunks take it from
    // a pointer that moves on; in the last one a row past the segment's end repeats the last. The sums, whose segments are whole
    // chunks, go from the last chunk to the first: what is read last is read first afterwards.
    auto is_v = [](int i) { return i >= KN && i < KN + VN; };
    auto place_of = [&](int i) { return i < KN ? i * T * 8 : is_v(i) ? C * DK + (i - KN) * T * 8 : C * (DK + DV) + (i - KN - VN) * T * 8; };
    auto slot_of = [&](int i) { return t + T * (i < KN ? i : is_v(i) ? i - KN : i - KN - VN); };
    auto row_of = [&](int i) { return slot_of(i) / (is_v(i) ? VP : KP); };
    auto stride_of = [&](int i) { return i < KN ? a.k_stride : is_v(i) ? a.v_stride : a.q_stride; };
    const bf16_t* src[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = row_of(i), piece = (slot_of(i) % (is_v(i) ? VP : KP)) ^ (is_v(i) ? turn<VP>(row) : turn<KP>(row));
        src[i] = (i < KN ? a.k + hk * DK : is_v(i) ? a.v + (ll)h * DV : a.q + hk * DK) + (row0 + (SUMS ? n - C : 0) + row) * stride_of(i) + 8 * piece;
    }
    u32x4_any held[FAST ? 1 : N];
    auto request = [&](int c, bf16_t* set) {
        auto one = [&](int i, const bf16_t* from) {
            if constexpr (FAST) to_lds(from, set + place_of(i) + wave * 512);
            else held[i] = *reinterpret_cast<const u32x4_any*>(from);
        };
        if (SUMS || (c + 1) * C <= n) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                one(i, src[i]);
                src[i] += (SUMS ? -C : C) * stride_of(i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) one(i, src[i] - max(c * C + row_of(i) - (n - 1), 0) * stride_of(i));
        }
    };
    auto place = [&](bf16_t* set) {               // the registers' pieces
        if constexpr (!FAST) {
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<kda::u32x4_t*>(set + place_of(i) + t * 8) = held[i];
        }
    };
    if (n > 0) request(0, lds);

    f32x4 s[KT][2];
    kda::u32x4_t raw[KT / 2][2];
    if constexpr (RAW) {
#pragma unroll
        for (int u = 0; u < KT / 2; ++u)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                raw[u][x] = *reinterpret_cast<const kda::u32x4_t*>(a.state_in + state_at + value_of(x, wave, col) * DK + 32 * u + 8 * grp);
    } else if constexpr (SUMS) {
#pragma unroll
        for (int m = 0; m < KT; ++m) s[m][0] = s[m][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    } else if (a.work) {
        const float* w = work_at<DK, NW>(a.work, ((ll)b * a.heads + h) * a.segs + seg);
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) s[m][x] = *reinterpret_cast<const f32x4*>(w + (2 * m + x) * 256);
    } else {
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) s[m][x] = load_tile<S, DK>(a.state_in + state_at, m, x);
    }

    // The decays of a whole chunk that this lane uses: of its rows of v to the chunk's end, of the chunk's start to its two
    // rows of outputs, and between the rows of its scores. The score tiles (rows, columns) on and below the diagonal are
    // (0, 0), (1, 0), (1, 1), tile m for wave m mod NW: a wave has tiles of one kind.
    const float in_tail = fade_of(g, C - 8 - 8 * grp);   // of the last of its eight rows; the others' by steps, alike in all lanes
    const int gap = (wave == 1 ? 16 : 0) + col - 4 * grp;   // from the first of its scores' four rows of k to their row of q
    float step[8], to_row[2], between[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) step[e] = uniform(fade_of(g, 7 - e));
    if constexpr (!SUMS) {
#pragma unroll
        for (int i = 0; i < 2; ++i) to_row[i] = a.scale * fade_of(g, 16 * i + col + 1);
#pragma unroll
        for (int e = 0; e < 4; ++e) between[e] = a.scale * fade_of(g, max(gap - e, 0));
    }
    const float whole = fade_of(g, C);

    // a lane's places in a set: row col at piece grp (+ 4 u: 32 elements further, under the turn; row 16 + col has the same turn),
    // and transposed row 8 grp + col / 4 at piece col mod 4 (four rows below two pieces further, under the turn)
    int at_row = col * DK + 8 * (grp ^ turn<KP>(col));
    const int tr = 8 * grp + (col >> 2), j = col & 3;
    int at_k = tr * DK + 8 * (j ^ turn<KP>(tr)), at_v = C * DK + tr * DV + 8 * ((4 * wave + j) ^ turn<VP>(tr));

    // its pieces of the scores; the tile above the diagonal is zeros, as the second piece of row 0 always is
    const int at_p0 = grp < 2 ? score_at(col, grp) : score_at(0, 1), at_p1 = score_at(16 + col, grp);

    int set = 0;
    bool odd = false;                             // a chunk's first row shows any infinity or NaN of its v
    for (int c = 0; c * C < n; ++c, set = SET - set) {               // SUMS: chunk n / C - 1 - c
        const int live = SUMS ? C : min(n - c * C, C);
        bf16_t* now = lds + set;
        // (not known from the chunk before: the compiler would keep every place of a piece in a register of its own)
        asm volatile("" : "+v"(at_row), "+v"(at_k), "+v"(at_v));
        const bf16_t* qs = now + C * (DK + DV);
        // this thread's part of the chunk is there; behind the barrier everybody's is, and the other set is free
        if constexpr (FAST) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else place(now);
        __syncthreads();
        if ((c + 1) * C < n) request(c + 1, lds + (SET - set));

        // v as an operand: two words of four rows, twice, for each half of the wave's values
        uint32_t vp[2][4];
        auto load_v = [&] {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                column(now + at_v + 4 * x, &vp[x][0]);
                column(now + (at_v ^ 16) + 4 * DV + 4 * x, &vp[x][2]);
            }
            if (live < C) {                       // rows past the last count as zeros
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int r = 8 * grp + 2 * m;
                    const uint32_t keep = (r < live ? 0x0000ffffu : 0u) | (r + 1 < live ? 0xffff0000u : 0u);
                    vp[0][m] &= keep, vp[1][m] &= keep;
                }
            }
        };
        if constexpr (SUMS) load_v();
        if constexpr (!SUMS) {
            // scores: key rows as the first operand, so that a lane holds four consecutive columns of a row
#pragma unroll
            for (int m = 0; m < 3; ++m) {
                if (m % NW != wave) continue;
                constexpr int tiles_i[3] = {0, 1, 1}, tiles_j[3] = {0, 0, 1};
                const int ti = tiles_i[m], tj = tiles_j[m];
                f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int u = 0; u < DK / 32; ++u)
                    p = product(operand(now + (at_row ^ (32 * u)) + 16 * DK * tj), operand(qs + (at_row ^ (32 * u)) + 16 * DK * ti), p);
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = gap < e ? 0.0f : p[e] * between[e];   // (a decay of 0 keeps a NaN)
                uint32_t w[TERMS][2];
                in_terms(y, w);
                bf16_t* to = scores + score_at(16 * ti + col, 2 * tj + grp / 2) + 4 * (grp & 1);
#pragma unroll
                for (int i = 0; i < TERMS; ++i) *reinterpret_cast<uint2*>(to + i * SCORES) = make_uint2(w[i][0], w[i][1]);
            }
            // what the chunk's start gives to its rows
            f32x4 o[2][2] = {};
#pragma unroll
            for (int u = 0; u < DK / 32; ++u) {
                const bf16x8 q0 = operand(qs + (at_row ^ (32 * u))), q1 = operand(qs + (at_row ^ (32 * u)) + 16 * DK);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if constexpr (RAW) {
                        o[x][0] = product(__builtin_bit_cast(bf16x8, raw[u][x]), q0, o[x][0]);
                        o[x][1] = product(__builtin_bit_cast(bf16x8, raw[u][x]), q1, o[x][1]);
                        continue;
                    }
                    float z[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = s[2 * u][x][e], z[4 + e] = s[2 * u + 1][x][e];
                    uint32_t w[TERMS][4];
                    in_terms(z, w);
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) {
                        o[x][0] = product(operand(w[i]), q0, o[x][0]);
                        o[x][1] = product(operand(w[i]), q1, o[x][1]);
                    }
                }
            }
            load_v();
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                bf16x8 p[TERMS];
#pragma unroll
                for (int m = 0; m < TERMS; ++m) p[m] = operand(scores + m * SCORES + (i ? at_p1 : at_p0));
#pragma unroll
                for (int x = 0; x < 2; ++x) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[x][i][e] *= to_row[i];
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) o[x][i] = product(operand(vp[x]), p[m], o[x][i]);
                }
                if (16 * i + col < live) {
                    const float y[8] = {o[0][i][0], o[0][i][1], o[0][i][2], o[0][i][3], o[1][i][0], o[1][i][1], o[1][i][2], o[1][i][3]};
                    bf16_t* at = a.out + (row0 + c * C + 16 * i + col) * a.out_stride + (ll)h * DV + 32 * wave + 8 * grp;
                    store_row<8>(at, y);
                }
            }
            odd |= !finite(o[0][0], o[1][0]);
            if (ONCE || (a.state_out == nullptr && last && (c + 1) * C >= n)) break;   // nobody reads the state behind the last rows
        }
        // v decayed to the chunk's end (SUMS: to the segment's, so that the sums need no decay), in terms
        uint32_t vd[2][TERMS][4];
        {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (SUMS ? in_tail * fade_of(g, c * C) : in_tail) * step[e];
            if (live < C) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = fade_of(g, max(live - 1 - (8 * grp + e), 0));
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float z[8];
#pragma unroll
                for (int m = 0; m < 4; ++m)
                    z[2 * m] = f[2 * m] * __uint_as_float(vp[x][m] << 16), z[2 * m + 1] = f[2 * m + 1] * __uint_as_float(vp[x][m] & 0xffff0000u);
                in_terms(z, vd[x]);
            }
        }
        // the state behind the chunk
        float by = whole;
        if (live < C) by = fade_of(g, live);
#pragma unroll
        for (int m = 0; m < KT; ++m) {
            uint32_t kf[4];
            column(now + (at_k ^ (32 * (m / 2))) + 4 * (m & 1), &kf[0]);
            column(now + (at_k ^ (32 * (m / 2) + 16)) + 4 * DK + 4 * (m & 1), &kf[2]);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[m][x][e] *= SUMS ? 1.0f : by;
#pragma unroll
                for (int i = 0; i < TERMS; ++i) s[m][x] = product(operand(kf), operand(vd[x][i]), s[m][x]);
            }
        }
    }

    if constexpr (SUMS) {
        float* w = work_at<DK, NW>(a.work, ((ll)b * a.heads + h) * a.segs + seg + 1);
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) *reinterpret_cast<f32x4*>(w + (2 * m + x) * 256) = s[m][x];
    } else {
        if (__any(odd)) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the outputs so far are written
            const float* start = a.work ? a.work + (((ll)b * a.heads + h) * a.segs + seg) * (DV * DK) : nullptr;
            outputs_by_rows<S, DK, NW>(a, a.state_in + state_at, start, row0, n, h, g);
        }
        if (ONCE || !last || !a.state_out) return;
#pragma unroll
        for (int m = 0; m < KT; ++m)
#pragma unroll
            for (int x = 0; x < 2; ++x) store_tile<S, DK>(a.state_out + state_at, m, x, s[m][x]);
    }
}

// The state at every segment's start: the one the request came with, and behind each segment what it adds.
template <typename S, int DK, int NW>
__global__ void __launch_bounds__(64 * NW) starts_kernel(const PrefillArgs<S> a) {
    const int h = blockIdx.x, b = blockIdx.y, t = blockIdx.z / 2, x = blockIdx.z % 2;
    const int rows = max(min(a.cu_rows[b + 1] - a.cu_rows[b], a.most), 0);
    const float by = fade_of(a.log_decay[h], a.seg_rows);
    f32x4 s = load_tile<S, DK>(a.state_in + a.state_off[b] + (ll)h * (32 * NW * DK), t, x);
    float* w = work_at<DK, NW>(a.work, ((ll)b * a.heads + h) * a.segs) + (2 * t + x) * 256;
    *reinterpret_cast<f32x4*>(w) = s;
    constexpr int AHEAD = 8;                      // segments requested at a time
    const int count = (int)(((ll)rows + a.seg_rows - 1) / a.seg_rows);
    for (int seg0 = 1; seg0 < count; seg0 += AHEAD) {
        f32x4 d[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
            if (seg0 + i < count) d[i] = *reinterpret_cast<const f32x4*>(w + (ll)(seg0 + i) * (32 * NW * DK));
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (seg0 + i >= count) break;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = __builtin_fmaf(by, s[e], d[i][e]);
            *reinterpret_cast<f32x4*>(w + (ll)(seg0 + i) * (32 * NW * DK)) = s;
        }
    }
}

inline int launched() { return (int)hipGetLastError(); }
inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool good_shape(int heads, int qk_heads, int dk, int dv, int batch) {
    return heads >= 1 && heads <= 65535 && qk_heads >= 1 && heads % qk_heads == 0 && (dk == 64 || dk == 128) &&
           (dv == 64 || dv == 128) && batch >= 1 && batch <= 65535;
}

template <typename S, int DK, int NROW, bool READ>
int launch_chain(const ChainArgs<S>& a, int layers, int batch, hipStream_t stream) {
    const dim3 grid((unsigned)((ll)layers * a.heads * (a.dv / NROW)), (unsigned)batch);
    chain_kernel<S, DK, NROW, READ><<<grid, THREADS, 0, stream>>>(a);
    return launched();
}

template <typename S, bool READ>
int launch_chain(const ChainArgs<S>& a, int dk, int layers, int batch, hipStream_t stream) {
    const bool fine = (ll)layers * a.heads * batch * (a.dv / 64) < 512;   // fewer than two workgroups per CU
    if (dk == 64) return fine ? launch_chain<S, 64, 32, READ>(a, layers, batch, stream) : launch_chain<S, 64, 64, READ>(a, layers, batch, stream);
    return fine ? launch_chain<S, 128, 32, READ>(a, layers, batch, stream) : launch_chain<S, 128, 64, READ>(a, layers, batch, stream);
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

// Segments of a call: as many as give every CU two workgroups, or with several requests four, so that requests of unequal
// length even out; a segment is 256 rows at least, since one costs a state's round through memory. Sizes alone decide, and they do
// not say whether the requests are alike. Two and four workgroups, us (64 heads of 128 but for the last two): one prompt of 8192
// rows 220 and 238; three of up to 4096 rows 281 and 240; nine of up to 1801 (32 heads, 64 keys) 132 and 100; but several equal
// ones 2 x 8192 400 and 423, 4 x 2048 203 and 231, 20 x 600 of 16 heads 79 and 123.
struct Cut {
    int segs, seg_rows;
};
Cut cut(int heads, int batch, int max_rows) {
    const ll groups = (ll)heads * batch, most = ((ll)max_rows + 255) / 256;
    ll segs = batch == 1 ? 512 / groups : (1024 + groups - 1) / groups;
    if (segs > most) segs = most;
    if (groups >= 512 || segs < 2) return {1, 0x7fffffc0};
    const ll rows = (((ll)max_rows + segs - 1) / segs + 63) / 64 * 64;
    return {(int)(((ll)max_rows + rows - 1) / rows), (int)rows};
}

template <typename S, int DK, int NW, bool FAST>
int launch_prefill(const PrefillArgs<S>& a, int batch, hipStream_t stream) {
    const dim3 grid((unsigned)((ll)a.heads * a.segs), (unsigned)batch);
    if (a.segs > 1) {
        segment_kernel<S, DK, NW, FAST, true, false><<<grid, 64 * NW, 0, stream>>>(a);
        starts_kernel<S, DK, NW><<<dim3((unsigned)a.heads, (unsigned)batch, 2 * (DK / 16)), 64 * NW, 0, stream>>>(a);
    }
    if (a.segs == 1 && a.state_out == nullptr && a.most <= C)
        segment_kernel<S, DK, NW, FAST, false, true><<<grid, 64 * NW, 0, stream>>>(a);
    else
        segment_kernel<S, DK, NW, FAST, false, false><<<grid, 64 * NW, 0, stream>>>(a);
    return launched();
}

template <typename S, int DK>
int launch_prefill(const PrefillArgs<S>& a, int dv, bool fast, int batch, hipStream_t stream) {
    if (dv == 64) return fast ? launch_prefill<S, DK, 2, true>(a, batch, stream) : launch_prefill<S, DK, 2, false>(a, batch, stream);
    return fast ? launch_prefill<S, DK, 4, true>(a, batch, stream) : launch_prefill<S, DK, 4, false>(a, batch, stream);
}

inline bool whole_pieces(const void* p, ll stride) { return aligned(p, 16) && stride % 8 == 0; }

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
    const bool fast = whole_pieces(r.q, r.q_stride) && whole_pieces(r.k, r.k_stride) && whole_pieces(r.v, r.v_stride);
    return dk == 64 ? launch_prefill<S, 64>(a, dv, fast, batch, stream) : launch_prefill<S, 128>(a, dv, fast, batch, stream);
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
