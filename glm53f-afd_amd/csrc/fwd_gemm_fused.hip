// BF16 matrix product with bias, activation and residual in its epilogue (gfx950), for any rows, n and k.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ext/glm53f_fwd_gemm.h"
#include "fwd_epilogue.h"
#include "fwd_stream.h"

namespace fwd_fused {
namespace {

using fwd_epilogue::Epilogue;
using fwd_stream::bf16x8;
using fwd_stream::dropped;
using fwd_stream::f32x4;
using fwd_stream::u32x4;
using fwd_stream::u32x4_any;

constexpr int kInvalid = 1;                       // hipErrorInvalidValue
constexpr int kCus = 256;
constexpr int kMostSize = 1 << 30;                // of rows, n and k: tiles' counts and ends stay below 2^31

struct Args {
    const uint16_t* x;
    long long ldx, x_gs;
    const uint16_t* w;
    long long ldw, w_gs;
    int groups, rows, n, k;
    Epilogue e;
    hipStream_t stream;
};

// What the streaming kernel's four outputs become.
struct Finish {
    Epilogue e;
    int n;
    __device__ __forceinline__ void operator()(int g, int row, int o, f32x4 s) const {
        fwd_epilogue::finish(e, fwd_epilogue::request(e, g, row, o, n), g, row, o, n, s);
    }
};

// ------------------------------------------------------------------------------------------------------- tiles

// 16 bytes per lane from global memory to LDS without a register in between: to lds + 16 lane (lds the same in all lanes).
// Written out because the compiler cannot tell the two sets of tiles apart and has every read of one wait for the
// loads of the other; whoever reads the set waits for its loads himself, before a barrier.
__device__ __forceinline__ void to_lds(const uint16_t* src, uint16_t* lds) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(at) : "memory");
}

// BM rows x BN outputs per workgroup of WM x WN waves, k in steps of BK, a ring of STAGES sets of LDS tiles: the steps ahead
// are requested before the current one's products, STAGES - 1 of them. A tile row is BK / 8 pieces of 16 bytes in LDS,
// swizzled by the row so that the sixteen rows of an operand's read fall on all banks. With 16-byte aligned rows and k a
// multiple of 8 (FAST) the tiles go straight to LDS, the swizzle in the lanes' addresses, and where k is no multiple of BK
// (TAIL) the pieces behind the rows' ends come from a piece of zeros (2048 rows 8200 -> 4096 136 us, through registers 163; 200
// rows 4104 -> 4096 23 and 31; 1024 rows, whose stride parts every row's run over two lines, 59 and 57); otherwise through
// registers, a piece that crosses the row's end shifted and filled with zeros. Rows past the last repeat it and are not
// stored.
__device__ const u32x4 kZeros[1] = {};

template <int BM, int BN, int WM, int WN, int KW, int BK, int STAGES, bool FAST, bool TAIL>
__global__ void __launch_bounds__(64 * WM * WN * KW) tile_kernel(const Args a) {
    constexpr int T = 64 * WM * WN * KW, MT = BM / WM / 16, NT = BN / WN / 16, PR = BK / 8;
    constexpr int XP = BM * PR / T, WP = BN * PR / T, P = XP + WP;   // pieces per thread of a step
    constexpr int AHEAD = FAST ? 1 : STAGES - 1;                     // steps that registers hold
    static_assert(XP * T == BM * PR && WP * T == BN * PR, "whole pieces");
    constexpr int SETS = FAST ? STAGES : 2, SET = (BM + BN) * BK;
    constexpr int PASSES = KW * BM * BN * 4 > (128 << 10) ? 2 : 1, ROWS = BM / PASSES;   // the outputs take the tiles' place, in passes
    constexpr bool DIRECT = KW == 1 && MT * NT <= 16;                // a wave's outputs stored as they lie
    constexpr int CELLS = DIRECT || SETS * SET > KW * ROWS * BN * 2 ? SETS * SET : KW * ROWS * BN * 2;
    constexpr int SPARE = FAST ? T * 8 : 0;               // where the residual's early requests go
    __shared__ __align__(16) uint16_t lds[CELLS + SPARE];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), g = blockIdx.z;
    // Consecutive workgroups go to the eight XCDs in turn: give each XCD a run of tiles, and order the tiles in bands of
    // eight rows of tiles, column by column, so that the tiles that run at a time on an XCD are a block of both operands
    // and its L2 serves most of what they read.
    constexpr unsigned BAND = 8;
    const unsigned row_tiles = (unsigned)((a.rows + (long long)BM - 1) / BM), col_tiles = (unsigned)((a.n + (long long)BN - 1) / BN);
    const unsigned total = gridDim.x, per = total / 8, id = blockIdx.x;
    const unsigned tile = id < per * 8 ? (id % 8) * per + id / 8 : id;
    const unsigned band = tile / (BAND * col_tiles), in_band = tile % (BAND * col_tiles), high = min(BAND, row_tiles - band * BAND);
    const long long m0 = (long long)(band * BAND + in_band % high) * BM;
    const int n0 = (int)(in_band / high) * BN;
    const uint16_t* x = a.x + g * a.x_gs;
    const uint16_t* w = a.w + g * a.w_gs;

    // piece i of this thread: LDS slot i T + t, row slot / PR, piece (slot mod PR) ^ swizzle of the step
    auto swizzle = [](int row) { return PR >= 8 ? (row >> 1) & 7 : (row >> 2) & 3; };
    const uint16_t* src[P];
    int col[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int slot = (i < XP ? i : i - XP) * T + t, row = slot / PR;
        col[i] = 8 * ((slot & (PR - 1)) ^ swizzle(row));
        src[i] = i < XP ? x + min(m0 + row, (long long)a.rows - 1) * a.ldx : w + (long long)min(n0 + row, a.n - 1) * a.ldw;
    }
    const int steps = (a.k + BK - 1) / BK;
    u32x4 held[AHEAD][FAST ? 1 : P];
    auto slot_of = [&](int i, int set) { return lds + set * SET + (i < XP ? i * T * 8 : BM * BK + (i - XP) * T * 8); };
    auto request_piece = [&](int i, int step, int set) {   // (behind the last step it is requested again: the waits count requests)
        step = min(step, steps - 1);
        const uint16_t* from = src[i] + step * BK + col[i];
        if constexpr (TAIL) from = step * BK + col[i] < a.k ? from : reinterpret_cast<const uint16_t*>(kZeros);
        if constexpr (FAST)
            to_lds(from, slot_of(i, set) + wave * 512);
        else
            held[set][i] = *reinterpret_cast<const u32x4_any*>(src[i] + min(step * BK + col[i], a.k - 8));
    };
    auto request = [&](int step, int set) {
#pragma unroll
        for (int i = 0; i < P; ++i) request_piece(i, step, set);
    };
    auto place = [&](int step, int from, int set) {   // the registers' pieces
        if constexpr (!FAST) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (step >= steps - 1) held[from][i] = dropped(held[from][i], max((steps - 1) * BK + col[i] - (a.k - 8), 0));
                *reinterpret_cast<u32x4*>(slot_of(i, set) + t * 8) = held[from][i];
            }
        }
    };
    f32x4 acc[MT][NT] = {};
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) % WN * (BN / WN), wk = wave / (WM * WN), r16 = lane & 15, q = lane >> 4;

    // One step's products; `between` is called P times, spread over them.
    auto products = [&](int set, auto between) {
        const uint16_t* xs = lds + set * SET + (wm + r16) * BK;
        const uint16_t* ws = lds + set * SET + BM * BK + (wn + r16) * BK;
        constexpr int KK = BK / 32 / KW, GROUPS = KK * MT;
        bf16x8 fx[KK][MT], fw[KK][NT];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int at = 8 * ((4 * (wk * KK + kk) + q) ^ swizzle(r16));
#pragma unroll
            for (int j = 0; j < NT; ++j) fw[kk][j] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(ws + 16 * j * BK + at));
#pragma unroll
            for (int i = 0; i < MT; ++i) fx[kk][i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(xs + 16 * i * BK + at));
        }
        if constexpr (FAST) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[kk][j], fx[kk][i], acc[i][j], 0, 0, 0);
                if constexpr (FAST) {
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int m = (kk * MT + i) * P / GROUPS; m < (kk * MT + i + 1) * P / GROUPS; ++m) between(m);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
    };
    // The residual's tile is asked for during the last steps, into a corner that nobody reads: the epilogue then finds it in the
    // caches (2048 rows 8192 -> 4096 134 -> 132 us, 129 without a residual; 1024 -> 4096 34.6 -> 33.1; 4096 rows 4096 -> 8192
    // 318 -> 298; 256 rows 4096 -> 4096 22.1 -> 21.2).
    const int res = a.e.early ? (a.e.out_f32 ? BM * BN / 4 / T : BM * BN / 8 / T) : 0, res_from = max(steps - res - 4, 0);
    auto early = [&](int step) {
        const int i = step - res_from, per = a.e.out_f32 ? 4 : 8, slot = i * T + t;
        if (i < 0 || i >= res) return;
        const long long row = min(m0 + slot / (BN / per), (long long)a.rows - 1);
        const int o = min(n0 + slot % (BN / per) * per, (a.n - per) & -per);
        const long long cell = g * a.e.r_gs + row * a.e.ldr + o;
        to_lds(static_cast<const uint16_t*>(a.e.residual) + (a.e.out_f32 ? 2 * cell : cell), lds + CELLS + wave * 512);
    };
    if constexpr (FAST && BK == 32) {
        // The operands of the next step are read while the current one's products run.
        bf16x8 f[2][MT + NT];
        auto read = [&](int set, bf16x8 (&to)[MT + NT]) {
            const uint16_t* xs = lds + set * SET + (wm + r16) * BK + 8 * (q ^ swizzle(r16));
            const uint16_t* ws = lds + set * SET + BM * BK + (wn + r16) * BK + 8 * (q ^ swizzle(r16));
#pragma unroll
            for (int i = 0; i < MT; ++i) to[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(xs + 16 * i * BK));
#pragma unroll
            for (int j = 0; j < NT; ++j) to[MT + j] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(ws + 16 * j * BK));
        };
        auto multiply = [&](const bf16x8 (&by)[MT + NT]) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(by[MT + j], by[i], acc[i][j], 0, 0, 0);
        };
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) request(s, s);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(P * (STAGES - 2)) : "memory");
        __syncthreads();
        read(0, f[0]);
        int set = 0;
        auto step = [&](int s, const bf16x8 (&now)[MT + NT], bf16x8 (&then)[MT + NT]) {
            // step s + 1 is there behind this barrier, and everybody has the operands of s - 1 in use: its set is filled anew
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(P * (STAGES - 3)) : "memory");
            __syncthreads();
            const int before = set == 0 ? STAGES - 1 : set - 1;
            set = set == STAGES - 1 ? 0 : set + 1;
            read(set, then);
            early(s);
            request(s + STAGES - 1, before);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
            multiply(now);
            __builtin_amdgcn_s_setprio(0);
        };
        int s = 0;
        for (; s + 1 < steps; s += 2) {
            step(s, f[0], f[1]);
            step(s + 1, f[1], f[0]);
        }
        if (s < steps) step(s, f[0], f[1]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else if constexpr (FAST) {
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) request(s, s);
        int set = 0;
        for (int s = 0; s < steps; ++s) {
            early(s);
            // this wave's part of the set is there once all but the newer steps' requests have come back; behind the
            // barrier everybody's is, and nobody reads the set before it any more, which the newest request fills
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(P * (STAGES - 2)) : "memory");
            __syncthreads();
            products(set, [&](int i) { request_piece(i, s + STAGES - 1, set == 0 ? STAGES - 1 : set - 1); });
            set = set == STAGES - 1 ? 0 : set + 1;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) request(s, s);
        place(0, 0, 0);
        request(AHEAD, 0);
        // LDS set s mod 2 holds step s; registers s + 1 .. s + AHEAD, step i in held[i mod AHEAD]
        for (int s0 = 0; s0 < steps; s0 += 2 * AHEAD) {
#pragma unroll
            for (int i = 0; i < 2 * AHEAD; ++i) {
                const int s = s0 + i;
                if (s >= steps) break;
                __syncthreads();
                products(i & 1, [](int) {});
                place(s + 1, (i + 1) % AHEAD, (i + 1) & 1);
                request(s + 1 + AHEAD, (i + 1) % AHEAD);
            }
        }
    }
    // acc[i][j][e]: row 16 i + lane % 16, output 16 j + 4 (lane / 16) + e of the wave's part. Where a wave has them whole and
    // the registers hold what is added to a row of tiles beside them, they are stored from there (2048 rows 2048 -> 4096 39.3 us,
    // through LDS 41.9; tiles of 256 x 256 spill).
    if constexpr (DIRECT) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const long long m = m0 + wm + 16 * i + r16;
            fwd_epilogue::Added added[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int o = n0 + wn + 16 * j + 4 * q;
                if (m < a.rows && o < a.n) added[j] = fwd_epilogue::request(a.e, g, m, o, a.n);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int o = n0 + wn + 16 * j + 4 * q;
                if (m < a.rows && o < a.n) fwd_epilogue::finish(a.e, added[j], g, m, o, a.n, acc[i][j]);
            }
        }
        return;
    }
    // Otherwise through LDS (pieces of four outputs, swizzled like the tiles), where the waves' parts of k meet and a wave stores
    // whole runs of a row.
    float* whole = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        __syncthreads();
        if (PASSES == 1 || wm / ROWS == pass) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int row = wm - pass * ROWS + 16 * i + r16, piece = (wn + 16 * j) / 4 + q;
                    *reinterpret_cast<f32x4*>(&whole[wk * (ROWS * BN) + row * BN + 4 * (piece ^ (row & 7))]) = acc[i][j];
                }
        }
        __syncthreads();
        // several pieces at a time: their bias and residual are requested together
        constexpr int U = ROWS * BN / 4 / T < 4 ? ROWS * BN / 4 / T : 4;
        static_assert(ROWS * BN / 4 % (U * T) == 0, "whole rounds");
        for (int s0 = t; s0 < ROWS * BN / 4; s0 += U * T) {
            fwd_epilogue::Added added[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long m = m0 + pass * ROWS + (s0 + u * T) / (BN / 4);
                const int o = n0 + 4 * ((s0 + u * T) % (BN / 4));
                if (m < a.rows && o < a.n) added[u] = fwd_epilogue::request(a.e, g, m, o, a.n);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int row = (s0 + u * T) / (BN / 4), piece = (s0 + u * T) % (BN / 4);
                const long long m = m0 + pass * ROWS + row;
                const int o = n0 + 4 * piece;
                if (m >= a.rows || o >= a.n) continue;
                const float* at = &whole[row * BN + 4 * (piece ^ (row & 7))];
                f32x4 y = *reinterpret_cast<const f32x4*>(at);
#pragma unroll
                for (int k = 1; k < KW; ++k) y += *reinterpret_cast<const f32x4*>(at + k * (ROWS * BN));
                fwd_epilogue::finish(a.e, added[u], g, m, o, a.n, y);
            }
        }
    }
}

// k below eight: one output per lane.
__global__ void __launch_bounds__(256) short_kernel(const Args a) {
    const int o = blockIdx.x * 256 + threadIdx.x, g = blockIdx.z;
    if (o >= a.n) return;
    for (long long m = blockIdx.y; m < a.rows; m += gridDim.y) {
        float y = 0.0f;
        for (int i = 0; i < a.k; ++i)
            y += fwd_epilogue::widen(a.x[g * a.x_gs + m * a.ldx + i]) * fwd_epilogue::widen(a.w[g * a.w_gs + (long long)o * a.ldw + i]);
        fwd_epilogue::finish(a.e, fwd_epilogue::request(a.e, g, m, o, o + 1), g, m, o, o + 1, f32x4{y, 0.0f, 0.0f, 0.0f});
    }
}

// ------------------------------------------------------------------------------------------------------- choices

template <int CK, int NT, int T, int KS, bool ANY>
int32_t stream(const Args& a) {
    const dim3 grid((unsigned)(((a.n + 15) / 16 + T - 1) / T), (unsigned)((a.rows + 16 * NT - 1) / (16 * NT)), (unsigned)a.groups);
    fwd_stream::stream_kernel<CK, NT, T, KS, ANY, Finish>
        <<<grid, 64 * KS, 0, a.stream>>>(a.x, a.ldx, a.x_gs, a.w, a.ldw, a.w_gs, a.rows, a.n, a.k, Finish{a.e, a.n});
    return (int32_t)hipGetLastError();
}

// The weight tiles per workgroup: the power of two (TMIN to TMAX) that brings the grid nearest to one workgroup per CU
// from above.
template <int CK, int NT, int KS, int TMIN, int TMAX, bool ANY>
int32_t stream_tiles(const Args& a) {
    const long long tiles = (long long)((a.n + 15) / 16) * a.groups;
    if constexpr (TMAX >= 8) if (tiles > 4 * kCus) return stream<CK, NT, 8, KS, ANY>(a);
    if constexpr (TMAX >= 4) if (tiles > 2 * kCus) return stream<CK, NT, 4, KS, ANY>(a);
    if constexpr (TMIN < 2) if (tiles > kCus) return stream<CK, NT, 2, KS, ANY>(a);
    return stream<CK, NT, TMIN, KS, ANY>(a);
}

// The waves per workgroup, which split k: eight where one tile each is at most a workgroup per CU and k is 1024 at least, four
// otherwise, one below 512; chunks of 256 where every wave has whole ones. The aligned form's waves have equal shares of whole
// chunks (whole_shares); the form for any address cuts the chunks as evenly as they go.
template <int NT, int TMAX, bool ANY>
int32_t stream_split(const Args& a) {
    const long long tiles = (long long)((a.n + 15) / 16) * a.groups;
    if (tiles <= kCus && (ANY ? a.k >= 1024 : a.k % 1024 == 0)) {
        // (sixteen rows a workgroup where they still are at most one per CU: 192 rows 2048 -> 1024 10.8 us otherwise, 7.7 so)
        const long long row_tiles = a.rows <= 64 ? NT : (a.rows + 15) / 16;
        if constexpr (!ANY) if (a.k % 2048 == 0 && (NT == 1 || tiles * row_tiles <= kCus)) return stream<256, 1, 1, 8, ANY>(a);
        return stream<128, NT, 1, 8, ANY>(a);
    }
    if (ANY ? a.k >= 512 : a.k % 512 == 0) {
        if constexpr (!ANY) if (a.k % 1024 == 0) return stream_tiles<256, NT, 4, 2, 8, ANY>(a);   // (more tiles than CUs)
        return stream_tiles<128, NT, 4, 1, TMAX, ANY>(a);
    }
    return stream_tiles<128, NT, 1, 1, TMAX, ANY>(a);
}

// The aligned form would need fewer waves for other k, and loses more by that than it gains by its loads (us, aligned and any):
//   1, 16, 64 rows 11,008 -> 4096 with one wave   52 52 99    any  19 21 34
//   1, 16, 64 rows 640 -> 4096 with one wave      5.2 5.3 9.4      5.0 4.9 5.2
//   1, 16, 64 rows 5632 -> 2048 with four waves   9.9 10.0 18.3    6.7 7.1 12.8
//   1, 16, 64 rows 5632 -> 4096 with four waves   10.9 11.0 19.2   10.4 11.7 18.6
bool whole_shares(const Args& a) {
    const long long tiles = (long long)((a.n + 15) / 16) * a.groups;
    return a.k < 512 || a.k % (tiles <= kCus && a.k >= 1024 ? 1024 : 512) == 0;
}

template <bool ANY>
int32_t stream_rows(const Args& a) {
    if (a.rows <= 16) return stream_split<1, 8, ANY>(a);
    if (a.rows <= 32) return stream_split<2, 4, ANY>(a);
    return stream_split<4, 4, ANY>(a);
}

template <int BM, int BN, int WM, int WN, int KW, int BK, int STAGES, bool FAST, bool TAIL = false>
int32_t tiles(const Args& a) {
    const long long count = (long long)((a.rows + (long long)BM - 1) / BM) * ((a.n + (long long)BN - 1) / BN);
    if (count > 0x7fffffff) return kInvalid;
    tile_kernel<BM, BN, WM, WN, KW, BK, STAGES, FAST, TAIL>
        <<<dim3((unsigned)count, 1, (unsigned)a.groups), 64 * WM * WN * KW, 0, a.stream>>>(a);
    return (int32_t)hipGetLastError();
}

// The tile of a product of more than 64 rows. Each shape runs a workgroup per CU, and a step of 64 k takes it about the
// time of the table, larger tiles less per output (fewer bytes through the CU's load path per product, which bounds them)
// but in whole rounds of 256: the shape whose rounds take least time is launched. Measured 8192 -> 4096, us:
//   rows            128   256   512  1024  2048  4096        at any address  128   256   512  1024  2048
//   64 x 32          28    53   106   197   355   707                         45    75   138   239   445
//   64 x 64          36    40    73   130   236   469                         56    59    97   166   311
//   128 x 64         50    52    53    93   178   349                         96    92    90   152   256
//   128 x 128        73    72    73    75   146   286                        131   124   119   113   199
//   128 x 256       114   113   112   112   126   251                        209   199   193   183   172
//   256 x 256       198   220   215   206   202   239
enum Shape { k64x32, k64x64, k128x64, k128x128, k128x256, k256x256 };
Shape shape_of(const Args& a, bool fast) {
    constexpr struct { int bm, bn; double aligned, any; } table[] = {{64, 32, 0.20, 0.33},   {64, 64, 0.29, 0.43},   {128, 64, 0.39, 0.67},
                                                                     {128, 128, 0.56, 0.85}, {128, 256, 0.96, 1.31}, {256, 256, 1.85, 0.0}};
    int best = 0;
    double least = 1e300;
    for (int i = 0; i < (fast ? 6 : 5); ++i) {
        const double count = (double)((a.rows + (long long)table[i].bm - 1) / table[i].bm) *
                             (double)((a.n + (long long)table[i].bn - 1) / table[i].bn) * a.groups;
        const double time = (double)(long long)((count + kCus - 1) / kCus) * (fast ? table[i].aligned : table[i].any);
        if (time < least) least = time, best = i;
    }
    return (Shape)best;
}

template <bool TAIL>
int32_t aligned_tiles(const Args& a, Shape shape) {
    switch (shape) {
        case k64x32: return tiles<64, 32, 2, 2, 2, 128, 4, true, TAIL>(a);
        case k64x64: return tiles<64, 64, 2, 2, 2, 128, 4, true, TAIL>(a);
        case k128x64: return tiles<128, 64, 2, 1, 4, 128, 3, true, TAIL>(a);
        case k128x128: return tiles<128, 128, 2, 2, 2, 64, 4, true, TAIL>(a);
        case k128x256: return tiles<128, 256, 2, 4, 1, 64, 3, true, TAIL>(a);
        default: return tiles<256, 256, 2, 4, 1, 32, 4, true, TAIL>(a);
    }
}

int32_t tiled(const Args& a, bool fast) {
    const Shape shape = shape_of(a, fast);
    // whole steps are of 128 k with the narrow tiles, whose four waves share a step's k, of 64 with the others
    const bool narrow = shape <= k128x64;
    if (fast) return a.k % (narrow ? 128 : 64) == 0 ? aligned_tiles<false>(a, shape) : aligned_tiles<true>(a, shape);
    switch (shape) {
        case k64x32: return tiles<64, 32, 2, 1, 4, 128, 2, false>(a);
        case k64x64: return tiles<64, 64, 2, 2, 2, 128, 2, false>(a);
        case k128x64: return tiles<128, 64, 2, 2, 2, 64, 3, false>(a);
        case k128x128: return tiles<128, 128, 2, 2, 2, 64, 2, false>(a);
        default: return tiles<128, 256, 2, 4, 1, 64, 3, false>(a);
    }
}

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace
}  // namespace fwd_fused

extern "C" int32_t glm53f_fwd_gemm_bf16_fused(const uint16_t* x, int64_t ldx, int64_t x_gstride, const uint16_t* w,
                                              int64_t ldw, int64_t w_gstride, int32_t groups, int32_t rows, int32_t n,
                                              int32_t k, const uint16_t* bias, int64_t b_gstride, int32_t act,
                                              const void* residual, int64_t ldr, int64_t r_gstride, void* out,
                                              int32_t out_f32, int64_t ldo, int64_t o_gstride, ihipStream_t* stream) {
    using namespace fwd_fused;
    if (groups < 1 || groups > 65535 || rows < 0 || n < 1 || k < 1 || rows > kMostSize || n > kMostSize || k > kMostSize ||
        act < GLM53F_ACT_NONE || act > GLM53F_ACT_SIGMOID)
        return kInvalid;
    if (ldx < k || ldw < k || ldo < n || x_gstride < 0 || w_gstride < 0 || o_gstride < 0 ||
        (bias && b_gstride < 0) || (residual && (ldr < n || r_gstride < 0)))
        return kInvalid;
    if (rows == 0) return 0;
    const unsigned cell = out_f32 ? 4 : 2;
    if (!x || !w || !out || !aligned(x, 2) || !aligned(w, 2) || !aligned(bias, 2) || !aligned(out, cell) ||
        !aligned(residual, cell))
        return kInvalid;
    if (residual == out && (ldr != ldo || (groups > 1 && r_gstride != o_gstride))) return kInvalid;
    Args a{x, ldx, x_gstride, w, ldw, w_gstride, groups, rows, n, k,
           Epilogue{bias, b_gstride, act, residual, ldr, r_gstride, out, out_f32, ldo, o_gstride, 0}, stream};
    if (k < 8) {
        short_kernel<<<dim3((unsigned)((n + 255LL) / 256), (unsigned)(rows < 1024 ? rows : 1024), (unsigned)groups), 256, 0, stream>>>(a);
        return (int32_t)hipGetLastError();
    }
    const int per = out_f32 ? 4 : 8;
    a.e.early = residual && n >= per && aligned(residual, 16) && ldr % per == 0 && r_gstride % per == 0;
    const bool fast = aligned(x, 16) && aligned(w, 16) && ldx % 8 == 0 && ldw % 8 == 0 && x_gstride % 8 == 0 &&
                      w_gstride % 8 == 0;
    // Up to 64 rows the weights stream past the rows once; with up to 256 too where a workgroup per sixteen outputs and 64 rows is at
    // most one per CU and k is long enough for more than one wave (200 rows 4096 -> 512: 10.9 us against 13.1 with tiles; 128 rows
    // 8192 -> 2048 20.6 and 25.3, 11,008 -> 1024 20.9 and 27.9, 1001 -> 1024 6.1 and 7.8, 640 -> 2048 4.7 and 4.9; but 384 -> 1024 6.3
    // and 4.5, 136 -> 512 6.5 and 4.6).
    const long long thin = (long long)((n + 15LL) / 16) * ((rows + 63LL) / 64) * groups;
    if (rows <= 64 || (rows <= 256 && thin <= kCus && k >= 512))
        return fast && n % 16 == 0 && k % 128 == 0 && whole_shares(a) ? stream_rows<false>(a) : stream_rows<true>(a);
    return tiled(a, fast && k % 8 == 0);
}
