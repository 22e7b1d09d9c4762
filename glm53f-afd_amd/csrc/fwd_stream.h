// The weight-streaming BF16 product for up to 64 rows a workgroup (gfx950): the projections of a decode or verify step with
// more rows than the GEMV takes. Like the GEMV it is bound by the weight stream - every weight byte is read from HBM once with 128-bit
// nontemporal loads - but the arithmetic runs on the matrix cores: with sixteen rows a weight piece of 1 KiB is one
// v_mfma_f32_16x16x32_bf16, so the vector units, which bound the GEMV from five rows up, do nothing here.
//
// Shape of the work. A workgroup owns T tiles of sixteen outputs; its KS waves split the K range; a wave walks its
// range in chunks of CK. Both operands reach the matrix core's fragment layout (lane l: row l % 16, k = 8 (l / 16)
// .. + 7 of a step of 32) through LDS, because the layout's natural load - sixteen rows of 64 bytes per instruction
// - asks the texture path for 64 cache lines per KiB: a kernel that loads fragments directly, activations from the
// L2 in the same way, reaches 2.9 TB/s of weights on 4096 -> 24,640 with sixteen rows, this one 6.4 TB/s. Here
//   - a load instruction covers whole runs of a row (CK = 256: two rows of 512 consecutive bytes, lanes 0..31 one
//     row, 32..63 the next; CK = 128: four rows of 256 bytes), CK / 32 of them a tile of sixteen rows x CK; the
//     wave writes the tile to its own LDS rows (2 CK + 16 bytes apart: a fragment read's sixteen rows then fall on
//     all 64 banks once) and reads it back as CK / 32 fragments. No workgroup barrier: a wave's LDS instructions
//     run in order, and the region is its own;
//   - the activations' tiles (NT of sixteen rows) go the same way once per chunk and stay in registers for the T
//     weight tiles, so their traffic from the L2 is NT / T of the weight stream;
//   - two sets of loads alternate over the items of a chunk (the NT activation tiles, then the T weight tiles):
//     the next item is requested before the current one is waited for.
// The launch takes T so that the grid is at most one workgroup per CU where the registers allow (measured: one
// round of 193 workgroups of four waves at T = 8 runs 4096 -> 24,640 in 31.3 us, 385 at T = 4 in 33.6, and 257 at
// T = 6 - one more than the CUs, so a second round of one - in 40.7).
#ifndef GLM53F_FWD_STREAM_H
#define GLM53F_FWD_STREAM_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fwd_stream {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(2)));   // at any element's address

__device__ __forceinline__ uint32_t f2bf2(float lo, float hi) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf2));
}

// Eight elements without the first `past` of them, zeros behind.
__device__ __forceinline__ u32x4 dropped(u32x4 v, int past) {
    uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
    if (past >= 4) lo = hi, hi = 0, past -= 4;
    if (past >= 4) return u32x4{0, 0, 0, 0};
    const int bits = 16 * past;
    if (bits) lo = lo >> bits | hi << (64 - bits), hi >>= bits;
    return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

template <int CK> struct Staged {
    static constexpr int N8 = CK / 32;            // loads of an item = fragments of an item
    static constexpr int LANES = CK / 8;          // lanes that cover one row's CK elements with 16 bytes each
    static constexpr int ROW = 2 * CK + 16;       // bytes between a staged tile's rows
    static constexpr int BYTES = 16 * ROW;        // a wave's staging region
};

// CK: k per chunk. NT: tiles of sixteen rows (rows <= 16 NT). T: tiles of sixteen outputs per workgroup. KS: waves
// of a workgroup, each with k / KS of the K range (a multiple of CK). Store: what becomes of four consecutive outputs of a
// row. ANY: every n, every k from 8 on, rows at any address: a weight row past the last repeats it, the waves share
// whole chunks, and in the last chunk a lane whose piece crosses the end of the row loads the row's last piece and shifts
// it, zeros behind. Its weights' rows share cache lines between chunks, so they are not loaded past the caches (sixteen rows
// 4104 -> 24,640 42 us, 45 past them; 1 row 4097 -> 4096 9.2 and 10.4).
template <int CK, int NT, int T, int KS, bool ANY, typename Store>
__global__ void __launch_bounds__(64 * KS) stream_kernel(const uint16_t* __restrict__ x, long long ldx, long long x_gs,
                                                         const uint16_t* __restrict__ w, long long ldw, long long w_gs,
                                                         int rows, int n, int k, const Store store) {
    using S = Staged<CK>;
    constexpr int N8 = S::N8, RPL = 64 / S::LANES, NI = NT + T;
    constexpr int PART = KS * T * NT * 1024;      // the partial tiles reuse the staging regions
    constexpr int LDS_BYTES = KS * S::BYTES > PART ? KS * S::BYTES : PART;
    __shared__ __align__(16) unsigned char lds[LDS_BYTES];
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int g = blockIdx.z, tiles = ANY ? (n + 15) / 16 : n / 16, tile0 = blockIdx.x * T;
    const int row0 = blockIdx.y * (16 * NT);      // gridDim.y > 1: the rows in groups of 16 NT, a workgroup each
    rows = min(rows - row0, 16 * NT);
    const int all = (k + CK - 1) / CK;            // ANY: chunks of the whole range, the waves' shares differ by one at most
    const int lo = ANY ? CK * (int)((long long)all * wave / KS) : wave * (k / KS);
    const int chunks = ANY ? (int)((long long)all * (wave + 1) / KS) - lo / CK : k / KS / CK;
    const int lrow = lane / S::LANES, lcol = 8 * (lane % S::LANES);
    unsigned char* stage = lds + wave * S::BYTES;
    unsigned char* put = stage + lrow * S::ROW + 2 * lcol;                        // + RPL j rows
    const unsigned char* get = stage + (lane & 15) * S::ROW + 16 * (lane >> 4);   // + 64 s

    // items 0 .. NT - 1 of a chunk: the activations' tiles (a row past the end repeats the last one: its column
    // is not stored); item NT + i: weight tile i of this workgroup (a tile past the last repeats it, not stored)
    const uint16_t* xsrc = x + g * x_gs + (long long)row0 * ldx + (ANY ? 0 : lo + lcol);
    const uint16_t* wsrc = w + g * w_gs + (ANY ? 0 : (long long)lrow * ldw + lo + lcol);
    auto request = [&](u32x4 (&set)[N8], int item, int c) {
        if constexpr (ANY) {
            const int col = min(lo + CK * c + lcol, k - 8);
            if (item < NT) {
#pragma unroll
                for (int j = 0; j < N8; ++j)
                    set[j] = *reinterpret_cast<const u32x4_any*>(xsrc + (long long)min(16 * item + RPL * j + lrow, rows - 1) * ldx + col);
            } else {
                const int row = 16 * min(tile0 + item - NT, tiles - 1) + lrow;
#pragma unroll
                for (int j = 0; j < N8; ++j)
                    set[j] = *reinterpret_cast<const u32x4_any*>(wsrc + (long long)min(row + RPL * j, n - 1) * ldw + col);
            }
        } else if (item < NT) {
#pragma unroll
            for (int j = 0; j < N8; ++j)
                set[j] = *reinterpret_cast<const u32x4*>(xsrc + (long long)min(16 * item + RPL * j + lrow, rows - 1) * ldx + CK * c);
        } else {
            const uint16_t* src = wsrc + (long long)(16 * min(tile0 + item - NT, tiles - 1)) * ldw + CK * c;
#pragma unroll
            for (int j = 0; j < N8; ++j)
                set[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + (long long)(RPL * j) * ldw));
        }
    };
    auto fragments = [&](u32x4 (&set)[N8], u32x4 (&frag)[N8], int c) {
        if constexpr (ANY) {
            if (lo + CK * (c + 1) > k) {          // the row's last chunk: entries past its end are zeros
                const int past = max(lo + CK * c + lcol - (k - 8), 0);
#pragma unroll
                for (int j = 0; j < N8; ++j) set[j] = dropped(set[j], past);
            }
        }
#pragma unroll
        for (int j = 0; j < N8; ++j) *reinterpret_cast<u32x4*>(put + RPL * j * S::ROW) = set[j];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < N8; ++s) frag[s] = *reinterpret_cast<const u32x4*>(get + 64 * s);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };

    f32x4 acc[T][NT];
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[i][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    u32x4 xf[NT][N8];

    // One chunk: `first` holds (or has in flight) the chunk's item 0, the sets alternate from there; the item
    // after the chunk's last (the next chunk's item 0; after the last chunk a repeat, not used) goes to the set
    // that the next call names `first`.
    auto chunk = [&](u32x4 (&first)[N8], u32x4 (&second)[N8], int c) {
#pragma unroll
        for (int item = 0; item < NI; ++item) {
            u32x4 (&cur)[N8] = (item & 1) ? second : first;
            u32x4 (&nxt)[N8] = (item & 1) ? first : second;
            if (item + 1 < NI) request(nxt, item + 1, c);
            else request(nxt, 0, ANY ? c + 1 : min(c + 1, chunks - 1));
            if (item < NT) {
                fragments(cur, xf[item], c);
            } else {
                u32x4 wf[N8];
                fragments(cur, wf, c);
#pragma unroll
                for (int s = 0; s < N8; ++s)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        f32x4& a = acc[item - NT][nt];
                        a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wf[s]),
                                                                    __builtin_bit_cast(bf16x8, xf[nt][s]), a, 0, 0, 0);
                    }
            }
        }
    };
    u32x4 sa[N8], sb[N8];
    request(sa, 0, 0);
    if constexpr (NI % 2 == 0) {                  // an even number of items: every chunk starts on the same set
        for (int c = 0; c < chunks; ++c) chunk(sa, sb, c);
    } else {
        int c = 0;
        for (; c + 1 < chunks; c += 2) {
            chunk(sa, sb, c);
            chunk(sb, sa, c + 1);
        }
        if (c < chunks) chunk(sa, sb, c);
    }

    // acc[i][nt][e] = C[output 16 (tile0 + i) + 4 (lane / 16) + e][row 16 nt + lane % 16]: the waves' partial tiles,
    // added in wave order (the staging regions are free once every wave has left the loop)
    float* part = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<f32x4*>(&part[(((wave * T + i) * NT + nt) * 64 + lane) * 4]) = acc[i][nt];
    __syncthreads();
    for (int e = t; e < T * NT * 64; e += 64 * KS) {
        const int tn = e >> 6, l = e & 63, i = tn / NT, nt = tn % NT;
        f32x4 s = *reinterpret_cast<const f32x4*>(&part[(tn * 64 + l) * 4]);
#pragma unroll
        for (int kk = 1; kk < KS; ++kk) {
            const f32x4 p = *reinterpret_cast<const f32x4*>(&part[((kk * T * NT + tn) * 64 + l) * 4]);
            s = f32x4{s[0] + p[0], s[1] + p[1], s[2] + p[2], s[3] + p[3]};
        }
        const int row = 16 * nt + (l & 15), o = 16 * (tile0 + i) + 4 * (l >> 4);
        if (row >= rows || tile0 + i >= tiles) continue;
        store(g, row0 + row, o, s);
    }
}

}  // namespace fwd_stream

#endif
