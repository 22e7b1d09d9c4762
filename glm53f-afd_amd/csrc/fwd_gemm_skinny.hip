// BF16 weight GEMM for 9 to 64 rows (gfx950): the projections of a decode or verify step with more rows than the
// GEMV takes. Like the GEMV it is bound by the weight stream - every weight byte is read from HBM once with 128-bit
// nontemporal loads - but the arithmetic runs on the matrix cores: with sixteen rows a weight piece of 1 KiB is one
// v_mfma_f32_16x16x32_bf16, so the vector units, which bound the GEMV from five rows up, do nothing here.
//
// The reference has no kernel for this range: its engine calls the vendor GEMM above 8 rows (crates/glm53f-forward/
// src/gemm.rs:228-234, :293-325). What this replaces there is that call, for 9..64 rows.
//
// Numerics: exact bf16 products, f32 accumulation on the matrix core over K in steps of 32 inside a wave's K range,
// the ranges of a workgroup's waves added in wave order; bf16 outputs rounded to nearest even. A row's result does
// not depend on the rows beside it or on their number. No bit-level contract (the reference has none above 8 rows: its own test holds
// the vendor GEMM to the GEMV within f32 rounding).
//
// The kernel is stream_kernel of fwd_stream.h; this file chooses its shape.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fwd_stream.h"
#include "glm53f_fwd_gemv.h"

namespace fwd_gemm {
namespace {

constexpr int kInvalid = 1;                       // hipErrorInvalidValue
constexpr int kCus = 256;

// The bare product: four outputs as f32, or as bf16 in two accesses.
struct Plain {
    void* out;
    int out_f32;
    long long ldo, o_gs;
    __device__ __forceinline__ void operator()(int g, int row, int o, fwd_stream::f32x4 s) const {
        if (out_f32) {
            float* dst = static_cast<float*>(out) + g * o_gs + (long long)row * ldo + o;
            dst[0] = s[0]; dst[1] = s[1]; dst[2] = s[2]; dst[3] = s[3];
        } else {
            uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(out) + g * o_gs + (long long)row * ldo + o);
            dst[0] = fwd_stream::f2bf2(s[0], s[1]);
            dst[1] = fwd_stream::f2bf2(s[2], s[3]);
        }
    }
};

struct Args {
    const uint16_t* x; long long ldx, x_gs;
    const uint16_t* w; long long ldw, w_gs;
    int groups, rows, n, k;
    void* out; int out_f32; long long ldo, o_gs;
    hipStream_t stream;
};

template <int CK, int NT, int T, int KS>
int32_t launch(const Args& a) {
    const dim3 grid((unsigned)((a.n / 16 + T - 1) / T), (unsigned)((a.rows + 16 * NT - 1) / (16 * NT)), (unsigned)a.groups);
    fwd_stream::stream_kernel<CK, NT, T, KS, false, Plain><<<grid, 64 * KS, 0, a.stream>>>(
        a.x, a.ldx, a.x_gs, a.w, a.ldw, a.w_gs, a.rows, a.n, a.k, Plain{a.out, a.out_f32, a.ldo, a.o_gs});
    return (int32_t)hipGetLastError();
}

// T: the power of two (at most TMAX) that brings the grid nearest to one workgroup per CU from above.
template <int CK, int NT, int KS, int TMAX>
int32_t launch_tiles(const Args& a) {
    const long long tiles = (long long)(a.n / 16) * a.groups;
    if constexpr (TMAX >= 8) if (tiles > 4 * kCus) return launch<CK, NT, 8, KS>(a);
    if constexpr (TMAX >= 4) if (tiles > 2 * kCus) return launch<CK, NT, 4, KS>(a);
    if constexpr (TMAX >= 2) if (tiles > kCus) return launch<CK, NT, 2, KS>(a);
    return launch<CK, NT, 1, KS>(a);
}

// The K split depends on n and k alone, so a row's bits do not change with the number of rows beside it: eight waves
// where the grid is at most one workgroup per CU even at one tile each (more loads in flight per CU), four otherwise,
// one where the K range is too short to split into chunks. The chunk is 256 k where the wave's range is a multiple
// of it and, with eight waves, where sixteen rows leave the registers for it; with four waves the workgroup may
// run alone on its CU (eight weight tiles x four row tiles: 426 registers, the accumulators in the AGPRs), which
// pays because the activations' L2 traffic falls with the tiles per workgroup: 4096 -> 24,640 with 64 rows
// 38 us at eight tiles against 45 at four.
template <int NT, int TMAX>
int32_t launch_split(const Args& a) {
    const long long tiles = (long long)(a.n / 16) * a.groups;
    if (tiles <= kCus && a.k % (8 * 128) == 0) {
        // A weight so small that a workgroup per tile and per sixteen rows still leaves CUs free (the gates' first
        // projection: 16 tiles) is bound by a wave's chain of items, not by bytes: the row tiles go to workgroups of
        // their own, which re-read the weight from the L2 (4096 -> 256 with 64 rows: 11 -> 6 us).
        if (a.k % (8 * 256) == 0 && (NT == 1 || tiles * NT <= kCus)) return launch<256, 1, 1, 8>(a);
        return launch<128, NT, 1, 8>(a);
    }
    if (a.k % (4 * 128) == 0) {
        if (a.k % (4 * 256) == 0) return launch_tiles<256, NT, 4, 8>(a);
        return launch_tiles<128, NT, 4, TMAX>(a);
    }
    return launch_tiles<128, NT, 1, TMAX>(a);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace fwd_gemm

extern "C" int32_t glm53f_fwd_gemm_bf16_skinny(const uint16_t* x, int64_t ldx, int64_t x_gstride, const uint16_t* w,
                                               int64_t ldw, int64_t w_gstride, int32_t groups, int32_t rows, int32_t n,
                                               int32_t k, void* out, int32_t out_f32, int64_t ldo, int64_t o_gstride,
                                               ihipStream_t* stream) {
    using namespace fwd_gemm;
    if (groups < 1 || groups > 65535 || rows < 1 || rows > 64 || n < 16 || n % 16 || k < 128 || k % 128) return kInvalid;
    if (!x || !w || !out || !aligned16(x) || !aligned16(w) || ldx % 8 || ldw % 8 || x_gstride % 8 || w_gstride % 8 ||
        ldx < k || ldw < k || ldo < n)
        return kInvalid;
    // bf16 outputs are stored two at a time (32 bits), f32 outputs one at a time
    if (!out_f32 && ((reinterpret_cast<uintptr_t>(out) & 3u) || ldo % 2 || o_gstride % 2)) return kInvalid;
    if (out_f32 && (reinterpret_cast<uintptr_t>(out) & 3u)) return kInvalid;
    const Args a{x, ldx, x_gstride, w, ldw, w_gstride, groups, rows, n, k, out, out_f32, ldo, o_gstride, stream};
    switch ((rows + 15) / 16) {                   // (the last argument bounds T where the chunk is 128 k)
        case 1: return launch_split<1, 8>(a);
        case 2: return launch_split<2, 4>(a);
        default: return launch_split<4, 4>(a);    // 33 to 48 rows too: a third tile's seven items per chunk need more
                                                  // registers than a fourth tile of repeated rows costs
    }
}
