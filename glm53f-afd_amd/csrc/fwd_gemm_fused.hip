// BF16 matrix product with bias, activation and residual in its epilogue (gfx950).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ext/glm53f_fwd_gemm.h"
#include "fwd_epilogue.h"

namespace fwd_fused {
namespace {

using fwd_epilogue::Epilogue;

constexpr int kInvalid = 1;                       // hipErrorInvalidValue

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const uint16_t* x;
    long long ldx, x_gs;
    const uint16_t* w;
    long long ldw, w_gs;
    int rows, n, k;
    Epilogue e;
};

// Any size, any stride: a workgroup of four waves owns 64 rows x 64 outputs, both operands pass through LDS in steps of
// 32 along k, zero beyond the edges. VEC: rows are read in pieces of 16 bytes.
template <bool VEC>
__global__ void __launch_bounds__(256) any_kernel(const Args a) {
    constexpr int BM = 64, BN = 64, BK = 32, LD = BK + 8;
    __shared__ __align__(16) uint16_t xs[BM * LD], ws[BN * LD];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, g = blockIdx.z;
    const long long m0 = (long long)blockIdx.y * BM;
    const int n0 = blockIdx.x * BN, tr = t >> 2, tc = (t & 3) * 8;
    const bool xin = m0 + tr < a.rows, win = n0 + tr < a.n;
    const uint16_t* x = a.x + g * a.x_gs + (xin ? m0 + tr : 0) * a.ldx;
    const uint16_t* w = a.w + g * a.w_gs + (long long)(win ? n0 + tr : 0) * a.ldw;
    auto piece = [&](const uint16_t* src, bool in, int k0) {
        u32x4 p = {0, 0, 0, 0};
        if (in) {
            if constexpr (VEC) {
                if (k0 < a.k) p = *reinterpret_cast<const u32x4*>(src + k0);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + i < a.k) p[i / 2] |= (uint32_t)src[k0 + i] << (16 * (i & 1));
            }
        }
        return p;
    };
    f32x4 acc[2][2] = {};
    const int mw = (wave & 1) * 32, nw = (wave >> 1) * 32;
    for (int k0 = 0; k0 < a.k; k0 += BK) {
        const u32x4 px = piece(x, xin, k0 + tc), pw = piece(w, win, k0 + tc);
        __syncthreads();
        *reinterpret_cast<u32x4*>(&xs[tr * LD + tc]) = px;
        *reinterpret_cast<u32x4*>(&ws[tr * LD + tc]) = pw;
        __syncthreads();
        bf16x8 fx[2], fw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fx[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(&xs[(mw + 16 * i + (lane & 15)) * LD + 8 * (lane >> 4)]));
            fw[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(&ws[(nw + 16 * i + (lane & 15)) * LD + 8 * (lane >> 4)]));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[j], fx[i], acc[i][j], 0, 0, 0);
    }
    // acc[i][j][c]: row 16 i + lane % 16, output 16 j + 4 (lane / 16) + c of the wave's tile
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const long long m = m0 + mw + 16 * i + (lane & 15);
                const int o = n0 + nw + 16 * j + 4 * (lane >> 4) + c;
                if (m < a.rows && o < a.n) fwd_epilogue::finish(a.e, g, m, o, acc[i][j][c]);
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
    if (groups < 1 || groups > 65535 || rows < 0 || n < 1 || k < 1 || act < GLM53F_ACT_NONE || act > GLM53F_ACT_SIGMOID)
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
    const Args a{x, ldx, x_gstride, w, ldw, w_gstride, rows, n, k,
                 Epilogue{bias, b_gstride, act, residual, ldr, r_gstride, out, out_f32, ldo, o_gstride}};
    const bool vec = aligned(x, 16) && aligned(w, 16) && ldx % 8 == 0 && ldw % 8 == 0 && x_gstride % 8 == 0 &&
                     w_gstride % 8 == 0 && k % 8 == 0;
    const unsigned row_tiles = ((unsigned)rows + 63) / 64, col_tiles = ((unsigned)n + 63) / 64;
    if (row_tiles > 65535) return kInvalid;
    const dim3 grid(col_tiles, row_tiles, (unsigned)groups);
    if (vec)
        any_kernel<true><<<grid, 256, 0, stream>>>(a);
    else
        any_kernel<false><<<grid, 256, 0, stream>>>(a);
    return (int32_t)hipGetLastError();
}
