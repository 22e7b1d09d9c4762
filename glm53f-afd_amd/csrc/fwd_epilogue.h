// What follows a projection's product (gfx950): bias, activation and residual in f32, one rounding to the outputs' type.
#ifndef GLM53F_FWD_EPILOGUE_H
#define GLM53F_FWD_EPILOGUE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ext/glm53f_fwd_gemm.h"

namespace fwd_epilogue {

struct Epilogue {
    const uint16_t* bias;                         // NULL: none
    long long b_gs;
    int act;
    const void* residual;                         // NULL: none; of the outputs' type
    long long ldr, r_gs;
    void* out;
    int out_f32;
    long long ldo, o_gs;
    int early;                                    // the residual may be requested in 16-byte pieces
};

__device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// y * sigmoid(z), by the hardware's exp2 and reciprocal (one rounding of the last place each). exp(-z) overflows to
// infinity where the sigmoid is below the smallest f32: the product is then 0.
__device__ __forceinline__ float gated(float y, float z) {
    return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
}

// y Phi(y), with e^(x^2) erfc(x) / 2 = t (c0 + c1 t + .. + c8 t^8), t = 1 / (1 + 0.4 x) for x >= 0: the polynomial of least
// relative error over all x (weighted least squares, the weights raised where the error is largest), off by at most 1.3e-7 of the
// value, so that the far left, which keeps the factor e^(-x^2), stays accurate too. 333 rows 1001 -> 1999 take 12.1 us with it, as
// with five terms that are 5e-5 of the value off at y = -3; the library's erfc took 4 us more.
__device__ __forceinline__ float gelu(float y) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.4f * 0.70710678118654752f, fabsf(y), 1.0f));
    float p = __builtin_fmaf(0.0251339953f, t, -0.0914624855f);
    p = __builtin_fmaf(p, t, 0.0845619738f);
    p = __builtin_fmaf(p, t, -0.00282036117f);
    p = __builtin_fmaf(p, t, 0.070723772f);
    p = __builtin_fmaf(p, t, 0.0842687935f);
    p = __builtin_fmaf(p, t, 0.103921659f);
    p = __builtin_fmaf(p, t, 0.112834781f);
    p = __builtin_fmaf(p, t, 0.112837933f);
    const float half = p * t * __builtin_amdgcn_exp2f(y * y * -0.72134752044448170f);   // erfc(|y| / sqrt 2) / 2
    return y * (y < 0.0f ? half : 1.0f - half);
}

// The switch is on a kernel argument: every lane of the launch takes the same way.
__device__ __forceinline__ float activate(float y, int act) {
    switch (act) {
        case GLM53F_ACT_RELU: return y < 0.0f ? 0.0f : y;
        case GLM53F_ACT_SILU: return gated(y, y);
        case GLM53F_ACT_GELU: return gelu(y);
        case GLM53F_ACT_GELU_TANH: return gated(y, 1.5957691216057308f * (y + 0.044715f * y * y * y));   // (1 + tanh u) / 2 = sigmoid(2u)
        case GLM53F_ACT_SIGMOID: return gated(1.0f, y);
        default: return y;
    }
}

// Vectors at any address that their elements may have.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));

__device__ __forceinline__ f32x4 widen4(const void* p) {
    const u32x2_any v = *static_cast<const u32x2_any*>(p);
    return f32x4{__uint_as_float(v[0] << 16), __uint_as_float(v[0] & 0xffff0000u), __uint_as_float(v[1] << 16),
                 __uint_as_float(v[1] & 0xffff0000u)};
}

__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf2));
}

// What four outputs o .. o + 3 of a row take in, requested ahead of their use.
struct Added {
    f32x4 bias, residual;
};
__device__ __forceinline__ Added request(const Epilogue& e, int g, long long m, int o, int n) {
    const long long from = g * e.r_gs + m * e.ldr + o;
    Added a{{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    if (o + 4 <= n) {
        if (e.bias) a.bias = widen4(e.bias + g * e.b_gs + o);
        if (e.residual)
            a.residual = e.out_f32 ? (f32x4)*reinterpret_cast<const f32x4_any*>(static_cast<const float*>(e.residual) + from)
                                   : widen4(static_cast<const uint16_t*>(e.residual) + from);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (o + i >= n) continue;
            if (e.bias) a.bias[i] = widen(e.bias[g * e.b_gs + o + i]);
            if (e.residual)
                a.residual[i] = e.out_f32 ? static_cast<const float*>(e.residual)[from + i]
                                          : widen(static_cast<const uint16_t*>(e.residual)[from + i]);
        }
    }
    return a;
}

// Outputs o .. o + 3 of row m of group g, those below n, from their sums y.
__device__ __forceinline__ void finish(const Epilogue& e, const Added& a, int g, long long m, int o, int n, f32x4 y) {
    const long long at = g * e.o_gs + m * e.ldo + o;
    if (e.bias) y += a.bias;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = activate(y[i], e.act);
    if (e.residual) y += a.residual;
    if (o + 4 <= n) {
        if (e.out_f32) *reinterpret_cast<f32x4_any*>(static_cast<float*>(e.out) + at) = y;
        else *reinterpret_cast<u32x2_any*>(static_cast<uint16_t*>(e.out) + at) = u32x2_any{narrow2(y[0], y[1]), narrow2(y[2], y[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (o + i >= n) continue;
        if (e.out_f32) static_cast<float*>(e.out)[at + i] = y[i];
        else static_cast<uint16_t*>(e.out)[at + i] = __builtin_bit_cast(uint16_t, (__bf16)y[i]);
    }
}

}  // namespace fwd_epilogue

#endif
