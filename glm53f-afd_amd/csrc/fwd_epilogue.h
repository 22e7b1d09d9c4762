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
};

__device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// y * sigmoid(z). exp(-z) overflows to infinity where the sigmoid is below the smallest f32: the quotient is then 0.
__device__ __forceinline__ float gated(float y, float z) { return y / (1.0f + expf(-z)); }

// The switch is on a kernel argument: every lane of the launch takes the same way.
__device__ __forceinline__ float activate(float y, int act) {
    switch (act) {
        case GLM53F_ACT_RELU: return y < 0.0f ? 0.0f : y;
        case GLM53F_ACT_SILU: return gated(y, y);
        case GLM53F_ACT_GELU: return 0.5f * y * erfcf(y * -0.70710678118654752f);   // Phi(y), exact in the far left too
        case GLM53F_ACT_GELU_TANH: return gated(y, 1.5957691216057308f * (y + 0.044715f * y * y * y));   // (1 + tanh u) / 2 = sigmoid(2u)
        case GLM53F_ACT_SIGMOID: return gated(1.0f, y);
        default: return y;
    }
}

// One output: row m, column o of group g.
__device__ __forceinline__ void finish(const Epilogue& e, int g, long long m, int o, float y) {
    if (e.bias) y += widen(e.bias[g * e.b_gs + o]);
    y = activate(y, e.act);
    if (e.out_f32) {
        if (e.residual) y = static_cast<const float*>(e.residual)[g * e.r_gs + m * e.ldr + o] + y;
        static_cast<float*>(e.out)[g * e.o_gs + m * e.ldo + o] = y;
    } else {
        if (e.residual) y = widen(static_cast<const uint16_t*>(e.residual)[g * e.r_gs + m * e.ldr + o]) + y;
        static_cast<uint16_t*>(e.out)[g * e.o_gs + m * e.ldo + o] = __builtin_bit_cast(uint16_t, (__bf16)y);
    }
}

}  // namespace fwd_epilogue

#endif
