// What the dense bf16 linears' kernels share: arguments of the epilogue, activations and their slopes.
#pragma once
#include "mx_device.h"

namespace mxl {

constexpr int kActSilu = MXL_ACT_SILU, kActGelu = MXL_ACT_GELU, kActRelu = MXL_ACT_RELU, kActNone = MXL_ACT_NONE;

// y = act(a . b^T + bias) + residual;  z = a . b^T + bias is kept for the backward if wanted
struct EpilogueArgs {
    const void* bias;           // [n], null: none
    const uint16_t* residual;   // [m, n] bf16, null: none
    uint16_t* z;                // [m, n] bf16, null: not kept
    int bias_f32;
};

// act in fp32.  SiLU and GELU as the gated activation's kernels compute them (hardware exp2 and reciprocal, about 1 ulp of fp32 each).
template <int ACT> __device__ __forceinline__ float epi_act(float z) {
    if constexpr (ACT == kActNone) return z;
    else if constexpr (ACT == kActRelu) return z != z ? z : fmaxf(z, 0.f);       // (a NaN stays one)
    else return act_fwd<ACT>(z);
}
// act'(z) in fp32
template <int ACT> __device__ __forceinline__ float epi_slope(float z) {
    if constexpr (ACT == kActNone) return 1.f;
    else if constexpr (ACT == kActRelu) return z != z ? z : (z > 0.f ? 1.f : 0.f);
    else if constexpr (ACT == kActSilu) {
        const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
        return s * (1.f + z * (1.f - s));
    } else {
        // Phi(z) + z phi(z); Phi from erfc_fit as in act_fwd, t exp(P(t)) exp(-z^2 / 2), whose last factor is phi's too
        const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.f + 0.5f * x);
        const float e = __builtin_amdgcn_exp2f(x * x * -1.4426950408889634f);
        const float tail = 0.5f * t * __builtin_amdgcn_exp2f(erfc_fit(t) * 1.4426950408889634f) * e;
        return fmaf(z * 0.39894228040143268f, e, z < 0.f ? tail : 1.f - tail);
    }
}

// bias of 4 columns from `col` on (a multiple of 4; the columns exist)
__device__ __forceinline__ v4f epi_bias4(const EpilogueArgs& e, int64_t col) {
    if (!e.bias) return v4f{0.f, 0.f, 0.f, 0.f};
    if (e.bias_f32) return *(const v4f*)((const float*)e.bias + col);
    const uint2 u = *(const uint2*)((const uint16_t*)e.bias + col);
    return v4f{bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)};
}
__device__ __forceinline__ uint2 pack4(const v4f& x) { return make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])); }
__device__ __forceinline__ v4f unpack4(const uint2& u) { return v4f{bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y)}; }

}  // namespace mxl
