// Reductions over aligned runs of lanes and loads of a float of any of the three types, shared by the routing and permutation kernels.
#pragma once
#include "mx_device.h"

namespace mxl {

// ---- reductions over aligned runs of lanes (every lane gets the result, and the same bits) ----
struct Pair32 { uint32_t a, b; };
__device__ __forceinline__ Pair32 swap16(uint32_t v) {      // rows of 16 lanes: {r0 r0 r2 r2}, {r1 r1 r3 r3}
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ Pair32 swap32(uint32_t v) {      // halves: {h0 h0}, {h1 h1}
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {r[0], r[1]};
}
struct OpMaxU {
    __device__ static __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
struct OpMinU {
    __device__ static __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return a < b ? a : b; }
};
struct OpMaxF {
    __device__ static __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
};
struct OpAddF {
    __device__ static __forceinline__ uint32_t f(uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }
};
template <class OP, int LANES> __device__ __forceinline__ uint32_t lanes_reduce(uint32_t v) {
    if constexpr (LANES > 1) v = OP::f(v, dpp_xor1(v));
    if constexpr (LANES > 2) v = OP::f(v, dpp_xor2(v));
    if constexpr (LANES > 4) v = OP::f(v, dpp_half_mirror(v));
    if constexpr (LANES > 8) v = OP::f(v, dpp_mirror(v));
    if constexpr (LANES > 16) { const Pair32 p = swap16(v); v = OP::f(p.a, p.b); }
    if constexpr (LANES > 32) { const Pair32 p = swap32(v); v = OP::f(p.a, p.b); }
    return v;
}
// the same with a number of lanes known at run time (a power of two, the same for the whole wave)
template <class OP> __device__ __forceinline__ uint32_t lanes_reduce(uint32_t v, int lanes) {
    if (lanes > 1) v = OP::f(v, dpp_xor1(v));
    if (lanes > 2) v = OP::f(v, dpp_xor2(v));
    if (lanes > 4) v = OP::f(v, dpp_half_mirror(v));
    if (lanes > 8) v = OP::f(v, dpp_mirror(v));
    if (lanes > 16) { const Pair32 p = swap16(v); v = OP::f(p.a, p.b); }
    if (lanes > 32) { const Pair32 p = swap32(v); v = OP::f(p.a, p.b); }
    return v;
}
template <int LANES> __device__ __forceinline__ float lanes_max(float v) { return __uint_as_float(lanes_reduce<OpMaxF, LANES>(__float_as_uint(v))); }
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) { return __uint_as_float(lanes_reduce<OpAddF, LANES>(__float_as_uint(v))); }

// element i of an array of MXL_DT_* type
__device__ __forceinline__ float load_dt(const void* p, int dtype, int64_t i) {
    if (dtype == MXL_DT_F32) return ((const float*)p)[i];
    if (dtype == MXL_DT_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void store_dt(void* p, int dtype, int64_t i, float x) {
    if (dtype == MXL_DT_F32) ((float*)p)[i] = x;
    else if (dtype == MXL_DT_BF16) ((__bf16*)p)[i] = (__bf16)x;
    else ((_Float16*)p)[i] = (_Float16)x;
}

}  // namespace mxl
