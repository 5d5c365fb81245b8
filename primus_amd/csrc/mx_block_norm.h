// What the two directions of the norms that join and end blocks share: sizes, rows and their workers, loads of eight columns.
#pragma once
#include "mx_lanes.h"

namespace mxl {

constexpr int BN_MAX_K = 16384;
constexpr int BN_VEC = 8;               // columns a lane takes at once
constexpr int BN_MAX_THREADS = 1024;
constexpr int BN_SMALL_K = 256;         // up to here a wave takes several rows
constexpr int BN_SMALL_THREADS = 256;

enum { GATE_NONE = 0, GATE_SCALAR = 1, GATE_VECTOR = 2 };

// The gate of row r is row (r / div) % mod of [mod, 1] or [mod, k]: rows = outer * mod * div.
struct Gate {
    const void* p;
    int kind;
    uint32_t div, mod;
};

template <int DT> struct DtOf;
template <> struct DtOf<MXL_DT_F32> { typedef float type; };
template <> struct DtOf<MXL_DT_BF16> { typedef __bf16 type; };
template <> struct DtOf<MXL_DT_F16> { typedef _Float16 type; };
template <int DT> constexpr int dt_bytes() { return DT == MXL_DT_F32 ? 4 : 2; }

// Eight elements as they lie in memory.  Rows of any length start at any element: the hardware takes 16-byte accesses at
// every address, so only a row's last, partial eight goes element by element.
template <int DT> struct Raw8 { uint32_t w[dt_bytes<DT>() * BN_VEC / 4]; };
typedef uint32_t bn_u32x4 __attribute__((ext_vector_type(4), aligned(2)));

template <int DT> __device__ __forceinline__ Raw8<DT> load8(const void* base, int64_t at, int left, bool streaming) {
    Raw8<DT> r;
    typedef typename DtOf<DT>::type E;
    const E* p = (const E*)base + at;
    if (left >= BN_VEC) {
#pragma unroll
        for (int i = 0; i < dt_bytes<DT>() / 2; ++i) {
            const bn_u32x4* s = (const bn_u32x4*)p + i;
            const bn_u32x4 v = streaming ? __builtin_nontemporal_load(s) : *s;
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
        }
    } else {
        E e[BN_VEC];
#pragma unroll
        for (int i = 0; i < BN_VEC; ++i) e[i] = i < left ? p[i] : (E)0.f;
        __builtin_memcpy(&r, e, sizeof(r));
    }
    return r;
}
template <int DT> __device__ __forceinline__ void store8(void* base, int64_t at, int left, const float* v) {
    typedef typename DtOf<DT>::type E;
    E* p = (E*)base + at;
    E e[BN_VEC];
#pragma unroll
    for (int i = 0; i < BN_VEC; ++i) e[i] = (E)v[i];
    if (left >= BN_VEC) {
        Raw8<DT> r;
        __builtin_memcpy(&r, e, sizeof(r));
#pragma unroll
        for (int i = 0; i < dt_bytes<DT>() / 2; ++i) {
            const bn_u32x4 t = {r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
            __builtin_nontemporal_store(t, (bn_u32x4*)p + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < BN_VEC; ++i)
            if (i < left) p[i] = e[i];
    }
}
template <int DT> __device__ __forceinline__ void unpack8(const Raw8<DT>& r, float* v) {
    typedef typename DtOf<DT>::type E;
    E e[BN_VEC];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < BN_VEC; ++i) v[i] = (float)e[i];
}
template <int DT> __device__ __forceinline__ Raw8<DT> none8() {
    Raw8<DT> r;
    __builtin_memset(&r, 0, sizeof(r));
    return r;
}

// Sums over a worker's lanes in a fixed order, every lane gets them.  SMALL: a worker is `lanes` lanes of a wave; otherwise the
// workgroup.  `part` holds two sets of N sums a wave, used in turn: one barrier a call.
template <int N, bool SMALL> struct RowSums {
    float (*part)[BN_MAX_THREADS / 64][N];
    int lanes, waves, turn;
    __device__ __forceinline__ RowSums(float (*part_)[BN_MAX_THREADS / 64][N], int lanes_) : part(part_), lanes(lanes_), waves((int)blockDim.x >> 6), turn(0) {}
    __device__ __forceinline__ void operator()(float* v) {
        if constexpr (SMALL) {
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = __uint_as_float(lanes_reduce<OpAddF>(__float_as_uint(v[n]), lanes));
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = lanes_sum<64>(v[n]);
            if (waves == 1) return;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int n = 0; n < N; ++n) part[turn][threadIdx.x >> 6][n] = v[n];
            }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float s = part[turn][0][n];
                for (int w = 1; w < waves; ++w) s += part[turn][w][n];
                v[n] = s;
            }
            turn ^= 1;
        }
    }
};

// ---- host side ----
inline bool bn_shape_ok(int64_t rows, int64_t k, int dtype, int stream_dtype) {
    return rows >= 0 && rows <= 0x7FFFFFFF && k > 0 && k <= BN_MAX_K && dtype >= MXL_DT_F32 && dtype <= MXL_DT_F16 &&
           (stream_dtype == dtype || stream_dtype == MXL_DT_F32);
}
inline bool bn_gate_ok(int64_t rows, int64_t k, const void* gate, int64_t div, int64_t mod, int64_t cols) {
    if (!gate) return true;
    if (cols != 1 && cols != k) return false;
    if (rows == 0) return true;
    return div > 0 && mod > 0 && div <= rows && mod <= rows / div && rows % (div * mod) == 0;
}
// (a gate [mod, 1] of rows of one column is a gate of vectors: each is its row's only element)
inline Gate bn_gate(const void* gate, int64_t rows, int64_t div, int64_t mod, int64_t cols, int64_t k) {
    if (!gate) return {nullptr, GATE_NONE, (uint32_t)(rows > 0 ? rows : 1), 1u};
    return {gate, cols == k ? GATE_VECTOR : GATE_SCALAR, (uint32_t)div, (uint32_t)mod};
}
// lanes of a row where a wave takes several (a power of two)
inline int bn_lanes(int64_t k) {
    int lanes = 8;
    while (lanes * BN_VEC < k) lanes *= 2;
    return lanes;
}
inline int bn_chunks(int64_t k) { return k <= BN_MAX_THREADS * BN_VEC ? 1 : 2; }
inline int bn_threads(int64_t k) {
    const int64_t per = (int64_t)BN_VEC * bn_chunks(k);
    return (int)((((k + per - 1) / per) + 63) / 64 * 64);
}

}  // namespace mxl
