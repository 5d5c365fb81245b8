// What the two directions of the norms that join and end blocks share: sizes, rows and their workers, loads of eight columns.
#pragma once
#include <initializer_list>

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

// Eight elements as they lie in memory.
template <int DT> struct Raw8 { uint32_t w[dt_bytes<DT>() * BN_VEC / 4]; };
typedef uint32_t bn_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t bn_u32x2 __attribute__((ext_vector_type(2)));

template <int DT> __device__ __forceinline__ Raw8<DT> none8() {
    Raw8<DT> r;
    __builtin_memset(&r, 0, sizeof(r));
    return r;
}
template <int DT> __device__ __forceinline__ void unpack8(const Raw8<DT>& r, float* v) {
    if constexpr (DT == MXL_DT_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = bf16_lo(r.w[i]), v[2 * i + 1] = bf16_hi(r.w[i]);
    } else {
        typedef typename DtOf<DT>::type E;
        E e[BN_VEC];
        __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < BN_VEC; ++i) v[i] = (float)e[i];
    }
}
template <int DT> __device__ __forceinline__ Raw8<DT> pack8(const float* v) {
    typedef typename DtOf<DT>::type E;
    E e[BN_VEC];
#pragma unroll
    for (int i = 0; i < BN_VEC; ++i) e[i] = (E)v[i];
    Raw8<DT> r;
    __builtin_memcpy(&r, e, sizeof(r));
    return r;
}

// Which columns a lane has: of every chunk eight, next to each other where all rows are of 16-bit types, and two fours where there are floats.
// So a store of a wave writes whole lines; streaming stores of every other sixteen bytes do not combine (both norms on a stream in fp32,
// [5403, 2880], forward: 36 us, 41 with eight floats in a row).
template <int S> struct Cols {
    static constexpr int WIDTH = S == MXL_DT_F32 ? 4 : 8, PIECES = BN_VEC / WIDTH;
    int lanes, lane, k;
    __device__ __forceinline__ int piece(int j, int q) const { return ((j * PIECES + q) * lanes + lane) * WIDTH; }
    __device__ __forceinline__ int operator()(int j, int e) const { return piece(j, e / WIDTH) + e % WIDTH; }
};

// From and to any element's address: a row's last, partial piece goes element by element, missing ones are zeros.
template <int DT, int WIDTH> __device__ __forceinline__ void load_any(const void* base, int64_t at, int left, uint32_t* w, bool streaming) {
    typedef typename DtOf<DT>::type E;
    constexpr int WORDS = WIDTH * dt_bytes<DT>() / 4;
    typedef uint32_t Words __attribute__((ext_vector_type(WORDS), aligned(2)));
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
    if (left <= 0 || base == nullptr) return;
    const E* p = (const E*)base + at;
    if (left >= WIDTH) {
        const Words v = streaming ? __builtin_nontemporal_load((const Words*)p) : *(const Words*)p;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) w[i] = v[i];
    } else {
        E e[WIDTH];
#pragma unroll
        for (int i = 0; i < WIDTH; ++i) e[i] = i < left ? p[i] : (E)0.f;
        __builtin_memcpy(w, e, sizeof(e));
    }
}
template <int DT, int WIDTH> __device__ __forceinline__ void store_any(void* base, int64_t at, int left, const uint32_t* w) {
    if (left <= 0 || base == nullptr) return;
    typedef typename DtOf<DT>::type E;
    constexpr int WORDS = WIDTH * dt_bytes<DT>() / 4;
    typedef uint32_t Words __attribute__((ext_vector_type(WORDS), aligned(2)));
    E* p = (E*)base + at;
    if (left >= WIDTH) {
        Words t;
#pragma unroll
        for (int i = 0; i < WORDS; ++i) t[i] = w[i];
        __builtin_nontemporal_store(t, (Words*)p);
    } else {
        E e[WIDTH];
        __builtin_memcpy(e, w, sizeof(e));
#pragma unroll
        for (int i = 0; i < WIDTH; ++i)
            if (i < left) p[i] = e[i];
    }
}
// a lane's columns of a vector [k]
template <int DT, int S> __device__ __forceinline__ Raw8<DT> load_vector(const void* base, const Cols<S>& cols, int j) {
    Raw8<DT> r;
#pragma unroll
    for (int q = 0; q < Cols<S>::PIECES; ++q)
        load_any<DT, Cols<S>::WIDTH>(base, cols.piece(j, q), cols.k - cols.piece(j, q), r.w + q * (Cols<S>::WIDTH * dt_bytes<DT>() / 4), false);
    return r;
}

// The rows of a tensor [rows, k], a lane's columns at a time.  On dwords (ANY false): through buffer descriptors, whose range check is dword
// by dword.  A lane past the row's end, a row's last columns and a tensor that is not there (null) then need no branch: nothing is
// read (zeros) or written.  That keeps the loop one basic block, so that the wait for a row's loads need not be one for the stores
// behind them.  SMALL: several rows a wave, one descriptor for the tensor (whole eights, below 2 GiB); otherwise a row has its own.
// ANY: from any element, with branches.
constexpr int BN_NT = 2;        // non-temporal
template <int DT, int S, bool SMALL, bool ANY> struct RowsOf {
    static constexpr int WIDTH = Cols<S>::WIDTH, PIECES = Cols<S>::PIECES, WORDS = WIDTH * dt_bytes<DT>() / 4;
    void* base;
    int64_t row0;               // element of the row's beginning
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ RowsOf(const void* base_, int64_t rows, int64_t row, int k) : base((void*)base_), row0(row * k) {
        constexpr int size = dt_bytes<DT>();
        if constexpr (!ANY) {
            if constexpr (SMALL) rsrc = __builtin_amdgcn_make_buffer_rsrc(base, 0, base ? (int)(rows * k * size) : 0, 0x00020000);
            else rsrc = __builtin_amdgcn_make_buffer_rsrc((uint8_t*)base + row0 * size, 0, base ? k * size : 0, 0x00020000);
        }
    }
    __device__ __forceinline__ int offset(int col, int k) const {
        if constexpr (SMALL) return col < k ? ((int)row0 + col) * dt_bytes<DT>() : (int)0x80000000;
        return col * dt_bytes<DT>();
    }
    template <int HINT> __device__ __forceinline__ Raw8<DT> load(const Cols<S>& cols, int j) const {
        Raw8<DT> r;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            const int col = cols.piece(j, q);
            uint32_t* w = r.w + q * WORDS;
            if constexpr (ANY) {
                load_any<DT, WIDTH>(base, row0 + col, cols.k - col, w, HINT == BN_NT);
            } else if constexpr (WORDS == 4) {
                const bn_u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, offset(col, cols.k), 0, HINT);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = v[i];
            } else {
                const bn_u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rsrc, offset(col, cols.k), 0, HINT);
                w[0] = v[0], w[1] = v[1];
            }
        }
        return r;
    }
    __device__ __forceinline__ void store(const Cols<S>& cols, int j, const float* v) const {
        const Raw8<DT> r = pack8<DT>(v);
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
            const int col = cols.piece(j, q);
            const uint32_t* w = r.w + q * WORDS;
            if constexpr (ANY) {
                store_any<DT, WIDTH>(base, row0 + col, cols.k - col, w);
            } else if constexpr (WORDS == 4) {
                const bn_u32x4 t = {w[0], w[1], w[2], w[3]};
                __builtin_amdgcn_raw_buffer_store_b128(t, rsrc, offset(col, cols.k), 0, BN_NT);
            } else {
                const bn_u32x2 t = {w[0], w[1]};
                __builtin_amdgcn_raw_buffer_store_b64(t, rsrc, offset(col, cols.k), 0, BN_NT);
            }
        }
    }
};

// Sums over a worker's lanes in a fixed order, every lane gets them.  SMALL: a worker is `lanes` lanes of a wave; otherwise the
// workgroup, whose waves' sums meet in shared memory and are added up by a tree over sixteen lanes again.  `part` holds two sets, used in
// turn: one barrier a call.
constexpr int BN_MAX_WAVES = BN_MAX_THREADS / 64;
template <int N, bool SMALL> struct RowSums {
    typedef float Part[BN_MAX_WAVES][N];
    Part* part;
    int lanes, waves, turn;
    __device__ __forceinline__ RowSums(Part* part_, int lanes_) : part(part_), lanes(lanes_), waves((int)blockDim.x >> 6), turn(0) {
        if constexpr (!SMALL) {     // (before the first call's barrier)
            if ((int)threadIdx.x < 2 * BN_MAX_WAVES && ((int)threadIdx.x & (BN_MAX_WAVES - 1)) >= waves) {
#pragma unroll
                for (int n = 0; n < N; ++n) part[threadIdx.x / BN_MAX_WAVES][threadIdx.x & (BN_MAX_WAVES - 1)][n] = 0.f;
            }
        }
    }
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
            for (int n = 0; n < N; ++n) v[n] = part[turn][threadIdx.x & (BN_MAX_WAVES - 1)][n];
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = lanes_sum<BN_MAX_WAVES>(v[n]);
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
// Whether the rows of tensors at these addresses can go through buffer descriptors: every row begins at a dword, and where a wave
// takes several, each is whole eights and the tensor's offsets fit 31 bits.
inline bool bn_on_dwords(int64_t rows, int64_t k, int dtype, std::initializer_list<const void*> ps) {
    if (dtype != MXL_DT_F32 && k % 2 != 0) return false;
    if (k <= BN_SMALL_K && (k % BN_VEC != 0 || rows * k >= ((int64_t)1 << 29))) return false;
    for (const void* p : ps)
        if ((uintptr_t)p % 4 != 0) return false;
    return true;
}
// lanes of a row where a wave takes several (a power of two)
inline int bn_lanes(int64_t k) {
    int lanes = 8;
    while (lanes * BN_VEC < k) lanes *= 2;
    return lanes;
}
inline int bn_threads(int64_t k, int chunks) {
    const int64_t per = (int64_t)BN_VEC * chunks;
    return (int)((((k + per - 1) / per) + 63) / 64 * 64);
}

}  // namespace mxl
