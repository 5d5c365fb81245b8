// The global norm of many tensors, and their clipping by it:
//
//   norm = sqrt(sum over tensors and elements of g^2)   or   max |g|          g *= min(1, max_norm / (norm + 1e-6))
//
// The tensors' addresses and sizes travel in the kernels' arguments, GN_TENSORS a launch: nothing is copied to the device and a
// captured launch keeps its own table.  A launch's tensors are cut into chunks, which its workgroups take in turn.
//
// Squares and sums are fp64: a float's square is exact there and neither overflows nor underflows, whatever the gradients' scale.
// Every workgroup leaves one sum, one workgroup adds them up in their order, and no atomics: which sums an element goes through depends on the sizes, the types and
// the addresses modulo 16 (a chunk's elements in front of its first whole sixteen bytes go by themselves), on nothing else.
//
// Bound by memory.  1.4e9 floats 813 us (6.9 TB/s), 2.2e8 bf16 elements 66 us (6.6); clipping those into floats 220 us (6.0 TB/s).  The fp64 work hides
// behind the loads.  (With loads behind branches, one after the other: 3520, 100 and, the output's sixteen bytes every 32, 312.)
#include <math.h>
#include <stdlib.h>

#include "mx_lanes.h"

namespace mxl {

constexpr int GN_TENSORS = 160;             // a launch: 20 bytes each, the arguments stay below 4 KB
constexpr int GN_THREADS = 256;
constexpr int GN_LOADS = 8;                 // 16-byte loads a lane asks for at once
constexpr int GN_CHUNK = GN_THREADS * GN_LOADS * 16;        // bytes
constexpr int GN_BLOCKS = 2048;
constexpr int GN_JOIN_THREADS = 1024;

typedef uint32_t gn_u32x4 __attribute__((ext_vector_type(4)));

struct NormTable {
    const void* p[GN_TENSORS];
    int64_t n[GN_TENSORS];                  // elements; the type code in the upper bits
    uint32_t end[GN_TENSORS];               // chunks up to and with this tensor's
    int count;
};
constexpr int GN_TYPE_SHIFT = 56;
static_assert(sizeof(NormTable) <= 4032, "kernel arguments");

__device__ __forceinline__ float half_lo(uint32_t v) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(v & 0xFFFFu)); }
__device__ __forceinline__ float half_hi(uint32_t v) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16)); }

// a sum of squares, or the largest magnitude's bits (those of a NaN are above those of every number)
template <bool MAX> struct Stat;
template <> struct Stat<false> {
    double a = 0., b = 0.;
    __device__ __forceinline__ void add(float x, float y) {
        a = fma((double)x, (double)x, a);
        b = fma((double)y, (double)y, b);
    }
    __device__ __forceinline__ void join(const Stat& o) { a += o.a, b += o.b; }
};
template <> struct Stat<true> {
    uint32_t a = 0;
    __device__ __forceinline__ void add(float x, float y) {
        const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu, v = __float_as_uint(y) & 0x7FFFFFFFu, m = u > v ? u : v;
        a = a > m ? a : m;
    }
};
template <int DT, bool MAX> __device__ __forceinline__ void add_vec(Stat<MAX>& s, const gn_u32x4& v) {
#pragma unroll
    for (int i = 0; i < 4; i += DT == MXL_DT_F32 ? 2 : 1) {
        if (DT == MXL_DT_F32) s.add(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
        else if (DT == MXL_DT_BF16) s.add(bf16_lo(v[i]), bf16_hi(v[i]));
        else s.add(half_lo(v[i]), half_hi(v[i]));
    }
}

// Elements [lo, hi) of a tensor: the 16-byte pieces among them, through a buffer descriptor that ends with the last (zeros arrive for
// pieces past it, which add nothing: no branches, so that all loads are on their way at once), and the elements before and behind.
template <int DT, bool MAX> __device__ __forceinline__ void chunk_stat(Stat<MAX>& s, const void* base, int64_t lo, int64_t hi) {
    constexpr int SIZE = DT == MXL_DT_F32 ? 4 : 2;
    const int64_t bytes = (hi - lo) * SIZE;
    const uint8_t* a = (const uint8_t*)base + lo * SIZE;
    int64_t head = -(int64_t)(uintptr_t)a & 15;
    if (head > bytes) head = bytes;
    const int vecs = (int)((bytes - head) / 16), tail = (int)(bytes - head - (int64_t)vecs * 16);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(a + head), 0, vecs * 16, 0x00020000);
    gn_u32x4 r[GN_LOADS];
#pragma unroll
    for (int u = 0; u < GN_LOADS; ++u) r[u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)threadIdx.x * 16, u * GN_THREADS * 16, 2);
    if (head | tail) {
        const int i = (int)threadIdx.x;
        if (i < (int)head / SIZE) s.add(load_dt(base, DT, lo + i), 0.f);
        else if (i >= 64 && i - 64 < tail / SIZE) s.add(load_dt(base, DT, hi - tail / SIZE + (i - 64)), 0.f);
    }
#pragma unroll
    for (int u = 0; u < GN_LOADS; ++u) add_vec<DT, MAX>(s, r[u]);
}

// Which tensor a chunk belongs to: the number of tensors that end at or before it.  The ends are in registers, some a lane.
template <int TENSORS> struct TensorOf {
    static constexpr int PER = (TENSORS + 63) / 64;
    uint32_t end[PER];
    __device__ __forceinline__ TensorOf(const uint32_t* ends, int count) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int t = i * 64 + ((int)threadIdx.x & 63);
            end[i] = t < count ? ends[t] : 0xFFFFFFFFu;
        }
    }
    __device__ __forceinline__ int operator()(uint32_t chunk) const {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) n += __builtin_popcountll(__ballot(end[i] <= chunk));
        return n;
    }
};

__device__ __forceinline__ double lanes_sum_f64(double v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
template <int THREADS> __device__ __forceinline__ double block_stat(double v, bool max) {     // thread 0 gets it
    __shared__ double part[THREADS / 64];
    if (max) {
        // (bits of a float as a double: whole numbers, in order)
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) v = fmax(v, __shfl_xor(v, m));
    } else {
        v = lanes_sum_f64(v);
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = part[0];
    if (threadIdx.x == 0)
        for (int i = 1; i < THREADS / 64; ++i) s = max ? fmax(s, part[i]) : s + part[i];
    return s;
}
__device__ __forceinline__ float norm_of(double total, bool max) { return max ? __uint_as_float((uint32_t)total) : (float)sqrt(total); }

// `out` set: the launch's only workgroup writes the norm itself.
template <bool MAX> __global__ __launch_bounds__(GN_THREADS) void grad_norm_kernel(NormTable t, double* partial, float* out) {
    Stat<MAX> s;
    const uint32_t chunks = t.end[t.count - 1];
    const TensorOf<GN_TENSORS> tensor_of(t.end, t.count);
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int at = tensor_of(c);
        const uint32_t first = at ? t.end[at - 1] : 0;
        const int64_t packed = t.n[at], n = packed & (((int64_t)1 << GN_TYPE_SHIFT) - 1);
        const int type = (int)(packed >> GN_TYPE_SHIFT);
        const int64_t per = type == MXL_DT_F32 ? GN_CHUNK / 4 : GN_CHUNK / 2, lo = (int64_t)(c - first) * per, hi = lo + per < n ? lo + per : n;
        if (type == MXL_DT_F32) chunk_stat<MXL_DT_F32, MAX>(s, t.p[at], lo, hi);
        else if (type == MXL_DT_BF16) chunk_stat<MXL_DT_BF16, MAX>(s, t.p[at], lo, hi);
        else chunk_stat<MXL_DT_F16, MAX>(s, t.p[at], lo, hi);
    }
    double v;
    if constexpr (MAX) v = (double)s.a;
    else v = s.a + s.b;
    v = block_stat<GN_THREADS>(v, MAX);
    if (threadIdx.x == 0) {
        if (out) *out = norm_of(v, MAX);
        else partial[blockIdx.x] = v;
    }
}

__global__ __launch_bounds__(GN_JOIN_THREADS) void grad_norm_join_kernel(const double* partial, int64_t n, int max, float* out) {
    double v = 0.;
    for (int64_t i = threadIdx.x; i < n; i += GN_JOIN_THREADS) v = max ? fmax(v, partial[i]) : v + partial[i];
    v = block_stat<GN_JOIN_THREADS>(v, max != 0);
    if (threadIdx.x == 0) *out = norm_of(v, max != 0);
}

// ---- clipping ----
constexpr int GC_TENSORS = 128;
struct ClipTable {
    const void* p[GC_TENSORS];
    void* out[GC_TENSORS];
    int64_t n[GC_TENSORS];                  // elements; the type codes, out's above the gradient's
    uint32_t end[GC_TENSORS];
    int count, in_place;                    // in_place: every output is its gradient
};
static_assert(sizeof(ClipTable) <= 4032, "kernel arguments");
constexpr int GC_PER = GN_THREADS * 32;     // elements of a chunk
// Workgroups of a launch.  As many as there are chunks is fastest where something is written (1.4e9 floats in place, launch after launch, 2057 us; 32768
// workgroups 2101, 2048 2152), but all of them have to come and go where the norm is within the bound (39, 9 and 5 us), the common case.
constexpr uint32_t GC_BLOCKS = 32768;

// The product is made in fp64 and rounded to fp32 (of a 16-bit type it is exact till then but for the factor's 53 bits), and once more to a 16-bit output.
// The factor as a float would lose bits, and all of them in the end, below 2^-126.
// us for 2.2e8 elements, with 16-bit ones scaled in fp32 and so: bf16 to bf16 139 and 138, to fp16 138 and 138, to fp32 238 and 220.
template <int DO> __device__ __forceinline__ float scaled(float g, double c) {
    float f = (float)((double)g * c);
    if (DO != MXL_DT_F32) asm("" : "+v"(f));    // (or both roundings become one from fp64, many instructions: bf16 to fp16 209 us)
    return f;
}

// Four or eight elements a lane and step (so that a store of a wave writes whole lines: streaming stores of every other sixteen bytes do not
// combine), through buffer descriptors of the chunk's whole steps' worth (past it nothing is read or written); the rest element by element.
// Two-byte elements that begin between two dwords: the descriptor begins a dword boundary later, the element in front goes by itself.
template <int DT, int DO> __device__ __forceinline__ void clip_chunk(const void* src, void* dst, int64_t lo, int64_t hi, double c) {
    constexpr int IN = DT == MXL_DT_F32 ? 4 : 2, OUT = DO == MXL_DT_F32 ? 4 : 2;    // bytes of an element
    constexpr int PER = IN == 2 && OUT == 2 ? 8 : 4, STEPS = GC_PER / PER / GN_THREADS;
    constexpr int IW = PER * IN / 4, OW = PER * OUT / 4;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const uint8_t* s = (const uint8_t*)src + lo * IN;
    uint8_t* d = (uint8_t*)dst + lo * OUT;
    const bool odd_in = IN == 2 && ((uintptr_t)s & 2), odd_out = OUT == 2 && ((uintptr_t)d & 2);
    const int n = (int)(hi - lo);
    if (IN == 2 && OUT == 2 && odd_in != odd_out) {     // one on dwords and the other between them
        for (int i = (int)threadIdx.x; i < n; i += GN_THREADS) store_dt(dst, DO, lo + i, scaled<DO>(load_dt(src, DT, lo + i), c));
        return;
    }
    const int head = odd_in || odd_out ? 1 : 0, whole = (n - head) / PER;
    const auto in = __builtin_amdgcn_make_buffer_rsrc((void*)(s + head * IN), 0, whole * PER * IN, 0x00020000);
    const auto out = __builtin_amdgcn_make_buffer_rsrc(d + head * OUT, 0, whole * PER * OUT, 0x00020000);
    uint32_t r[STEPS][IW];
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
        if constexpr (IW == 4) {
            const gn_u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(in, (int)threadIdx.x * 16, u * GN_THREADS * 16, 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) r[u][j] = v[j];
        } else {
            const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(in, (int)threadIdx.x * 8, u * GN_THREADS * 8, 2);
            r[u][0] = v[0], r[u][1] = v[1];
        }
    }
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
        float f[PER];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (DT == MXL_DT_F32) f[j] = __uint_as_float(r[u][j % IW]);
            else if (DT == MXL_DT_BF16) f[j] = j & 1 ? bf16_hi(r[u][j / 2]) : bf16_lo(r[u][j / 2]);
            else f[j] = j & 1 ? half_hi(r[u][j / 2]) : half_lo(r[u][j / 2]);
            f[j] = scaled<DO>(f[j], c);
        }
        uint32_t o[OW];
#pragma unroll
        for (int j = 0; j < OW; ++j) {
            if (DO == MXL_DT_F32) o[j] = __float_as_uint(f[j % PER]);
            else if (DO == MXL_DT_BF16) o[j] = pack_bf16(f[2 * j % PER], f[(2 * j + 1) % PER]);
            else o[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j % PER]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[(2 * j + 1) % PER]) << 16);
        }
        // (No scalar offset: a store of more than 8 bytes fetches its data after it has issued, and only without one does the compiler keep two wait states
        // in front of an instruction that writes those registers.)
        if constexpr (OW == 4) {
            const gn_u32x4 t = {o[0], o[1], o[2], o[3]};
            __builtin_amdgcn_raw_buffer_store_b128(t, out, (int)threadIdx.x * 16 + u * GN_THREADS * 16, 0, 2);
        } else {
            const u32x2 t = {o[0], o[1]};
            __builtin_amdgcn_raw_buffer_store_b64(t, out, (int)threadIdx.x * 8, u * GN_THREADS * 8, 2);
        }
    }
    const int rest = n - head - whole * PER;
    if (head + rest) {
        const int t = (int)threadIdx.x;
        if (t < head || (t >= 64 && t - 64 < rest)) {
            const int64_t i = t < head ? lo : hi - rest + (t - 64);
            store_dt(dst, DO, i, scaled<DO>(load_dt(src, DT, i), c));
        }
    }
}

__global__ __launch_bounds__(GN_THREADS) void clip_kernel(ClipTable t, const float* norm, double max_norm) {
    const double raw = max_norm / ((double)*norm + 1e-6);
    const bool within = raw >= 1.;          // (a NaN is not)
    const double c = within ? 1. : raw;
    if (within && t.in_place) return;
    const uint32_t chunks = t.end[t.count - 1];
    const TensorOf<GC_TENSORS> tensor_of(t.end, t.count);
    for (uint32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
        const int at = tensor_of(i);
        const void* src = t.p[at];
        void* dst = t.out[at];
        if (within && src == dst) continue;
        const int64_t packed = t.n[at], n = packed & (((int64_t)1 << GN_TYPE_SHIFT) - 1);
        const int types = (int)(packed >> GN_TYPE_SHIFT), in = types & 3, out = types >> 2;
        const uint32_t first = at ? t.end[at - 1] : 0;
        const int64_t lo = (int64_t)(i - first) * GC_PER, hi = lo + GC_PER < n ? lo + GC_PER : n;
#define MXL_CLIP(DT, DO) clip_chunk<DT, DO>(src, dst, lo, hi, c)
        switch (in * 4 + out) {
            case MXL_DT_F32 * 4 + MXL_DT_F32: MXL_CLIP(MXL_DT_F32, MXL_DT_F32); break;
            case MXL_DT_F32 * 4 + MXL_DT_BF16: MXL_CLIP(MXL_DT_F32, MXL_DT_BF16); break;
            case MXL_DT_F32 * 4 + MXL_DT_F16: MXL_CLIP(MXL_DT_F32, MXL_DT_F16); break;
            case MXL_DT_BF16 * 4 + MXL_DT_F32: MXL_CLIP(MXL_DT_BF16, MXL_DT_F32); break;
            case MXL_DT_BF16 * 4 + MXL_DT_BF16: MXL_CLIP(MXL_DT_BF16, MXL_DT_BF16); break;
            case MXL_DT_BF16 * 4 + MXL_DT_F16: MXL_CLIP(MXL_DT_BF16, MXL_DT_F16); break;
            case MXL_DT_F16 * 4 + MXL_DT_F32: MXL_CLIP(MXL_DT_F16, MXL_DT_F32); break;
            case MXL_DT_F16 * 4 + MXL_DT_BF16: MXL_CLIP(MXL_DT_F16, MXL_DT_BF16); break;
            default: MXL_CLIP(MXL_DT_F16, MXL_DT_F16); break;
        }
#undef MXL_CLIP
    }
}

static int gn_size(int dtype) { return dtype == MXL_DT_F32 ? 4 : 2; }
static bool gn_list_ok(const void* const* p, const int64_t* n, const int32_t* dtypes, int count) {
    if (count < 0 || (count > 0 && (!p || !n || !dtypes))) return false;
    for (int i = 0; i < count; ++i)
        if (n[i] < 0 || n[i] >= ((int64_t)1 << 36) || dtypes[i] < MXL_DT_F32 || dtypes[i] > MXL_DT_F16 ||
            (n[i] > 0 && (!p[i] || (uintptr_t)p[i] % gn_size(dtypes[i])))) return false;
    return true;
}

struct Span {
    uintptr_t lo, hi;
    int written;
};
static int span_order(const void* a, const void* b) {
    const Span *x = (const Span*)a, *y = (const Span*)b;
    return x->lo < y->lo ? -1 : x->lo > y->lo;
}
// MXL_OK if what is written shares no byte with anything else that is read, the norm too, or written (a gradient that is its own output is one span).
static int clip_spans_apart(const void* const* p, void* const* out, const int64_t* n, const int32_t* dtypes, const int32_t* out_dtypes, int count,
                            const float* norm) {
    Span* s = (Span*)malloc((size_t)(2 * (int64_t)count + 1) * sizeof(Span));
    if (!s) return MXL_ENOMEM;
    int64_t m = 0;
    s[m++] = {(uintptr_t)norm, (uintptr_t)norm + sizeof(float), 0};
    for (int i = 0; i < count; ++i) {
        if (n[i] == 0) continue;
        const bool same = p[i] == out[i] && dtypes[i] == out_dtypes[i];
        if (!same) s[m++] = {(uintptr_t)p[i], (uintptr_t)p[i] + (uintptr_t)n[i] * gn_size(dtypes[i]), 0};
        s[m++] = {(uintptr_t)out[i], (uintptr_t)out[i] + (uintptr_t)n[i] * gn_size(out_dtypes[i]), 1};
    }
    qsort(s, (size_t)m, sizeof(Span), span_order);
    uintptr_t read_end = 0, write_end = 0;
    int apart = 1;
    for (int64_t i = 0; i < m && apart; ++i) {
        if (s[i].lo < write_end || (s[i].written && s[i].lo < read_end)) apart = 0;
        uintptr_t& end = s[i].written ? write_end : read_end;
        if (s[i].hi > end) end = s[i].hi;
    }
    free(s);
    return apart ? MXL_OK : MXL_EINVAL;
}

}  // namespace mxl

using namespace mxl;

extern "C" int64_t mxl_grad_norm_workspace_bytes(int count) {
    if (count < 0) return -1;
    return ((int64_t)count + GN_TENSORS - 1) / GN_TENSORS * GN_BLOCKS * 8;
}

extern "C" int mxl_grad_norm(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int count, int kind, float* norm, void* workspace,
                             int64_t workspace_bytes, void* stream) {
    if (!gn_list_ok(grads, sizes, dtypes, count) || (kind != MXL_NORM_L2 && kind != MXL_NORM_MAX) || !norm || ((uintptr_t)norm & 3)) return MXL_EINVAL;
    if (workspace_bytes < mxl_grad_norm_workspace_bytes(count) || (count > 0 && (!workspace || ((uintptr_t)workspace & 7) != 0))) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    hipStream_t st = (hipStream_t)stream;
    const bool max = kind == MXL_NORM_MAX;
    double* partial = (double*)workspace;
    int64_t partials = 0;
    int i = 0;
    while (i < count) {
        NormTable t;
        t.count = 0;
        uint32_t chunks = 0;
        for (; i < count && t.count < GN_TENSORS; ++i) {
            if (sizes[i] == 0) continue;
            const int64_t per = GN_CHUNK / gn_size(dtypes[i]), more = (sizes[i] + per - 1) / per;
            if (more + chunks > 0x7FFFFFFF) break;
            chunks += (uint32_t)more;
            t.p[t.count] = grads[i];
            t.n[t.count] = sizes[i] | ((int64_t)dtypes[i] << GN_TYPE_SHIFT);
            t.end[t.count++] = chunks;
        }
        if (t.count == 0) break;
        const int blocks = (int)(chunks < (uint32_t)GN_BLOCKS ? chunks : (uint32_t)GN_BLOCKS);
        float* out = i == count && partials == 0 && blocks == 1 ? norm : nullptr;
        if (max) hipLaunchKernelGGL(grad_norm_kernel<true>, dim3((unsigned)blocks), dim3(GN_THREADS), 0, st, t, partial + partials, out);
        else hipLaunchKernelGGL(grad_norm_kernel<false>, dim3((unsigned)blocks), dim3(GN_THREADS), 0, st, t, partial + partials, out);
        if (hipGetLastError() != hipSuccess) return MXL_ELAUNCH;
        if (out) return MXL_OK;
        partials += blocks;
    }
    hipLaunchKernelGGL(grad_norm_join_kernel, dim3(1), dim3(GN_JOIN_THREADS), 0, st, partial, partials, (int)max, norm);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

extern "C" int mxl_clip_grads(const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* dtypes, const int32_t* out_dtypes,
                              int count, double max_norm, const float* norm, void* stream) {
    if (!gn_list_ok(grads, sizes, dtypes, count) || !gn_list_ok(outs, sizes, out_dtypes, count) || !norm || ((uintptr_t)norm & 3) || !(max_norm >= 0.)) return MXL_EINVAL;
    const int apart = clip_spans_apart(grads, outs, sizes, dtypes, out_dtypes, count, norm);
    if (apart != MXL_OK) return apart;
    if (!device_is_gfx950()) return MXL_ENODEV;
    hipStream_t st = (hipStream_t)stream;
    int i = 0;
    while (i < count) {
        ClipTable t;
        t.count = 0;
        t.in_place = 1;
        uint32_t chunks = 0;
        for (; i < count && t.count < GC_TENSORS; ++i) {
            if (sizes[i] == 0) continue;
            const int64_t more = (sizes[i] + GC_PER - 1) / GC_PER;
            if (more + chunks > 0x7FFFFFFF) break;
            chunks += (uint32_t)more;
            t.p[t.count] = grads[i];
            t.out[t.count] = outs[i];
            t.in_place &= grads[i] == outs[i];
            t.n[t.count] = sizes[i] | ((int64_t)(dtypes[i] | (out_dtypes[i] << 2)) << GN_TYPE_SHIFT);
            t.end[t.count++] = chunks;
        }
        if (t.count == 0) break;
        hipLaunchKernelGGL(clip_kernel, dim3(chunks < GC_BLOCKS ? chunks : GC_BLOCKS), dim3(GN_THREADS), 0, st, t, norm, max_norm);
        if (hipGetLastError() != hipSuccess) return MXL_ELAUNCH;
    }
    return MXL_OK;
}
