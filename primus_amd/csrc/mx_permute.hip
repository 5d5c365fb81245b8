// Rows of tokens into the order of their experts and back, on the device: the grouped linears take each expert's rows back to back
// (primus/backends/megatron/core/transformer/experts.py:179-268), the router says which experts a token goes to.
//
//   entry i = t * topk + k of `indices` (expert e_i) goes to row  off[e_i] + #{j < i : e_j = e_i}
// off = prefix sums of the experts' counts, each rounded up to `align`; an entry whose expert is outside [0, experts) goes
// nowhere (row -1), a row that no entry goes to is zero.  The host does not know the counts, so the buffer is sized for the
// worst case and the rows behind the last expert's padding count as the last expert's, as in mxl_pad_groups.
//
//   permute:    rows[row_of[t, k]] = x[t]                            gradient: combine without probabilities
//   combine:    y[t] = sum_k p[t, k] rows[row_of[t, k]]              gradient: drows[row_of[t, k]] = p[t, k] dy[t],
//                                                                              dp[t, k] = <rows[row_of[t, k]], dy[t]>
//
// All of them are bound by the rows' bytes.  They go by tokens, not by rows of the permuted buffer: a token's row is read (or
// written) once and its topk copies come out of (or go into) registers, which is the least there is to move.  us (TB/s): 16384 tokens of
// 4096, two rows each, permute 76 (5.3), combine 85 (4.7), counting and placing 3.8 + 7.9; 8192 of 7168, eight each with probabilities,
// combine 193 (5.5), its gradient 406 (4.9; a row at a time 536); 32 tokens of 2880, four each, 3.7 and 3.6 for placing.  A large copy
// reaches 4.8-5.1 TB/s.
#include "mx_lanes.h"

namespace mxl {

constexpr int PM_MAX_TOPK = 32;
constexpr int PM_THREADS = 1024, PM_WAVES = 16;     // of the planning kernels
constexpr int PM_CHUNK = 4096;                      // entries per workgroup, while that gives at most
constexpr int PM_MAX_BLOCKS = 256;                  // so many workgroups

typedef uint32_t m32x4 __attribute__((ext_vector_type(4)));

struct PlanArgs {
    const int64_t* indices;
    int64_t entries, rows;
    int experts, align, key_bits;
    int chunk;                  // entries per workgroup, a multiple of PM_THREADS
    int* partial;               // [workgroups, experts] counts (unused with one workgroup)
    int64_t* row_of;
    int* entry_of;
    int64_t* group_lens;
    const void* probs;          // null: none
    void* row_probs;
    int prob_bytes;
};

__global__ __launch_bounds__(PM_THREADS) void permute_count_kernel(PlanArgs p) {
    __shared__ int hist[MXL_MAX_GROUPS];
    for (int e = threadIdx.x; e < p.experts; e += PM_THREADS) hist[e] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * p.chunk, end = lo + p.chunk < p.entries ? lo + p.chunk : p.entries;
    for (int64_t i = lo + threadIdx.x; i < end; i += PM_THREADS) {
        const int64_t e = p.indices[i];
        if (e >= 0 && e < p.experts) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.experts; e += PM_THREADS) p.partial[(int64_t)blockIdx.x * p.experts + e] = hist[e];
}

__device__ __forceinline__ void put_prob(const PlanArgs& p, int64_t row, int64_t entry) {      // entry < 0: zero
    if (p.prob_bytes == 4) ((uint32_t*)p.row_probs)[row] = entry < 0 ? 0u : ((const uint32_t*)p.probs)[entry];
    else ((uint16_t*)p.row_probs)[row] = entry < 0 ? (uint16_t)0 : ((const uint16_t*)p.probs)[entry];
}

// Every workgroup derives its experts' first rows from the counts of all chunks, gives each of its waves a run of its chunk, and
// the waves hand out rows 64 entries at a time in the entries' order.
__global__ __launch_bounds__(PM_THREADS) void permute_place_kernel(PlanArgs p) {
    extern __shared__ int lds[];
    const int E = p.experts;
    int* cnt = lds;                             // [waves][experts]: counts, then the next row of the wave's run
    int* total = lds + PM_WAVES * E;            // [experts] entries
    int* before = total + E;                    // [experts] entries in earlier chunks, then the chunk's first row
    int* off = before + E;                      // [experts + 1] first rows
    const int t = threadIdx.x, w = t >> 6, lane = t & 63;
    for (int i = t; i < (PM_WAVES + 2) * E; i += PM_THREADS) lds[i] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * p.chunk, end = lo + p.chunk < p.entries ? lo + p.chunk : p.entries;
    const int run = p.chunk / PM_WAVES;         // a multiple of 64
    const int64_t w_lo = lo + (int64_t)w * run;
    for (int64_t i = w_lo + lane; i < w_lo + run && i < end; i += 64) {
        const int64_t e = p.indices[i];
        if (e >= 0 && e < E) atomicAdd(&cnt[w * E + e], 1);
    }
    if (gridDim.x > 1) {
        const int n = (int)gridDim.x * E;
        const int mine = (int)blockIdx.x * E;
        for (int i = t; i < n; i += PM_THREADS) {
            const int c = p.partial[i], e = i % E;
            if (c) {
                atomicAdd(&total[e], c);
                if (i < mine) atomicAdd(&before[e], c);
            }
        }
    }
    __syncthreads();
    if (gridDim.x == 1) {
        for (int e = t; e < E; e += PM_THREADS) {
            int c = 0;
            for (int i = 0; i < PM_WAVES; ++i) c += cnt[i * E + e];
            total[e] = c;
        }
        __syncthreads();
    }
    if (w == 0) {
        uint32_t base = 0;
        for (int c = 0; c < E; c += 64) {
            const int e = c + lane;
            const uint32_t padded = e < E ? (uint32_t)((total[e] + p.align - 1) / p.align * p.align) : 0u;
            const uint32_t incl = wave_prefix(padded) + base;
            if (e < E) off[e] = (int)(incl - padded);
            base = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
        }
        if (lane == 0) off[E] = (int)base;      // <= rows: the buffer is sized for the worst case
    }
    __syncthreads();
    for (int e = t; e < E; e += PM_THREADS) {
        int at = off[e] + before[e];
        for (int i = 0; i < PM_WAVES; ++i) {
            const int c = cnt[i * E + e];
            cnt[i * E + e] = at;
            at += c;
        }
        if (blockIdx.x == 0) p.group_lens[e] = e == E - 1 ? p.rows - off[e] : off[e + 1] - off[e];
    }
    __syncthreads();
    for (int64_t i0 = w_lo; i0 < w_lo + run && i0 < end; i0 += 64) {
        const int64_t i = i0 + lane;
        const int64_t e64 = i < end ? p.indices[i] : -1;
        const bool live = e64 >= 0 && e64 < E;
        const int e = live ? (int)e64 : 0;
        uint64_t peers = __ballot(live);        // lanes with this lane's expert
        for (int b = 0; b < p.key_bits; ++b) {
            const uint64_t set = __ballot((e >> b) & 1);
            peers &= ((e >> b) & 1) ? set : ~set;
        }
        const int rank = __builtin_popcountll(peers & (((uint64_t)1 << lane) - 1));
        const int at = live ? cnt[w * E + e] + rank : -1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (live && rank == 0) cnt[w * E + e] = at + __builtin_popcountll(peers);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (i < end) p.row_of[i] = at;
        if (live) {
            p.entry_of[at] = (int)i;
            if (p.probs) put_prob(p, at, i);
        }
    }
    // rows that no entry goes to: padding inside the experts' runs, and the rest of the buffer
    for (int e = (int)blockIdx.x * PM_THREADS + t; e < E; e += (int)gridDim.x * PM_THREADS)
        for (int r = off[e] + total[e]; r < off[e + 1]; ++r) {      // fewer than align rows
            p.entry_of[r] = -1;
            if (p.probs) put_prob(p, r, -1);
        }
    for (int64_t r = off[E] + (int64_t)blockIdx.x * PM_THREADS + t; r < p.rows; r += (int64_t)gridDim.x * PM_THREADS) {
        p.entry_of[r] = -1;
        if (p.probs) put_prob(p, r, -1);
    }
}

struct MoveArgs {
    const uint8_t* x;           // permute: [tokens, row_bytes];  combine: rows [rows, hidden]
    uint8_t* out;               // permute: [rows, row_bytes];    combine: y [tokens, hidden]
    const int64_t* row_of;      // [tokens, topk]
    const int* entry_of;        // [rows]
    const void* probs;          // combine: [tokens, topk], null: none
    const void* row_probs;      // combine: if set, probs_out[t, k] = row_probs[row_of[t, k]]
    void* probs_out;
    const uint8_t* dy;          // gradient of combine: [tokens, hidden]; out = drows
    float* dprobs;
    int64_t tokens, rows, row_bytes;
    int hidden, topk, dtype, probs_dtype;
};

constexpr int MV_THREADS = 256, MV_WAVES = 4, MV_UNROLL = 4;

template <typename V> __device__ __forceinline__ V zero_of() {
    V z;
    __builtin_memset(&z, 0, sizeof(V));
    return z;
}
// zero rows of `out` that no entry goes to: 64 rows of entry_of at a time
template <typename V> __device__ __forceinline__ void zero_rows(const MoveArgs& p, int64_t wave, int64_t waves) {
    const int lane = threadIdx.x & 63;
    const int64_t vecs = p.row_bytes / (int64_t)sizeof(V);
    for (int64_t r0 = wave * 64; r0 < p.rows; r0 += waves * 64) {
        const int64_t r = r0 + lane;
        uint64_t empty = __ballot(r < p.rows && p.entry_of[r < p.rows ? r : 0] < 0);
        while (empty) {
            const int b = __builtin_ctzll(empty);
            empty &= empty - 1;
            V* o = (V*)(p.out + (r0 + b) * p.row_bytes);
            for (int64_t v = lane; v < vecs; v += 64) o[v] = zero_of<V>();
        }
    }
}

// a wave takes MV_UNROLL x 64 vectors of a token's row and stores them to its topk places
template <typename V>
__global__ __launch_bounds__(MV_THREADS) void permute_rows_kernel(MoveArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * MV_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int64_t)gridDim.x * MV_WAVES;
    const int64_t vecs = p.row_bytes / (int64_t)sizeof(V), pieces = (vecs + 64 * MV_UNROLL - 1) / (64 * MV_UNROLL);
    for (int64_t it = wave; it < p.tokens * pieces; it += waves) {
        const int64_t t = it / pieces, v0 = (it - t * pieces) * (64 * MV_UNROLL) + lane;
        const V* src = (const V*)(p.x + t * p.row_bytes);
        V d[MV_UNROLL];
#pragma unroll
        for (int u = 0; u < MV_UNROLL; ++u) d[u] = v0 + u * 64 < vecs ? __builtin_nontemporal_load(src + v0 + u * 64) : zero_of<V>();
        for (int k = 0; k < p.topk; ++k) {
            const int64_t r = p.row_of[t * p.topk + k];
            if (r < 0 || r >= p.rows) continue;
            V* o = (V*)(p.out + r * p.row_bytes);
#pragma unroll
            for (int u = 0; u < MV_UNROLL; ++u)
                if (v0 + u * 64 < vecs) __builtin_nontemporal_store(d[u], o + v0 + u * 64);
        }
    }
    zero_rows<V>(p, wave, waves);
}

// N elements at p as floats, and back (N = 16 bytes' worth, or 1)
template <int DT, int N> __device__ __forceinline__ void load_n(const uint8_t* p, float (&x)[N]) {
    if constexpr (N == 1) {
        x[0] = load_dt(p, DT, 0);
    } else {
        const m32x4 v = __builtin_nontemporal_load((const m32x4*)p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MXL_DT_F32) x[i] = __uint_as_float(v[i]);
            else if constexpr (DT == MXL_DT_BF16) x[2 * i] = bf16_lo(v[i]), x[2 * i + 1] = bf16_hi(v[i]);
            else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = __builtin_bit_cast(h2, (uint32_t)v[i]);
                x[2 * i] = (float)h[0], x[2 * i + 1] = (float)h[1];
            }
        }
    }
}
template <int DT, int N> __device__ __forceinline__ void store_n(uint8_t* p, const float (&x)[N]) {
    if constexpr (N == 1) {
        store_dt(p, DT, 0, x[0]);
    } else {
        m32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MXL_DT_F32) v[i] = __float_as_uint(x[i]);
            else if constexpr (DT == MXL_DT_BF16) v[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
            else {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                const h2 h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
                v[i] = __builtin_bit_cast(uint32_t, h);
            }
        }
        __builtin_nontemporal_store(v, (m32x4*)p);
    }
}

// a wave takes 64 vectors of a token's output row; its topk input rows are summed in fp32 in the order of k and rounded once
template <int DT, int N>
__global__ __launch_bounds__(MV_THREADS) void combine_rows_kernel(MoveArgs p) {
    constexpr int SIZE = DT == MXL_DT_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * MV_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int64_t)gridDim.x * MV_WAVES;
    const int64_t vecs = p.hidden / N, pieces = (vecs + 63) / 64;
    for (int64_t it = wave; it < p.tokens * pieces; it += waves) {
        const int64_t t = it / pieces, piece = it - t * pieces, v = piece * 64 + lane;
        if (p.probs_out && piece == 0 && lane < p.topk) {
            const int64_t r = p.row_of[t * p.topk + lane];
            const float x = r >= 0 && r < p.rows ? load_dt(p.row_probs, p.probs_dtype, r) : 0.f;
            store_dt(p.probs_out, p.probs_dtype, t * p.topk + lane, x);
        }
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
        if (v >= vecs) continue;
        for (int k = 0; k < p.topk; ++k) {
            const int64_t r = p.row_of[t * p.topk + k];
            if (r < 0 || r >= p.rows) continue;
            const float w = p.probs ? load_dt(p.probs, p.probs_dtype, t * p.topk + k) : 1.f;
            float x[N];
            load_n<DT, N>(p.x + (r * p.hidden + v * N) * SIZE, x);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = fmaf(w, x[i], acc[i]);
        }
        store_n<DT, N>(p.out + (t * p.hidden + v * N) * SIZE, acc);
    }
}

// the probabilities' part of the above alone: a thread an entry.  A launch and one wait: 32768 entries 2.4 us, 65536 2.7 (graph replays)
__global__ __launch_bounds__(MV_THREADS) void entry_probs_kernel(MoveArgs p) {
    const int64_t i = (int64_t)blockIdx.x * MV_THREADS + threadIdx.x;
    if (i >= p.tokens * p.topk) return;
    const int64_t r = p.row_of[i];
    store_dt(p.probs_out, p.probs_dtype, i, r >= 0 && r < p.rows ? load_dt(p.row_probs, p.probs_dtype, r) : 0.f);
}

// gradient of combine with probabilities: a workgroup takes a token, whose row of dy is scaled into its topk rows of drows and
// multiplied with their rows for the probabilities' gradients (fp32; the sum's order is fixed by the row length).  Eight rows at a
// time, so that a thread has nine loads on their way.
constexpr int CB_ROWS = 8;
template <int DT, int N>
__global__ __launch_bounds__(MV_THREADS) void combine_rows_bwd_kernel(MoveArgs p) {
    constexpr int SIZE = DT == MXL_DT_F32 ? 4 : 2;
    __shared__ float part[MV_WAVES][PM_MAX_TOPK];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, threads = (int)blockDim.x, block_waves = threads >> 6;
    const int64_t vecs = p.hidden / N;
    for (int64_t t = blockIdx.x; t < p.tokens; t += gridDim.x) {
        const uint8_t* dy = p.dy + t * p.hidden * SIZE;
        for (int k0 = 0; k0 < p.topk; k0 += CB_ROWS) {
            int64_t at[CB_ROWS];
            float pr[CB_ROWS], dot[CB_ROWS];
#pragma unroll
            for (int k = 0; k < CB_ROWS; ++k) {
                const int64_t r = k0 + k < p.topk ? p.row_of[t * p.topk + k0 + k] : -1;
                at[k] = r >= 0 && r < p.rows ? r * p.hidden * SIZE : -1;
                pr[k] = k0 + k < p.topk ? load_dt(p.probs, p.probs_dtype, t * p.topk + k0 + k) : 0.f;
                dot[k] = 0.f;
            }
            for (int64_t v = threadIdx.x; v < vecs; v += threads) {
                float d[N], a[CB_ROWS][N];
                load_n<DT, N>(dy + v * N * SIZE, d);
                if (p.dprobs) {
#pragma unroll
                    for (int k = 0; k < CB_ROWS; ++k)
                        if (at[k] >= 0) load_n<DT, N>(p.x + at[k] + v * N * SIZE, a[k]);
                }
#pragma unroll
                for (int k = 0; k < CB_ROWS; ++k) {
                    if (at[k] < 0) continue;
                    if (p.dprobs) {
#pragma unroll
                        for (int i = 0; i < N; ++i) dot[k] = fmaf(a[k][i], d[i], dot[k]);
                    }
                    if (p.out) {
                        float o[N];
#pragma unroll
                        for (int i = 0; i < N; ++i) o[i] = d[i] * pr[k];
                        store_n<DT, N>(p.out + at[k] + v * N * SIZE, o);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < CB_ROWS; ++k) {
                const float s = lanes_sum<64>(dot[k]);
                if (lane == 0 && k0 + k < p.topk) part[w][k0 + k] = s;
            }
        }
        __syncthreads();
        if (p.dprobs && (int)threadIdx.x < p.topk) {
            float s = 0.f;
            for (int i = 0; i < block_waves; ++i) s += part[i][threadIdx.x];
            p.dprobs[t * p.topk + threadIdx.x] = s;
        }
        __syncthreads();
    }
    if (!p.out) return;
    const int64_t wave = (int64_t)blockIdx.x * block_waves + w;
    if constexpr (N == 1) {
        if constexpr (SIZE == 2) zero_rows<uint16_t>(p, wave, (int64_t)gridDim.x * block_waves);
        else zero_rows<uint32_t>(p, wave, (int64_t)gridDim.x * block_waves);
    } else {
        zero_rows<m32x4>(p, wave, (int64_t)gridDim.x * block_waves);
    }
}

static int64_t plan_blocks(int64_t entries) {
    int64_t b = (entries + PM_CHUNK - 1) / PM_CHUNK;
    return b < 1 ? 1 : b < PM_MAX_BLOCKS ? b : PM_MAX_BLOCKS;
}
static int64_t plan_lds(int experts) { return ((int64_t)(PM_WAVES + 3) * experts + 1) * 4; }

static bool move_sizes_ok(int64_t tokens, int topk, int64_t rows) {
    return tokens >= 0 && topk >= 1 && topk <= PM_MAX_TOPK && tokens <= 0x3FFFFFFF / topk && rows >= 0 && rows <= 0x7FFFFFFF;
}
static int64_t move_blocks(int64_t items) {
    int64_t b = (items + MV_WAVES - 1) / MV_WAVES;
    return b < 1 ? 1 : b < 256 * 8 ? b : 256 * 8;
}

}  // namespace mxl

using namespace mxl;

extern "C" int64_t mxl_permute_plan_workspace_bytes(int64_t entries, int num_experts) {
    if (entries < 0 || num_experts < 1 || num_experts > MXL_MAX_GROUPS) return -1;
    const int64_t blocks = plan_blocks(entries);
    return blocks > 1 ? blocks * num_experts * 4 : 0;
}

extern "C" int mxl_permute_plan(const int64_t* indices, int64_t entries, int num_experts, int align, int64_t rows, int64_t* row_of,
                                int32_t* entry_of, int64_t* group_lens, const void* probs, int prob_bytes, void* row_probs, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    if (entries < 0 || entries > 0x3FFFFFFF || num_experts < 1 || num_experts > MXL_MAX_GROUPS || align < 1 || align > (1 << 20)) return MXL_EINVAL;
    if (rows < mxl_padded_rows_bound(entries, num_experts, align) || rows > 0x7FFFFFFF || !group_lens) return MXL_EINVAL;
    if ((entries > 0 && (!indices || !row_of)) || (rows > 0 && !entry_of)) return MXL_EINVAL;
    if (row_probs && ((prob_bytes != 2 && prob_bytes != 4) || (entries > 0 && !probs))) return MXL_EINVAL;
    const int64_t need = mxl_permute_plan_workspace_bytes(entries, num_experts);
    if (need > 0 && (workspace_bytes < need || !workspace)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    PlanArgs a{};
    a.indices = indices, a.entries = entries, a.rows = rows, a.experts = num_experts, a.align = align;
    while ((1 << a.key_bits) < num_experts) ++a.key_bits;
    const int64_t blocks = plan_blocks(entries);
    a.chunk = (int)((((entries + blocks - 1) / blocks) + PM_THREADS - 1) / PM_THREADS * PM_THREADS);
    if (a.chunk == 0) a.chunk = PM_THREADS;
    a.partial = (int*)workspace, a.row_of = row_of, a.entry_of = entry_of, a.group_lens = group_lens;
    a.probs = row_probs ? probs : nullptr, a.row_probs = row_probs, a.prob_bytes = prob_bytes;
    // (no entries: the rows' probabilities are all zero, and probs may be null)
    if (row_probs && !a.probs) a.probs = row_probs;
    hipStream_t st = (hipStream_t)stream;
    static std::atomic<bool> attr_set[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return MXL_ELAUNCH;
    if (!attr_set[dev & 63].load(std::memory_order_acquire)) {
        if (hipFuncSetAttribute((const void*)permute_place_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)plan_lds(MXL_MAX_GROUPS)) != hipSuccess)
            return MXL_ELAUNCH;
        attr_set[dev & 63].store(true, std::memory_order_release);
    }
    if (blocks > 1) hipLaunchKernelGGL(permute_count_kernel, dim3((unsigned)blocks), dim3(PM_THREADS), 0, st, a);
    hipLaunchKernelGGL(permute_place_kernel, dim3((unsigned)blocks), dim3(PM_THREADS), (unsigned)plan_lds(num_experts), st, a);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

extern "C" int mxl_permute_rows(const void* x, int64_t tokens, int64_t row_bytes, const int64_t* row_of, int topk, const int32_t* entry_of,
                                int64_t rows, void* out, void* stream) {
    if (!move_sizes_ok(tokens, topk, rows) || row_bytes < 1 || row_bytes > (1 << 24)) return MXL_EINVAL;
    if (rows == 0) return MXL_OK;
    if ((tokens > 0 && (!x || !row_of)) || !entry_of || !out) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    MoveArgs a{};
    a.x = (const uint8_t*)x, a.out = (uint8_t*)out, a.row_of = row_of, a.entry_of = entry_of, a.tokens = tokens, a.rows = rows, a.row_bytes = row_bytes, a.topk = topk;
    const uintptr_t bits = (uintptr_t)x | (uintptr_t)out | (uintptr_t)row_bytes;
    const int size = (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1;
    const int64_t pieces = (row_bytes / size + 64 * MV_UNROLL - 1) / (64 * MV_UNROLL);
    int64_t items = tokens * pieces;
    if (items < (rows + 63) / 64) items = (rows + 63) / 64;
    const dim3 grid((unsigned)move_blocks(items)), block(MV_THREADS);
    hipStream_t st = (hipStream_t)stream;
    if (size == 16) hipLaunchKernelGGL(permute_rows_kernel<m32x4>, grid, block, 0, st, a);
    else if (size == 4) hipLaunchKernelGGL(permute_rows_kernel<uint32_t>, grid, block, 0, st, a);
    else if (size == 2) hipLaunchKernelGGL(permute_rows_kernel<uint16_t>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(permute_rows_kernel<uint8_t>, grid, block, 0, st, a);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

extern "C" int mxl_permute_tokens(const void* x, int64_t tokens, int64_t row_bytes, const int64_t* indices, int topk, int num_experts, int align,
                                  int64_t rows, int64_t* row_of, int32_t* entry_of, int64_t* group_lens, const void* probs, int prob_bytes,
                                  void* row_probs, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!move_sizes_ok(tokens, topk, rows) || row_bytes < 1 || row_bytes > (1 << 24) || (tokens > 0 && !x) || (rows > 0 && !out)) return MXL_EINVAL;
    const int rc = mxl_permute_plan(indices, tokens * topk, num_experts, align, rows, row_of, entry_of, group_lens, probs, prob_bytes, row_probs,
                                    workspace, workspace_bytes, stream);
    return rc != MXL_OK ? rc : mxl_permute_rows(x, tokens, row_bytes, row_of, topk, entry_of, rows, out, stream);
}

// launches `kernel<DT, N>` for a type and whether rows are made of aligned 16-byte pieces
#define MXL_BY_TYPE(kernel, wide, grid, threads, st, a)                                                                       \
    do {                                                                                                                      \
        if (a.dtype == MXL_DT_F32) {                                                                                          \
            if (wide) hipLaunchKernelGGL((kernel<MXL_DT_F32, 4>), grid, dim3(threads), 0, st, a);                             \
            else hipLaunchKernelGGL((kernel<MXL_DT_F32, 1>), grid, dim3(threads), 0, st, a);                                  \
        } else if (a.dtype == MXL_DT_BF16) {                                                                                  \
            if (wide) hipLaunchKernelGGL((kernel<MXL_DT_BF16, 8>), grid, dim3(threads), 0, st, a);                            \
            else hipLaunchKernelGGL((kernel<MXL_DT_BF16, 1>), grid, dim3(threads), 0, st, a);                                 \
        } else {                                                                                                              \
            if (wide) hipLaunchKernelGGL((kernel<MXL_DT_F16, 8>), grid, dim3(threads), 0, st, a);                             \
            else hipLaunchKernelGGL((kernel<MXL_DT_F16, 1>), grid, dim3(threads), 0, st, a);                                  \
        }                                                                                                                     \
    } while (0)

static bool move_types_ok(int hidden, int dtype, int probs_dtype) {
    return hidden >= 1 && hidden <= (1 << 22) && dtype >= MXL_DT_F32 && dtype <= MXL_DT_F16 && probs_dtype >= MXL_DT_F32 && probs_dtype <= MXL_DT_F16;
}

extern "C" int mxl_combine_rows(const void* rows_in, int64_t rows, int hidden, int dtype, const int64_t* row_of, int64_t tokens, int topk,
                                const void* probs, const void* row_probs, void* probs_out, int probs_dtype, void* y, void* stream) {
    if (!move_sizes_ok(tokens, topk, rows) || !move_types_ok(hidden, dtype, probs_dtype)) return MXL_EINVAL;
    if (tokens == 0) return MXL_OK;         // (empty outputs, which may have no address, beside rows that are there)
    if ((row_probs != nullptr) != (probs_out != nullptr) || !row_of || (y ? rows > 0 && !rows_in : !probs_out)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    MoveArgs a{};
    a.x = (const uint8_t*)rows_in, a.out = (uint8_t*)y, a.row_of = row_of, a.probs = probs, a.row_probs = row_probs, a.probs_out = probs_out;
    a.tokens = tokens, a.rows = rows, a.hidden = hidden, a.topk = topk, a.dtype = dtype, a.probs_dtype = probs_dtype;
    if (!y) {
        hipLaunchKernelGGL(entry_probs_kernel, dim3((unsigned)((tokens * topk + MV_THREADS - 1) / MV_THREADS)), dim3(MV_THREADS), 0, (hipStream_t)stream, a);
        return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
    }
    const int size = dtype == MXL_DT_F32 ? 4 : 2;
    const bool wide = (((uintptr_t)rows_in | (uintptr_t)y | (uintptr_t)((int64_t)hidden * size)) & 15) == 0;
    const int64_t pieces = (hidden / (wide ? 16 / size : 1) + 63) / 64;
    const dim3 grid((unsigned)move_blocks(tokens * pieces));
    MXL_BY_TYPE(combine_rows_kernel, wide, grid, MV_THREADS, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}

extern "C" int mxl_combine_rows_bwd(const void* dy, const void* rows_in, int64_t rows, int hidden, int dtype, const int64_t* row_of,
                                    const int32_t* entry_of, int64_t tokens, int topk, const void* probs, int probs_dtype, void* drows,
                                    float* dprobs, void* stream) {
    if (!move_sizes_ok(tokens, topk, rows) || !move_types_ok(hidden, dtype, probs_dtype)) return MXL_EINVAL;
    if ((tokens == 0 && rows == 0) || (!drows && !dprobs)) return MXL_OK;
    if ((tokens > 0 && (!dy || !row_of || !probs)) || (rows > 0 && ((dprobs && !rows_in) || (drows && !entry_of)))) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    MoveArgs a{};
    const int size = dtype == MXL_DT_F32 ? 4 : 2;
    a.x = (const uint8_t*)rows_in, a.dy = (const uint8_t*)dy, a.out = (uint8_t*)drows, a.row_of = row_of, a.entry_of = entry_of, a.probs = probs, a.dprobs = dprobs;
    a.tokens = tokens, a.rows = rows, a.hidden = hidden, a.topk = topk, a.dtype = dtype, a.probs_dtype = probs_dtype, a.row_bytes = (int64_t)hidden * size;
    const bool wide = (((uintptr_t)rows_in | (uintptr_t)dy | (uintptr_t)drows | (uintptr_t)a.row_bytes) & 15) == 0;
    int64_t blocks = tokens > (rows + 255) / 256 ? tokens : (rows + 255) / 256;
    if (blocks > 256 * 8) blocks = 256 * 8;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks));
    // rows of up to 128 vectors: half the threads (20000 tokens of 512, two each, 77 -> 46 us; 16384 of 4096 136 with all, 138 with half)
    const int threads = hidden / (wide ? 16 / size : 1) <= MV_THREADS / 2 ? MV_THREADS / 2 : MV_THREADS;
    MXL_BY_TYPE(combine_rows_bwd_kernel, wide, grid, threads, (hipStream_t)stream, a);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}
