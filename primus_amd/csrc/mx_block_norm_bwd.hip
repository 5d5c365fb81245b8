// Gradient of the norms where blocks meet (mx_block_norm.hip).  With t the gradient of h, f = scale * gate, g = dy * weight,
// hh = h * r, xh = x * rp and n = xh * post_weight (n = x without one), means over a row:
//
//   t = dh + r * (g - hh * mean(g * hh))         dresidual = t        dweight = sum_rows dy * hh
//   dgate = scale * sum n * t over what the gate is broadcast over
//   dx = rp * (f * t * post_weight - xh * mean(f * n * t))            dpost_weight = sum_rows f * t * xh        (dx = f * t without)
//
// mean(f n t) needs t and t needs mean(g hh), but sum q t = sum q dh + r * (sum q g - mean(g hh) * sum q hh): all four sums of a
// row go through one reduction.  hh is made from h as it was stored.
//
// Workers (workgroups, or runs of lanes where rows are short) each own rows of one gate after the other, so that the gate's gradient
// is a sum in registers like the weights'.  Sums that several workers share go through float rows in the workspace, which a second
// kernel adds up in their order: no atomics.
#include "mx_block_norm.h"

namespace mxl {

struct BlockNormBwdArgs {
    const void *dy, *dh, *x, *h, *post_weight, *weight;
    const float *post_rstd, *rstd;
    Gate gate;
    float scale;
    int k, ldk, lanes;
    // rows of group g: (i / gdiv) * groups * gdiv + g * gdiv + i % gdiv, i < each; worker w has i = w % share, + share, ... of group
    // w / share, then of the groups gstep further on
    int64_t groups, each, share, gstep, gdiv, active;
    void *dx, *dres, *dgate;
    float *part_w, *part_p, *part_g;
};

template <int T, int S, int CH, bool PRE, bool POST, bool GATEV, bool SMALL>
__global__ __launch_bounds__(SMALL ? BN_SMALL_THREADS : BN_MAX_THREADS) void block_norm_bwd_kernel(BlockNormBwdArgs p) {
    constexpr int NS = PRE && POST ? 4 : 1;
    __shared__ float part[2][BN_MAX_THREADS / 64][NS];
    const int lanes = SMALL ? p.lanes : (int)blockDim.x;
    const int lane = SMALL ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
    const int64_t worker = SMALL ? (int64_t)blockIdx.x * (BN_SMALL_THREADS / lanes) + threadIdx.x / lanes : blockIdx.x;
    RowSums<NS, SMALL> sums(part, lanes);
    const int k = p.k;
    const float inv_k = 1.0f / (float)k;
    int col[CH], left[CH];
    Raw8<T> w[CH], wp[CH], gv[CH];
    float aw[CH][BN_VEC], ap[CH][BN_VEC], ag[CH][BN_VEC], ags = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        col[j] = (j * lanes + lane) * BN_VEC;
        left[j] = k - col[j];
        w[j] = wp[j] = gv[j] = none8<T>();
        if (left[j] > 0) {
            if (PRE) w[j] = load8<T>(p.weight, col[j], left[j], false);
            if (POST) wp[j] = load8<T>(p.post_weight, col[j], left[j], false);
        }
#pragma unroll
        for (int e = 0; e < BN_VEC; ++e) aw[j][e] = ap[j][e] = ag[j][e] = 0.f;
    }
    const bool gate_wanted = p.dgate != nullptr;
    const bool need_x = POST || gate_wanted;
    Raw8<T> xn[CH], dyn[CH];
    Raw8<S> hn[CH], dhn[CH];
    float rn = 0.f, rpn = 0.f;
    auto row_of = [&](int64_t g, int64_t i) -> int64_t {
        if (p.gdiv == p.each) return g * p.each + i;
        const uint32_t q = (uint32_t)i / (uint32_t)p.gdiv;
        return (int64_t)q * p.groups * p.gdiv + g * p.gdiv + ((uint32_t)i - q * (uint32_t)p.gdiv);
    };
    auto request = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            xn[j] = dyn[j] = none8<T>();
            hn[j] = dhn[j] = none8<S>();
            if (left[j] > 0) {
                const int64_t at = row * k + col[j];
                if (need_x) xn[j] = load8<T>(p.x, at, left[j], true);
                if (p.dh) dhn[j] = load8<S>(p.dh, at, left[j], true);
                if (PRE) {
                    dyn[j] = load8<T>(p.dy, at, left[j], true);
                    hn[j] = load8<S>(p.h, at, left[j], true);
                }
            }
        }
        if (PRE) rn = p.rstd[row];
        if (POST) rpn = p.post_rstd[row];
    };
    int64_t g = worker / p.share, i = worker - g * p.share, gate_row = -1;
    const int64_t first = i;
    bool live = worker < p.active && g < p.groups && i < p.each;
    int64_t row = live ? row_of(g, i) : 0;
    constexpr bool AHEAD = CH == 1;     // (two chunks a lane, a row ahead: more than 128 registers)
    if (AHEAD && live) request(row);
    while (live) {
        Raw8<T> xr[CH], dyr[CH];
        Raw8<S> hr[CH], dhr[CH];
        if (!AHEAD) request(row);
#pragma unroll
        for (int j = 0; j < CH; ++j) xr[j] = xn[j], dyr[j] = dyn[j], hr[j] = hn[j], dhr[j] = dhn[j];
        const float r = rn, rp = rpn;
        float factor = p.scale;
        if (p.gate.kind != GATE_NONE) {
            const int64_t gr = (uint32_t)row / p.gate.div % p.gate.mod;
            if (p.gate.kind == GATE_SCALAR) {
                factor *= (float)((const typename DtOf<T>::type*)p.gate.p)[gr];
            } else if (gr != gate_row) {
#pragma unroll
                for (int j = 0; j < CH; ++j)
                    if (left[j] > 0) gv[j] = load8<T>(p.gate.p, gr * k + col[j], left[j], false);
                gate_row = gr;
            }
        }
        int64_t gn = g, in = i + p.share;
        if (in >= p.each) {
            in = first;
            gn += p.gstep;
        }
        const int64_t row_now = row;
        live = gn < p.groups;
        if (live) {
            row = row_of(gn, in);
            if (AHEAD) request(row);
        }
        const bool vec = p.gate.kind == GATE_VECTOR;
        // the row's sums (columns past the row hold zeros in x, dy, h and dh; their factors may be infinite)
        float v[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) v[n] = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float xh[BN_VEC], dh[BN_VEC], dy[BN_VEC], hh[BN_VEC], ww[BN_VEC], wpp[BN_VEC], gg[BN_VEC];
            unpack8<S>(dhr[j], dh);
            if (PRE) {
                unpack8<T>(dyr[j], dy);
                unpack8<S>(hr[j], hh);
                unpack8<T>(w[j], ww);
            }
            if (POST) {
                unpack8<T>(xr[j], xh);
                unpack8<T>(wp[j], wpp);
                unpack8<T>(gv[j], gg);
            }
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                const bool in_row = col[j] + e < k;
                float q = 0.f;
                if (POST) {
                    q = xh[e] * rp * wpp[e];
                    if (vec) q *= factor * gg[e];
                }
                if (PRE) {
                    const float d = dy[e] * ww[e], n = hh[e] * r;
                    if (in_row) {
                        v[0] += d * n;
                        if (POST) {
                            v[NS - 3] += q * dh[e];
                            v[NS - 2] += q * d;
                            v[NS - 1] += q * n;
                        }
                    }
                } else if (in_row) {
                    v[0] += q * dh[e];
                }
            }
        }
        sums(v);
        // mean(g hh), and sum q t (q without a gate that is the same for the whole row)
        const float c1 = PRE ? v[0] * inv_k : 0.f;
        float qt = 0.f;
        if (POST) qt = PRE ? v[NS - 3] + r * (v[NS - 2] - c1 * v[NS - 1]) : v[0];
        const float c2 = vec ? qt * inv_k : factor * qt * inv_k;
        float nt = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float x[BN_VEC], t[BN_VEC], dy[BN_VEC], hh[BN_VEC], ww[BN_VEC], wpp[BN_VEC], gg[BN_VEC], o[BN_VEC];
            unpack8<S>(dhr[j], t);
            unpack8<T>(xr[j], x);
            unpack8<T>(gv[j], gg);
            if (PRE) {
                unpack8<T>(dyr[j], dy);
                unpack8<S>(hr[j], hh);
                unpack8<T>(w[j], ww);
            }
            if (POST) unpack8<T>(wp[j], wpp);
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                if (PRE) {
                    const float n = hh[e] * r;
                    t[e] += r * (dy[e] * ww[e] - n * c1);
                    aw[j][e] += dy[e] * n;
                }
                const float ft = (vec ? factor * gg[e] : factor) * t[e];
                if (POST) {
                    x[e] *= rp;
                    o[e] = rp * (ft * wpp[e] - x[e] * c2);
                    ap[j][e] += ft * x[e];
                    if (GATEV) ag[j][e] += x[e] * wpp[e] * t[e];
                } else {
                    o[e] = ft;
                    if (GATEV) ag[j][e] += x[e] * t[e];
                    else if (gate_wanted && col[j] + e < k) nt += x[e] * t[e];
                }
            }
            if (left[j] > 0) {
                if (p.dx) store8<T>(p.dx, row_now * k + col[j], left[j], o);
                if (p.dres) store8<S>(p.dres, row_now * k + col[j], left[j], t);
            }
        }
        if (!GATEV && gate_wanted) {
            if (POST) {
                nt = qt;
            } else {
                float s[NS];
                s[0] = nt;
                sums(s);
                nt = s[0];
            }
            ags += nt;
        }
        if (gate_wanted && p.share == 1 && gn != g) {
            if (GATEV) {
#pragma unroll
                for (int j = 0; j < CH; ++j) {
#pragma unroll
                    for (int e = 0; e < BN_VEC; ++e) ag[j][e] *= p.scale;
                    if (left[j] > 0) store8<T>(p.dgate, g * k + col[j], left[j], ag[j]);
#pragma unroll
                    for (int e = 0; e < BN_VEC; ++e) ag[j][e] = 0.f;
                }
            } else {
                if (lane == 0) ((typename DtOf<T>::type*)p.dgate)[g] = (typename DtOf<T>::type)(ags * p.scale);
                ags = 0.f;
            }
        }
        g = gn;
        i = in;
    }
    // what several workers share, for the second kernel: a row of a workgroup or, of short rows, of a wave
    int64_t to = blockIdx.x;
    bool writes = true;
    if (SMALL) {
        for (int m = lanes; m < 64; m *= 2) {
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                if (PRE) aw[0][e] += __shfl_xor(aw[0][e], m);
                if (POST) ap[0][e] += __shfl_xor(ap[0][e], m);
                if (GATEV) ag[0][e] += __shfl_xor(ag[0][e], m);
            }
            ags += __shfl_xor(ags, m);
        }
        to = (int64_t)blockIdx.x * (BN_SMALL_THREADS / 64) + (threadIdx.x >> 6);
        writes = (threadIdx.x & 63) < lanes;
    }
    if (!writes) return;
    auto put = [&](float* base, const float* v, int c) {
        float* d = base + to * p.ldk + c;
        *(float4*)d = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
    };
#pragma unroll
    for (int j = 0; j < CH; ++j)
        if (left[j] > 0) {
            if (PRE && p.part_w) put(p.part_w, aw[j], col[j]);
            if (POST && p.part_p) put(p.part_p, ap[j], col[j]);
            if (GATEV && p.part_g) put(p.part_g, ag[j], col[j]);
        }
    if (!GATEV && p.part_g && lane == 0) p.part_g[to] = ags;
}

// Column sums of float rows: up to two of the weights over all `rows`, and those of the gate over `gate_share` rows a gate.  A workgroup
// owns 32 columns: thread (bg, cg) adds rows bg, bg + 32, ... of four columns, then the 32 sums are added, in order.
struct BlockNormSumArgs {
    const float* part[2];
    void* out[2];
    int jobs, dtype, k, ldk, blocks_x;
    int64_t rows;
    const float* part_g;
    void* dgate;
    int64_t gates, gate_share;
    int gate_scalar;
    float scale;
};
constexpr int BS_THREADS = 256, BS_LOADS = 16;

__global__ __launch_bounds__(BS_THREADS) void block_norm_sum_kernel(BlockNormSumArgs p) {
    __shared__ float4 part[32][8];
    int64_t job = blockIdx.x / p.blocks_x;
    int cb = blockIdx.x - (int)job * p.blocks_x;
    const float* src;
    void* dst;
    int64_t rows = p.rows, at = 0;
    float scale = 1.f;
    if (job < p.jobs) {
        src = p.part[job];
        dst = p.out[job];
    } else if (!p.gate_scalar) {
        const int64_t gate = job - p.jobs;
        src = p.part_g + gate * p.gate_share * p.ldk;
        rows = p.gate_share;
        dst = p.dgate;
        at = gate * p.k;
        scale = p.scale;
    } else {
        // a wave a gate
        const int64_t gate = ((int64_t)blockIdx.x - (int64_t)p.jobs * p.blocks_x) * (BS_THREADS / 64) + (threadIdx.x >> 6);
        if (gate >= p.gates) return;
        float s = 0.f;
        for (int64_t r = threadIdx.x & 63; r < p.gate_share; r += 64) s += p.part_g[gate * p.gate_share + r];
        s = lanes_sum<64>(s);
        if ((threadIdx.x & 63) == 0) store_dt(p.dgate, p.dtype, gate, s * p.scale);
        return;
    }
    const int cg = threadIdx.x & 7, bg = threadIdx.x >> 3;
    const int c = cb * 32 + 4 * cg;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < p.k) {
        for (int64_t b0 = bg; b0 < rows; b0 += 32 * BS_LOADS) {
            float4 v[BS_LOADS];
#pragma unroll
            for (int u = 0; u < BS_LOADS; ++u) {
                v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (b0 + 32 * u < rows) v[u] = *(const float4*)(src + (b0 + 32 * u) * p.ldk + c);
            }
#pragma unroll
            for (int u = 0; u < BS_LOADS; ++u) {
                s.x += v[u].x;
                s.y += v[u].y;
                s.z += v[u].z;
                s.w += v[u].w;
            }
        }
    }
    part[bg][cg] = s;
    __syncthreads();
    if (bg == 0 && c < p.k) {
        float4 t = part[0][cg];
        for (int i = 1; i < 32; ++i) {
            const float4 v = part[i][cg];
            t.x += v.x;
            t.y += v.y;
            t.z += v.z;
            t.w += v.w;
        }
        const float o[4] = {t.x, t.y, t.z, t.w};
        for (int e = 0; e < 4; ++e)
            if (c + e < p.k) store_dt(dst, p.dtype, at + c + e, o[e] * scale);
    }
}

// How the rows are dealt out, by the sizes alone.
struct BlockNormPlan {
    int64_t groups, each, share, gstep, gdiv, active;
    int blocks, threads, lanes, ldk;
    int64_t part_rows;      // float rows of a weight's sums
};
static BlockNormPlan block_norm_plan(int64_t rows, int64_t k, bool gate_wanted, int64_t div, int64_t mod) {
    BlockNormPlan q;
    const bool small = k <= BN_SMALL_K;
    q.lanes = small ? bn_lanes(k) : 0;
    q.threads = small ? BN_SMALL_THREADS : bn_threads(k);
    q.ldk = (int)((k + 7) / 8 * 8);
    const int64_t per_block = small ? BN_SMALL_THREADS / q.lanes : 1, per_wave = small ? 64 / q.lanes : 1;
    q.groups = gate_wanted ? mod : 1;
    q.gdiv = gate_wanted ? div : rows;
    q.each = rows / q.groups;
    int64_t cap = small ? 1024 : 256 * 1024 / q.threads;
    if (small) {
        const int64_t want = (rows + per_block * 4 - 1) / (per_block * 4);
        cap = want < cap ? want : cap;
    }
    const int64_t workers = cap * per_block;
    int64_t share = (workers + q.groups - 1) / q.groups;
    if (share > q.each) share = q.each;
    if (share > 1) share = (share + per_wave - 1) / per_wave * per_wave;
    q.share = share;
    if (share > 1 || q.groups <= workers) {
        q.active = q.groups * share;
        q.gstep = q.groups;
    } else {
        q.active = q.gstep = workers;
    }
    q.blocks = (int)((q.active + per_block - 1) / per_block);
    q.part_rows = small ? (int64_t)q.blocks * (BN_SMALL_THREADS / 64) : q.blocks;
    return q;
}
static int64_t block_norm_gate_rows(const BlockNormPlan& q) {       // float rows (or floats) of the gate's sums
    return q.share > 1 ? q.part_rows : 0;
}

template <int T, int S, int CH, bool GATEV, bool SMALL>
static void block_norm_bwd_launch(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st) {
    const dim3 g((unsigned)q.blocks), b((unsigned)q.threads);
    if (p.weight && p.post_weight) hipLaunchKernelGGL((block_norm_bwd_kernel<T, S, CH, true, true, GATEV, SMALL>), g, b, 0, st, p);
    else if (p.weight) hipLaunchKernelGGL((block_norm_bwd_kernel<T, S, CH, true, false, GATEV, SMALL>), g, b, 0, st, p);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<T, S, CH, false, true, GATEV, SMALL>), g, b, 0, st, p);
}
template <int T, int S> static void block_norm_bwd_launch(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st) {
    const bool gv = p.dgate && p.gate.kind == GATE_VECTOR;
    if (q.lanes) {
        if (gv) block_norm_bwd_launch<T, S, 1, true, true>(p, q, st);
        else block_norm_bwd_launch<T, S, 1, false, true>(p, q, st);
    } else if (bn_chunks(p.k) == 1) {
        if (gv) block_norm_bwd_launch<T, S, 1, true, false>(p, q, st);
        else block_norm_bwd_launch<T, S, 1, false, false>(p, q, st);
    } else {
        if (gv) block_norm_bwd_launch<T, S, 2, true, false>(p, q, st);
        else block_norm_bwd_launch<T, S, 2, false, false>(p, q, st);
    }
}

}  // namespace mxl

using namespace mxl;

static int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

extern "C" int64_t mxl_block_norm_bwd_workspace_bytes(int64_t rows, int64_t k, int has_weight, int has_post_weight, int64_t gate_div, int64_t gate_mod,
                                                      int64_t gate_cols) {
    static const int any = 0;
    if (!bn_shape_ok(rows, k, MXL_DT_F32, MXL_DT_F32) || !bn_gate_ok(rows, k, gate_cols ? &any : nullptr, gate_div, gate_mod, gate_cols)) return -1;
    if (rows == 0) return 0;
    const BlockNormPlan q = block_norm_plan(rows, k, gate_cols != 0, gate_div, gate_mod);
    int64_t n = (int64_t)((has_weight != 0) + (has_post_weight != 0)) * q.part_rows * q.ldk * 4;
    if (gate_cols) n += block_norm_gate_rows(q) * (gate_cols == k ? q.ldk : 1) * 4;
    return round16(n);
}

extern "C" int mxl_block_norm_bwd(const void* dy, const void* dh, const void* x, const void* h, int64_t rows, int64_t k, int dtype, int stream_dtype,
                                  const void* post_weight, const float* post_rstd, const void* gate, int64_t gate_div, int64_t gate_mod,
                                  int64_t gate_cols, float scale, const void* weight, const float* rstd, void* dx, void* dresidual, void* dweight,
                                  void* dpost_weight, void* dgate, void* workspace, int64_t workspace_bytes, void* stream) {
    if (!bn_shape_ok(rows, k, dtype, stream_dtype) || (!weight && !post_weight) || (dgate && !gate)) return MXL_EINVAL;
    if (!bn_gate_ok(rows, k, gate, gate_div, gate_mod, gate_cols)) return MXL_EINVAL;
    if ((dweight && !weight) || (dpost_weight && !post_weight)) return MXL_EINVAL;
    if (rows == 0) {
        // sums over no rows, written by the second kernel
        if (!dweight && !dpost_weight) return MXL_OK;
        if (!device_is_gfx950()) return MXL_ENODEV;
    }
    BlockNormPlan q;
    const int64_t need = mxl_block_norm_bwd_workspace_bytes(rows, k, dweight != nullptr, dpost_weight != nullptr, gate_div, gate_mod, dgate ? gate_cols : 0);
    if (rows > 0) {
        if ((weight && (!dy || !h || !rstd)) || (post_weight && (!x || !post_rstd)) || (dgate && !x)) return MXL_EINVAL;
        if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)) return MXL_EINVAL;
        if (!device_is_gfx950()) return MXL_ENODEV;
        q = block_norm_plan(rows, k, dgate != nullptr, gate_div, gate_mod);
    } else {
        q = BlockNormPlan{};
        q.ldk = (int)((k + 7) / 8 * 8);
    }
    hipStream_t st = (hipStream_t)stream;
    float* ws = (float*)workspace;
    float *part_w = nullptr, *part_p = nullptr, *part_g = nullptr;
    if (dweight) part_w = ws, ws += q.part_rows * q.ldk;
    if (dpost_weight) part_p = ws, ws += q.part_rows * q.ldk;
    const bool gate_joined = rows > 0 && dgate && q.share > 1;
    if (gate_joined) part_g = ws;
    if (rows > 0) {
        BlockNormBwdArgs p = {dy, dh, x, h, post_weight, weight, post_rstd, rstd, bn_gate(gate, rows, gate_div, gate_mod, gate_cols, k), scale, (int)k, q.ldk,
                              q.lanes, q.groups, q.each, q.share, q.gstep, q.gdiv, q.active, dx, dresidual, dgate, part_w, part_p, part_g};
        if (dtype == MXL_DT_F32) block_norm_bwd_launch<MXL_DT_F32, MXL_DT_F32>(p, q, st);
        else if (dtype == MXL_DT_BF16 && stream_dtype == MXL_DT_BF16) block_norm_bwd_launch<MXL_DT_BF16, MXL_DT_BF16>(p, q, st);
        else if (dtype == MXL_DT_BF16) block_norm_bwd_launch<MXL_DT_BF16, MXL_DT_F32>(p, q, st);
        else if (stream_dtype == MXL_DT_F16) block_norm_bwd_launch<MXL_DT_F16, MXL_DT_F16>(p, q, st);
        else block_norm_bwd_launch<MXL_DT_F16, MXL_DT_F32>(p, q, st);
        if (hipGetLastError() != hipSuccess) return MXL_ELAUNCH;
    }
    BlockNormSumArgs s = {};
    if (dweight) s.part[s.jobs] = part_w, s.out[s.jobs++] = dweight;
    if (dpost_weight) s.part[s.jobs] = part_p, s.out[s.jobs++] = dpost_weight;
    s.dtype = dtype, s.k = (int)k, s.ldk = q.ldk, s.blocks_x = (int)((k + 31) / 32), s.rows = q.part_rows, s.scale = scale;
    int64_t grid = (int64_t)s.jobs * s.blocks_x;
    if (gate_joined) {
        s.part_g = part_g, s.dgate = dgate, s.gates = q.groups;
        s.gate_scalar = gate_cols != k;
        // (a wave of short rows has summed its workers' sums)
        s.gate_share = q.share / (q.lanes ? 64 / q.lanes : 1);
        grid += s.gate_scalar ? (s.gates + BS_THREADS / 64 - 1) / (BS_THREADS / 64) : s.gates * s.blocks_x;
    }
    if (grid == 0) return MXL_OK;
    hipLaunchKernelGGL(block_norm_sum_kernel, dim3((unsigned)grid), dim3(BS_THREADS), 0, st, s);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}
