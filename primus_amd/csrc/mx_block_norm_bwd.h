// Gradient of the norms where blocks meet (mx_block_norm.hip); a source file for each type instantiates the kernels.
// With t the gradient of h, f = scale * gate, g = dy * weight, hh = h * r, xh = x * rp and n = xh * post_weight (n = x without one), means
// over a row:
//
//   t = dh + r * (g - hh * mean(g * hh))         dresidual = t        dweight = sum_rows dy * hh
//   dgate = scale * sum n * t over what the gate is broadcast over
//   dx = rp * (f * t * post_weight - xh * mean(f * n * t))            dpost_weight = sum_rows f * t * xh        (dx = f * t without)
//
// mean(f n t) needs t and t needs mean(g hh), but sum q t = sum q dh + r * (sum q g - mean(g hh) * sum q hh): all four sums of a
// row go through one reduction.
//
// hh is made from h as it was stored where that is in fp32, and where dweight is not wanted.  Otherwise h is summed again from x and the residual: the
// rounding of h to 16 bits in every hh is as large as dweight's own, [16384, 4096] bf16 2.4e-3 of its norm off, 1.8e-3 so.  Nothing more is read with
// post_weight or a gate's gradient, x is read for those anyway; without them a tensor more, us from h and so: [16384, 4096] 90 and 113, [8192, 7168] 78 and 99.
//
// Workers (workgroups, or runs of lanes where rows are short) each own rows of one gate after the other, so that the gate's gradient
// is a sum in registers like the weights'.  Sums that several workers share go through float rows in the workspace, which a second
// kernel adds up in their order: no atomics.
//
// Bound by memory, and near to it by instructions: a row's floats are made once and stay in registers over the reduction, and what a whole row
// multiplies is applied to the sums.  us (TB/s) from memory: add and norm [16384, 4096] 113 (5.9); norm and add with a gate a channel [8192, 7168]
// 63 (5.6); both norms, a gate a sequence, the stream in fp32 [5403, 2880] 57 (4.9).  A row ahead pays where a CU holds one workgroup (over 512
// threads: [8192, 7168] from h 93 -> 78 us), and costs where it holds more ([16384, 4096] 90 -> 96): others' loads are on their way then anyway.
#pragma once
#include "mx_block_norm.h"

namespace mxl {

struct BlockNormBwdArgs {
    const void *dy, *dh, *x, *h, *post_weight, *weight;
    const float *post_rstd, *rstd;
    Gate gate;
    float scale;
    int k, ldk, lanes;
    int64_t rows;
    // rows of group g: (i / gdiv) * groups * gdiv + g * gdiv + i % gdiv, i < each; worker w has i = w % share, + share, ... of group
    // w / share, then of the groups gstep further on
    int64_t groups, each, share, gstep, gdiv, active;
    bool summed;        // h is the residual: with x it makes h as the forward had it (16-bit streams)
    void *dx, *dres, *dgate;
    float *part_w, *part_p, *part_g;
};

// Whether a lane has the weights and their sums in registers.  Two chunks of both norms, or of a norm and a gate of vectors, do not fit: the
// weights are loaded again for every row (from the caches) and their sums are in shared memory, 64 bytes a lane each.  us, in registers (spilt)
// and so, [2730, 12288]: both norms 158 and 109, and a stream in fp32 and a gate 263 and 199, a norm and a gate a row 122 and 111; a norm without
// one 62 and 69.  Two chunks use scratch all the same, by the compiler's report, bytes a lane: both norms and a gate of vectors 100 to 264, both norms without one
// up to 84, one norm up to 88.
constexpr bool bn_bwd_keeps(int chunks, bool pre, bool post, bool gate) { return chunks == 1 || !pre || !(post || gate); }

// SAME: no gradient of x apart from the residual's.  GATEV: the gate is a vector, and groups are its rows.  AHEAD: the next row is asked for
// before the present one is worked on.
template <int T, int S, int CH, bool PRE, bool POST, bool SAME, bool GATEV, bool SMALL, bool ANY, int BOUND, bool AHEAD>
__global__ __launch_bounds__(BOUND) void block_norm_bwd_kernel(BlockNormBwdArgs p) {
    constexpr int NS = PRE && POST ? 4 : 1;
    constexpr bool SUM = PRE && S != MXL_DT_F32;        // h may have to be summed again
    __shared__ float part[2][BN_MAX_WAVES][NS];
    const int lanes = SMALL ? p.lanes : (int)blockDim.x;
    const int lane = SMALL ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
    const int64_t worker = SMALL ? (int64_t)blockIdx.x * (BN_SMALL_THREADS / lanes) + threadIdx.x / lanes : blockIdx.x;
    RowSums<NS, SMALL> sums(part, lanes);
    const int k = p.k;
    const float inv_k = 1.0f / (float)k;
    typedef RowsOf<T, S, SMALL, ANY> RowsT;
    typedef RowsOf<S, S, SMALL, ANY> RowsS;
    const Cols<S> cols = {lanes, lane, k};
    constexpr bool KEEP = bn_bwd_keeps(CH, PRE, POST, GATEV);
    // wq: post_weight times the gate where that is a vector.  au: sum of xh t (x t without post_weight) over the rows of one gate, whose
    // gradient is scale * post_weight times that, and dpost_weight's part of them scale * gate times it.
    float w[CH][BN_VEC], wp[CH][BN_VEC], wq[CH][BN_VEC];
    Raw8<T> gv[CH];
    float aw[CH][BN_VEC], ap[CH][BN_VEC], au[CH][BN_VEC], ags = 0.f;
    extern __shared__ __attribute__((aligned(16))) uint8_t bn_lds[];
    float4* const sums_of = (float4*)bn_lds + lane;
    auto add = [&](float (&reg)[CH][BN_VEC], int which, int j, const float* v) {
        if constexpr (KEEP) {
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) reg[j][e] += v[e];
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float4* s = sums_of + ((which * CH + j) * 2 + q) * lanes;
                const float4 o = *s;
                *s = make_float4(o.x + v[4 * q], o.y + v[4 * q + 1], o.z + v[4 * q + 2], o.w + v[4 * q + 3]);
            }
        }
    };
    auto weight = [&](const void* base, int j, float* v) { unpack8<T>(load_vector<T>(base, cols, j), v); };
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        gv[j] = none8<T>();
        if (KEEP && PRE) weight(p.weight, j, w[j]);
        if (KEEP && POST) weight(p.post_weight, j, wp[j]);
#pragma unroll
        for (int e = 0; e < BN_VEC; ++e) aw[j][e] = ap[j][e] = au[j][e] = 0.f;
        if (!KEEP) {        // (a lane has its sums to itself: no barrier)
#pragma unroll
            for (int q = 0; q < 2 * (PRE + POST); ++q) sums_of[(q / 2 * CH * 2 + j * 2 + q % 2) * lanes] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    const bool gate_wanted = p.dgate != nullptr;
    const bool summed = SUM && p.summed;
    const void* x_in = POST || gate_wanted || summed ? p.x : nullptr;

    // a row as it lies in memory
    Raw8<T> xn[CH], dyn[CH];
    Raw8<S> hn[CH], dhn[CH];
    float rn = 0.f, rpn = 0.f;
    auto request = [&](int64_t row) {
        const RowsT in_x(x_in, p.rows, row, k), in_dy(p.dy, p.rows, row, k);
        const RowsS in_h(p.h, p.rows, row, k), in_dh(p.dh, p.rows, row, k);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            if (!SAME || SUM) xn[j] = in_x.template load<BN_NT>(cols, j);
            dhn[j] = in_dh.template load<BN_NT>(cols, j);
            if (PRE) {
                dyn[j] = in_dy.template load<BN_NT>(cols, j);
                hn[j] = in_h.template load<BN_NT>(cols, j);
            }
        }
        if (PRE) rn = p.rstd[row];
        if (POST) rpn = p.post_rstd[row];
    };
    // this worker's rows
    struct At {
        int64_t g, i, row;
        bool live;
    };
    const int64_t g0 = worker / p.share, first = worker - g0 * p.share;
    auto row_of = [&](At& a) {
        if (p.gdiv == p.each) {
            a.row = a.g * p.each + a.i;
        } else {
            const uint32_t q = (uint32_t)a.i / (uint32_t)p.gdiv;
            a.row = (int64_t)q * p.groups * p.gdiv + a.g * p.gdiv + ((uint32_t)a.i - q * (uint32_t)p.gdiv);
        }
    };
    auto advance = [&](At& a) {
        a.i += p.share;
        if (a.i >= p.each) {
            a.i = first;
            a.g += p.gstep;
        }
        a.live = a.g < p.groups;
        if (a.live) row_of(a);
    };
    At at = {g0, first, 0, worker < p.active && g0 < p.groups && first < p.each}, ahead;
    if (at.live) row_of(at);
    ahead = at;
    if (AHEAD && ahead.live) {
        request(ahead.row);
        advance(ahead);
    }
    int64_t gate_row = -1;
    auto gated = [&](int j) {       // wq of a vector gate
        float f[BN_VEC];
        unpack8<T>(gv[j], f);
#pragma unroll
        for (int e = 0; e < BN_VEC; ++e) wq[j][e] = POST ? p.scale * f[e] * wp[j][e] : p.scale * f[e];
    };
    auto gate_done = [&](int j, float* dgate) {     // what the rows of one gate have added up to
        float f[BN_VEC];
        if (POST) unpack8<T>(gv[j], f);
        if (!KEEP && POST) weight(p.post_weight, j, wp[j]);
#pragma unroll
        for (int e = 0; e < BN_VEC; ++e) {
            if (POST) f[e] *= p.scale * au[j][e];
            dgate[e] = p.scale * (POST ? wp[j][e] * au[j][e] : au[j][e]);
            au[j][e] = 0.f;
        }
        if (POST) add(ap, PRE, j, f);
    };

    while (at.live) {
        if (!AHEAD) request(at.row);
        // the row's chunks as floats, x (with post_weight) and h normalised
        float x[CH][BN_VEC], t[CH][BN_VEC], dy[CH][BN_VEC], hh[CH][BN_VEC];
        const float r = rn, rp = rpn;
        auto weights_again = [&](int j) {
            const void *pw = p.weight, *pp = p.post_weight;
            asm volatile("" : "+s"(pw), "+s"(pp));      // (or they are loaded in front of the loop, and kept)
            if (PRE) weight(pw, j, w[j]);
            if (POST) weight(pp, j, wp[j]);
            if (GATEV) gated(j);
        };
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            unpack8<S>(dhn[j], t[j]);
            if (!SAME || SUM) unpack8<T>(xn[j], x[j]);
            if (PRE) {
                unpack8<T>(dyn[j], dy[j]);
                unpack8<S>(hn[j], hh[j]);
            }
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                if (POST) x[j][e] *= rp;
                if (PRE && !SUM) hh[j][e] *= r;
            }
        }
        const int64_t row = at.row;
        float factor = p.scale;
        if (GATEV) {
            if (at.g != gate_row) {
                const RowsT in_g(p.gate.p, p.groups, at.g, k);
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    gv[j] = in_g.template load<0>(cols, j);
                    if (KEEP) gated(j);
                }
                gate_row = at.g;
            }
        } else if (p.gate.kind == GATE_SCALAR) {
            const int64_t gr = gate_wanted ? at.g : (int64_t)((uint32_t)row / p.gate.div % p.gate.mod);
            factor *= (float)((const typename DtOf<T>::type*)p.gate.p)[gr];
        }
        if (AHEAD && ahead.live) {
            request(ahead.row);
            advance(ahead);
        }
        const float whole = GATEV ? 1.f : factor;       // of f: what wq does not have
        // The row's sums.  (Columns past the row hold zeros in all that is read, a gate's vector too.  A factor of the whole row, which may
        // be infinite, is applied behind the sums; r and rp are infinite for a row of zeros without eps alone, whose gradients are NaN.)
        float v[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) v[n] = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            if (!KEEP) weights_again(j);
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                float q = 0.f;
                if (POST) {
                    q = x[j][e] * (GATEV ? wq[j][e] : wp[j][e]);
                }
                if (SUM) {
                    const float n = POST ? q : GATEV ? x[j][e] * wq[j][e] : x[j][e];
                    hh[j][e] = (summed ? hh[j][e] + n * whole : hh[j][e]) * r;
                }
                if (PRE) {
                    const float d = dy[j][e] * w[j][e];
                    v[0] += d * hh[j][e];
                    if (POST) {
                        v[NS - 3] += q * t[j][e];
                        v[NS - 2] += q * d;
                        v[NS - 1] += q * hh[j][e];
                    }
                } else {
                    v[0] += q * t[j][e];
                }
            }
        }
        sums(v);
        // mean(g hh), and sum q t of q = f n without what f has for the whole row
        const float c1 = PRE ? v[0] * inv_k : 0.f;
        float qt = 0.f;
        if (POST) qt = PRE ? v[NS - 3] + r * (v[NS - 2] - c1 * v[NS - 1]) : v[0];
        const float rc1 = r * c1, rw = rp * whole, rc2 = rw * (qt * inv_k);
        float nt = 0.f;
        const RowsT out_x(p.dx, p.rows, row, k);
        const RowsS out_r(p.dres, p.rows, row, k);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float o[BN_VEC], of_w[BN_VEC], of_p[BN_VEC];
            if (!KEEP) weights_again(j);
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                if (PRE) {
                    t[j][e] += r * (dy[j][e] * w[j][e]);
                    t[j][e] -= hh[j][e] * rc1;
                    of_w[e] = dy[j][e] * hh[j][e];
                }
                if (POST) {
                    o[e] = t[j][e] * (GATEV ? wq[j][e] : wp[j][e]) * rw - x[j][e] * rc2;
                    if (GATEV) au[j][e] += x[j][e] * t[j][e];
                    else of_p[e] = x[j][e] * t[j][e] * whole;
                } else {
                    if (GATEV) au[j][e] += x[j][e] * t[j][e];
                    else if (!SAME) nt += x[j][e] * t[j][e];
                    if (!SAME) o[e] = t[j][e] * (GATEV ? wq[j][e] : factor);
                }
            }
            if (PRE) add(aw, 0, j, of_w);
            if (POST && !GATEV) add(ap, PRE, j, of_p);
            if (!SAME) out_x.store(cols, j, o);
            if (PRE) out_r.store(cols, j, t[j]);
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
        const int64_t g = at.g;
        advance(at);
        if ((GATEV || gate_wanted) && p.share == 1 && at.g != g) {
            if (GATEV) {
                const RowsT out_g(p.dgate, p.groups, g, k);
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    float o[BN_VEC];
                    gate_done(j, o);
                    out_g.store(cols, j, o);
                }
            } else {
                if (lane == 0) ((typename DtOf<T>::type*)p.dgate)[g] = (typename DtOf<T>::type)(ags * p.scale);
                ags = 0.f;
            }
        }
    }
    // what several workers share, for the second kernel: a row of a workgroup or, of short rows, of a wave
    float ag[CH][BN_VEC];
    if (GATEV) {
        // (a worker that has its gates to itself is done with each of them; once more, with sums of zero, an infinite gate would add NaN)
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            if (p.share > 1) {
                gate_done(j, ag[j]);
            } else {
#pragma unroll
                for (int e = 0; e < BN_VEC; ++e) ag[j][e] = 0.f;
            }
        }
    }
    if (!KEEP) {
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (PRE) *(float4*)&aw[j][4 * q] = sums_of[(j * 2 + q) * lanes];
                if (POST) *(float4*)&ap[j][4 * q] = sums_of[((PRE * CH + j) * 2 + q) * lanes];
            }
    }
    int64_t to = blockIdx.x;
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
        if ((int)(threadIdx.x & 63) >= lanes) return;
    }
    auto put = [&](float* base, const float* v, int j) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
            if (cols(j, 4 * q) < k) *(float4*)(base + to * p.ldk + cols(j, 4 * q)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    };
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        if (PRE && p.part_w) put(p.part_w, aw[j], j);
        if (POST && p.part_p) put(p.part_p, ap[j], j);
        if (GATEV && p.part_g) put(p.part_g, ag[j], j);
    }
    if (!GATEV && p.part_g && lane == 0) p.part_g[to] = ags;
}

// How the rows are dealt out, by the sizes alone.  grouped: by the gate's rows.
struct BlockNormPlan {
    int64_t groups, each, share, gstep, gdiv, active;
    int blocks, threads, lanes, ldk, chunks;
    int64_t part_rows;      // float rows of a weight's sums
};
inline BlockNormPlan block_norm_plan(int64_t rows, int64_t k, bool grouped, int64_t div, int64_t mod) {
    BlockNormPlan q;
    const bool small = k <= BN_SMALL_K;
    q.lanes = small ? bn_lanes(k) : 0;
    q.chunks = k <= BN_MAX_THREADS * BN_VEC ? 1 : 2;
    q.threads = small ? BN_SMALL_THREADS : bn_threads(k, q.chunks);
    q.ldk = (int)((k + 7) / 8 * 8);
    const int64_t per_block = small ? BN_SMALL_THREADS / q.lanes : 1, per_wave = small ? 64 / q.lanes : 1;
    q.groups = grouped ? mod : 1;
    q.gdiv = grouped ? div : rows;
    q.each = rows / q.groups;
    // as many workgroups as the chip holds at once (sixteen waves a CU at the kernels' registers), each with all its rows: one more is
    // another round.  [8192, 7168] gradient of the norm after a block, 256 workgroups 126 us, 292 154.
    int64_t cap = small ? 1024 : 256 * (BN_MAX_THREADS / q.threads);
    if (small) {
        const int64_t want = (rows + per_block * 4 - 1) / (per_block * 4);
        cap = want < cap ? want : cap;
    }
    const int64_t workers = cap * per_block;
    int64_t share = workers / q.groups;
    if (share > q.each) share = q.each;
    if (share > 1) share = (share + per_wave - 1) / per_wave * per_wave;
    if (share < 1) share = 1;
    q.share = share;
    q.active = q.groups <= workers ? q.groups * share : workers;
    q.gstep = q.groups <= workers ? q.groups : workers;
    q.blocks = (int)((q.active + per_block - 1) / per_block);
    q.part_rows = small ? (int64_t)q.blocks * (BN_SMALL_THREADS / 64) : q.blocks;
    return q;
}
inline int64_t block_norm_gate_rows(const BlockNormPlan& q) {       // float rows (or floats) of the gate's sums
    return q.share > 1 ? q.part_rows : 0;
}

template <int T, int S> int block_norm_bwd_launch(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st);

}  // namespace mxl
