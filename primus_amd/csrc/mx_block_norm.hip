// RMSNorms where blocks meet, with the residual add, the block's gate and its residual scale:
//
//   n = x * rp * post_weight,  rp = 1 / sqrt(mean_j x^2 + post_eps)     (n = x without post_weight)
//   h = residual + scale * gate * n
//   y = h * r * weight,        r = 1 / sqrt(mean_j h^2 + eps)           (not without weight)
//
// fp32 from the inputs to y and h, which are rounded once each: y is the norm of the sums before their rounding.  A row stays in
// registers from its load to its last store.
#include "mx_block_norm.h"

namespace mxl {

struct BlockNormArgs {
    const void *x, *residual, *post_weight, *weight;
    Gate gate;
    float scale, post_eps, eps;
    int64_t rows, row0;         // this launch's first row
    int k, lanes;
    void *y, *h;
    float *post_rstd, *rstd;
};

// T: type of x, y, weights and gate; S: of residual and h.  A workgroup a row (a run of lanes where rows are short), CH chunks of eight
// columns a lane, all loads asked for at once.
//
// Bound by memory: x and residual in, y and h out.  us (TB/s) from memory: [16384, 4096] add and norm 89 (6.0), norm and add 69 (5.8); [8192,
// 7168] 80 (5.9) and 63 (5.6); both norms [11651, 2880] 50 (5.3).  Against workgroups that stay and ask for their next row while they work on
// the present one: 96, 69, 85, 69 and 52.
template <int T, int S, int CH, bool PRE, bool POST, bool SMALL, bool ANY>
__global__ __launch_bounds__(SMALL ? BN_SMALL_THREADS : BN_MAX_THREADS) void block_norm_kernel(BlockNormArgs p) {
    __shared__ float part[2][BN_MAX_WAVES][1];
    const int lanes = SMALL ? p.lanes : (int)blockDim.x;
    const int lane = SMALL ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
    const int64_t row = p.row0 + (SMALL ? (int64_t)blockIdx.x * (BN_SMALL_THREADS / lanes) + threadIdx.x / lanes : blockIdx.x);
    if (SMALL && row >= p.rows) return;
    RowSums<1, SMALL> sums(part, lanes);
    const int k = p.k;
    const float inv_k = 1.0f / (float)k;
    typedef RowsOf<T, S, SMALL, ANY> RowsT;
    typedef RowsOf<S, S, SMALL, ANY> RowsS;
    const Cols<S> cols = {lanes, lane, k};
    const bool vec = p.gate.kind == GATE_VECTOR;
    const int64_t g = p.gate.kind == GATE_NONE ? 0 : (int64_t)((uint32_t)row / p.gate.div % p.gate.mod);
    const RowsT in_x(p.x, p.rows, row, k), in_g(vec ? p.gate.p : nullptr, p.gate.mod, g, k);
    const RowsS in_r(p.residual, p.rows, row, k);
    Raw8<T> xr[CH], gr[CH], wr[CH], wpr[CH];
    Raw8<S> rr[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        xr[j] = in_x.template load<BN_NT>(cols, j);
        rr[j] = in_r.template load<BN_NT>(cols, j);
        if (POST) wpr[j] = load_vector<T>(p.post_weight, cols, j);
        gr[j] = in_g.template load<0>(cols, j);
        if (PRE) wr[j] = load_vector<T>(p.weight, cols, j);
    }
    float factor = p.scale;
    if (p.gate.kind == GATE_SCALAR) factor *= (float)((const typename DtOf<T>::type*)p.gate.p)[g];
    float x[CH][BN_VEC], h[CH][BN_VEC];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        unpack8<T>(xr[j], x[j]);
        unpack8<S>(rr[j], h[j]);
    }
    if (POST) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) ss += x[j][e] * x[j][e];
        sums(&ss);
        const float rp = 1.0f / sqrtf(ss * inv_k + p.post_eps);
        if (p.post_rstd && lane == 0) p.post_rstd[row] = rp;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float w[BN_VEC];
            unpack8<T>(wpr[j], w);
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) x[j][e] = x[j][e] * rp * w[e];
        }
    }
    float ss = 0.f;
    const RowsS out_h(p.h, p.rows, row, k);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        if (vec) {
            float f[BN_VEC];
            unpack8<T>(gr[j], f);
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) h[j][e] += factor * f[e] * x[j][e];
        } else {
            // (past the row there are zeros, which an infinite factor must not meet)
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) h[j][e] += (cols(j, e) < k ? factor : 0.f) * x[j][e];
        }
#pragma unroll
        for (int e = 0; e < BN_VEC; ++e) ss += h[j][e] * h[j][e];
        out_h.store(cols, j, h[j]);
    }
    if (PRE) {
        sums(&ss);
        const float r = 1.0f / sqrtf(ss * inv_k + p.eps);
        if (p.rstd && lane == 0) p.rstd[row] = r;
        const RowsT out_y(p.y, p.rows, row, k);
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float w[BN_VEC];
            unpack8<T>(wr[j], w);
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) h[j][e] = h[j][e] * r * w[e];
            out_y.store(cols, j, h[j]);
        }
    }
}

// Columns a lane.  Two chunks: fewer waves to wait for each other, from 4096 columns on ([8192, 7168] 96 -> 80 us), and of both norms, which
// wait twice, above 512 ([11651, 2880] 61 -> 50) unless the chip is not full anyway ([64, 4096] 6.5 and 7.0).
static int block_norm_chunks(const BlockNormArgs& p) {
    if (p.k > BN_MAX_THREADS * BN_VEC / 2) return 2;
    return p.weight && p.post_weight && p.k > 512 && p.rows > 512 ? 2 : 1;
}

// `per` rows a workgroup; a launch has fewer than 2^32 threads
template <int T, int S, int CH, bool SMALL, bool ANY>
static void block_norm_launch(BlockNormArgs& p, int64_t per, int threads, hipStream_t st) {
    const int64_t most = 0xFFFFFFFFll / threads * per;
    for (p.row0 = 0; p.row0 < p.rows; p.row0 += most) {
        const int64_t rows = p.rows - p.row0 < most ? p.rows - p.row0 : most;
        const dim3 g((unsigned)((rows + per - 1) / per)), b((unsigned)threads);
        if (p.weight && p.post_weight) hipLaunchKernelGGL((block_norm_kernel<T, S, CH, true, true, SMALL, ANY>), g, b, 0, st, p);
        else if (p.weight) hipLaunchKernelGGL((block_norm_kernel<T, S, CH, true, false, SMALL, ANY>), g, b, 0, st, p);
        else hipLaunchKernelGGL((block_norm_kernel<T, S, CH, false, true, SMALL, ANY>), g, b, 0, st, p);
    }
}
template <int T, int S, bool ANY> static void block_norm_launch(BlockNormArgs& p, hipStream_t st) {
    if (p.k <= BN_SMALL_K) {
        p.lanes = bn_lanes(p.k);
        block_norm_launch<T, S, 1, true, ANY>(p, BN_SMALL_THREADS / p.lanes, BN_SMALL_THREADS, st);
    } else if (block_norm_chunks(p) == 1) {
        block_norm_launch<T, S, 1, false, ANY>(p, 1, bn_threads(p.k, 1), st);
    } else {
        block_norm_launch<T, S, 2, false, ANY>(p, 1, bn_threads(p.k, 2), st);
    }
}
template <int T, int S> static void block_norm_launch(BlockNormArgs& p, hipStream_t st) {
    if (bn_on_dwords(p.rows, p.k, T, {p.x, p.residual, p.gate.kind == GATE_VECTOR ? p.gate.p : nullptr, p.y, p.h})) block_norm_launch<T, S, false>(p, st);
    else block_norm_launch<T, S, true>(p, st);
}

}  // namespace mxl

using namespace mxl;

extern "C" int mxl_block_norm(const void* x, const void* residual, int64_t rows, int64_t k, int dtype, int stream_dtype, const void* post_weight,
                              float post_eps, const void* gate, int64_t gate_div, int64_t gate_mod, int64_t gate_cols, float scale,
                              const void* weight, float eps, void* y, void* h, float* post_rstd, float* rstd, void* stream) {
    if (!bn_shape_ok(rows, k, dtype, stream_dtype) || (!weight && !post_weight) || !(eps >= 0.f) || !(post_eps >= 0.f)) return MXL_EINVAL;
    if (!bn_gate_ok(rows, k, gate, gate_div, gate_mod, gate_cols)) return MXL_EINVAL;
    if (rows == 0) return MXL_OK;
    if (!x || !residual || !h || (weight && !y)) return MXL_EINVAL;
    if (!device_is_gfx950()) return MXL_ENODEV;
    BlockNormArgs p = {x, residual, post_weight, weight, bn_gate(gate, rows, gate_div, gate_mod, gate_cols, k), scale, post_eps, eps, rows, 0, (int)k, 0,
                       y, h, post_rstd, rstd};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == MXL_DT_F32) block_norm_launch<MXL_DT_F32, MXL_DT_F32>(p, st);
    else if (dtype == MXL_DT_BF16 && stream_dtype == MXL_DT_BF16) block_norm_launch<MXL_DT_BF16, MXL_DT_BF16>(p, st);
    else if (dtype == MXL_DT_BF16) block_norm_launch<MXL_DT_BF16, MXL_DT_F32>(p, st);
    else if (stream_dtype == MXL_DT_F16) block_norm_launch<MXL_DT_F16, MXL_DT_F16>(p, st);
    else block_norm_launch<MXL_DT_F16, MXL_DT_F32>(p, st);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}
