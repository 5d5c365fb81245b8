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
    int64_t rows;
    int k, lanes;
    void *y, *h;
    float *post_rstd, *rstd;
};

// T: type of x, y, weights and gate; S: of residual and h.  CH chunks of eight columns a lane.
template <int T, int S, int CH, bool PRE, bool POST, bool SMALL>
__global__ __launch_bounds__(SMALL ? BN_SMALL_THREADS : BN_MAX_THREADS) void block_norm_kernel(BlockNormArgs p) {
    __shared__ float part[2][BN_MAX_THREADS / 64][1];
    const int lanes = SMALL ? p.lanes : (int)blockDim.x;
    const int lane = SMALL ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
    const int64_t workers = SMALL ? (int64_t)gridDim.x * (BN_SMALL_THREADS / lanes) : gridDim.x;
    const int64_t worker = SMALL ? (int64_t)blockIdx.x * (BN_SMALL_THREADS / lanes) + threadIdx.x / lanes : blockIdx.x;
    RowSums<1, SMALL> sums(part, lanes);
    const int k = p.k;
    const float inv_k = 1.0f / (float)k;
    int col[CH], left[CH];
    Raw8<T> w[CH], wp[CH], gv[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        col[j] = (j * lanes + lane) * BN_VEC;
        left[j] = k - col[j];
        w[j] = wp[j] = gv[j] = none8<T>();
        if (left[j] > 0) {
            if (PRE) w[j] = load8<T>(p.weight, col[j], left[j], false);
            if (POST) wp[j] = load8<T>(p.post_weight, col[j], left[j], false);
        }
    }
    Raw8<T> xn[CH];
    Raw8<S> rn[CH];
    auto request = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            xn[j] = none8<T>();
            rn[j] = none8<S>();
            if (left[j] > 0) {
                xn[j] = load8<T>(p.x, row * k + col[j], left[j], true);
                rn[j] = load8<S>(p.residual, row * k + col[j], left[j], true);
            }
        }
    };
    int64_t gate_row = -1;
    if (worker < p.rows) request(worker);
    for (int64_t row = worker; row < p.rows; row += workers) {
        float x[CH][BN_VEC], h[CH][BN_VEC];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            unpack8<T>(xn[j], x[j]);
            unpack8<S>(rn[j], h[j]);
        }
        float factor = p.scale;
        if (p.gate.kind != GATE_NONE) {
            const int64_t g = (uint32_t)row / p.gate.div % p.gate.mod;
            if (p.gate.kind == GATE_SCALAR) {
                factor *= (float)((const typename DtOf<T>::type*)p.gate.p)[g];
            } else if (g != gate_row) {
#pragma unroll
                for (int j = 0; j < CH; ++j)
                    if (left[j] > 0) gv[j] = load8<T>(p.gate.p, g * k + col[j], left[j], false);
                gate_row = g;
            }
        }
        if (row + workers < p.rows) request(row + workers);
        if (POST) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int e = 0; e < BN_VEC; ++e) ss += x[j][e] * x[j][e];
            sums(&ss);
            const float rp = 1.0f / sqrtf(ss * inv_k + p.post_eps);
            if (lane == 0 && p.post_rstd) p.post_rstd[row] = rp;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                float v[BN_VEC];
                unpack8<T>(wp[j], v);
#pragma unroll
                for (int e = 0; e < BN_VEC; ++e) x[j][e] = x[j][e] * rp * v[e];
            }
        }
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            float f[BN_VEC];
            if (p.gate.kind == GATE_VECTOR) {
                unpack8<T>(gv[j], f);
#pragma unroll
                for (int e = 0; e < BN_VEC; ++e) f[e] *= factor;
            } else {
#pragma unroll
                for (int e = 0; e < BN_VEC; ++e) f[e] = factor;
            }
#pragma unroll
            for (int e = 0; e < BN_VEC; ++e) {
                h[j][e] += f[e] * x[j][e];
                if (col[j] + e < k) ss += h[j][e] * h[j][e];    // (past the row: an infinite factor times the zeros there)
            }
            if (left[j] > 0) store8<S>(p.h, row * k + col[j], left[j], h[j]);
        }
        if (PRE) {
            sums(&ss);
            const float r = 1.0f / sqrtf(ss * inv_k + p.eps);
            if (lane == 0 && p.rstd) p.rstd[row] = r;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                float v[BN_VEC];
                unpack8<T>(w[j], v);
#pragma unroll
                for (int e = 0; e < BN_VEC; ++e) v[e] = h[j][e] * r * v[e];
                if (left[j] > 0) store8<T>(p.y, row * k + col[j], left[j], v);
            }
        }
    }
}

template <int T, int S, int CH, bool SMALL>
static void block_norm_launch(const BlockNormArgs& p, int blocks, int threads, hipStream_t st) {
    const dim3 g((unsigned)blocks), b((unsigned)threads);
    if (p.weight && p.post_weight) hipLaunchKernelGGL((block_norm_kernel<T, S, CH, true, true, SMALL>), g, b, 0, st, p);
    else if (p.weight) hipLaunchKernelGGL((block_norm_kernel<T, S, CH, true, false, SMALL>), g, b, 0, st, p);
    else hipLaunchKernelGGL((block_norm_kernel<T, S, CH, false, true, SMALL>), g, b, 0, st, p);
}
template <int T, int S> static void block_norm_launch(BlockNormArgs& p, hipStream_t st) {
    if (p.k <= BN_SMALL_K) {
        p.lanes = bn_lanes(p.k);
        const int64_t per = BN_SMALL_THREADS / p.lanes, want = (p.rows + per - 1) / per;
        block_norm_launch<T, S, 1, true>(p, (int)(want < 2048 ? want : 2048), BN_SMALL_THREADS, st);
        return;
    }
    const int threads = bn_threads(p.k);
    const int64_t cap = 256 * 2048 / threads;
    const int blocks = (int)(p.rows < cap ? p.rows : cap);
    if (bn_chunks(p.k) == 1) block_norm_launch<T, S, 1, false>(p, blocks, threads, st);
    else block_norm_launch<T, S, 2, false>(p, blocks, threads, st);
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
    BlockNormArgs p = {x, residual, post_weight, weight, bn_gate(gate, rows, gate_div, gate_mod, gate_cols, k), scale, post_eps, eps, rows, (int)k, 0,
                       y, h, post_rstd, rstd};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == MXL_DT_F32) block_norm_launch<MXL_DT_F32, MXL_DT_F32>(p, st);
    else if (dtype == MXL_DT_BF16 && stream_dtype == MXL_DT_BF16) block_norm_launch<MXL_DT_BF16, MXL_DT_BF16>(p, st);
    else if (dtype == MXL_DT_BF16) block_norm_launch<MXL_DT_BF16, MXL_DT_F32>(p, st);
    else if (stream_dtype == MXL_DT_F16) block_norm_launch<MXL_DT_F16, MXL_DT_F16>(p, st);
    else block_norm_launch<MXL_DT_F16, MXL_DT_F32>(p, st);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}
