// Gradient of the norms where blocks meet: the sums that workers share, and the entry points.
#include "mx_block_norm_bwd.h"

namespace mxl {

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
    if (job < p.jobs) {
        src = p.part[job];
        dst = p.out[job];
    } else if (!p.gate_scalar) {
        const int64_t gate = job - p.jobs;
        src = p.part_g + gate * p.gate_share * p.ldk;
        rows = p.gate_share;
        dst = p.dgate;
        at = gate * p.k;
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
            if (c + e < p.k) store_dt(dst, p.dtype, at + c + e, o[e]);
    }
}

}  // namespace mxl


using namespace mxl;

static int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

extern "C" int64_t mxl_block_norm_bwd_workspace_bytes(int64_t rows, int64_t k, int has_weight, int has_post_weight, int64_t gate_div, int64_t gate_mod,
                                                      int64_t gate_cols, int need_dgate) {
    static const int any = 0;
    if (!bn_shape_ok(rows, k, MXL_DT_F32, MXL_DT_F32) || !bn_gate_ok(rows, k, gate_cols ? &any : nullptr, gate_div, gate_mod, gate_cols)) return -1;
    if (rows == 0) return 0;
    const BlockNormPlan q = block_norm_plan(rows, k, gate_cols != 0 && (need_dgate || gate_cols == k), gate_div, gate_mod);
    int64_t n = (int64_t)((has_weight != 0) + (has_post_weight != 0)) * q.part_rows * q.ldk * 4;
    if (gate_cols && need_dgate) n += block_norm_gate_rows(q) * (gate_cols == k ? q.ldk : 1) * 4;
    return round16(n);
}

extern "C" int mxl_block_norm_bwd(const void* dy, const void* dh, const void* x, const void* h, int64_t rows, int64_t k, int dtype, int stream_dtype,
                                  const void* post_weight, const float* post_rstd, const void* gate, int64_t gate_div, int64_t gate_mod,
                                  int64_t gate_cols, float scale, const void* weight, const float* rstd, void* dx, void* dresidual, void* dweight,
                                  void* dpost_weight, void* dgate, void* workspace, int64_t workspace_bytes, void* stream) {
    const bool summed = (stream_dtype & MXL_NORM_SUMMED) != 0;
    stream_dtype &= ~MXL_NORM_SUMMED;
    if (!bn_shape_ok(rows, k, dtype, stream_dtype) || (!weight && !post_weight) || (dgate && !gate) || (dresidual && !weight)) return MXL_EINVAL;
    if (summed && (!weight || stream_dtype == MXL_DT_F32)) return MXL_EINVAL;
    if (!bn_gate_ok(rows, k, gate, gate_div, gate_mod, gate_cols)) return MXL_EINVAL;
    if ((dweight && !weight) || (dpost_weight && !post_weight)) return MXL_EINVAL;
    if (rows == 0) {
        // sums over no rows, written by the second kernel
        if (!dweight && !dpost_weight) return MXL_OK;
        if (!device_is_gfx950()) return MXL_ENODEV;
    }
    BlockNormPlan q;
    const int64_t need = mxl_block_norm_bwd_workspace_bytes(rows, k, dweight != nullptr, dpost_weight != nullptr, gate_div, gate_mod, gate ? gate_cols : 0, dgate != nullptr);
    if (rows > 0) {
        if ((weight && (!dy || !h || !rstd)) || (post_weight && (!x || !post_rstd)) || ((dgate || summed) && !x)) return MXL_EINVAL;
        if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)) return MXL_EINVAL;
        if (!device_is_gfx950()) return MXL_ENODEV;
        q = block_norm_plan(rows, k, dgate || (gate && gate_cols == k), gate_div, gate_mod);
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
                              q.lanes, rows, q.groups, q.each, q.share, q.gstep, q.gdiv, q.active, summed, dx, dresidual, dgate, part_w, part_p, part_g};
        int rc;
        if (dtype == MXL_DT_F32) rc = block_norm_bwd_launch<MXL_DT_F32, MXL_DT_F32>(p, q, st);
        else if (dtype == MXL_DT_BF16 && stream_dtype == MXL_DT_BF16) rc = block_norm_bwd_launch<MXL_DT_BF16, MXL_DT_BF16>(p, q, st);
        else if (dtype == MXL_DT_BF16) rc = block_norm_bwd_launch<MXL_DT_BF16, MXL_DT_F32>(p, q, st);
        else if (stream_dtype == MXL_DT_F16) rc = block_norm_bwd_launch<MXL_DT_F16, MXL_DT_F16>(p, q, st);
        else rc = block_norm_bwd_launch<MXL_DT_F16, MXL_DT_F32>(p, q, st);
        if (rc != MXL_OK) return rc;
    }
    BlockNormSumArgs s = {};
    if (dweight) s.part[s.jobs] = part_w, s.out[s.jobs++] = dweight;
    if (dpost_weight) s.part[s.jobs] = part_p, s.out[s.jobs++] = dpost_weight;
    s.dtype = dtype, s.k = (int)k, s.ldk = q.ldk, s.blocks_x = (int)((k + 31) / 32), s.rows = q.part_rows;
    int64_t grid = (int64_t)s.jobs * s.blocks_x;
    if (gate_joined) {
        s.part_g = part_g, s.dgate = dgate, s.gates = q.groups;
        s.gate_scalar = gate_cols != k;
        s.scale = scale;
        // (a wave of short rows has summed its workers' sums)
        s.gate_share = q.share / (q.lanes ? 64 / q.lanes : 1);
        grid += s.gate_scalar ? (s.gates + BS_THREADS / 64 - 1) / (BS_THREADS / 64) : s.gates * s.blocks_x;
    }
    if (grid == 0) return MXL_OK;
    hipLaunchKernelGGL(block_norm_sum_kernel, dim3((unsigned)grid), dim3(BS_THREADS), 0, st, s);
    return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
}
