// The launches of the gradient's kernels, for the source files that instantiate them.
#pragma once
#include "mx_block_norm_bwd.h"

namespace mxl {

template <int T, int S, int CH, bool SMALL, bool ANY, int BOUND, bool AHEAD>
static int block_norm_bwd_modes(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st) {
    const dim3 g((unsigned)q.blocks), b((unsigned)q.threads);
    const bool gv = p.gate.kind == GATE_VECTOR;
    // the weights' sums, where they are in shared memory
    const int lds = bn_bwd_keeps(CH, p.weight, p.post_weight, gv) ? 0 : (1 + (p.post_weight != nullptr)) * CH * BN_VEC * 4 * q.threads;
    auto launch = [&](void (*kernel)(BlockNormBwdArgs)) -> int {
        if (lds > 0 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return MXL_ELAUNCH;
        hipLaunchKernelGGL(kernel, g, b, lds, st, p);
        return hipGetLastError() == hipSuccess ? MXL_OK : MXL_ELAUNCH;
    };
    // (both norms and a gate of vectors: a row ahead does not fit the registers of a workgroup of over 512 threads)
#define MXL_BN_BWD(PRE, POST, SAME, GATEV) launch(block_norm_bwd_kernel<T, S, CH, PRE, POST, SAME, GATEV, SMALL, ANY, BOUND, AHEAD && !(PRE && POST && GATEV)>)
    if (p.weight && p.post_weight) return gv ? MXL_BN_BWD(true, true, false, true) : MXL_BN_BWD(true, true, false, false);
    if (p.weight) return gv ? MXL_BN_BWD(true, false, false, true) : p.dx || p.dgate ? MXL_BN_BWD(true, false, false, false) : MXL_BN_BWD(true, false, true, false);
    return gv ? MXL_BN_BWD(false, true, false, true) : MXL_BN_BWD(false, true, false, false);
#undef MXL_BN_BWD
}
template <int T, int S> int block_norm_bwd_launch(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st) {
    if (bn_on_dwords(p.rows, p.k, T, {p.dy, p.dh, p.x, p.h, p.gate.kind == GATE_VECTOR ? p.gate.p : nullptr, p.dx, p.dres, p.gate.kind == GATE_VECTOR ? p.dgate : nullptr})) {
        if (q.lanes) return block_norm_bwd_modes<T, S, 1, true, false, BN_SMALL_THREADS, true>(p, q, st);
        if (q.chunks == 2) return block_norm_bwd_modes<T, S, 2, false, false, BN_MAX_THREADS, false>(p, q, st);
        if (q.threads > BN_MAX_THREADS / 2) return block_norm_bwd_modes<T, S, 1, false, false, BN_MAX_THREADS, true>(p, q, st);
        return block_norm_bwd_modes<T, S, 1, false, false, BN_MAX_THREADS / 2, false>(p, q, st);
    }
    if (q.lanes) return block_norm_bwd_modes<T, S, 1, true, true, BN_SMALL_THREADS, false>(p, q, st);
    if (q.chunks == 2) return block_norm_bwd_modes<T, S, 2, false, true, BN_MAX_THREADS, false>(p, q, st);
    return block_norm_bwd_modes<T, S, 1, false, true, BN_MAX_THREADS, false>(p, q, st);
}

}  // namespace mxl
