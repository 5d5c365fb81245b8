// The launches of the gradient's kernels, for the source files that instantiate them.
#pragma once
#include "mx_block_norm_bwd.h"

namespace mxl {

template <int T, int S, int CH, bool SMALL, bool ANY, int BOUND, int DEPTH>
static void block_norm_bwd_modes(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st) {
    const dim3 g((unsigned)q.blocks), b((unsigned)q.threads);
    const bool gv = p.gate.kind == GATE_VECTOR;
#define MXL_BN_BWD(PRE, POST, SAME, GATEV) hipLaunchKernelGGL((block_norm_bwd_kernel<T, S, CH, PRE, POST, SAME, GATEV, SMALL, ANY, BOUND, (PRE && POST && GATEV ? 0 : DEPTH)>), g, b, 0, st, p)
    if (p.weight && p.post_weight) {
        if (gv) MXL_BN_BWD(true, true, false, true);
        else MXL_BN_BWD(true, true, false, false);
    } else if (p.weight) {
        if (gv) MXL_BN_BWD(true, false, false, true);
        else if (p.dx) MXL_BN_BWD(true, false, false, false);
        else MXL_BN_BWD(true, false, true, false);
    } else {
        if (gv) MXL_BN_BWD(false, true, false, true);
        else MXL_BN_BWD(false, true, false, false);
    }
#undef MXL_BN_BWD
}
template <int T, int S> void block_norm_bwd_launch(const BlockNormBwdArgs& p, const BlockNormPlan& q, hipStream_t st) {
    if (bn_on_dwords(p.rows, p.k, T, {p.dy, p.dh, p.x, p.h, p.gate.kind == GATE_VECTOR ? p.gate.p : nullptr, p.dx, p.dres, p.gate.kind == GATE_VECTOR ? p.dgate : nullptr})) {
        if (q.lanes) block_norm_bwd_modes<T, S, 1, true, false, BN_SMALL_THREADS, 1>(p, q, st);
        else if (q.chunks == 2) block_norm_bwd_modes<T, S, 2, false, false, BN_MAX_THREADS, 0>(p, q, st);
        else if (q.threads > BN_MAX_THREADS / 2) block_norm_bwd_modes<T, S, 1, false, false, BN_MAX_THREADS, 1>(p, q, st);
        else block_norm_bwd_modes<T, S, 1, false, false, BN_MAX_THREADS / 2, 0>(p, q, st);
    } else {
        if (q.lanes) block_norm_bwd_modes<T, S, 1, true, true, BN_SMALL_THREADS, 0>(p, q, st);
        else if (q.chunks == 2) block_norm_bwd_modes<T, S, 2, false, true, BN_MAX_THREADS, 0>(p, q, st);
        else block_norm_bwd_modes<T, S, 1, false, true, BN_MAX_THREADS, 0>(p, q, st);
    }
}

}  // namespace mxl
