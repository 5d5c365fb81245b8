// Arguments of the bf16 GEMMs' kernels, and the dense linear on their 256-row tiles.
#pragma once
#include "mx_epilogue.h"

namespace mxl {

struct Bf16Args {
    const uint8_t* a;      // forward: activations [total_m, k];   wgrad: p [total_m, m_out]
    const uint8_t* b;      // forward: weights [G, n, k] or [G, k, n];   wgrad: q [total_m, n_out]
    void* c;
    const int64_t* group_lens;
    int num_groups;
    int64_t total_m;
    int64_t m;             // wgrad: m_out
    int64_t n;             // forward: n;  wgrad: n_out
    int64_t k;             // forward: contraction length
    EpilogueArgs epi;      // dense forward only
};

// act(a . b^T + bias) + residual with one group, 256-row tiles (MXL_ACT_*)
int launch_bf16_linear_tall(const Bf16Args& a, int act, hipStream_t st);

}  // namespace mxl
