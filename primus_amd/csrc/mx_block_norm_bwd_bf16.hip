// Gradient of the norms where blocks meet: the kernels of bf16 operands.
#include "mx_block_norm_bwd_kernels.h"

template int mxl::block_norm_bwd_launch<MXL_DT_BF16, MXL_DT_BF16>(const mxl::BlockNormBwdArgs&, const mxl::BlockNormPlan&, hipStream_t);
template int mxl::block_norm_bwd_launch<MXL_DT_BF16, MXL_DT_F32>(const mxl::BlockNormBwdArgs&, const mxl::BlockNormPlan&, hipStream_t);
