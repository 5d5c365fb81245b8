// Gradient of the norms where blocks meet: the kernels of f32 operands.
#include "mx_block_norm_bwd_kernels.h"

template int mxl::block_norm_bwd_launch<MXL_DT_F32, MXL_DT_F32>(const mxl::BlockNormBwdArgs&, const mxl::BlockNormPlan&, hipStream_t);
