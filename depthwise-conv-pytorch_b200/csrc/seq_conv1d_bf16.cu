// Causal depthwise convolution of sequences: bf16.
#include "seq_conv1d_kernels.cuh"

namespace dwb {
DWB_CONV1D_INSTANTIATE(__nv_bfloat16)
}  // namespace dwb
