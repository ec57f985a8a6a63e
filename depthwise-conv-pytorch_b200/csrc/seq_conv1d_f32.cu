// Causal depthwise convolution of sequences: fp32.
#include "seq_conv1d_kernels.cuh"

namespace dwb {
DWB_CONV1D_INSTANTIATE(float)
}  // namespace dwb
