// Causal depthwise convolution of sequences: fp16.
#include "seq_conv1d_kernels.cuh"

namespace dwb {
DWB_CONV1D_INSTANTIATE(__half)
}  // namespace dwb
