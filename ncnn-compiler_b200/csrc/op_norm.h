// Group norm as the layers of a loaded graph have it (op_norm.cu).
#pragma once

#include "act_ref.cuh"

namespace nb {

// Whether k_group_norm takes groups of this size (a group's channels have to fit the threads of a CTA).
bool group_norm_fits(int channels, int groups);

// images x pixels x channels, channel-last, dense, in any format of a graph's tensors; act is ACT_NONE, ACT_RELU, ACT_SWISH or
// ACT_GELU.
cudaError_t launch_group_norm(const ActRef& in, const ActRef& out, long long images, long long pixels, int channels, int groups, const float* gamma,
                              const float* beta, float eps, int act, int device, cudaStream_t st);

}  // namespace nb
