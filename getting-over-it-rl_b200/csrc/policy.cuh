// The policy's side of a batch of worlds (delta_*.cu, clip.cu): parameters shared by the kernels and the C entries.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/goib2d.h"

namespace gb {

// ---- the gated delta rule (delta_step.cu, delta_forward.cu, delta_backward.cu)

cudaError_t launch_delta_step(const goib2d_delta_desc &d, cudaStream_t s);
cudaError_t launch_delta_forward(const goib2d_delta_desc &d, void *saved, cudaStream_t s);
cudaError_t launch_delta_backward(const goib2d_delta_desc &d, const goib2d_delta_grads &gr, const void *saved,
                                  void *workspace, cudaStream_t s);
int64_t delta_saved_bytes(const goib2d_delta_desc &d);
int64_t delta_workspace_bytes(const goib2d_delta_desc &d);

// ---- gradient clipping (clip.cu)

cudaError_t launch_clip(const goib2d_grad *grads, int32_t n, float max_norm, float *norm, void *workspace,
                        cudaStream_t s);
int64_t clip_workspace_bytes(const goib2d_grad *grads, int32_t n);

}  // namespace gb
