// Host API of the multi-tensor gradient norm / clipping kernels (grad_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <vector>

#include "transformer_api.h"

namespace dca {
struct GradTensor {
  void* p;
  int64_t n;
  TDtype dt;
};
enum class NormKind : int { kL2 = 0, kL1 = 1, kMax = 2 };
// doubles of workspace for these tensors
int64_t grad_norm_workspace(const std::vector<GradTensor>& t);
// norm[0] = the norm over all tensors (fp32); `partial`: the workspace.
void grad_norm(const std::vector<GradTensor>& t, NormKind kind, double* partial, float* norm, hipStream_t st);
// every tensor *= min(1, max_norm / (norm + 1e-6)); nothing is written where that is 1.
void grad_clip(const std::vector<GradTensor>& t, const float* norm, float max_norm, hipStream_t st);
}  // namespace dca
