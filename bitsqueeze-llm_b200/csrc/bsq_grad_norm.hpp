// Norm over all elements of many tensors, and the tensors scaled so that it is at most a given one (bsq_grad_norm.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bsq {

constexpr size_t kNormScratchBytes = 16384;                      // a double for each CTA of the pass that finds the norm
// types: OpType values (bsq_fp4.hpp).  norm_kind 2: square root of the sum of squares, 0: largest magnitude.  outs (nullable: the norm alone):
// out[i] = in[i] * min(1, max_norm / (norm + 1e-6)), in the type of in[i]; out[i] is in[i] itself or lies apart from every input and output
// (norm_layout_ok).
bool norm_layout_ok(const void *const *ins, const uint64_t *counts, const int *types, int n, void *const *outs);
cudaError_t grad_norm_clip(const void *const *ins, const uint64_t *counts, const int *types, int n, void *const *outs, double max_norm, int norm_kind, float *norm,
                           void *scratch, int sm_count, cudaStream_t stream);

}  // namespace bsq
