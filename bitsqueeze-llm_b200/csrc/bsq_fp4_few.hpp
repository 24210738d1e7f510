// The gradient of the input for few rows (bsq_fp4_few.cu).
#pragma once

#include "bsq_fp4.hpp"

namespace bsq {

constexpr uint64_t kFewRowsMax = 16;
// R at most kFewRowsMax; dy's rows start on 16 bytes
cudaError_t fp4_grad_few(int format, const void *dy, int R, uint64_t ld_dy, const uint8_t *packed, uint64_t D, uint64_t C, void *out, int type, uint64_t ld,
                         int sm_count, cudaStream_t stream);

}  // namespace bsq
