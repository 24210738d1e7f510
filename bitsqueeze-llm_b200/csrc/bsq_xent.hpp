// Softmax cross entropy of x W^T without the logits, and its gradient (bsq_xent.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bsq {

enum XentReduction : int { kXentNone = 0, kXentSum = 1, kXentMean = 2 };

// Sums in tensor memory are in chains of 1024 of K or so (logits of the loss) or 4096 (logits of the gradient, dx and dW).  At most so many columns, and tokens in FP16 and BF16
constexpr uint64_t kXentMaxCols = 65536;
inline uint64_t xent_max_tokens(int type) { return type == 1 ? 65536 : 524288; }

struct XentCall {
    int type;                                                    // kF16 or kBf16
    const void *x, *w;                                           // tokens x cols, vocab x cols
    uint64_t tokens, cols, vocab, ld_x, ld_w;
    const long long *target;
    long long ignore;
    double smoothing;
    int reduction;
};

size_t xent_scratch_bytes(const XentCall &c, int sm_count);
size_t xent_grad_scratch_bytes(const XentCall &c, bool dx, int sm_count);
// loss: one float, or one for each token (kXentNone).  stats: 2 * tokens + 1 floats for the gradient.
cudaError_t xent_loss(const XentCall &c, float *loss, float *stats, void *scratch, unsigned *status, int sm_count, cudaStream_t stream);
// grad: of the loss, one float or one for each token.  dx, dw nullable.
cudaError_t xent_grad(const XentCall &c, const float *stats, const float *grad, void *dx, uint64_t ld_dx, void *dw, uint64_t ld_dw, void *scratch, unsigned *status,
                      int sm_count, cudaStream_t stream);

}  // namespace bsq
