// Matrices made orthogonal by Newton-Schulz steps (bsq_orth.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bsq {

constexpr uint64_t kOrthMaxDim = 65536;
constexpr int kOrthMaxSteps = 64;

struct OrthMatrix {
    const void *in;
    void *out;
    uint64_t rows, cols, ld_in, ld_out;
    int type;                                                    // of the input
};
// Coefficients a, b, c of each step: X <- a X + (b A + c A^2) X
struct OrthCall {
    const OrthMatrix *m;
    int n, out_type, steps;
    const float *coefficients;
    double eps;
    float scale;
};

size_t orth_scratch_bytes(const OrthCall &c);
// Whether the steps keep singular values that start within 0 and 1 below 1000
bool orth_steps_ok(const float *coefficients, int steps);
// ... else cudaErrorInvalidValue: nothing is launched then
cudaError_t orthogonalize(const OrthCall &c, void *scratch, unsigned *status, int sm_count, cudaStream_t stream);

}  // namespace bsq
