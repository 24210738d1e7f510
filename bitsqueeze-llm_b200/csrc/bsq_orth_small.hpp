// Newton-Schulz steps of matrices with a short side of up to 128 (bsq_orth_small.cu), as bsq_orth.cu calls them.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "bsq_orth.hpp"

namespace bsq {

constexpr int kOrthMost = 64;                                    // matrices of a launch
constexpr int kOrthSmallSide = 128;

// Matrices of one shape: s on the short side, l on the long one
struct OrthSmall {
    const void *in[kOrthMost];
    void *out[kOrthMost];
    uint64_t ld[kOrthMost], ld_out[kOrthMost];
    int s, l;
    const double *parts;                                         // part_count shares of each matrix's sum of squares
    int part_count;
    double eps;
};
// A step as products of operands that are held times powers of two: factors of the accumulators and operands
struct OrthSmallStep {
    int a;                                                       // A is held times 2^a
    float square, linear, constant;                              // of A A, A and I in M
    float first_q;                                               // Q = M of the first step
    float of_q, of_t, of_a;                                      // M Q, M A, M (M A)
    float out;                                                   // Q of the last step
};
struct OrthSmallSteps {
    OrthSmallStep step[kOrthMaxSteps];
    int steps;
};
struct OrthSmallRoom {
    int slices, per;                                             // of the long side, and how long each is
    float *sums, *sum, *q;                                       // count x slices x s x s, count x s x s each
};

int orth_small_slices(uint64_t l, int *per);
cudaError_t orth_small(const OrthSmall &g, bool tall, int type, const OrthSmallSteps &t, int count, const OrthSmallRoom &r, unsigned *status, cudaStream_t stream);

}  // namespace bsq
