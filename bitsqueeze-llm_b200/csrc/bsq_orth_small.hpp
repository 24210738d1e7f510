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
    float square, linear;                                        // of A A and A in N
    float first_r;                                               // R = N of the first step
    float r_product, r_self, r_n;                                // of N R, R and N in the next R, or in the result's
    float t_product, t_self;                                     // of N A and A in T
    float a_product, a_self;                                     // of N T and T in the next A
};
struct OrthSmallSteps {
    OrthSmallStep step[kOrthMaxSteps];
    float identity;                                              // q of the result
    int steps;
};
struct OrthSmallRoom {
    int slices, per;                                             // of the long side, and how long each is
    float *sums, *sum, *r, *identity;                            // count x slices x s x s, count x s x s each, count
};

int orth_small_slices(uint64_t l, int *per);
cudaError_t orth_small(const OrthSmall &g, bool tall, int type, const OrthSmallSteps &t, int count, const OrthSmallRoom &r, unsigned *status, cudaStream_t stream);

}  // namespace bsq
