// Microscaled 4-bit matrices (MXFP4, NVFP4): their packed form and the launchers of the kernels that make and read it.
//
// Elements are e2m1 (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) times the scale of their block along the row times the scale of the
// matrix.  MXFP4: blocks of 32, scales 2^(byte - 127), matrix scale 1.  NVFP4: blocks of 16, E4M3 scales, an FP32 matrix scale.
//
// Packed form (one allocation, 16-byte aligned):
//   head     128 bytes; the first word is the matrix scale
//   codes    rows x fp4_ld(cols) bytes, 16 bytes for 32 columns, the even column in the low nibble; what is behind `cols` is 0
//   scales   from the next multiple of 128 bytes on, tiles of 128 rows x 4 blocks of 512 bytes, tiles of a group of rows one
//            behind the other: row r, block b of a tile at (r % 32) * 16 + (r / 32) * 4 + b -- what tcgen05.cp takes into
//            tensor memory for a block-scaled MMA, so that a product copies scales as they are.  Blocks behind the
//            last one of a row are 0 up to the end of its tile; rows behind the last one are never written.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bsq {

enum Fp4Format : int { kMxFp4 = 8, kNvFp4 = 9 };                 // quantization_method_t MXFP4, NVFP4
enum OpType : int { kF32 = 0, kF16 = 1, kBf16 = 2 };

constexpr uint64_t kFp4Head = 128, kFp4ScaleTile = 512;

__host__ __device__ constexpr int fp4_block(int format) { return format == kMxFp4 ? 32 : 16; }
__host__ __device__ constexpr uint64_t fp4_ld(uint64_t cols) { return (cols + 31) / 32 * 16; }
__host__ __device__ constexpr uint64_t fp4_quads(int format, uint64_t cols) {         // scale tiles along a row
    return (cols + 4 * fp4_block(format) - 1) / (4 * fp4_block(format));
}
__host__ __device__ constexpr uint64_t fp4_scales_at(uint64_t rows, uint64_t cols) { return (kFp4Head + rows * fp4_ld(cols) + 127) / 128 * 128; }
__host__ __device__ constexpr uint64_t fp4_packed_bytes(int format, uint64_t rows, uint64_t cols) {
    return fp4_scales_at(rows, cols) + (rows + 127) / 128 * fp4_quads(format, cols) * kFp4ScaleTile;
}
constexpr uint64_t kFp4MaxDim = 0x7fffff00ull;                   // rows and columns: TMA coordinates are 32-bit and signed
inline bool fp4_shape_ok(int format, uint64_t rows, uint64_t cols) {
    return (format == kMxFp4 || format == kNvFp4) && rows <= kFp4MaxDim && cols >= 1 && cols <= kFp4MaxDim;
}
inline int op_bytes(int type) { return type == kF32 ? 4 : (type == kF16 || type == kBf16) ? 2 : 0; }

// One float per CTA of the pass that finds the largest magnitude of an NVFP4 matrix.
constexpr int kFp4Partials = 1024;
// Up to this many bytes every CTA of an NVFP4 quantiser finds the largest magnitude by itself instead of a pass of its own in front.
constexpr uint64_t kFp4OwnAmaxBytes = 64 << 10;
inline size_t fp4_quantize_scratch(int format, int type, uint64_t rows, uint64_t cols) {
    return format == kNvFp4 && rows * cols * (uint64_t)op_bytes(type) > kFp4OwnAmaxBytes ? kFp4Partials * sizeof(float) : 0;
}

// Tries after which the epilogues of the products give up a wait for accumulators: `usual`, or fewer where a test has set them (bsq_test_limit_waits).
void limit_epilogue_tries(unsigned tries);
unsigned epilogue_tries(unsigned usual);

// amax (nullable, NVFP4): a device word with the largest magnitude the caller reckons with; larger elements saturate.
cudaError_t fp4_quantize(int format, const void *x, int type, uint64_t rows, uint64_t cols, uint64_t ld, const float *amax, void *packed,
                         void *scratch, int sm_count, cudaStream_t stream);
cudaError_t fp4_dequantize(int format, const void *packed, uint64_t rows, uint64_t cols, void *out, int type, uint64_t ld, int sm_count,
                           cudaStream_t stream);
// out (M x N) = A (M x K) B (N x K)^T
cudaError_t fp4_matmul(int format, const void *a, uint64_t M, const void *b, uint64_t N, uint64_t K, void *out, int type, uint64_t ld,
                       unsigned *status, int sm_count, cudaStream_t stream);
// out (M x K) = dy (M x N) W (N x K);  out (N x K) = dy (M x N)^T X (M x K): dy in BF16, W and X packed.
size_t fp4_grad_scratch_bytes(uint64_t M, uint64_t N, const void *dy, uint64_t ld_dy);
cudaError_t fp4_grad_input(int format, const void *dy, uint64_t M, uint64_t ld_dy, const void *w, uint64_t N, uint64_t K, void *out, int type,
                           uint64_t ld, void *scratch, unsigned *status, int sm_count, cudaStream_t stream);
cudaError_t fp4_grad_weight(int format, const void *dy, uint64_t M, uint64_t N, uint64_t ld_dy, const void *x, uint64_t K, void *out, int type,
                            uint64_t ld, void *scratch, unsigned *status, int sm_count, cudaStream_t stream);

}  // namespace bsq
