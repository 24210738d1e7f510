// What the tensor-core products of microscaled 4-bit matrices share: the way of a tile out of tensor memory, the addition of the partial
// tiles of a cluster, tensor maps of packed codes.
#pragma once

#include <cooperative_groups.h>

#include <atomic>

#include "bsq_fp4.cuh"
#include "bsq_gemm_tc.cuh"
#include "bsq_tma.cuh"

namespace bsq {
namespace {

namespace cg = cooperative_groups;

// Tensor memory of a CTA, or of both CTAs of a pair (a warp of each executes it)
template <int CTAS> __device__ __forceinline__ void tmem_alloc(unsigned *base, unsigned cols) {
    if (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(base)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CTAS> __device__ __forceinline__ void tmem_free(unsigned base, unsigned cols) {
    if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}

// 16 neighbouring accumulators of this thread's row; NaN for a tile that was given up
__device__ __forceinline__ void read16(unsigned taddr, unsigned (&r)[16], bool ok) {
    if (ok) tmem_ld16(taddr, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    if (!ok) {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0x7fffffffu;
    }
}

// 16 neighbouring accumulators of this thread's row, written (visible to reads behind a tcgen05.wait::st)
__device__ __forceinline__ void tmem_st16(unsigned taddr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};\n" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
        "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// ... added to what is in registers, rounded
__device__ __forceinline__ void add16(unsigned taddr, unsigned (&r)[16]) {
    unsigned q[16];
    read16(taddr, q, true);
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(q[j]));
}

// The two factors of a result (matrix scales) as one where their product is a normal number; else the larger one comes first, so that a result within the range of
// FP32 does not leave it on the way: sums up to 2^40 times 2^117 times 2^-110.
struct Factors {
    float first, second;
};
__device__ __forceinline__ Factors join_factors(float a, float b) {
    const float c = a * b;
    if (fabsf(c) >= 1.17549435e-38f && fabsf(c) <= 3.402823466e+38f) return {c, 1.0f};
    return fabsf(a) >= fabsf(b) ? Factors{a, b} : Factors{b, a};
}

__device__ __forceinline__ void store_one(void *out, int type, long at, float v) {
    if (type == kF32) store_elem<kF32>(out, (uint64_t)at, v);
    else if (type == kBf16) store_elem<kBf16>(out, (uint64_t)at, v);
    else store_elem<kF16>(out, (uint64_t)at, v);
}

// A box of 32 rows x 128 bytes, as the epilogues of the products leave it in shared memory (16-byte piece i of row r at piece i ^ (r & 7)), to a result whose rows
// TMA cannot take (stride or start off 16 bytes): a row at a time, neighbouring lanes neighbouring elements.  (A row per lane and element after element, as it
// lies in the registers, touches 32 lines with every store: 1031 x 3001 results of 1501 products took 57 us, this way 27.)
__device__ __forceinline__ void box_out(const unsigned char *box, int lane, void *out, int size, long at, long ld, int rows, int cols) {
    const int per_lane = 128 / size / 32;                        // elements of a row for each lane: 1 (FP32) or 2
    __syncwarp();
#pragma unroll 4
    for (int r = 0; r < min(rows, 32); ++r) {
        const unsigned w = *reinterpret_cast<const unsigned *>(box + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
        const long to = at + (long)r * ld + lane * per_lane;
        if (size == 4) {
            if (lane < cols) static_cast<unsigned *>(out)[to] = w;
        } else {
            if (2 * lane < cols) static_cast<unsigned short *>(out)[to] = (unsigned short)w;
            if (2 * lane + 1 < cols) static_cast<unsigned short *>(out)[to + 1] = (unsigned short)(w >> 16);
        }
    }
    __syncwarp();
}
// ... added to what is there (FP32): by the same lane as what it wrote before, so in its order, the same bits every time.  (Additions without an answer: a load, an addition
// and a store would each wait for the one before.)
__device__ __forceinline__ void box_add(const unsigned char *box, int lane, float *out, long at, long ld, int rows, int cols) {
    __syncwarp();
#pragma unroll 4
    for (int r = 0; r < min(rows, 32); ++r) {
        const float v = *reinterpret_cast<const float *>(box + r * 128 + ((((lane >> 2) ^ (r & 7)) << 4) | ((lane & 3) << 2)));
        if (lane < cols) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(out + at + (long)r * ld + lane), "f"(v) : "memory");
    }
    __syncwarp();
}

// The rows that fall to CTA `rank` of a tile whose partial sums lie in the shared memory of the `splits` (at most 8) CTAs of a cluster, each `rows` x `run` with
// `run` along memory: added in the order of the CTAs' ranks, and written.  read(i, c): four values from element i of CTA c's partial sums on (i a multiple of
// 4).  A value comes from another SM in some 1000 clocks, so a thread asks for all of four columns at once (one value at a time: 777 x 1031 x 5120 18.6 us, this way
// 14.0).
template <int THREADS, class Read>
__device__ __forceinline__ void add_parts(const Read &read, int rank, int ld_part, int rows, int run, int splits, float scale0, float scale1, void *out, int type, long at,
                                          long ld) {
    const Factors f = join_factors(scale0, scale1);
    const int per = (rows + splits - 1) / splits, r0 = rank * per, r1 = min(rows, r0 + per), fours = (run + 3) / 4;
    const int size = type == kF32 ? 4 : 2;
    const bool whole = ((reinterpret_cast<uintptr_t>(out) + (uintptr_t)(at * size)) | (uintptr_t)(ld * size)) % (unsigned)(4 * size) == 0;
    for (int i = r0 * fours + (int)threadIdx.x; i < r1 * fours; i += THREADS) {
        const int row = i / fours, col = (i - row * fours) * 4;
        float4 p[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
            if (c < splits) p[c] = read(row * ld_part + col, c);
        float4 v = p[0];
#pragma unroll
        for (int c = 1; c < 8; ++c)
            if (c < splits) v = make_float4(v.x + p[c].x, v.y + p[c].y, v.z + p[c].z, v.w + p[c].w);
        const float o[4] = {v.x * f.first * f.second, v.y * f.first * f.second, v.z * f.first * f.second, v.w * f.first * f.second};
        const long to = at + (long)row * ld + col;
        if (whole && col + 4 <= run) {
            if (type == kF32) *reinterpret_cast<float4 *>(static_cast<float *>(out) + to) = make_float4(o[0], o[1], o[2], o[3]);
            else *reinterpret_cast<uint2 *>(static_cast<unsigned short *>(out) + to) =
                     type == kBf16 ? make_uint2(pack_pair<kBf16>(o[0], o[1]), pack_pair<kBf16>(o[2], o[3])) : make_uint2(pack_pair<kF16>(o[0], o[1]), pack_pair<kF16>(o[2], o[3]));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < run) store_one(out, type, to + j, o[j]);
        }
    }
}

// A partial tile that was given up
template <int THREADS> __device__ __forceinline__ void nan_part(float *part, int count) {
    for (int i = (int)threadIdx.x; i < count; i += THREADS) part[i] = __uint_as_float(0x7fffffffu);
}

inline bool map_codes(CUtensorMap *map, const uint8_t *packed, uint64_t rows, uint64_t cols, unsigned box_rows) {
    const cuuint64_t dims[2] = {fp4_ld(cols), rows}, strides[1] = {fp4_ld(cols)};
    const cuuint32_t box[2] = {128u, box_rows}, estr[2] = {1, 1};
    return encode_tiled() && encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(packed) + kFp4Head, dims, strides, box, estr,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether a result can leave by TMA: rows that start on 16 bytes and end on 16.  A tiled store leaves out what lies behind the last column only in whole pieces of 16
// bytes; a row that ends inside one would have up to 14 bytes behind it overwritten.
inline bool tma_can_write(const void *out, uint64_t row_stride, uint64_t row_bytes) {
    return (reinterpret_cast<uintptr_t>(out) | row_stride | row_bytes) % 16 == 0;
}

// Lets a kernel have all of an SM's shared memory, or `bytes` of it, once for each device.
template <class F> cudaError_t allow_smem(F *kernel, std::atomic<uint64_t> *done, int bytes = 227 * 1024) {
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    const uint64_t bit = 1ull << (device & 63);
    if (device < 64 && (done->load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess && device < 64) done->fetch_or(bit, std::memory_order_relaxed);
    return err;
}

// A chained launch (launch_chained) in clusters of `ctas` along x
template <class... P, class... A>
cudaError_t launch_cluster(void (*fn)(P...), unsigned grid, unsigned block, int ctas, size_t smem, cudaStream_t stream, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...);
}

}  // namespace
}  // namespace bsq
