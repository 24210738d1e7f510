// What the tensor-core products of microscaled 4-bit matrices share: the way of a tile out of tensor memory, the addition of the partial
// tiles of a cluster, tensor maps of packed codes.
#pragma once

#include <cooperative_groups.h>

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

// 16 neighbouring results (one row of the tile) to memory
__device__ __forceinline__ void store_run16(void *out, int type, long at, const unsigned (&r)[16], float f0, float f1, int have, bool wide) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]) * f0 * f1;
    if (type == kF32) {
        float *dst = static_cast<float *>(out) + at;
        if (wide && have == 16) {
            st_global_v8(dst, make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]));
            st_global_v8(dst + 8, make_float4(v[8], v[9], v[10], v[11]), make_float4(v[12], v[13], v[14], v[15]));
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < have) dst[j] = v[j];
        }
        return;
    }
    unsigned w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = type == kBf16 ? pack_pair<kBf16>(v[2 * j], v[2 * j + 1]) : pack_pair<kF16>(v[2 * j], v[2 * j + 1]);
    unsigned short *dst = static_cast<unsigned short *>(out) + at;
    if (wide && have == 16) {
        st_words8(dst, w);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (j < have) dst[j] = (unsigned short)(j & 1 ? w[j >> 1] >> 16 : w[j >> 1]);
    }
}
__device__ __forceinline__ void store_one(void *out, int type, long at, float v) {
    if (type == kF32) store_elem<kF32>(out, (uint64_t)at, v);
    else if (type == kBf16) store_elem<kBf16>(out, (uint64_t)at, v);
    else store_elem<kF16>(out, (uint64_t)at, v);
}

// The rows that fall to CTA `rank` of a tile whose partial sums lie in the shared memory of the `splits` CTAs of a cluster (each `rows` x `run`, `run`
// along memory): added in the order of the CTAs' ranks, and written.  read(i, c): element i of CTA c's partial sums.
template <int THREADS, class Read>
__device__ __forceinline__ void add_parts(const Read &read, int rank, int ld_part, int rows, int run, int splits, float f0, float f1, void *out, int type, long at, long ld) {
    const int per = (rows + splits - 1) / splits, r0 = rank * per, r1 = min(rows, r0 + per);
    for (int i = r0 + (int)(threadIdx.x >> 5); i < r1; i += THREADS / 32)
        for (int j = (int)(threadIdx.x & 31); j < run; j += 32) {
            float v = 0.0f;
            for (int c = 0; c < splits; ++c) v += read(i * ld_part + j, c);
            store_one(out, type, at + (long)i * ld + j, v * f0 * f1);
        }
}

inline bool map_codes(CUtensorMap *map, const uint8_t *packed, uint64_t rows, uint64_t cols, unsigned box_rows) {
    const cuuint64_t dims[2] = {fp4_ld(cols), rows}, strides[1] = {fp4_ld(cols)};
    const cuuint32_t box[2] = {128u, box_rows}, estr[2] = {1, 1};
    return encode_tiled() && encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(packed) + kFp4Head, dims, strides, box, estr,
                                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
