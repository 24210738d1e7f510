// What the TMA-fed tensor-core kernels share: tiled copies and their tensor maps, operand descriptors of 128-byte-swizzled
// shared memory, positions in rings of stages.
#pragma once

#include <cuda.h>

#include <mutex>

#include "bsq_device.cuh"

namespace bsq {
namespace {

// K-major operand in 128-byte-swizzled shared memory: rows of 128 B, groups of 8 rows 1024 B apart (stride byte
// offset), leading byte offset unused, descriptor version 1, layout type 2 (128-byte swizzle).  Steps of 8 along K
// inside the 128-byte row are steps of 32 B of the start address.
__device__ __forceinline__ uint64_t smem_desc_sw128(unsigned addr_bytes) {
    return (uint64_t)((addr_bytes >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void tma_load_2d(void *dst_smem, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_u32(dst_smem)),
                 "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, int x, int y, const void *src_smem) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(smem_u32(src_smem))
                 : "memory");
}
// ... added to what is there (FP32)
__device__ __forceinline__ void tma_add_2d(const CUtensorMap *map, int x, int y, const void *src_smem) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(smem_u32(src_smem))
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// One lane of a warp whose lanes are all here.  The warp that issues MMAs walks its loops with all lanes and lets one of them issue: addresses and
// descriptors then stay in uniform registers, which is where these instructions take them from.  In a branch of one lane every operand was moved
// there one by one, some 100 clocks for each instruction (12 copies of scales and 4 MMAs per stage: 2300 clocks instead of 960).
__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// ---- pairs of CTAs (cta_group::2): one MMA over both, issued by the CTA of even rank in the cluster, the leader ----
// A tiled copy into this CTA's shared memory that counts itself off on a barrier of either CTA of the pair (a shared::cluster address)
__device__ __forceinline__ void tma_load_2d_pair(void *dst_smem, const CUtensorMap *map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst_smem)),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// An arrival on a barrier of either CTA of the pair.  What it announces stays where it is and is read by the tensor core of the SM that wrote it (operands in
// this CTA's shared memory, behind a proxy fence; accumulators that have been read out): nothing has to become visible to threads of the other SM, so the
// release stays within the CTA.  One of cluster scope waits some 900 clocks for all stores of the SM: a stage of 64 of K then took 2180 clocks instead of 960.
__device__ __forceinline__ void mbar_arrive_pair(unsigned bar) {
    asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// mbar_wait_bounded for the many warps of a kernel that wait most of the time: a try that finds the barrier closed sleeps up to 20 us before it answers, where the
// default has it asked again and again.  What that costs is issue slots and, under the power limit, clock: the gradient products took 2 to 10 % longer.
// 65536 tries of 20 us, or 1.3 s, are the bound.
constexpr unsigned kWaitTries = 1u << 16;
// ... of a role that has given up, for what it has under way itself: 82 ms
constexpr unsigned kDrainTries = 1u << 12;
__device__ __forceinline__ bool mbar_wait_asleep(uint64_t *bar, unsigned parity, unsigned *status, unsigned tries = kWaitTries) {
    for (unsigned i = 0; i < tries; ++i) {
        unsigned ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
            : "memory");
        if (ok) return true;
    }
    if (status) atomicOr(status, kStatusBarrierTimeout);
    return false;
}
// Position in a ring of `n` stages and the parity of its current round.  Every role walks its rings with one of these:
// a division and a remainder by the (run-time) ring length per stage were most of what the single threads that issue
// the copies and the MMAs executed per stage.
struct Ring {
    int pos = 0, n;
    unsigned par = 0;            // parity of the round `pos` is in
    bool wrapped = false;        // the ring has been around at least once: the stage at `pos` has a previous use
    __device__ __forceinline__ explicit Ring(int stages) : n(stages) {}
    __device__ __forceinline__ void next() {
        if (++pos == n) { pos = 0; par ^= 1u; wrapped = true; }
    }
};
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// ... on the barriers at this offset in both CTAs of the pair; `mask`: their ranks in the cluster
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar, unsigned short mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(mask) : "memory");
}

// cuTensorMapEncodeTiled from the driver, looked up once (the library links the runtime only).  It wants a current context, which a host thread has only after its first call of
// the runtime that needs one: without it an operator that was the first thing a thread asked for, the thread of a backward pass say, failed.
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
typedef CUresult (*CurrentContextFn)(CUcontext *);
inline EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static CurrentContextFn current = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        const auto look_up = [](const char *name) {
            void *p = nullptr;
            cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
            if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) return p;
            cudaGetLastError();
            return (void *)nullptr;
        };
        current = reinterpret_cast<CurrentContextFn>(look_up("cuCtxGetCurrent"));
        fn = reinterpret_cast<EncodeTiledFn>(look_up("cuTensorMapEncodeTiled"));
    });
    CUcontext context = nullptr;
    int device = 0;
    if (fn && (!current || current(&context) != CUDA_SUCCESS || !context) && (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess)) {
        cudaGetLastError();
        return nullptr;
    }
    return fn;
}

}  // namespace
}  // namespace bsq
