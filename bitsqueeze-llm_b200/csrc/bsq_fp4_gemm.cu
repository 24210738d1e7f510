// Product of two microscaled 4-bit matrices (sm_100a): out[M x N] = A[M x K] B[N x K]^T with both operands packed
// (bsq_fp4.hpp), on the block-scaled tensor-core instructions: tcgen05.mma kind::mxf4nvf4 with a scale for 16 of K (NVFP4),
// kind::mxf4 with one for 32 (MXFP4).  Products of codes and block scales are exact, sums are FP32 in tensor memory; the
// matrix scales are multiplied in when a tile leaves, and the result is rounded once.
//
// One CTA per SM, ten warps that meet only through mbarriers: warp 0 brings a stage of 256 of K (128 rows of P and up to 256 of Q
// by tiled TMA copies with 128-byte swizzle, their scale tiles by plain bulk copies), warp 1 copies the scales into tensor
// memory (tcgen05.cp, which runs in order with the MMAs of the same thread) and issues four MMAs of 64 of K, warps 2 to 9 take the
// accumulators out.  P is the operand whose rows are the 128 lanes of a tile, Q the one whose rows are its columns: P = A for
// training sizes; for a few tokens P = B, so that the tile's width follows the number of tokens and nothing is
// computed for rows that are not there.  Where there are fewer tiles than SMs, a cluster of 2 to 8 CTAs shares a tile: each
// takes a slice of K, the partial tiles are added through distributed shared memory in a fixed order.
// Every wait is bounded; a tile whose wait ran out is written as NaN.  No multicast.
#include "bsq_fp4.cuh"
#include "bsq_fp4_tile.cuh"
#include "bsq_internal.hpp"

namespace bsq {
namespace {

constexpr int kStageK = 256;                                     // of K per stage: one 128-byte row of codes
constexpr int kGemmThreads = 10 * 32;
constexpr int kEpilogueWarps = 8;
constexpr int kMaxStages = 10;

struct Fp4Gemm {
    int P, Q, K;                     // rows of P (tiles of 128), rows of Q (tiles of q_tile), columns of both
    int q_tile;                      // multiple of 16, up to 256; below 128 there is one tile of Q
    int p_tiles, q_tiles, stages, ring, sets;
    int k_stages, splits, stages_per_split;
    unsigned quads;                  // scale tiles along a row
    const uint8_t *p_scales, *q_scales;
    const float *p_head, *q_head;
    void *out;
    long ld;
    int type;
    bool lanes_contiguous;           // out[q * ld + p] instead of out[p * ld + q]
};

struct Fp4Bars {
    uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
    unsigned tmem_base, failed;
};

template <int FMT>
__device__ __forceinline__ void mma_fp4(unsigned tmem_d, uint64_t desc_a, uint64_t desc_b, unsigned idesc, unsigned sfa, unsigned sfb, bool accumulate) {
    const unsigned acc = accumulate ? 1u : 0u;
    if (FMT == kNvFp4)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
            : "memory");
}
// a scale tile (128 rows x 4 scales, 512 bytes) into four columns of tensor memory, the same in all four quarters of the lanes
__device__ __forceinline__ void copy_scales(unsigned tmem, unsigned smem) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(smem_desc(smem, 16u, 128u)) : "memory");
}

template <int FMT, bool SPLIT>
__global__ void __launch_bounds__(kGemmThreads, 1) fp4_gemm_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                                                                   const Fp4Gemm g, unsigned *status) {
    chain_begin();
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *base = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    constexpr int kQuads = FMT == kNvFp4 ? 4 : 2;                // scale tiles along K in a stage
    const int q_groups = (g.q_tile + 127) / 128;                 // scale tiles across the rows of a tile of Q
    const unsigned p_bytes = 128u * 128u, q_bytes = (unsigned)g.q_tile * 128u;
    const unsigned sp_at = p_bytes + ((q_bytes + 1023u) & ~1023u), sq_at = sp_at + kQuads * 512u;
    const unsigned stage_bytes = (sq_at + (unsigned)q_groups * kQuads * 512u + 1023u) & ~1023u;
    Fp4Bars &bars = *reinterpret_cast<Fp4Bars *>(base + (size_t)g.ring * stage_bytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = SPLIT ? (int)(blockIdx.x % (unsigned)g.splits) : 0;
    const int tiles = g.p_tiles * g.q_tiles;
    const int first = SPLIT ? (int)(blockIdx.x / (unsigned)g.splits) : (int)blockIdx.x, step = SPLIT ? tiles : (int)gridDim.x;
    const int k0 = rank * g.stages_per_split, k1 = min(g.k_stages, k0 + g.stages_per_split);

    const unsigned sf_cols = (unsigned)kQuads * 4u * (1u + (unsigned)q_groups);          // scales of a stage in tensor memory
    const unsigned acc_cols = (unsigned)((g.q_tile + 31) & ~31);
    const unsigned need = (unsigned)g.sets * acc_cols + 2u * sf_cols;
    const unsigned tmem_cols = need <= 128u ? 128u : need <= 256u ? 256u : 512u;
    if (tid == 0) {
        for (int i = 0; i < g.ring; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.acc_full[i], 1);
            mbar_init(&bars.acc_empty[i], kEpilogueWarps);
        }
        mbar_init(&bars.drain, 1);
        bars.failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars.tmem_base, tmem_sf = tmem + (unsigned)g.sets * acc_cols;
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            Ring r(g.ring);
            int filled = 0;
            const int p_limit = (g.P + 127) / 128, q_limit = (g.Q + 127) / 128;
            for (int t = first; t < tiles && ok; t += step) {
                const int pt = t % g.p_tiles, qt = t / g.p_tiles, q_first = qt * g.q_tile / 128;
                for (int k = k0; k < k1; ++k, ++filled, r.next()) {
                    if (r.wrapped) ok = mbar_wait_bounded(&bars.empty[r.pos], r.par ^ 1u, status);
                    if (!ok) break;
                    unsigned char *s = base + (size_t)r.pos * stage_bytes;
                    const unsigned quad = (unsigned)k * kQuads, sf = min((unsigned)kQuads, g.quads - quad) * 512u;
                    const int groups = min(q_groups, q_limit - q_first);
                    uint64_t *bar = &bars.full[r.pos];
                    mbar_expect_tx(bar, p_bytes + q_bytes + sf * (1u + (unsigned)groups));
                    tma_load_2d(s, &map_p, k * 128, pt * 128, bar);
                    tma_load_2d(s + p_bytes, &map_q, k * 128, qt * g.q_tile, bar);
                    bulk_g2s(s + sp_at, g.p_scales + ((size_t)min(pt, p_limit - 1) * g.quads + quad) * 512, sf, bar);
                    for (int i = 0; i < groups; ++i)
                        bulk_g2s(s + sq_at + (unsigned)i * kQuads * 512u, g.q_scales + ((size_t)(q_first + i) * g.quads + quad) * 512, sf, bar);
                }
            }
            if (!ok) {                                           // copies in flight must have landed before this CTA's shared memory goes away
                atomicOr(&bars.failed, 1u);
                for (int c = max(0, filled - g.ring); c < filled; ++c) mbar_wait_bounded(&bars.full[c % g.ring], (unsigned)(c / g.ring) & 1u, status);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // E2M1 x E2M1, scales UE4M3 (NVFP4) or UE8M0, FP32 sums, Q >> 3, P >> 7
            const unsigned idesc0 = (1u << 7) | (1u << 10) | ((unsigned)(g.q_tile >> 3) << 17) | (FMT == kMxFp4 ? 1u << 23 : 0u) | (1u << 27);
            Ring r(g.ring), rs(g.sets);
            unsigned buf = 0;
            for (int t = first; t < tiles && ok; t += step, rs.next()) {
                const unsigned acc = tmem + (unsigned)rs.pos * acc_cols;
                if (rs.wrapped) ok = mbar_wait_bounded(&bars.acc_empty[rs.pos], rs.par ^ 1u, status);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int k = k0; k < k1; ++k, r.next(), buf ^= 1u) {
                    ok = mbar_wait_bounded(&bars.full[r.pos], r.par, status);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned s = smem_u32(base + (size_t)r.pos * stage_bytes);
                    const unsigned sfp = tmem_sf + buf * sf_cols, sfq = sfp + (unsigned)kQuads * 4u;
                    const int quads = (int)min((unsigned)kQuads, g.quads - (unsigned)k * kQuads);
                    for (int i = 0; i < quads; ++i) {
                        copy_scales(sfp + (unsigned)i * 4u, s + sp_at + (unsigned)i * 512u);
                        for (int j = 0; j < q_groups; ++j)
                            copy_scales(sfq + (unsigned)(i * q_groups + j) * 4u, s + sq_at + (unsigned)(j * kQuads + i) * 512u);
                    }
                    const uint64_t dp = smem_desc_sw128(s), dq = smem_desc_sw128(s + p_bytes);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (k * kStageK + kk * 64 >= g.K) break;
                        const int quad = FMT == kNvFp4 ? kk : kk >> 1;
                        const unsigned id = FMT == kNvFp4 ? 0u : (unsigned)(kk & 1) * 2u;        // MXFP4: the scales of a 64 are half of a tile's four
                        mma_fp4<FMT>(acc, dp + (uint64_t)(kk * 2), dq + (uint64_t)(kk * 2), idesc0 | (id << 4) | (id << 29), sfp + (unsigned)quad * 4u,
                                     sfq + (unsigned)(quad * q_groups) * 4u, k > k0 || kk > 0);
                    }
                    tc_commit(&bars.empty[r.pos]);
                }
                if (ok) tc_commit(&bars.acc_full[rs.pos]);
            }
            if (!ok) {
                atomicOr(&bars.failed, 1u);
                tc_commit(&bars.drain);                          // MMAs under way must be done before tensor memory is given back
                mbar_wait_bounded(&bars.drain, 0, status);
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;    // the lanes this warp may read; which half of the columns
        const int chunks = g.q_tile / 16, c_first = half ? (chunks + 1) / 2 : 0, c_count = half ? chunks / 2 : (chunks + 1) / 2;
        const float f0 = *g.p_head, f1 = *g.q_head;
        const int size = g.type == kF32 ? 4 : 2;
        const bool wide = (reinterpret_cast<uintptr_t>(g.out) | (uintptr_t)(g.ld * size)) % 32 == 0;
        Ring rs(g.sets);
        for (int t = first; t < tiles; t += step, rs.next()) {
            const int pt = t % g.p_tiles, qt = t / g.p_tiles;
            if (ok) ok = __all_sync(kFullMask, mbar_wait_bounded(&bars.acc_full[rs.pos], rs.par, status)) != 0;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned taddr = tmem + (unsigned)rs.pos * acc_cols + ((unsigned)(quarter * 32) << 16) + (unsigned)c_first * 16u;
            if constexpr (SPLIT) {
                // stages are free: every copy has landed and every MMA has read them
                float *part = reinterpret_cast<float *>(base);
                const int row = quarter * 32 + lane, ldp = g.q_tile + 4;
                for (int c = 0; c < c_count; ++c) {
                    unsigned r[16];
                    read16(taddr + (unsigned)c * 16u, r, ok);
                    if (g.lanes_contiguous) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) part[((c_first + c) * 16 + j) * 128 + row] = __uint_as_float(r[j]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            *reinterpret_cast<uint4 *>(part + row * ldp + (c_first + c) * 16 + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                    }
                }
            } else {
                unsigned r[8][16];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c < c_count && ok) tmem_ld16(taddr + (unsigned)c * 16u, r[c]);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (!ok) {
#pragma unroll
                    for (int c = 0; c < 8; ++c)
#pragma unroll
                        for (int j = 0; j < 16; ++j) r[c][j] = 0x7fffffffu;
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.acc_empty[rs.pos]);  // the accumulators are in registers: the next tile may begin
                const int p = pt * 128 + quarter * 32 + lane;
                if (p >= g.P) continue;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int q = qt * g.q_tile + (c_first + c) * 16, have = c < c_count ? min(16, g.Q - q) : 0;
                    if (have <= 0) continue;
                    if (g.lanes_contiguous) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (j < have) store_one(g.out, g.type, (long)(q + j) * g.ld + p, __uint_as_float(r[c][j]) * f0 * f1);
                    } else {
                        store_run16(g.out, g.type, (long)p * g.ld + q, r[c], f0, f1, have, wide);
                    }
                }
            }
        }
        if (!ok && lane == 0) atomicOr(&bars.failed, 1u);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols) : "memory");

    if (SPLIT) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int pt = first % g.p_tiles, qt = first / g.p_tiles;
        const int n_p = min(128, g.P - pt * 128), n_q = min(g.q_tile, g.Q - qt * g.q_tile);
        const auto read = [&](int i, int c) { return *cluster.map_shared_rank(reinterpret_cast<const float *>(base) + i, c); };
        if (g.lanes_contiguous)
            add_parts<kGemmThreads>(read, rank, 128, n_q, n_p, g.splits, *g.p_head, *g.q_head, g.out, g.type, (long)(qt * g.q_tile) * g.ld + pt * 128, g.ld);
        else
            add_parts<kGemmThreads>(read, rank, g.q_tile + 4, n_p, n_q, g.splits, *g.p_head, *g.q_head, g.out, g.type, (long)(pt * 128) * g.ld + qt * g.q_tile, g.ld);
        cluster.sync();                                          // nobody leaves while its shared memory is being read
    }
}

template <int FMT, bool SPLIT>
cudaError_t launch_fp4_gemm(const CUtensorMap &map_p, const CUtensorMap &map_q, const Fp4Gemm &g, unsigned grid, size_t smem, unsigned *status, cudaStream_t stream) {
    cudaError_t err = cudaFuncSetAttribute(fp4_gemm_kernel<FMT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return err;
    if (!SPLIT) return launch_chained(fp4_gemm_kernel<FMT, SPLIT>, grid, kGemmThreads, smem, stream, map_p, map_q, g, status);
    return launch_cluster(fp4_gemm_kernel<FMT, SPLIT>, grid, kGemmThreads, g.splits, smem, stream, map_p, map_q, g, status);
}

}  // namespace

cudaError_t fp4_matmul(int format, const void *a, uint64_t M, const void *b, uint64_t N, uint64_t K, void *out, int type, uint64_t ld,
                       unsigned *status, int sm_count, cudaStream_t stream) {
    if (M == 0 || N == 0) return cudaSuccess;
    const uint8_t *pa = static_cast<const uint8_t *>(a), *pb = static_cast<const uint8_t *>(b);
    const bool swap = M <= 64;                                   // few tokens: their number is the tile's width
    const uint64_t P = swap ? N : M, Q = swap ? M : N;
    const uint8_t *pp = swap ? pb : pa, *pq = swap ? pa : pb;
    Fp4Gemm g = {};
    g.P = (int)P; g.Q = (int)Q; g.K = (int)K;
    g.q_tile = swap ? (int)((Q + 15) / 16 * 16) : Q <= 128 ? 128 : 256;
    const uint64_t p_tiles = (P + 127) / 128, q_tiles = (Q + g.q_tile - 1) / g.q_tile;
    if (p_tiles * q_tiles > 0x7fffffffull / 8) return cudaErrorInvalidValue;
    g.p_tiles = (int)p_tiles; g.q_tiles = (int)q_tiles;
    g.k_stages = (int)((K + kStageK - 1) / kStageK);
    g.quads = (unsigned)fp4_quads(format, K);
    g.p_scales = pp + fp4_scales_at(P, K); g.q_scales = pq + fp4_scales_at(Q, K);
    g.p_head = reinterpret_cast<const float *>(pp); g.q_head = reinterpret_cast<const float *>(pq);
    g.out = out; g.ld = (long)ld; g.type = type; g.lanes_contiguous = swap;
    const int tiles = g.p_tiles * g.q_tiles;
    g.splits = 1;
    while (g.splits < 8 && tiles * g.splits * 2 <= sm_count && g.k_stages >= g.splits * 4) g.splits *= 2;
    g.stages_per_split = (g.k_stages + g.splits - 1) / g.splits;
    g.splits = (g.k_stages + g.stages_per_split - 1) / g.stages_per_split;               // no slice is empty
    g.sets = g.splits > 1 || g.q_tile > 128 ? 1 : 2;
    const int kQuads = format == kNvFp4 ? 4 : 2, q_groups = (g.q_tile + 127) / 128;
    const size_t stage = ((size_t)128 * 128 + ((size_t)g.q_tile * 128 + 1023) / 1024 * 1024 + (size_t)kQuads * 512 * (1 + q_groups) + 1023) / 1024 * 1024;
    const size_t room = (size_t)227 * 1024 - 1024 - sizeof(Fp4Bars) - 64;
    g.ring = (int)(room / stage < (size_t)kMaxStages ? room / stage : (size_t)kMaxStages);
    size_t smem = 1024 + g.ring * stage + sizeof(Fp4Bars) + 64;
    CUtensorMap map_p, map_q;
    if (!map_codes(&map_p, pp, P, K, 128u) || !map_codes(&map_q, pq, Q, K, (unsigned)g.q_tile)) return cudaErrorInvalidValue;
    if (g.splits > 1) {
        const unsigned grid = (unsigned)(tiles * g.splits);
        return format == kNvFp4 ? launch_fp4_gemm<kNvFp4, true>(map_p, map_q, g, grid, smem, status, stream)
                                : launch_fp4_gemm<kMxFp4, true>(map_p, map_q, g, grid, smem, status, stream);
    }
    const unsigned grid = (unsigned)(tiles < sm_count ? tiles : sm_count);
    return format == kNvFp4 ? launch_fp4_gemm<kNvFp4, false>(map_p, map_q, g, grid, smem, status, stream)
                            : launch_fp4_gemm<kMxFp4, false>(map_p, map_q, g, grid, smem, status, stream);
}

}  // namespace bsq
