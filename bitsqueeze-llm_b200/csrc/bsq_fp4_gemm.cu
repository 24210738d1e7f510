// Product of two microscaled 4-bit matrices (sm_100a): out[M x N] = A[M x K] B[N x K]^T with both operands packed
// (bsq_fp4.hpp), on the block-scaled tensor-core instructions: tcgen05.mma kind::mxf4nvf4 with a scale for 16 of K (NVFP4),
// kind::mxf4 with one for 32 (MXFP4).  Products of codes and block scales are exact, sums are FP32 in tensor memory; the
// matrix scales are multiplied in when a tile leaves, and the result is rounded once (FP32 results of more than 4096 of K: once for each chain, see kChainF32).
//
// Where there are tiles enough a pair of CTAs on two SMs shares one of 256 x 256 (cta_group::2): each brings 128 rows of either operand, so that shared memory
// is read 64 bytes a clock by the MMAs and written as fast by the copies; alone, with 128 x 256, it is 96 and 96, more than the 128 it can do.
// Ten warps that meet only through mbarriers: warp 0 brings a stage of 256 of K (tiled TMA copies, codes with 128-byte swizzle, scale tiles as
// they are), warp 1 of the leader copies the scales into tensor memory (tcgen05.cp, which runs in order with the MMAs of the same thread) and issues four
// MMAs of 64 of K, warps 2 to 9 take the accumulators into registers, so that the next tile may begin, and then write them.  P is the operand whose rows are
// the lanes of a tile, Q the one whose rows are its columns: P = A for training sizes; for a few tokens P = B, so that the tile's width follows the
// number of tokens.  Where there are fewer tiles than SMs, a cluster of 2 to 8 CTAs shares a tile: each takes a slice of K, the partial tiles are
// added through distributed shared memory in a fixed order.  Every wait is bounded; a tile whose wait ran out is written as NaN.  No load
// is a multicast; of a pair's MMAs only the word that they are done goes to both CTAs.
//
// NVFP4 4096 x 14336 x 4096: 99 us, 4.9 PFLOP/s, three times the measured rate of a BF16 library product.  The tensor pipe is busy for 0.78 of a tile's time; without
// MMAs and copies of scales the same loads take 82 us, so the rest is what shared memory is filled with (14 TB/s over all SMs), and some 600 clocks per
// tile in which the accumulators are read.  One row against 14336 x 4096: 9.4 us with the weight in the L2, 11.2 from memory (3.0 TB/s; 112 tiles on 148 SMs).
#include "bsq_fp4.cuh"
#include "bsq_fp4_tile.cuh"
#include "bsq_internal.hpp"

namespace bsq {
namespace {

constexpr int kStageK = 256;                                     // of K per stage: one 128-byte row of codes
constexpr int kGemmThreads = 10 * 32;
constexpr int kEpilogueWarps = 8;
constexpr int kMaxStages = 10;
// Longest chain of additions in one accumulator, in stages.  The tensor core cuts additions off instead of rounding them, 1.5e-8 of the sum each (one addition for 64 of K):
// 64 of them for FP32 results, as in the gradient products.  2048 x 4096 x 131072 with a column that is large in both matrices: 0.3e-6 off 64 bits, as rounded FP32 sums are
// (3.9e-6 in chains of 256).  Pairs pay for it, as the additions in memory take their share of what the operands need: 4096 x 4096 x 14336 94 to 117 us, with 4097 columns,
// whose rows TMA cannot add to, 104 to 206 (tiles of 128 columns and an accumulator for the total: 190).  16-bit
// results: 4096 additions where FP16's rounding hides them, 32768 for BF16.
constexpr int kChainF32 = 64 * 64 / kStageK, kChainF16 = 64 * kChainF32, kChainBf16 = 8 * kChainF16;
enum : int { kOneChain = 0, kInMemory, kInTotal };               // chains of a tile: one, added up in memory (pairs with FP32 results), in an accumulator of their own

struct Fp4Gemm {
    int P, Q, K;                     // rows of P, rows of Q, columns of both
    int q_tile;                      // multiple of 16, up to 256; below 128 there is one tile of Q
    int p_tiles, q_tiles, ring, sets;
    int k_stages, splits, stages_per_split, chain;       // (chain: stages that are summed in one accumulator)
    const float *p_head, *q_head;
    void *out;
    long ld;
    int type;
    bool lanes_contiguous;           // out[q * ld + p] instead of out[p * ld + q]
    bool boxes;                      // the result can be written by TMA
    unsigned epilogue_tries;         // of the waits for accumulators (kWaitTries but in tests)
};
struct GemmMaps {
    CUtensorMap p, q, p_scales, q_scales, out;
};

struct Fp4Bars {
    uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
    unsigned tmem_base, failed;
};
constexpr unsigned kBoxBytes = 32 * 128;                         // 32 rows x 128 bytes of the result on their way out, one box for each epilogue warp

// Bytes of a stage: codes of P and Q, scales of P and Q
template <int FMT, int CTAS> __host__ __device__ inline unsigned stage_bytes_of(int q_tile) {
    const unsigned quads = FMT == kNvFp4 ? 4 : 2, q = ((unsigned)q_tile / CTAS * 128u + 1023u) & ~1023u;
    return (128u * 128u + q + quads * 512u * (1u + ((unsigned)q_tile + 127u) / 128u) + 1023u) & ~1023u;
}

template <int FMT, int CTAS>
__device__ __forceinline__ void mma_fp4(unsigned tmem_d, uint64_t desc_a, uint64_t desc_b, unsigned idesc, unsigned sfa, unsigned sfb, bool accumulate) {
    const unsigned acc = accumulate ? 1u : 0u;
#define BSQ_MMA_FP4(KIND)                                                                                                                          \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma." KIND " [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(tmem_d), \
                 "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)                                                                \
                 : "memory")
    if (FMT == kNvFp4 && CTAS == 2) BSQ_MMA_FP4("cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X");
    else if (FMT == kNvFp4) BSQ_MMA_FP4("cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X");
    else if (CTAS == 2) BSQ_MMA_FP4("cta_group::2.kind::mxf4.block_scale.scale_vec::2X");
    else BSQ_MMA_FP4("cta_group::1.kind::mxf4.block_scale.scale_vec::2X");
#undef BSQ_MMA_FP4
}
// a scale tile (128 rows x 4 scales, 512 bytes) into four columns of tensor memory, the same in all four quarters of the lanes; of a pair: each CTA's own
template <int CTAS> __device__ __forceinline__ void copy_scales(unsigned tmem, uint64_t desc) {
    if (CTAS == 2) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// CTAS: 1, or 2 for a pair.  SPLIT: the CTAs of a cluster share a tile, each with a slice of K.
template <int FMT, int CTAS, bool SPLIT, int CHAINS>
__global__ void __launch_bounds__(kGemmThreads, 1) fp4_gemm_kernel(const __grid_constant__ GemmMaps maps, const Fp4Gemm g, unsigned *status) {
    static_assert(CTAS == 1 ? CHAINS != kInMemory : !SPLIT && CHAINS != kInTotal, "pairs do not share tiles and leave no room for a total");
    constexpr bool TOTAL = CHAINS == kInTotal;
    chain_begin();
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *base = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    constexpr int kQuads = FMT == kNvFp4 ? 4 : 2;                // scale tiles along K in a stage
    const int q_groups = (g.q_tile + 127) / 128;                 // scale tiles across the rows of a tile of Q
    const unsigned p_bytes = 128u * 128u, q_bytes = (unsigned)(g.q_tile / CTAS) * 128u;
    const unsigned sp_at = p_bytes + ((q_bytes + 1023u) & ~1023u), sq_at = sp_at + kQuads * 512u;
    const unsigned stage_bytes = stage_bytes_of<FMT, CTAS>(g.q_tile);
    unsigned char *boxes = base + (size_t)g.ring * stage_bytes;
    Fp4Bars &bars = *reinterpret_cast<Fp4Bars *>(boxes + (SPLIT || g.lanes_contiguous ? 0u : kEpilogueWarps * kBoxBytes));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int side = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;      // which CTA of the pair
    const bool leader = side == 0;
    const int rank = SPLIT ? (int)(blockIdx.x % (unsigned)g.splits) : 0;
    const int tiles = g.p_tiles * g.q_tiles;
    const int first = (int)(blockIdx.x / (SPLIT ? (unsigned)g.splits : (unsigned)CTAS)), step = SPLIT ? tiles : (int)(gridDim.x / CTAS);
    const int k0 = rank * g.stages_per_split, k1 = min(g.k_stages, k0 + g.stages_per_split);

    const unsigned sf_cols = (unsigned)kQuads * 4u * (1u + (unsigned)q_groups);          // scales of a stage in tensor memory
    const unsigned acc_cols = (unsigned)((g.q_tile + 31) & ~31);
    const unsigned total_at = (unsigned)g.sets * acc_cols, need = total_at + (TOTAL ? acc_cols : 0u) + 2u * sf_cols;
    const unsigned tmem_cols = need <= 128u ? 128u : need <= 256u ? 256u : 512u;
    if (tid == 0) {
        for (int i = 0; i < g.ring; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.acc_full[i], 1);
            mbar_init(&bars.acc_empty[i], CTAS * kEpilogueWarps);
        }
        mbar_init(&bars.drain, 1);
        bars.failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<CTAS>(&bars.tmem_base, tmem_cols);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CTAS == 2) cg::this_cluster().sync();          // the other CTA's barriers are ready too
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars.tmem_base, tmem_sf = tmem + need - 2u * sf_cols;
    const unsigned lead = CTAS == 2 ? cluster_addr(smem_u32(base), 0u) - smem_u32(base) : 0u;       // from an address here to the leader's
    bool ok = true;

    if (warp == 0) {
        if (lane == 0) {
            Ring r(g.ring);
            int filled = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const int p_row = ((t % g.p_tiles) * CTAS + side) * 128, q_row = (t / g.p_tiles) * g.q_tile;
                for (int k = k0; k < k1; ++k, ++filled, r.next()) {
                    if (r.wrapped) ok = mbar_wait_asleep(&bars.empty[r.pos], r.par ^ 1u, status);
                    if (!ok) break;
                    unsigned char *s = base + (size_t)r.pos * stage_bytes;
                    uint64_t *bar = &bars.full[r.pos];
                    // (boxes count in full, also where they reach past the matrix and are filled with zeros)
                    if (leader) mbar_expect_tx(bar, CTAS * (p_bytes + q_bytes + (unsigned)kQuads * 512u * (1u + (unsigned)q_groups)));
                    if (CTAS == 2) {
                        const unsigned lead_bar = smem_u32(bar) + lead;
                        tma_load_2d_pair(s, &maps.p, k * 128, p_row, lead_bar);
                        tma_load_2d_pair(s + p_bytes, &maps.q, k * 128, q_row + side * (g.q_tile / 2), lead_bar);
                        tma_load_2d_pair(s + sp_at, &maps.p_scales, k * kQuads * 64, p_row / 128, lead_bar);
                        tma_load_2d_pair(s + sq_at, &maps.q_scales, k * kQuads * 64, q_row / 128, lead_bar);
                    } else {
                        tma_load_2d(s, &maps.p, k * 128, p_row, bar);
                        tma_load_2d(s + p_bytes, &maps.q, k * 128, q_row, bar);
                        tma_load_2d(s + sp_at, &maps.p_scales, k * kQuads * 64, p_row / 128, bar);
                        tma_load_2d(s + sq_at, &maps.q_scales, k * kQuads * 64, q_row / 128, bar);
                    }
                }
            }
            // copies in flight must have landed before this CTA's shared memory goes away, also where whoever reads them has given up
            if (leader)
                for (int c = max(0, filled - g.ring); c < filled; ++c) mbar_wait_asleep(&bars.full[c % g.ring], (unsigned)(c / g.ring) & 1u, status, ok ? kWaitTries : kDrainTries);
        }
    } else if (warp == 1) {
        if (leader) {
            // E2M1 x E2M1, scales UE4M3 (NVFP4) or UE8M0, FP32 sums, Q >> 3, P >> 7
            const unsigned idesc0 = (1u << 7) | (1u << 10) | ((unsigned)(g.q_tile >> 3) << 17) | (FMT == kMxFp4 ? 1u << 23 : 0u) | ((unsigned)CTAS << 27);
            const unsigned sq_quad = (unsigned)q_groups * 4u;    // columns of tensor memory for the scales of Q in a scale tile's K
            Ring r(g.ring), rs(g.sets);
            unsigned buf = 0;
            // (a tile's chains one behind the other: SPLIT has one tile)
            for (int t = first, c0 = k0; t < tiles && ok; rs.next()) {
                const unsigned acc = tmem + (unsigned)rs.pos * acc_cols;
                if (rs.wrapped) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.acc_empty[rs.pos], rs.par ^ 1u, status)) != 0;
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int c1 = CHAINS == kOneChain ? k1 : min(k1, c0 + g.chain);
                for (int k = c0; k < c1; ++k, r.next(), buf ^= 1u) {
                    ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.full[r.pos], r.par, status)) != 0;
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned s = smem_u32(base) + (unsigned)r.pos * stage_bytes;
                    const unsigned sfp = tmem_sf + buf * sf_cols, sfq = sfp + (unsigned)kQuads * 4u;
                    const uint64_t dsp = smem_desc(s + sp_at, 16u, 128u), dsq = smem_desc(s + sq_at, 16u, 128u);
                    const uint64_t dp = smem_desc_sw128(s), dq = smem_desc_sw128(s + p_bytes);
                    const int steps = min(4, (g.K - k * kStageK + 63) / 64);
                    if (elect_one()) {
                        // (tiles of scales behind the last one are zeros, so that a whole stage can be copied)
#pragma unroll
                        for (int i = 0; i < kQuads; ++i) {
                            copy_scales<CTAS>(sfp + (unsigned)i * 4u, dsp + (uint64_t)(i * 32));
                            copy_scales<CTAS>(sfq + (unsigned)i * sq_quad, dsq + (uint64_t)(i * 32));
                            if (q_groups == 2) copy_scales<CTAS>(sfq + (unsigned)i * sq_quad + 4u, dsq + (uint64_t)((kQuads + i) * 32));
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            const int quad = FMT == kNvFp4 ? kk : kk >> 1;
                            const unsigned id = FMT == kNvFp4 ? 0u : (unsigned)(kk & 1) * 2u;    // MXFP4: the scales of a 64 are half of a tile's four
                            if (kk < steps)
                                mma_fp4<FMT, CTAS>(acc, dp + (uint64_t)(kk * 2), dq + (uint64_t)(kk * 2), idesc0 | (id << 4) | (id << 29), sfp + (unsigned)quad * 4u,
                                                   sfq + (unsigned)quad * sq_quad, k > c0 || kk > 0);
                        }
                        if (CTAS == 2) tc_commit_pair(&bars.empty[r.pos], 3);
                        else tc_commit(&bars.empty[r.pos]);
                    }
                    __syncwarp();
                }
                if (ok && elect_one()) {
                    if (CTAS == 2) tc_commit_pair(&bars.acc_full[rs.pos], 3);
                    else tc_commit(&bars.acc_full[rs.pos]);
                }
                __syncwarp();
                c0 = c1;
                if (CHAINS == kOneChain || c0 >= k1) {
                    c0 = k0;
                    t += step;
                }
            }
            if (elect_one()) {                                   // MMAs under way must be done before tensor memory is given back, also where the epilogue has given up
                if (CTAS == 2) tc_commit_pair(&bars.drain, 1);
                else tc_commit(&bars.drain);
            }
            __syncwarp();
            mbar_wait_asleep(&bars.drain, 0, status);
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;    // the lanes this warp may read; which half of the columns
        const int chunks = g.q_tile / 16, c_first = half ? (chunks + 1) / 2 : 0, c_count = half ? chunks / 2 : (chunks + 1) / 2;
        const Factors f = join_factors(*g.p_head, *g.q_head);
        const int size = g.type == kF32 ? 4 : 2;
        Ring rs(g.sets);
        for (int t = first, c0 = k0; t < tiles; rs.next()) {
            const int p0 = ((t % g.p_tiles) * CTAS + side) * 128 + quarter * 32, q0 = (t / g.p_tiles) * g.q_tile;
            if (ok) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.acc_full[rs.pos], rs.par, status, g.epilogue_tries)) != 0;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned lanes = tmem + ((unsigned)(quarter * 32) << 16) + (unsigned)c_first * 16u;
            unsigned taddr = lanes + (unsigned)rs.pos * acc_cols;
            const bool more = TOTAL && k1 - c0 > g.chain, add = CHAINS == kInMemory && c0 > k0;    // not the last chain of this tile; (FP32) to what this warp wrote before
            if (TOTAL && (more || c0 > k0)) {
                for (int c = 0; c < c_count; ++c) {
                    unsigned r[16];
                    read16(taddr + (unsigned)c * 16u, r, ok);
                    if (c0 > k0) add16(lanes + total_at + (unsigned)c * 16u, r);
                    tmem_st16(lanes + total_at + (unsigned)c * 16u, r);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                taddr = lanes + total_at;
            }
            if (more) {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (ok && lane == 0) mbar_arrive(&bars.acc_empty[rs.pos]);
            } else if constexpr (SPLIT) {
                // stages are free: every copy has landed and every MMA has read them (without the accumulators nobody knows: nothing is written then)
                float *part = reinterpret_cast<float *>(base);
                const int row = quarter * 32 + lane, ldp = g.q_tile + 4;
                for (int c = 0; ok && c < c_count; ++c) {
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
                    for (int c = 0; c < 8; ++c) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) r[c][j] = 0x7fffffffu;
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                // the accumulators are in registers: the next tile may begin.  (Not where this warp has given up: it runs ahead from here on, and its arrivals would
                // let the next tile begin while others still read.)
                if (ok && lane == 0) {
                    if (CTAS == 2) mbar_arrive_pair(smem_u32(&bars.acc_empty[rs.pos]) + lead);
                    else mbar_arrive(&bars.acc_empty[rs.pos]);
                }
                if (!g.lanes_contiguous) {
                    // (tiles of Q of 128 or 256: a warp has 64 or 128 columns, boxes of 128 bytes a row, 16-byte pieces swizzled as the tensor map says)
                    // What was written to this tile before has to be there before it is added to: in that order every time, the same bits every time.
                    if (add && lane == 0) bulk_wait_all();
                    unsigned char *box = boxes + (unsigned)(warp - 2) * kBoxBytes;
                    uint4 *line = reinterpret_cast<uint4 *>(box + lane * 128);
                    const int per = 8 / size;                    // chunks of 16 columns in a box
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        if (c < c_count) {
                            const int in_box = c & (per - 1);
                            if (in_box == 0) {
                                if (lane == 0) bulk_wait_read_all();     // the box's last copy has been read
                                __syncwarp();
                            }
                            float v[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[c][j]) * f.first * f.second;
                            if (g.type == kF32) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float4 o = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                                    line[(in_box * 4 + j) ^ (lane & 7)] = *reinterpret_cast<const uint4 *>(&o);
                                }
                            } else {
                                unsigned w[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) w[j] = g.type == kBf16 ? pack_pair<kBf16>(v[2 * j], v[2 * j + 1]) : pack_pair<kF16>(v[2 * j], v[2 * j + 1]);
                                line[(in_box * 2) ^ (lane & 7)] = make_uint4(w[0], w[1], w[2], w[3]);
                                line[(in_box * 2 + 1) ^ (lane & 7)] = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                            if (in_box == per - 1) {
                                const int col = q0 + (c_first + c + 1 - per) * 16;
                                if (p0 < g.P && col < g.Q) {
                                    if (g.boxes) {
                                        fence_proxy_async_smem();
                                        __syncwarp();
                                        if (lane == 0) {
                                            if (add) tma_add_2d(&maps.out, col, p0, line);
                                            else tma_store_2d(&maps.out, col, p0, line);
                                            bulk_commit();
                                        }
                                    } else {
                                        if (add) box_add(box, lane, static_cast<float *>(g.out), (long)p0 * g.ld + col, g.ld, g.P - p0, g.Q - col);
                                        else box_out(box, lane, g.out, size, (long)p0 * g.ld + col, g.ld, g.P - p0, g.Q - col);
                                    }
                                }
                            }
                        }
                    }
                } else if (p0 + lane < g.P) {
                    const int p = p0 + lane;
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const int q = q0 + (c_first + c) * 16, have = c < c_count ? min(16, g.Q - q) : 0;
                        if (have > 0) {
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (j < have) store_one(g.out, g.type, (long)(q + j) * g.ld + p, __uint_as_float(r[c][j]) * f.first * f.second);
                        }
                    }
                }
            }
            c0 += g.chain;
            if (CHAINS == kOneChain || c0 >= k1) {
                c0 = k0;
                t += step;
            }
        }
        if (!SPLIT && lane == 0) bulk_wait_all();
        if (SPLIT && !ok && lane == 0) atomicOr(&bars.failed, 1u);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CTAS == 2) cg::this_cluster().sync();          // the leader's MMAs are done with this CTA's memory, the other's arrivals have landed
    if (warp == 1) tmem_free<CTAS>(tmem, tmem_cols);

    if constexpr (SPLIT) {
        // given up: NaN for the whole partial tile, now that nothing is on its way into the stages any more
        if (bars.failed) nan_part<kGemmThreads>(reinterpret_cast<float *>(base), 128 * (g.q_tile + 4));
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int pt = first % g.p_tiles, qt = first / g.p_tiles;
        const int n_p = min(128, g.P - pt * 128), n_q = min(g.q_tile, g.Q - qt * g.q_tile);
        const auto read = [&](int i, int c) { return *reinterpret_cast<const float4 *>(cluster.map_shared_rank(reinterpret_cast<const float *>(base) + i, c)); };
        if (g.lanes_contiguous)
            add_parts<kGemmThreads>(read, rank, 128, n_q, n_p, g.splits, *g.p_head, *g.q_head, g.out, g.type, (long)(qt * g.q_tile) * g.ld + pt * 128, g.ld);
        else
            add_parts<kGemmThreads>(read, rank, g.q_tile + 4, n_p, n_q, g.splits, *g.p_head, *g.q_head, g.out, g.type, (long)(pt * 128) * g.ld + qt * g.q_tile, g.ld);
        cluster.sync();                                          // nobody leaves while its shared memory is being read
    }
}

// Scale tiles as 64-bit elements: a row of the map for each group of 128 rows
template <int FMT> bool map_scales(CUtensorMap *map, const uint8_t *packed, uint64_t rows, uint64_t cols, unsigned box_groups) {
    const uint64_t quads = fp4_quads(FMT, cols);
    const cuuint64_t dims[2] = {quads * 64, (rows + 127) / 128}, strides[1] = {quads * 512};
    const cuuint32_t box[2] = {FMT == kNvFp4 ? 256u : 128u, box_groups}, estr[2] = {1, 1};
    return encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<uint8_t *>(packed) + fp4_scales_at(rows, cols), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int FMT, int CTAS, bool SPLIT, int CHAINS = kOneChain>
cudaError_t launch_fp4_gemm(GemmMaps &maps, Fp4Gemm &g, const uint8_t *p, const uint8_t *q, int sm_count, unsigned *status, cudaStream_t stream) {
    if (!map_codes(&maps.p, p, (uint64_t)g.P, (uint64_t)g.K, 128u) || !map_codes(&maps.q, q, (uint64_t)g.Q, (uint64_t)g.K, (unsigned)(g.q_tile / CTAS)) ||
        !map_scales<FMT>(&maps.p_scales, p, (uint64_t)g.P, (uint64_t)g.K, 1u) || !map_scales<FMT>(&maps.q_scales, q, (uint64_t)g.Q, (uint64_t)g.K, (unsigned)(g.q_tile + 127) / 128))
        return cudaErrorInvalidValue;
    const size_t stage = stage_bytes_of<FMT, CTAS>(g.q_tile), fixed = 1024 + sizeof(Fp4Bars) + 64 + (SPLIT || g.lanes_contiguous ? 0 : kEpilogueWarps * kBoxBytes);
    const size_t room = ((size_t)227 * 1024 - fixed) / stage;
    g.ring = (int)(room < (size_t)kMaxStages ? room : (size_t)kMaxStages);
    const size_t smem = fixed + g.ring * stage;
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = allow_smem(fp4_gemm_kernel<FMT, CTAS, SPLIT, CHAINS>, &done);
    if (err != cudaSuccess) return err;
    const int tiles = g.p_tiles * g.q_tiles, units = sm_count / CTAS;
    if (SPLIT) return launch_cluster(fp4_gemm_kernel<FMT, CTAS, SPLIT, CHAINS>, (unsigned)(tiles * g.splits), kGemmThreads, g.splits, smem, stream, maps, g, status);
    const unsigned grid = (unsigned)((tiles < units ? tiles : units) * CTAS);
    if (CTAS == 2) return launch_cluster(fp4_gemm_kernel<FMT, CTAS, SPLIT, CHAINS>, grid, kGemmThreads, CTAS, smem, stream, maps, g, status);
    return launch_chained(fp4_gemm_kernel<FMT, CTAS, SPLIT, CHAINS>, grid, kGemmThreads, smem, stream, maps, g, status);
}
template <int FMT>
cudaError_t launch_format(int ctas, GemmMaps &maps, Fp4Gemm &g, const uint8_t *p, const uint8_t *q, int sm_count, unsigned *status, cudaStream_t stream) {
    const bool chains = g.stages_per_split > g.chain;
    if (ctas == 2) return chains ? launch_fp4_gemm<FMT, 2, false, kInMemory>(maps, g, p, q, sm_count, status, stream)
                                 : launch_fp4_gemm<FMT, 2, false>(maps, g, p, q, sm_count, status, stream);
    if (chains) return g.splits > 1 ? launch_fp4_gemm<FMT, 1, true, kInTotal>(maps, g, p, q, sm_count, status, stream)
                                    : launch_fp4_gemm<FMT, 1, false, kInTotal>(maps, g, p, q, sm_count, status, stream);
    return g.splits > 1 ? launch_fp4_gemm<FMT, 1, true>(maps, g, p, q, sm_count, status, stream) : launch_fp4_gemm<FMT, 1, false>(maps, g, p, q, sm_count, status, stream);
}

}  // namespace

cudaError_t fp4_matmul(int format, const void *a, uint64_t M, const void *b, uint64_t N, uint64_t K, void *out, int type, uint64_t ld,
                       unsigned *status, int sm_count, cudaStream_t stream) {
    if (M == 0 || N == 0) return cudaSuccess;
    const uint8_t *pa = static_cast<const uint8_t *>(a), *pb = static_cast<const uint8_t *>(b);
    const bool swap = M <= 128;                                  // few tokens: their number is the tile's width (100 x 4096 x 4096: 17.7 us without, 8.1 with)
    const uint64_t P = swap ? N : M, Q = swap ? M : N;
    const uint8_t *pp = swap ? pb : pa, *pq = swap ? pa : pb;
    Fp4Gemm g = {};
    g.P = (int)P; g.Q = (int)Q; g.K = (int)K;
    g.k_stages = (int)((K + kStageK - 1) / kStageK);
    g.p_head = reinterpret_cast<const float *>(pp); g.q_head = reinterpret_cast<const float *>(pq);
    g.out = out; g.ld = (long)ld; g.type = type; g.lanes_contiguous = swap;
    g.epilogue_tries = epilogue_tries(kWaitTries);
    const uint64_t row_bytes = ld * op_bytes(type);
    const bool tma_out = !swap && tma_can_write(out, row_bytes, N * op_bytes(type));
    const int longest = type == kF32 ? kChainF32 : type == kF16 ? kChainF16 : kChainBf16;
    int ctas = 1;
    const auto plan = [&](int q_tile) {
        g.q_tile = q_tile;
        // a pair per tile of 256 x 256 where that fills the device
        ctas = q_tile == 256 && P > 128 && ((P + 255) / 256) * ((Q + 255) / 256) * 2 >= (uint64_t)sm_count * 2 / 3 ? 2 : 1;
        const uint64_t p_rows = (uint64_t)128 * ctas, p_tiles = (P + p_rows - 1) / p_rows, q_tiles = (Q + q_tile - 1) / q_tile;
        if (p_tiles * q_tiles > 0x7fffffffull / 8) return false;
        g.p_tiles = (int)p_tiles; g.q_tiles = (int)q_tiles;
        const int tiles = g.p_tiles * g.q_tiles;
        g.splits = 1;
        if (ctas == 1)
            while (g.splits < 8 && tiles * g.splits * 2 <= sm_count && g.k_stages >= g.splits * 4) g.splits *= 2;
        g.stages_per_split = (g.k_stages + g.splits - 1) / g.splits;
        g.splits = (g.k_stages + g.stages_per_split - 1) / g.stages_per_split;           // no slice is empty
        return true;
    };
    if (!plan(swap ? (int)((Q + 15) / 16 * 16) : Q <= 128 ? 128 : 256)) return cudaErrorInvalidValue;
    // Longer sums are several chains.  Pairs with FP32 results add them up in memory; else that takes an accumulator more, for which tiles of 256 columns leave no room.
    if (g.stages_per_split > longest && g.q_tile == 256 && !(ctas == 2 && type == kF32) && !plan(128)) return cudaErrorInvalidValue;
    g.chain = g.stages_per_split < longest ? g.stages_per_split : longest;
    g.sets = ctas == 1 && g.stages_per_split > g.chain ? 2 : g.splits > 1 || g.q_tile > 128 ? 1 : 2;
    if (!encode_tiled()) return cudaErrorInvalidValue;
    GemmMaps maps = {};
    g.boxes = tma_out && g.splits == 1;
    if (g.boxes) {
        const cuuint64_t dims[2] = {N, M}, strides[1] = {row_bytes};
        const cuuint32_t box[2] = {128u / (unsigned)op_bytes(type), 32u}, estr[2] = {1, 1};
        if (encode_tiled()(&maps.out, type == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out,
                           dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    return format == kNvFp4 ? launch_format<kNvFp4>(ctas, maps, g, pp, pq, sm_count, status, stream)
                            : launch_format<kMxFp4>(ctas, maps, g, pp, pq, sm_count, status, stream);
}

}  // namespace bsq
