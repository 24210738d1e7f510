// Gradient products of a linear layer whose weight and parked activations are held in 4 bits (sm_100a):
//   input    out[M x K] = dY[M x N] W[N x K]        weight   out[N x K] = dY[M x N]^T X[M x K]
// with dY in BF16 and W, X packed (bsq_fp4.hpp).  Both are out[R x C] = op(dY)[R x D] B[D x C], where B's blocks lie along C, not along the
// dimension D that is summed over, so the block-scaled instructions of bsq_fp4_gemm.cu do not apply: B is decoded to BF16.  A code
// times its block scale has 6 significant bits and BF16's exponent covers every MXFP4 scale (NVFP4: held 2^12 smaller), so decoding is exact;
// sums are FP32 in tensor memory, the matrix scale is multiplied in when a tile leaves, and the result is rounded once.  The tensor core
// cuts every addition off instead of rounding it, and what is lost grows with the length of the chain: results in FP32 leave tensor memory every 1024 of D
// and are added up rounded (4096 of D: 1.0e-6 off 64 bits in chains of 2048, 0.4e-6 in chains of 1024, a rounded FP32 product 0.3e-6).  Where CTAs share a tile, a
// slice of more than four such chains adds them up in tensor memory (1024 x 1024 from 65536: 0.2e-6 off, 2.6e-6 in the four chains of 8192 that it had; 199 us, 189).
// 16-bit results are one chain up to 65536 (FP16) or 524288 terms (BF16), and several that are added up in the same way beyond.
//
// Where there are enough tiles, a pair of CTAs on two SMs shares one (cta_group::2): of 512 x 256 for 16-bit results, so that an element of B is decoded once for
// 512 rows, of 256 x 256 for FP32 ones, which leaves a second set of accumulators for the next 1024 of D while one is taken out.  Each CTA has half of the rows of dY
// and decodes 128 columns of B.  Per 64 of D warp 0 brings the packed codes and scales of 64 rows of B (5 KB instead of 16), warp 2 boxes of dY (128-byte
// swizzle, in the orientation that memory has; the tensor core reads either), groups of four warps decode a stage each into the swizzled operand (contiguous
// along C), warp 1 of the leader issues the MMAs, four warps take finished tiles out.  Small results: one CTA per tile of 128 x 128, and clusters that share a
// tile along D (partial sums through distributed shared memory).
//
// Bound by the tensor core, then by power: dX of 4096 x 14336 x 4096 in BF16 325 us from rest (1480 TFLOP/s, 0.90 of the measured burst rate of a library product), 358
// sustained at 1.5 GHz (1345, 0.97 of the sustained rate); 128 tiles on 74 pairs are 0.86 of two full rounds.  dW of 4096 x 4096 x 14336 in FP32 455 us.  On the way
// here: one CTA per 128 x 256 with eight warps decoding 774 us (decoding waited for itself), pairs 1020 (every remote arrival waited for all stores of the SM), with
// arrivals that do not 453, decoded before the operand's place is waited for 418, left shifts 379, tiles of 512 rows 325.
#include "bsq_fp4_decode.cuh"
#include "bsq_fp4_few.hpp"
#include "bsq_fp4_tile.cuh"
#include "bsq_internal.hpp"

#include <algorithm>

namespace bsq {
namespace {

// warp 0: copies of B, 1: MMAs (in the other CTA of a pair: the word that a stage is ready), 2: copies of dY, 4-7: epilogue, 8-: decode
constexpr int kDecodeWarps = 4;                                  // at one stage
constexpr int kEpilogueWarps = 4, kFirstDecode = 4 + kEpilogueWarps;
constexpr int kTileC = 128, kStageD = 64;                        // a CTA's columns of B; of D per stage
constexpr int kMaxRing = 5, kMaxRawRing = 8;
constexpr unsigned kBoxBytes = 32 * 128;                         // 32 rows x 128 bytes of the result on their way out: two for each epilogue warp
constexpr unsigned kBoxesBytes = kEpilogueWarps * 2 * kBoxBytes;
constexpr unsigned kABytes = 128 * kStageD * 2, kBBytes = kStageD * kTileC * 2;
constexpr unsigned kCodeBytes = kStageD * kTileC / 2, kRawBytes = kCodeBytes + 1024;
constexpr int kChainStages = 1024 / kStageD;                     // FP32 results: longest chain of additions in tensor memory
// ... of 16-bit results: 65536 terms lose 0.3e-4, all to one side, a sixth of what FP16's rounding takes (2.1e-4); 262144 lose 1.9e-4.  BF16 has three bits fewer.
// (Longer chains than need be cost less: a second one rules tiles of 512 rows out, 4096 x 4096 from 65536 1360 us with them, 1700 without.)
constexpr int kChainStagesF16 = 65536 / kStageD, kChainStagesBf16 = 8 * kChainStagesF16;

// A stage: MT blocks of 128 rows of dY, 128 columns of B
__host__ __device__ constexpr unsigned op_bytes_of(int mt) { return (unsigned)mt * kABytes + kBBytes; }
__host__ __device__ constexpr int ring_of(int mt) { return mt == 2 ? 3 : 4; }
// Groups of decoding warps, each with a stage of its own.  They wait by the parity of barriers, which tells one round from the next and no more:
//   * a stage's MMAs are done in order, so a group that has done its last stage may wait for the next one if that lies no further on than a round: never more groups
//     than operand stages;
//   * copies land in ANY order, so nothing that a group has seen of other places says how far the copies of its next one are: every place of the raw ring always goes
//     to the same group, the ring a multiple of the groups.  (With six places and four groups a group could find the copy before last in a place whose last one
//     was still under way: about one product in 100000 had a tile with a stage of old values.)
__host__ __device__ constexpr int groups_of(int mt) { return mt == 2 ? 3 : 4; }
__host__ __device__ constexpr int raw_ring_of(int mt) { return mt == 2 ? 6 : 8; }
__host__ __device__ constexpr int grad_threads(int mt) { return (kFirstDecode + kDecodeWarps * groups_of(mt)) * 32; }
template <int MT> constexpr bool rings_fit() {
    return groups_of(MT) <= ring_of(MT) && raw_ring_of(MT) % groups_of(MT) == 0 && ring_of(MT) <= kMaxRing && raw_ring_of(MT) <= kMaxRawRing;
}
static_assert(rings_fit<1>() && rings_fit<2>(), "a wait could take one round for another");

struct Fp4Grad {
    int R, C, D;                     // rows and columns of the result, the dimension that is summed over
    int r_tiles, c_tiles, d_stages, splits, stages_per_split;
    bool a_kmajor;                   // dY contiguous along D (input gradient) or along R (weight gradient)
    int chain;                       // stages that are summed in one accumulator
    unsigned quads;                  // scale tiles along a row of B
    const uint8_t *scales;
    const float *head;
    void *out;
    long ld;
    int type;
    bool boxes;                      // the result can be written by TMA
    unsigned epilogue_tries;         // of the waits for accumulators (kWaitTries but in tests)
};

struct GradBars {
    uint64_t full[kMaxRing], empty[kMaxRing], ready[kMaxRing], raw_full[kMaxRawRing], raw_empty[kMaxRawRing], acc_full[2], acc_empty[2], drain;
    unsigned tmem_base, failed;
};

// Operand contiguous along M / N in 128-byte-swizzled shared memory: groups of 64 elements (128 bytes) x 64 of K, 8192 bytes apart (leading
// byte offset); within one, groups of 8 of K 1024 bytes apart (stride byte offset).  A step of 16 along K is 2048 bytes of the start address.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(unsigned addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(8192u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ void mma_f16_pair(unsigned tmem_d, uint64_t desc_a, uint64_t desc_b, unsigned idesc, bool accumulate) {
    const unsigned acc = accumulate ? 1u : 0u;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(0u)
        : "memory");
}

// 16 columns of accumulators, decode8's order of columns undone
__device__ __forceinline__ void read_columns(unsigned taddr, unsigned (&r)[16], bool ok) {
    unsigned p[16];
    read16(taddr, p, ok);
#pragma unroll
    for (int j = 0; j < 16; ++j) r[j] = p[(j & 8) | ((j & 3) << 1) | ((j & 4) >> 2)];
}

// CTAS: 1, or 2 for a pair.  MT: blocks of 128 rows of a CTA, each with accumulators of its own.  SPLIT: the CTAs of a cluster share a tile, each with a slice of D.
// TOTAL: chains are added up in tensor memory, in an accumulator of their own.
template <int FMT, int CTAS, int MT, bool SPLIT, bool TOTAL>
__global__ void __launch_bounds__(grad_threads(MT), 1) fp4_grad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                   const __grid_constant__ CUtensorMap map_c, const Fp4Grad g, unsigned *status) {
    static_assert((CTAS == 1 || !SPLIT) && (MT == 1 || CTAS == 2) && (MT == 1 || !TOTAL), "pairs do not share tiles, single CTAs have one block of rows, two blocks leave no room for a total");
    chain_begin();
    constexpr int kRing = ring_of(MT), kRawRing = raw_ring_of(MT);
    constexpr unsigned kOpBytes = op_bytes_of(MT);
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *base = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    unsigned char *raw = base + kRing * kOpBytes, *boxes = raw + kRawRing * kRawBytes;
    GradBars &bars = *reinterpret_cast<GradBars *>(boxes + kBoxesBytes);
    constexpr int kQuads = FMT == kNvFp4 ? 2 : 1;                // scale tiles across a CTA's 128 columns
    constexpr unsigned kAccCols = CTAS * kTileC;                 // columns of an accumulator
    // Accumulators that chains take in turn.  SPLIT: a slice of up to four chains leaves them side by side, one accumulator each, and they are added once; of a longer
    // one (TOTAL) they take two accumulators in turn, and a third holds what they have come to.
    constexpr int kSets = SPLIT ? 4 : 2 / MT, kTurns = SPLIT ? (TOTAL ? 2 : 1) : TOTAL ? 1 : kSets;
    constexpr unsigned kTotal = kTurns * kAccCols;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int half = CTAS == 2 ? (int)(blockIdx.x & 1) : 0, unit = (int)(blockIdx.x / (SPLIT ? (unsigned)g.splits : (unsigned)CTAS));
    const int rank = SPLIT ? (int)(blockIdx.x % (unsigned)g.splits) : 0;
    const int tiles = g.r_tiles * g.c_tiles;
    const int first = unit, step = SPLIT ? tiles : (int)(gridDim.x / CTAS);
    const int d0 = rank * g.stages_per_split, d1 = min(g.d_stages, d0 + g.stages_per_split);
    const bool leader = half == 0;

    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&bars.full[i], 1 + kDecodeWarps + (CTAS == 2 ? 1 : 0));
            mbar_init(&bars.empty[i], 1);
            mbar_init(&bars.ready[i], kDecodeWarps);
        }
        for (int i = 0; i < kRawRing; ++i) {
            mbar_init(&bars.raw_full[i], 1);
            mbar_init(&bars.raw_empty[i], kDecodeWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.acc_full[i], 1);
            mbar_init(&bars.acc_empty[i], CTAS * kEpilogueWarps);
        }
        mbar_init(&bars.drain, 1);
        bars.failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<CTAS>(&bars.tmem_base, 512u);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CTAS == 2) cg::this_cluster().sync();          // the other CTA's barriers are ready too
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars.tmem_base;
    const unsigned lead = CTAS == 2 ? cluster_addr(smem_u32(base), 0u) - smem_u32(base) : 0u;       // from an address here to the leader's
    bool ok = true;

    if (warp == 0) {
        // ---- codes and scales of this CTA's columns, up to kRawRing stages ahead ----
        if (lane == 0) {
            Ring r(kRawRing);
            int filled = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const int c_tile = (t / g.r_tiles) * CTAS + half;
                const unsigned quad = (unsigned)c_tile * kQuads, sf = quad < g.quads ? min((unsigned)kQuads, g.quads - quad) * 512u : 0u;
                for (int d = d0; d < d1; ++d, ++filled, r.next()) {
                    if (r.wrapped) ok = mbar_wait_asleep(&bars.raw_empty[r.pos], r.par ^ 1u, status);
                    if (!ok) break;
                    unsigned char *s = raw + (size_t)r.pos * kRawBytes;
                    mbar_expect_tx(&bars.raw_full[r.pos], kCodeBytes + sf);
                    tma_load_2d(s, &map_b, c_tile * (kTileC / 2), d * kStageD, &bars.raw_full[r.pos]);
                    if (sf) bulk_g2s(s + kCodeBytes, g.scales + ((size_t)(d >> 1) * g.quads + quad) * 512, sf, &bars.raw_full[r.pos]);
                }
            }
            // copies in flight must have landed before this CTA's shared memory goes away, also where whoever reads them has given up
            for (int c = max(0, filled - kRawRing); c < filled; ++c)
                mbar_wait_asleep(&bars.raw_full[c % kRawRing], (unsigned)(c / kRawRing) & 1u, status, ok ? kWaitTries : kDrainTries);
        }
    } else if (warp == 1) {
        if (lane == 0 && !leader) {
            // this CTA's decoded stages are announced to the leader by one thread: an arrival there waits for all stores in front of it
            Ring r(kRing);
            for (int t = first; t < tiles && ok; t += step)
                for (int d = d0; d < d1; ++d, r.next()) {
                    ok = mbar_wait_asleep(&bars.ready[r.pos], r.par, status);
                    if (!ok) break;
                    mbar_arrive_pair(smem_u32(&bars.full[r.pos]) + lead);
                }
        }
        if (leader) {
            // BF16 x BF16, FP32 sums, B contiguous along N, A along K or along M, N >> 3, M >> 4
            const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | (g.a_kmajor ? 0u : 1u << 15) | (1u << 16) | (kAccCols >> 3 << 17) | ((CTAS * 128u >> 4) << 24);
            const uint64_t a_step = g.a_kmajor ? 2u : 128u;
            Ring r(kRing), rs(kTurns);
            for (int t = first; t < tiles && ok; t += step) {
                for (int c0 = d0; c0 < d1 && ok; c0 += SPLIT && !TOTAL ? d1 - d0 : g.chain, rs.next()) {
                    const int c1 = SPLIT && !TOTAL ? d1 : min(d1, c0 + g.chain);
                    if (rs.wrapped) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.acc_empty[rs.pos], rs.par ^ 1u, status)) != 0;
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    int set = SPLIT && !TOTAL ? 0 : rs.pos, left = g.chain;                  // (SPLIT: up to four accumulators, one behind the other)
                    bool fresh = true;
                    for (int d = c0; d < c1; ++d, r.next()) {
                        ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.full[r.pos], r.par, status)) != 0;
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned s = smem_u32(base) + (unsigned)r.pos * kOpBytes;
                        const uint64_t da = g.a_kmajor ? smem_desc_sw128(s) : smem_desc_mn_sw128(s), db = smem_desc_mn_sw128(s + MT * kABytes);
                        const unsigned acc = tmem + (unsigned)set * kAccCols;
                        if (elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < kStageD / 16; ++kk)
#pragma unroll
                                for (int m = 0; m < MT; ++m) {
                                    const uint64_t dam = da + a_step * (uint64_t)kk + (uint64_t)(m * (kABytes >> 4));
                                    if (CTAS == 2) mma_f16_pair(acc + (unsigned)m * kAccCols, dam, db + (uint64_t)(kk * 128), idesc, !fresh || kk > 0);
                                    else mma_f16(acc, dam, db + (uint64_t)(kk * 128), idesc, !fresh || kk > 0);
                                }
                            if (CTAS == 2) tc_commit_pair(&bars.empty[r.pos], 3);
                            else tc_commit(&bars.empty[r.pos]);
                        }
                        __syncwarp();
                        fresh = false;
                        if (SPLIT && !TOTAL && --left == 0) {
                            ++set;
                            left = g.chain;
                            fresh = true;
                        }
                    }
                    if (ok && elect_one()) {
                        if (CTAS == 2) tc_commit_pair(&bars.acc_full[rs.pos], 3);
                        else tc_commit(&bars.acc_full[rs.pos]);
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) {                                   // MMAs under way must be done before tensor memory is given back, also where the epilogue has given up
                if (CTAS == 2) tc_commit_pair(&bars.drain, 1);
                else tc_commit(&bars.drain);
            }
            __syncwarp();
            mbar_wait_asleep(&bars.drain, 0, status);
        }
    } else if (warp == 2) {
        // ---- dY ----
        if (lane == 0) {
            Ring r(kRing);
            int filled = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const int row = ((t % g.r_tiles) * CTAS * MT + half) * 128;
                for (int d = d0; d < d1; ++d, ++filled, r.next()) {
                    if (r.wrapped) ok = mbar_wait_asleep(&bars.empty[r.pos], r.par ^ 1u, status);
                    if (!ok) break;
                    unsigned char *s = base + (size_t)r.pos * kOpBytes;
                    uint64_t *bar = &bars.full[r.pos];
                    if (leader) mbar_expect_tx(bar, CTAS * MT * kABytes);
#pragma unroll
                    for (int m = 0; m < MT; ++m, s += kABytes) {
                        const int r0 = row + m * CTAS * 128;
                        if (CTAS == 2) {
                            const unsigned lead_bar = smem_u32(bar) + lead;
                            if (g.a_kmajor) {
                                tma_load_2d_pair(s, &map_a, d * kStageD, r0, lead_bar);
                            } else {
                                tma_load_2d_pair(s, &map_a, r0, d * kStageD, lead_bar);
                                tma_load_2d_pair(s + kABytes / 2, &map_a, r0 + 64, d * kStageD, lead_bar);
                            }
                        } else if (g.a_kmajor) {
                            tma_load_2d(s, &map_a, d * kStageD, r0, bar);
                        } else {
                            tma_load_2d(s, &map_a, r0, d * kStageD, bar);
                            tma_load_2d(s + kABytes / 2, &map_a, r0 + 64, d * kStageD, bar);
                        }
                    }
                }
            }
            // (as above; a stage also waits for its decoding warps, which may have given up)
            if (leader)
                for (int c = max(0, filled - kRing); c < filled; ++c)
                    mbar_wait_asleep(&bars.full[c % kRing], (unsigned)(c / kRing) & 1u, status, ok ? kWaitTries : kDrainTries);
        }
    } else if (warp >= kFirstDecode) {
        // ---- decode: groups of four warps take the stages in turn.  A thread has one row of B and, twice, 32 of its columns; the lanes of a warp have
        // rows beside one another, so that neither the swizzled codes nor the swizzled operand see a bank conflict ----
        const int w = (warp - kFirstDecode) % kDecodeWarps, d_in = (w & 1) * 32 + lane, turn = (warp - kFirstDecode) / kDecodeWarps;
        Ring r(kRing), rr(kRawRing);
        int n = 0;
        for (int t = first; t < tiles && ok; t += step) {
            for (int d = d0; d < d1; ++d, n = n + 1 == groups_of(MT) ? 0 : n + 1, r.next(), rr.next()) {
                if (n != turn) continue;
                constexpr int kUnits = 8 / kDecodeWarps;         // of 32 columns for each thread
                ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.raw_full[rr.pos], rr.par, status)) != 0;
                if (!ok) break;
                const unsigned char *s = raw + (size_t)rr.pos * kRawBytes;
                const int row = (d & 1) * 64 + d_in;             // in its scale tile
                const unsigned char *sf = s + kCodeBytes + (row & 31) * 16 + (row >> 5) * 4;
                const bool live = d * kStageD + d_in < g.D;      // (scales behind the last row are anything)
                uint4 v[kUnits][4];
#pragma unroll
                for (int j = 0; j < kUnits; ++j) {
                    const int u = (w >> 1) + j * (kDecodeWarps / 2);
                    const uint4 c = *reinterpret_cast<const uint4 *>(s + d_in * 64 + ((u ^ ((d_in >> 1) & 3)) << 4));
                    unsigned s0, s1;
                    if (FMT == kMxFp4) {
                        const unsigned one = live ? sf[u] : 0u;
                        s0 = s1 = decode_scales<FMT>(one, one);
                    } else {
                        const unsigned two = live ? *reinterpret_cast<const unsigned short *>(sf + (u >> 1) * 512 + (u & 1) * 2) : 0u;
                        const unsigned both = decode_scales<FMT>(two & 0xffu, two >> 8);
                        s0 = __byte_perm(both, both, 0x1010);
                        s1 = __byte_perm(both, both, 0x3232);
                    }
                    v[j][0] = decode8<FMT>(c.x, s0);
                    v[j][1] = decode8<FMT>(c.y, s0);
                    v[j][2] = decode8<FMT>(c.z, s1);
                    v[j][3] = decode8<FMT>(c.w, s1);
                }
                // only then the operand's place is waited for: what follows is all that a free stage waits for on this side
                if (r.wrapped) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.empty[r.pos], r.par ^ 1u, status)) != 0;
                if (!ok) break;
                unsigned char *b = base + (size_t)r.pos * kOpBytes + MT * kABytes + d_in * 128;
#pragma unroll
                for (int j = 0; j < kUnits; ++j) {
                    const int u = (w >> 1) + j * (kDecodeWarps / 2);
#pragma unroll
                    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(b + (u >> 1) * 8192 + ((((u & 1) * 4 + i) ^ (d_in & 7)) << 4)) = v[j][i];
                }
                fence_proxy_async_smem();                        // stores before the tensor core's reads, reads before the next copy's writes
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(leader ? &bars.full[r.pos] : &bars.ready[r.pos]);
                    mbar_arrive(&bars.raw_empty[rr.pos]);
                }
            }
        }
        if (SPLIT && !ok && lane == 0) atomicOr(&bars.failed, 1u);                           // (as the epilogue does: this tile is not whole)
    } else if (warp >= 4) {
        const int quarter = warp & 3;                            // the lanes of tensor memory this warp may read
        const Factors f = join_factors(*g.head, FMT == kNvFp4 ? kNvHold : 1.0f);
        const int size = g.type == kF32 ? 4 : 2;
        int which = 0;
        Ring rs(kTurns);
        for (int t = first; t < tiles; t += step) {
            const int row = ((t % g.r_tiles) * CTAS * MT + half) * 128 + quarter * 32, col = (t / g.r_tiles) * (int)kAccCols;
            for (int c0 = d0; c0 < d1; c0 += SPLIT && !TOTAL ? d1 - d0 : g.chain, rs.next()) {
                if (ok) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.acc_full[rs.pos], rs.par, status, g.epilogue_tries)) != 0;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const unsigned lanes = tmem + ((unsigned)(quarter * 32) << 16);
                unsigned taddr = lanes + (SPLIT && !TOTAL ? 0u : (unsigned)rs.pos * kAccCols);
                const bool add = !SPLIT && !TOTAL && c0 > d0;    // (FP32 only: to what this warp wrote before)
                const bool more = TOTAL && d1 - c0 > g.chain;    // not the last chain of this tile
                if (TOTAL && (more || c0 > d0)) {
                    for (int c = 0; c < (int)kAccCols; c += 16) {
                        unsigned r[16];
                        read16(taddr + (unsigned)c, r, ok);
                        if (c0 > d0) add16(lanes + kTotal + (unsigned)c, r);
                        tmem_st16(lanes + kTotal + (unsigned)c, r);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    taddr = lanes + kTotal;
                }
                if (more) {
                } else if constexpr (SPLIT) {
                    // (without the accumulators nobody knows whether the stages are free: nothing is written then)
                    for (int c = 0; ok && c < (int)kAccCols; c += 16) {
                        unsigned r[16];
                        read_columns(taddr + (unsigned)c, r, ok);
                        for (int i = 1; !TOTAL && i < kSets && i * g.chain < d1 - d0; ++i) {
                            unsigned q[16];
                            read_columns(taddr + (unsigned)i * kAccCols + (unsigned)c, q, ok);
#pragma unroll
                            for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(q[j]));
                        }
                        // operand stages are free: every copy has landed and every MMA has read them
                        float *part = reinterpret_cast<float *>(base) + (quarter * 32 + lane) * (kTileC + 4) + c;
#pragma unroll
                        for (int j = 0; j < 16; j += 4) *reinterpret_cast<uint4 *>(part + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                    }
                } else {
                    // through boxes in shared memory, 16-byte pieces swizzled as the tensor map says, written (or added) by TMA as whole lines.  What was written to
                    // this tile before has to be there before it is added to: in that order every time, the same bits every time.
                    const int per = 128 / size;
                    if (add && lane == 0) bulk_wait_all();
                    for (int at = 0; at < MT * (int)kAccCols; at += per) {
                        const int m = at / (int)kAccCols, c = at - m * (int)kAccCols, row0 = row + m * CTAS * 128;
                        if (row0 >= g.R || col + c >= g.C) continue;
                        // The two boxes take turns with what is really copied: all copies but the newest have been read, so this box's last one has.  (A box that is
                        // written and not copied would put the count out by one, and the next would overwrite what is still being read.)
                        unsigned char *box = boxes + (unsigned)((warp - 4) * 2 + which) * kBoxBytes;
                        which ^= 1;
                        if (lane == 0) bulk_wait_read_1();
                        __syncwarp();
                        uint4 *line = reinterpret_cast<uint4 *>(box + lane * 128);
#pragma unroll 1
                        for (int h = 0; h < per; h += 16) {
                            unsigned r[16];
                            read_columns(taddr + (unsigned)(at + h), r, ok);
                            float v[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]) * f.first * f.second;
                            if (g.type == kF32) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float4 o = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                                    line[(h / 4 + j) ^ (lane & 7)] = *reinterpret_cast<const uint4 *>(&o);
                                }
                            } else {
                                unsigned w[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j) w[j] = g.type == kBf16 ? pack_pair<kBf16>(v[2 * j], v[2 * j + 1]) : pack_pair<kF16>(v[2 * j], v[2 * j + 1]);
                                line[(h / 8) ^ (lane & 7)] = make_uint4(w[0], w[1], w[2], w[3]);
                                line[(h / 8 + 1) ^ (lane & 7)] = make_uint4(w[4], w[5], w[6], w[7]);
                            }
                        }
                        if (g.boxes) {
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                if (add) tma_add_2d(&map_c, col + c, row0, box);
                                else tma_store_2d(&map_c, col + c, row0, box);
                                bulk_commit();
                            }
                        } else if (add) {
                            box_add(box, lane, static_cast<float *>(g.out), (long)row0 * g.ld + col + c, g.ld, g.R - row0, g.C - col - c);
                        } else {
                            box_out(box, lane, g.out, size, (long)row0 * g.ld + col + c, g.ld, g.R - row0, g.C - col - c);
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                // (not where this warp has given up: it runs ahead from here on, and its arrivals would let accumulators be overwritten that others still read)
                if (ok && lane == 0) {
                    if (CTAS == 2) mbar_arrive_pair(smem_u32(&bars.acc_empty[rs.pos]) + lead);
                    else mbar_arrive(&bars.acc_empty[rs.pos]);
                }
            }
        }
        if (!SPLIT && lane == 0) bulk_wait_all();
        if (SPLIT && !ok && lane == 0) atomicOr(&bars.failed, 1u);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CTAS == 2) cg::this_cluster().sync();          // the leader's MMAs are done with this CTA's memory, the other's arrivals have landed
    if (warp == 1) tmem_free<CTAS>(tmem, 512u);

    if constexpr (SPLIT) {
        // given up: NaN for the whole partial tile, now that nothing is on its way into the stages any more
        if (bars.failed) nan_part<grad_threads(MT)>(reinterpret_cast<float *>(base), 128 * (kTileC + 4));
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int rt = first % g.r_tiles, ct = first / g.r_tiles;
        const auto read = [&](int i, int c) { return *reinterpret_cast<const float4 *>(cluster.map_shared_rank(reinterpret_cast<const float *>(base) + i, c)); };
        add_parts<grad_threads(MT)>(read, rank, kTileC + 4, min(128, g.R - rt * 128), min(kTileC, g.C - ct * kTileC), g.splits, *g.head, FMT == kNvFp4 ? kNvHold : 1.0f, g.out,
                                g.type, (long)(rt * 128) * g.ld + ct * kTileC, g.ld);
        cluster.sync();                                          // nobody leaves while its shared memory is being read
    }
}

// Rows of 16-bit elements whose stride or start TMA cannot take, copied to rows of `ld_out` elements
__global__ void __launch_bounds__(256) pad_rows_kernel(const unsigned short *in, uint64_t rows, uint64_t cols, uint64_t ld, unsigned short *out, uint64_t ld_out) {
    chain_begin();
    for (uint64_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (uint64_t c = (uint64_t)blockIdx.x * 2048 + threadIdx.x; c < min(cols, (uint64_t)(blockIdx.x + 1) * 2048); c += 256) out[r * ld_out + c] = in[r * ld + c];
}

template <int FMT, int CTAS, int MT, bool SPLIT, bool TOTAL = false>
cudaError_t launch_grad(const CUtensorMap &map_a, const CUtensorMap &map_b, const CUtensorMap &map_c, const Fp4Grad &g, int sm_count, unsigned *status, cudaStream_t stream) {
    constexpr size_t smem = 1024 + ring_of(MT) * op_bytes_of(MT) + raw_ring_of(MT) * kRawBytes + kBoxesBytes + sizeof(GradBars) + 64;
    static_assert(smem <= 227 * 1024, "stages do not fit");
    static_assert((size_t)128 * (kTileC + 4) * 4 <= (size_t)ring_of(MT) * op_bytes_of(MT), "partial tile does not fit");
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = allow_smem(fp4_grad_kernel<FMT, CTAS, MT, SPLIT, TOTAL>, &done);
    if (err != cudaSuccess) return err;
    const int tiles = g.r_tiles * g.c_tiles;
    if (SPLIT) return launch_cluster(fp4_grad_kernel<FMT, CTAS, MT, SPLIT, TOTAL>, (unsigned)(tiles * g.splits), grad_threads(MT), g.splits, smem, stream, map_a, map_b, map_c, g, status);
    const int units = sm_count / CTAS, grid = (tiles < units ? tiles : units) * CTAS;
    if (CTAS == 2) return launch_cluster(fp4_grad_kernel<FMT, CTAS, MT, SPLIT, TOTAL>, (unsigned)grid, grad_threads(MT), CTAS, smem, stream, map_a, map_b, map_c, g, status);
    return launch_chained(fp4_grad_kernel<FMT, CTAS, MT, SPLIT, TOTAL>, (unsigned)grid, grad_threads(MT), smem, stream, map_a, map_b, map_c, g, status);
}
template <int FMT>
cudaError_t launch_grad_format(int ctas, int blocks, const CUtensorMap &map_a, const CUtensorMap &map_b, const CUtensorMap &map_c, const Fp4Grad &g, int sm_count, unsigned *status, cudaStream_t stream) {
    // chains that can neither lie side by side (FP32 results of shared tiles: up to four) nor be added up in memory (FP32 results)
    const bool total = g.type != kF32 ? g.stages_per_split > g.chain : g.splits > 1 && g.stages_per_split > 4 * g.chain;
    if (ctas == 2 && blocks == 2) return launch_grad<FMT, 2, 2, false>(map_a, map_b, map_c, g, sm_count, status, stream);
    if (ctas == 2) return total ? launch_grad<FMT, 2, 1, false, true>(map_a, map_b, map_c, g, sm_count, status, stream)
                                : launch_grad<FMT, 2, 1, false>(map_a, map_b, map_c, g, sm_count, status, stream);
    if (total) return g.splits > 1 ? launch_grad<FMT, 1, 1, true, true>(map_a, map_b, map_c, g, sm_count, status, stream)
                                   : launch_grad<FMT, 1, 1, false, true>(map_a, map_b, map_c, g, sm_count, status, stream);
    return g.splits > 1 ? launch_grad<FMT, 1, 1, true>(map_a, map_b, map_c, g, sm_count, status, stream) : launch_grad<FMT, 1, 1, false>(map_a, map_b, map_c, g, sm_count, status, stream);
}

bool needs_padding(const void *dy, uint64_t rows, uint64_t ld) { return reinterpret_cast<uintptr_t>(dy) % 16 != 0 || (rows > 1 && ld % 8 != 0); }

// out[R x C] = op(dY) B; dY is M x N, B is D x C packed
cudaError_t grad_product(int format, bool a_kmajor, const void *dy, uint64_t M, uint64_t N, uint64_t ld_dy, const uint8_t *b, uint64_t C, void *out, int type,
                         uint64_t ld, void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    const uint64_t R = a_kmajor ? M : N, D = a_kmajor ? N : M;
    if (R == 0) return cudaSuccess;
    if (D == 0) return cudaMemset2DAsync(out, ld * op_bytes(type), 0, C * op_bytes(type), R, stream);
    uint64_t ld_a = M > 1 ? ld_dy : (N + 7) / 8 * 8;             // (a single row: any stride will do)
    if (needs_padding(dy, M, ld_dy)) {
        ld_a = (N + 7) / 8 * 8;
        const dim3 grid((unsigned)((N + 2047) / 2048), (unsigned)(M < 4096 ? M : 4096));
        const cudaError_t err = launch_chained(pad_rows_kernel, grid, 256, 0, stream, static_cast<const unsigned short *>(dy), M, N, ld_dy,
                                               static_cast<unsigned short *>(scratch), ld_a);
        if (err != cudaSuccess) return err;
        dy = scratch;
    }
    // few rows: decoded in the registers of the MMAs (16 x 4096 x 14336 in MXFP4 18.5 us there, 30 here; one row in NVFP4 16.8 / 37; 5 x 1024 x 1024 5.6 / 6.8)
    if (a_kmajor && R <= kFewRowsMax) return fp4_grad_few(format, dy, (int)R, ld_a, b, D, C, out, type, ld, sm_count, stream);
    Fp4Grad g = {};
    g.R = (int)R; g.C = (int)C; g.D = (int)D;
    const uint64_t r128 = (R + 127) / 128, c128 = (C + kTileC - 1) / kTileC;
    if (r128 * c128 > 0x7fffffffull / 8) return cudaErrorInvalidValue;
    // a pair per tile of 256 x 256 where that fills the device
    const int ctas = r128 > 1 && ((r128 + 1) / 2) * ((c128 + 1) / 2) * 2 >= (uint64_t)sm_count * 2 / 3 ? 2 : 1;
    g.d_stages = (int)((D + kStageD - 1) / kStageD);
    const int longest = type == kF32 ? kChainStages : type == kF16 ? kChainStagesF16 : kChainStagesBf16;
    // ... of 512 x 256 where that does too: an element is then decoded once for 512 rows, but no accumulators are left for the next tile while one is taken out, or for a
    // second chain
    const int blocks = ctas == 2 && type != kF32 && g.d_stages <= longest && ((r128 + 3) / 4) * ((c128 + 1) / 2) * 2 >= (uint64_t)sm_count * 2 / 3 ? 2 : 1;
    g.r_tiles = (int)((r128 + ctas * blocks - 1) / (ctas * blocks)); g.c_tiles = (int)((c128 + ctas - 1) / ctas);
    g.a_kmajor = a_kmajor;
    g.quads = (unsigned)fp4_quads(format, C);
    g.scales = b + fp4_scales_at(D, C);
    g.head = reinterpret_cast<const float *>(b);
    g.out = out; g.ld = (long)ld; g.type = type;
    g.epilogue_tries = epilogue_tries(kWaitTries);
    const int tiles = g.r_tiles * g.c_tiles;
    g.splits = 1;
    if (ctas == 1)
        while (g.splits < 8 && tiles * g.splits * 2 <= sm_count && g.d_stages >= g.splits * 4) g.splits *= 2;
    g.stages_per_split = (g.d_stages + g.splits - 1) / g.splits;
    g.splits = (g.d_stages + g.stages_per_split - 1) / g.stages_per_split;               // no slice is empty
    g.chain = type != kF32 ? std::min(g.stages_per_split, longest) : g.splits > 1 ? std::min((g.stages_per_split + 3) / 4, longest) : longest;
    CUtensorMap map_a, map_b, map_c;
    const cuuint64_t dims_a[2] = {N, M}, strides_a[1] = {ld_a * 2}, dims_b[2] = {fp4_ld(C), D}, strides_b[1] = {fp4_ld(C)};
    const cuuint32_t box_a[2] = {64u, a_kmajor ? 128u : 64u}, box_b[2] = {kTileC / 2, kStageD}, estr[2] = {1, 1};
    if (!encode_tiled() ||
        encode_tiled()(&map_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(dy), dims_a, strides_a, box_a, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
        encode_tiled()(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(b) + kFp4Head, dims_b, strides_b, box_b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    map_c = map_a;                                               // (not looked at without boxes)
    const uint64_t row_bytes = (R == 1 ? C : ld) * op_bytes(type);
    g.boxes = tma_can_write(out, row_bytes, C * op_bytes(type));
    if (g.boxes) {
        const cuuint64_t dims_c[2] = {C, R}, strides_c[1] = {row_bytes};
        const cuuint32_t box_c[2] = {128u / (unsigned)op_bytes(type), 32u};
        if (encode_tiled()(&map_c, type == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out,
                           dims_c, strides_c, box_c, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    return format == kNvFp4 ? launch_grad_format<kNvFp4>(ctas, blocks, map_a, map_b, map_c, g, sm_count, status, stream)
                            : launch_grad_format<kMxFp4>(ctas, blocks, map_a, map_b, map_c, g, sm_count, status, stream);
}

}  // namespace

size_t fp4_grad_scratch_bytes(uint64_t M, uint64_t N, const void *dy, uint64_t ld_dy) { return needs_padding(dy, M, ld_dy) ? M * ((N + 7) / 8 * 8) * 2 : 0; }

cudaError_t fp4_grad_input(int format, const void *dy, uint64_t M, uint64_t ld_dy, const void *w, uint64_t N, uint64_t K, void *out, int type, uint64_t ld,
                           void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    return grad_product(format, true, dy, M, N, ld_dy, static_cast<const uint8_t *>(w), K, out, type, ld, scratch, status, sm_count, stream);
}

cudaError_t fp4_grad_weight(int format, const void *dy, uint64_t M, uint64_t N, uint64_t ld_dy, const void *x, uint64_t K, void *out, int type, uint64_t ld,
                            void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    return grad_product(format, false, dy, M, N, ld_dy, static_cast<const uint8_t *>(x), K, out, type, ld, scratch, status, sm_count, stream);
}

}  // namespace bsq
