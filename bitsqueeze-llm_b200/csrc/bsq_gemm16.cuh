// Products of 16-bit matrices on the tensor cores with an epilogue of the caller's choice (sm_100a): C[M x N] = A[M x K] B[N x K]^T for one matrix or a stack of them,
// FP32 sums in tensor memory.  What becomes of a tile is the epilogue's: statistics of a softmax, gradients of logits, a step of an iteration.
//
// Where there are enough tiles, a pair of CTAs on two SMs shares one of 256 x 256 (cta_group::2): each brings 128 rows of A and 128 of B, so that an element from
// the L2 feeds 256 multiplications.  Small results: one CTA per tile of 128 x 128.  Warp 0 brings stages of 64 of K by TMA (128-byte swizzle, five stages of 32 KB or seven; operands that are
// contiguous along K or along M / N, whichever they are in memory: the tensor core reads either), warp 1 of the leader issues the MMAs, warps 2 to 9 take finished
// tiles out while the next one is summed in the other half of tensor memory, each 32 rows and half of the columns.  (Four warps with all columns took 20 us for a tile that read
// and wrote two FP16 matrices, more than the 17 us of its 4096 of K.)
//
// The tensor core cuts additions off instead of rounding them: epilogues that want FP32's digits (kChained) get the sums every 1024 of K or so and add them up rounded, in registers.
// Others have no room for 128 sums beside what they hold (up to 4 KB a thread spill).  kBack: a function of its own adds them up and writes them back to where the last chain lies; the tile is taken from
// there while the next one's first chain is summed.  kTotals (chains of Gemm16::chain): they are added up, rounded, in the other half of tensor memory, where the tile is then taken from.
//
// An operand may come in two parts, high + low (splits): the product is then high x high + high x low + low x high, three walks along K into the same sums; or two, with the low part of one operand only.
//
// Bound by the tensor core, then by power: see the products that use it.
#pragma once

#include "bsq_fp4_tile.cuh"

namespace bsq {
namespace {

constexpr int kG16MaxStages = 7, kG16K = 64;                     // stages in flight at most, of K each
constexpr unsigned kG16Half = 128 * kG16K * 2, kG16Stage = 2 * kG16Half;
constexpr int kG16Warps = 8, kG16First = 2, kG16Threads = 32 * (kG16First + kG16Warps);       // epilogue warps, the last eight (ten in all: 200 registers a thread)
constexpr int kG16Chain = 1024 / kG16K;                          // stages of a chain of sums, about (kChained)
// ... (kBack).  A tile that is taken out holds the half that the next tile's second chain wants: loss and gradients of 4096 x 4096 x 32000 took 3270 us with one chain, 3310 this way, 3610 with chains of
// 2048, 4500 with 1024.  What is lost of sums of one sign, 2e-5 of them in FP16, is a tenth of a rounding to it.
constexpr int kG16BackChain = 4096 / kG16K;
constexpr unsigned kG16Box = 32 * 128;                           // 32 rows x 128 bytes on their way in or out: two for each epilogue warp, or none (EPI::kBoxes)
constexpr int kG16Band = 16;                                     // rows of tiles that are walked together, column after column

struct Gemm16 {
    int M, N;                        // of one matrix of the stack
    int m_tiles, n_tiles, batch;
    int k_stages, parts;             // stages along K of a tile, walks along K (1, 2 with one operand's low part, or 3 of split operands)
    bool low_a;                      // of two walks: the low part is A's, else B's
    int chain;                       // stages of a chain of sums, about; 0: one chain (kTotals)
    int splits;                      // a matrix's tiles are this many, each with k_stages of K, one behind the other: z = matrix * splits + slice
    bool a_kmajor, b_kmajor;         // contiguous along K, or along M / N
    bool lower;                      // the result is symmetric: tiles on and below the diagonal only
    bool bf16;
    unsigned tries;                  // of the epilogue's waits (kWaitTries but in tests)
};

struct Gemm16Maps {
    CUtensorMap a[2], b[2];          // high and low parts (low: with more than one walk)
};

struct Gemm16Bars {
    uint64_t full[kG16MaxStages], empty[kG16MaxStages], acc_full[2], acc_empty[2], fetched[kG16Warps], drain;
    unsigned tmem_base;
};

__device__ __forceinline__ void tma_load_3d(void *dst_smem, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst_smem)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void *dst_smem, const CUtensorMap *map, int x, int y, int z, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst_smem)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, int x, int y, int z, const void *src_smem) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(src_smem))
                 : "memory");
}
__device__ __forceinline__ void tma_add_3d(const CUtensorMap *map, int x, int y, int z, const void *src_smem) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(src_smem))
                 : "memory");
}

// Operand contiguous along M / N in 128-byte-swizzled shared memory: groups of 64 elements (128 bytes) x 64 of K, 8192 bytes apart (leading
// byte offset); within one, groups of 8 of K 1024 bytes apart (stride byte offset).  A step of 16 along K is 2048 bytes of the start address.
__device__ __forceinline__ uint64_t g16_desc_mn(unsigned addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(8192u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <int CTAS> __device__ __forceinline__ void g16_mma(unsigned tmem_d, uint64_t desc_a, uint64_t desc_b, unsigned idesc, bool accumulate) {
    const unsigned acc = accumulate ? 1u : 0u;
    if (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(tmem_d),
            "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc), "r"(0u)
            : "memory");
    else
        mma_f16(tmem_d, desc_a, desc_b, idesc, accumulate);
}
// All threads of both CTAs of a pair
__device__ __forceinline__ void pair_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Chains of sums, the last one half to one and a half of the others' length (one stage behind one of 16 kept the epilogue's warps as busy as a whole chain)
__device__ __forceinline__ int chains_of(int stages, int chain) { return chain ? max(1, (stages + chain / 2) / chain) : 1; }

// Where a tile lies
struct TileAt {
    int z, i, j;                     // matrix of the stack (and slice of K), row and column of tiles
};
__device__ __forceinline__ TileAt tile_at(const Gemm16 &g, int t) {
    const int per = g.lower ? g.m_tiles * (g.m_tiles + 1) / 2 : g.m_tiles * g.n_tiles;
    TileAt at;
    at.z = t / per;
    t -= at.z * per;
    if (g.lower) {
        int i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
        while ((i + 1) * (i + 2) / 2 <= t) ++i;
        while (i * (i + 1) / 2 > t) --i;
        at.i = i;
        at.j = t - i * (i + 1) / 2;
        return at;
    }
    const int band = t / (kG16Band * g.n_tiles), rows = min(kG16Band, g.m_tiles - band * kG16Band);
    t -= band * kG16Band * g.n_tiles;
    at.j = t / rows;
    at.i = band * kG16Band + t - at.j * rows;
    return at;
}

// What an epilogue is given: a warp has 32 rows of a tile (from `row` on; the thread's own is row + lane) and half of its columns, from `col` on.
struct TileOut {
    int z, row, col, lane;
    unsigned taddr;                  // accumulators of its rows
    bool ok;                         // not: the tile was given up, everything that it would give is NaN
    unsigned char *boxes;            // two boxes of this warp
    int *which;                      // the box that is next (box_next)
    uint64_t *fetched;               // boxes that were asked for are there
    unsigned *fetches;               // how many times
    unsigned *status;
};
// The box that is next, free to be written.  (The two take turns with what is really copied: a box that is asked for is copied out by TMA, box_send, or read by
// the warp itself before the next one is asked for.)
__device__ __forceinline__ unsigned char *box_next(const TileOut &t) {
    unsigned char *box = t.boxes + (unsigned)*t.which * kG16Box;
    *t.which ^= 1;
    if (t.lane == 0) bulk_wait_read_1();
    __syncwarp();
    return box;
}
__device__ __forceinline__ void box_send(const TileOut &t, const CUtensorMap *map, int x, int y, const unsigned char *box, bool add = false) {
    fence_proxy_async_smem();
    __syncwarp();
    if (t.lane == 0) {
        if (add) tma_add_3d(map, x, y, t.z, box);
        else tma_store_3d(map, x, y, t.z, box);
        bulk_commit();
    }
}
// The other way to use the two boxes: both at a time, first for what comes in.  (Rows of matrices that a thread reads and writes 32 bytes at a time touch 32 lines with every
// instruction: a tile that read and wrote two FP16 matrices took 14 us that way, more than 1024 of K; copies move whole lines.)  Asks for boxes of 64 columns x 32 rows of one or two matrices.
__device__ __forceinline__ void boxes_ask(const TileOut &o, const CUtensorMap *first, const CUtensorMap *second, int x) {
    fence_proxy_async_smem();                                    // this thread's reads and writes of the boxes come before the copies'
    __syncwarp();
    if (o.lane == 0) {
        bulk_wait_read_all();
        mbar_expect_tx(o.fetched, second ? 2 * kG16Box : kG16Box);
        tma_load_3d(o.boxes, first, x, o.row, o.z, o.fetched);
        if (second) tma_load_3d(o.boxes + kG16Box, second, x, o.row, o.z, o.fetched);
    }
    __syncwarp();
}
// The tile with boxes that are there (one that is given up where they do not come)
__device__ __forceinline__ TileOut boxes_wait(const TileOut &o) {
    TileOut t = o;
    t.ok = __all_sync(kFullMask, mbar_wait_asleep(o.fetched, *o.fetches & 1u, o.status)) != 0 && o.ok;
    ++*o.fetches;
    return t;
}
// ... free to be written without anything that came in
__device__ __forceinline__ void boxes_free(const TileOut &o) {
    if (o.lane == 0) bulk_wait_read_all();
    __syncwarp();
}
__device__ __forceinline__ uint4 *box_piece(const TileOut &o, int which, int i) { return reinterpret_cast<uint4 *>(o.boxes + (unsigned)which * kG16Box + o.lane * 128) + (i ^ (o.lane & 7)); }
// 16 FP16 values of the thread's row, two to a word: in, out
__device__ __forceinline__ void box_take16(const TileOut &o, int which, int h, unsigned (&w)[8]) {
    const uint4 a = *box_piece(o, which, 2 * h), b = *box_piece(o, which, 2 * h + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
}
__device__ __forceinline__ void box_give16(const TileOut &o, int which, int h, const unsigned (&w)[8]) {
    *box_piece(o, which, 2 * h) = make_uint4(w[0], w[1], w[2], w[3]);
    *box_piece(o, which, 2 * h + 1) = make_uint4(w[4], w[5], w[6], w[7]);
}
// A box as box_out takes it, 16 bytes at a time where rows start on 16 bytes
__device__ __forceinline__ void box_out_rows(const unsigned char *box, int lane, void *out, int size, long at, long ld, int rows, int cols) {
    if ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(ld * size) | (uintptr_t)(at * size)) % 16 != 0 || cols * size < 128) {
        box_out(box, lane, out, size, at, ld, rows, cols);
        return;
    }
    __syncwarp();
    const int piece = lane & 7;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        const uint4 q = *reinterpret_cast<const uint4 *>(box + r * 128 + ((piece ^ (r & 7)) << 4));
        if (r < rows) *reinterpret_cast<uint4 *>(static_cast<unsigned char *>(out) + (at + (long)r * ld) * size + piece * 16) = q;
    }
    __syncwarp();
}
// 16 values of the thread's row to places 16 h .. of its line of a box of 16-bit elements
template <int TYPE> __device__ __forceinline__ void box_put16(unsigned char *box, int lane, int h, const float (&v)[16]) {
    uint4 *line = reinterpret_cast<uint4 *>(box + lane * 128);
    unsigned w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = pack_pair<TYPE>(v[2 * j], v[2 * j + 1]);
    line[(2 * h) ^ (lane & 7)] = make_uint4(w[0], w[1], w[2], w[3]);
    line[(2 * h + 1) ^ (lane & 7)] = make_uint4(w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void read16f(unsigned taddr, float (&v)[16], bool ok) {
    unsigned r[16];
    read16(taddr, r, ok);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
}
// What a warp of the epilogue does before it takes a tile of several chains (kBack): all but the last one are added up in registers and given back, the last one's place gets the total.
// The ring is at the tile's first chain; the last one is still to be given back.  False: a wait has run out.
template <int COLS, int CTAS>
__device__ __noinline__ bool sum_chains(Gemm16Bars *bars, Ring rs, int chains, unsigned taddr, unsigned lead, bool mine, unsigned *status, unsigned tries, bool ok) {
    float sums[COLS];
    for (int n = 0;; ++n, rs.next()) {
        if (ok) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars->acc_full[rs.pos], rs.par, status, tries)) != 0;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (!ok || n + 1 == chains) break;
        if (mine) {
#pragma unroll
            for (int c = 0; c < COLS; c += 16) {
                float v[16];
                read16f(taddr + (unsigned)rs.pos * 256u + (unsigned)c, v, true);
#pragma unroll
                for (int j = 0; j < 16; ++j) sums[c + j] = n ? sums[c + j] + v[j] : v[j];
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            if (CTAS == 2) mbar_arrive_pair(smem_u32(&bars->acc_empty[rs.pos]) + lead);
            else mbar_arrive(&bars->acc_empty[rs.pos]);
        }
    }
    if (mine && ok) {
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
            const unsigned at = taddr + (unsigned)rs.pos * 256u + (unsigned)c;
            unsigned w[16];
            read16(at, w, true);
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(sums[c + j] + __uint_as_float(w[j]));
            tmem_st16(at, w);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
    return ok;
}
template <class EPI> __host__ __device__ constexpr int g16_stages() { return EPI::kBoxes ? 5 : kG16MaxStages; }
// EPI: a functor, called by whole warps:
//   kChained, kBack, kTotals                                          how chains of sums come together (one of them, or none: one chain)
//   template <int COLS> void tile(const TileOut &, Ahead &) const     takes COLS columns out; kChained: tile(const TileOut &, float (&sums)[COLS])
//   template <int COLS> void ahead(const TileOut &, Ahead &) const    what can be asked for while the tile is still being summed (not kChained)
//   void begin() const                                                by one thread of the launch (kChained)
// CTAS: 1, or 2 for a pair.
struct NoAhead {};
template <class EPI, int CTAS>
__global__ void __launch_bounds__(kG16Threads, 1) gemm16_kernel(const __grid_constant__ Gemm16Maps maps, const __grid_constant__ EPI epi, const Gemm16 g, unsigned *status) {
    chain_begin();
    constexpr int kTile = 128 * CTAS, kCols = kTile / 2, kStages = g16_stages<EPI>();
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *base = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    unsigned char *boxes = base + kStages * kG16Stage;
    Gemm16Bars &bars = *reinterpret_cast<Gemm16Bars *>(boxes + (EPI::kBoxes ? kG16Warps * 2 * kG16Box : 0));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int half = CTAS == 2 ? (int)(blockIdx.x & 1) : 0, first = (int)(blockIdx.x / CTAS), step = (int)(gridDim.x / CTAS);
    const int tiles = g.batch * g.splits * (g.lower ? g.m_tiles * (g.m_tiles + 1) / 2 : g.m_tiles * g.n_tiles);
    const int stages = g.k_stages * g.parts, chain = EPI::kChained ? kG16Chain : EPI::kBack ? kG16BackChain : EPI::kTotals ? g.chain : 0, chains = chains_of(stages, chain);
    const bool totals = EPI::kTotals && chains > 1;              // the MMAs write one half of tensor memory, the other one has the tile's total; else they write both by turns
    const bool leader = half == 0;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&bars.full[i], 1);
            mbar_init(&bars.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.acc_full[i], 1);
            mbar_init(&bars.acc_empty[i], CTAS * kG16Warps);
        }
        for (int i = 0; i < kG16Warps; ++i) mbar_init(&bars.fetched[i], 1);
        mbar_init(&bars.drain, 1);
        mbar_fence_init();
        if constexpr (EPI::kChained) {
            if (blockIdx.x == 0) epi.begin();
        }
    }
    if (warp == 1) tmem_alloc<CTAS>(&bars.tmem_base, 512u);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CTAS == 2) pair_meet();                        // the other CTA's barriers are ready too
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars.tmem_base;
    const unsigned lead = CTAS == 2 ? cluster_addr(smem_u32(base), 0u) - smem_u32(base) : 0u;       // from an address here to the leader's
    bool ok = true;

    if (warp == 0) {
        // ---- operands: this CTA's 128 rows of A and 128 of B ----
        if (lane == 0) {
            Ring r(kStages);
            int filled = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const TileAt at = tile_at(g, t);
                const int a0 = at.i * kTile + half * 128, b0 = at.j * kTile + half * 128, z = at.z / g.splits, d0 = at.z % g.splits * g.k_stages;
                for (int p = 0; p < g.parts && ok; ++p) {
                    const bool low_a = p == 2 || (p == 1 && g.low_a);
                    const CUtensorMap *ma = &maps.a[low_a], *mb = &maps.b[p && !low_a];
                    for (int d = 0; d < g.k_stages; ++d, ++filled, r.next()) {
                        if (r.wrapped) ok = mbar_wait_asleep(&bars.empty[r.pos], r.par ^ 1u, status);
                        if (!ok) break;
                        unsigned char *s = base + (size_t)r.pos * kG16Stage;
                        uint64_t *bar = &bars.full[r.pos];
                        if (leader) mbar_expect_tx(bar, CTAS * kG16Stage);
                        const int k = (d0 + d) * kG16K;
                        const unsigned lead_bar = smem_u32(bar) + lead;
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const CUtensorMap *m = o ? mb : ma;
                            const int r0 = o ? b0 : a0;
                            unsigned char *to = s + (unsigned)o * kG16Half;
                            if (o ? g.b_kmajor : g.a_kmajor) {
                                if (CTAS == 2) tma_load_3d_pair(to, m, k, r0, z, lead_bar);
                                else tma_load_3d(to, m, k, r0, z, bar);
                            } else if (CTAS == 2) {
                                tma_load_3d_pair(to, m, r0, k, z, lead_bar);
                                tma_load_3d_pair(to + kG16Half / 2, m, r0 + 64, k, z, lead_bar);
                            } else {
                                tma_load_3d(to, m, r0, k, z, bar);
                                tma_load_3d(to + kG16Half / 2, m, r0 + 64, k, z, bar);
                            }
                        }
                    }
                }
            }
            // copies in flight must have landed before shared memory goes away, also where whoever reads them has given up.  (Those of the other CTA count here too:
            // it does not leave before this one has been here.)
            if (leader)
                for (int c = max(0, filled - kStages); c < filled; ++c)
                    mbar_wait_asleep(&bars.full[c % kStages], (unsigned)(c / kStages) & 1u, status, ok ? kWaitTries : kDrainTries);
        }
    } else if (warp == 1) {
        if (leader) {
            // 16-bit operands of one type, FP32 sums, N >> 3, M >> 4
            const unsigned type = g.bf16 ? 1u : 0u;
            const unsigned idesc = (1u << 4) | (type << 7) | (type << 10) | (g.a_kmajor ? 0u : 1u << 15) | (g.b_kmajor ? 0u : 1u << 16) | ((unsigned)kTile >> 3 << 17) |
                                   ((unsigned)kTile >> 4 << 24);
            const uint64_t a_step = g.a_kmajor ? 2u : 128u, b_step = g.b_kmajor ? 2u : 128u;
            Ring r(kStages), rs(totals ? 1 : 2);
            for (int t = first; t < tiles && ok; t += step) {
                for (int n = 0, c0 = 0; n < chains && ok; ++n, c0 += chain, rs.next()) {
                    if (rs.wrapped) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.acc_empty[rs.pos], rs.par ^ 1u, status)) != 0;
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned acc = tmem + (unsigned)rs.pos * 256u;
                    const int c1 = n + 1 == chains ? stages : c0 + chain;
                    for (int d = c0; d < c1; ++d, r.next()) {
                        ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.full[r.pos], r.par, status)) != 0;
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const unsigned s = smem_u32(base) + (unsigned)r.pos * kG16Stage;
                        const uint64_t da = g.a_kmajor ? smem_desc_sw128(s) : g16_desc_mn(s), db = g.b_kmajor ? smem_desc_sw128(s + kG16Half) : g16_desc_mn(s + kG16Half);
                        if (elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < kG16K / 16; ++kk) g16_mma<CTAS>(acc, da + a_step * (uint64_t)kk, db + b_step * (uint64_t)kk, idesc, d > c0 || kk > 0);
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
        const int quarter = warp & 3, part = (warp - kG16First) >> 2;    // the lanes of tensor memory this warp may read, its half of the columns
        int which = 0;
        unsigned fetches = 0;
        Ring rs(totals ? 1 : 2);
        for (int t = first; t < tiles; t += step) {
            const TileAt at = tile_at(g, t);
            TileOut out = {at.z, at.i * kTile + half * 128 + quarter * 32, at.j * kTile + part * kCols, lane, 0, ok, boxes + (unsigned)(warp - kG16First) * 2 * kG16Box, &which,
                           &bars.fetched[warp - kG16First], &fetches, status};
            const bool mine = out.row < g.M && out.col < g.N;
            float sums[EPI::kChained ? kCols : 1];
            typename EPI::Ahead ahead;
            if constexpr (!EPI::kChained) {
                if (mine) epi.template ahead<kCols>(out, ahead);
            }
            const auto empty = [&] {
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                // (not where this warp has given up: it runs ahead from here on, and its arrivals would let accumulators be overwritten that others still read)
                if (ok && lane == 0) {
                    if (CTAS == 2) mbar_arrive_pair(smem_u32(&bars.acc_empty[rs.pos]) + lead);
                    else mbar_arrive(&bars.acc_empty[rs.pos]);
                }
            };
            if constexpr (EPI::kBack) {
                if (chains > 1) {
                    ok = sum_chains<kCols, CTAS>(&bars, rs, chains, tmem + (unsigned)(part * kCols) + ((unsigned)(quarter * 32) << 16), lead, mine, status, g.tries, ok);
                    for (int n = 1; n < chains; ++n) rs.next();
                }
            }
            for (int n = 0; n < chains; ++n, rs.next()) {
                if (ok && !(EPI::kBack && chains > 1)) ok = __all_sync(kFullMask, mbar_wait_asleep(&bars.acc_full[rs.pos], rs.par, status, g.tries)) != 0;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                out.taddr = tmem + (unsigned)rs.pos * 256u + (unsigned)(part * kCols) + ((unsigned)(quarter * 32) << 16);
                out.ok = ok;
                if constexpr (EPI::kChained) {
                    if (mine) {
#pragma unroll
                        for (int c = 0; c < kCols; c += 16) {
                            float v[16];                         // (32 at a time spill: 1264 -> 1634 us for 8192 x 4096 x 32000)
                            read16f(out.taddr + (unsigned)c, v, ok);
#pragma unroll
                            for (int j = 0; j < 16; ++j) sums[c + j] = n ? sums[c + j] + v[j] : v[j];
                        }
                    }
                } else if (totals && mine && ok) {
                    const unsigned total = out.taddr + 256u;
#pragma unroll 2
                    for (unsigned c = 0; c < (unsigned)kCols; c += 16) {
                        unsigned v[16];
                        read16(out.taddr + c, v, true);
                        if (n) add16(total + c, v);
                        tmem_st16(total + c, v);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                if (!EPI::kChained && !totals) break;
                empty();
            }
            if constexpr (EPI::kChained) {
                if (mine) epi.template tile<kCols>(out, sums);
            } else {
                if (totals) out.taddr += 256u;
                if (mine) epi.template tile<kCols>(out, ahead);
                if (!totals) {
                    empty();
                    rs.next();
                }
            }
        }
        if (lane == 0) bulk_wait_all();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CTAS == 2) pair_meet();                        // the leader's MMAs are done with this CTA's memory, the other's arrivals have landed
    if (warp == 1) tmem_free<CTAS>(tmem, 512u);
}

// ---- host ----
inline uint64_t padded(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }
// Scratch, handed out piece by piece on 128 bytes
struct Scratch {
    unsigned char *base;
    size_t used = 0;
    template <class T> T *take(uint64_t count) {
        T *p = reinterpret_cast<T *>(base + used);
        used += padded(count * sizeof(T), 128);
        return p;
    }
};
template <class EPI> constexpr size_t g16_smem() { return 1024 + g16_stages<EPI>() * kG16Stage + (EPI::kBoxes ? kG16Warps * 2 * kG16Box : 0) + sizeof(Gemm16Bars) + 64; }

// A stack of matrices of 16- or 32-bit elements in memory: `rows` rows of `cols` elements, `ld` apart, matrices `apart` elements apart
struct Stack {
    const void *at;
    uint64_t cols, rows, ld, batch, apart;
};
// A box of it as a tiled copy moves it
inline bool map_stack(CUtensorMap *map, const Stack &s, int type, unsigned box_cols, unsigned box_rows, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    const uint64_t size = (uint64_t)op_bytes(type), ld = s.rows > 1 ? s.ld : (s.cols * size + 15) / 16 * 16 / size, apart = s.batch > 1 ? s.apart : s.rows * ld;
    const cuuint64_t dims[3] = {s.cols, s.rows, s.batch}, strides[2] = {ld * size, apart * size};
    const cuuint32_t box[3] = {box_cols, box_rows, 1}, estr[3] = {1, 1, 1};
    const CUtensorMapDataType t = type == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode_tiled() && encode_tiled()(map, t, 3, const_cast<void *>(s.at), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// An operand: K-major stacks have K as their columns
inline bool map_operand(CUtensorMap *map, const Stack &s, bool bf16, bool kmajor) { return map_stack(map, s, bf16 ? kBf16 : kF16, kG16K, kmajor ? 128u : 64u); }

// Whether pairs of CTAs fill the device with tiles of 256 x 256
inline bool g16_pairs(uint64_t M, uint64_t N, uint64_t batch, bool lower, int sm_count) {
    const uint64_t i = (M + 255) / 256, j = (N + 255) / 256;
    return M > 128 && batch * (lower ? i * (i + 1) / 2 : i * j) * 2 >= (uint64_t)sm_count * 2 / 3;
}

template <class EPI, int CTAS>
cudaError_t launch_gemm16_ctas(const Gemm16Maps &maps, const EPI &epi, const Gemm16 &g, unsigned *status, int sm_count, cudaStream_t stream) {
    static_assert(g16_smem<EPI>() <= 227 * 1024, "stages do not fit");
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = allow_smem(gemm16_kernel<EPI, CTAS>, &done);
    if (err != cudaSuccess) return err;
    const long tiles = (long)g.batch * g.splits * (g.lower ? (long)g.m_tiles * (g.m_tiles + 1) / 2 : (long)g.m_tiles * g.n_tiles);
    if (tiles > 0x7fffffff / 2 || g.k_stages < 1) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)std::min<long>(tiles, sm_count / CTAS) * CTAS;
    if (CTAS == 2) return launch_cluster(gemm16_kernel<EPI, CTAS>, grid, kG16Threads, CTAS, g16_smem<EPI>(), stream, maps, epi, g, status);
    return launch_chained(gemm16_kernel<EPI, CTAS>, grid, kG16Threads, g16_smem<EPI>(), stream, maps, epi, g, status);
}
// M, N, batch, parts, splits and the flags of `g` are set; pairs: g16_pairs
template <class EPI>
cudaError_t launch_gemm16(const Gemm16Maps &maps, const EPI &epi, Gemm16 g, uint64_t K, bool pairs, unsigned *status, int sm_count, cudaStream_t stream) {
    const int tile = pairs ? 256 : 128;
    g.m_tiles = (g.M + tile - 1) / tile;
    g.n_tiles = (g.N + tile - 1) / tile;
    const int stages = (int)((K + kG16K - 1) / kG16K);
    g.k_stages = (stages + g.splits - 1) / g.splits;
    g.tries = epilogue_tries(kWaitTries);
    return pairs ? launch_gemm16_ctas<EPI, 2>(maps, epi, g, status, sm_count, stream) : launch_gemm16_ctas<EPI, 1>(maps, epi, g, status, sm_count, stream);
}

}  // namespace
}  // namespace bsq
