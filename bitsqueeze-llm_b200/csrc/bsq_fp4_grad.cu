// Gradient products of a linear layer whose weight and parked activations are held in 4 bits (sm_100a):
//   input    out[M x K] = dY[M x N] W[N x K]        weight   out[N x K] = dY[M x N]^T X[M x K]
// with dY in BF16 and W, X packed (bsq_fp4.hpp).  Both are out[R x C] = op(dY)[R x D] B[D x C], where B's blocks lie along C, not along the
// dimension D that is summed over, so the block-scaled instructions of bsq_fp4_gemm.cu do not apply: B is decoded to BF16.  A code
// times its block scale has 6 significant bits and BF16's exponent covers every MXFP4 scale (NVFP4: held 2^12 smaller), so decoding is exact;
// sums are FP32 in tensor memory, the matrix scale is multiplied in when a tile leaves, and the result is rounded once.  FP32 results are
// summed in two accumulators, one for each half of D: the tensor core cuts every addition off, which is what such a sum is off by.
//
// One CTA per SM walks over tiles of 128 x 256; per 64 of D warp 0 brings a box of dY (128-byte swizzle, in the orientation that memory
// has; the tensor core reads either) and the packed codes and scales of 64 rows of B (10 KB instead of 32), eight warps decode them into the
// swizzled operand (contiguous along C), warp 1 issues the MMAs, four warps take finished tiles out.  Decoding costs about as many issue
// slots as the MMAs take (64 x 256 elements at 3.4 instructions per 32 of them against 512 clocks), so it bounds the kernel together with them.
// Fewer tiles than SMs: clusters share a tile along D as in bsq_fp4_gemm.cu.
#include "bsq_fp4_tile.cuh"
#include "bsq_internal.hpp"

namespace bsq {
namespace {

constexpr int kGradThreads = 15 * 32;                            // warp 0: copies of B, 1: MMAs, 2-9: decode, 10-13: epilogue, 14: copies of dY
constexpr int kDecodeWarps = 8;
constexpr int kTileC = 256, kStageD = 64;
constexpr int kRing = 3, kRawRing = 6;
constexpr unsigned kABytes = 128 * kStageD * 2, kBBytes = kStageD * kTileC * 2, kOpBytes = kABytes + kBBytes;
constexpr unsigned kCodeBytes = kStageD * kTileC / 2, kRawBytes = kCodeBytes + 2048;
constexpr float kNvHold = 4096.0f;                               // NVFP4: decoded values are held 2^12 smaller

struct Fp4Grad {
    int R, C, D;                     // rows and columns of the result, the dimension that is summed over
    int r_tiles, c_tiles, d_stages, splits, stages_per_split;
    bool a_kmajor;                   // dY contiguous along D (input gradient) or along R (weight gradient)
    bool halves;                     // two accumulators per tile, instead of two tiles in turn
    unsigned quads;                  // scale tiles along a row of B
    const uint8_t *scales;
    const float *head;
    void *out;
    long ld;
    int type;
};

struct GradBars {
    uint64_t a_full[kRing], ready[kRing], empty[kRing], raw_full[kRawRing], raw_empty[kRawRing], acc_full[2], acc_empty[2], drain;
    unsigned tmem_base, failed;
};

// Operand contiguous along M / N in 128-byte-swizzled shared memory: groups of 64 elements (128 bytes) x 64 of K, 8192 bytes apart (leading
// byte offset); within one, groups of 8 of K 1024 bytes apart (stride byte offset).  A step of 16 along K is 2048 bytes of the start address.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(unsigned addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(8192u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

__device__ __forceinline__ unsigned mul_bf16x2(unsigned a, unsigned b) {
    unsigned r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// Eight codes to BF16, times a scale.  Sign and the three magnitude bits are moved to where BF16 has its sign, the last two bits of its exponent and
// the first of its mantissa: read as BF16 that is the element times 2^-126 (also for 0 and 0.5, which are subnormal in both), and multiplying brings it
// back.  Word i holds elements i and i + 4: columns of a group of 8 come out in the order 0 4 1 5 2 6 3 7, which the epilogue undoes for nothing.
template <int FMT> __device__ __forceinline__ uint4 decode8(unsigned x, unsigned scale2) {
    unsigned w[4];
    w[0] = ((x << 12) & 0x80008000u) | ((x << 6) & 0x01C001C0u);
    w[1] = ((x << 8) & 0x80008000u) | ((x << 2) & 0x01C001C0u);
    w[2] = ((x << 4) & 0x80008000u) | ((x >> 2) & 0x01C001C0u);
    w[3] = (x & 0x80008000u) | ((x >> 6) & 0x01C001C0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (FMT == kMxFp4) w[i] = mul_bf16x2(w[i], 0x7E807E80u);  // 2^126: the element itself, exact; the scale's range needs a product of its own
        w[i] = mul_bf16x2(w[i], scale2);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// The factor of decode8 from a scale byte, in both halves of a word
template <int FMT> __device__ __forceinline__ unsigned decode_scale(unsigned byte) {
    unsigned h;
    if (FMT == kMxFp4) {
        h = byte == 0 ? 0x0040u : byte == 255 ? 0x7FFFu : byte << 7;
    } else {
        byte &= 0x7fu;                                           // s * 2^(126 - 12), exact in BF16
        h = byte == 0x7fu ? 0x7FFFu : __float_as_uint(e4m3_decode(byte) * 2.076918743413931e34f) >> 16;
    }
    return h | (h << 16);
}

template <int FMT, bool SPLIT>
__global__ void __launch_bounds__(kGradThreads, 1) fp4_grad_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                   const Fp4Grad g, unsigned *status) {
    chain_begin();
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *base = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
    unsigned char *raw = base + kRing * kOpBytes;
    GradBars &bars = *reinterpret_cast<GradBars *>(raw + kRawRing * kRawBytes);
    constexpr int kQuads = FMT == kNvFp4 ? 4 : 2;                // scale tiles across a tile's 256 columns
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = SPLIT ? (int)(blockIdx.x % (unsigned)g.splits) : 0;
    const int tiles = g.r_tiles * g.c_tiles;
    const int first = SPLIT ? (int)(blockIdx.x / (unsigned)g.splits) : (int)blockIdx.x, step = SPLIT ? tiles : (int)gridDim.x;
    const int d0 = rank * g.stages_per_split, d1 = min(g.d_stages, d0 + g.stages_per_split);
    const int sets = g.halves ? 1 : 2, d_half = g.halves ? d0 + (d1 - d0 + 1) / 2 : d1;

    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(&bars.a_full[i], 1);
            mbar_init(&bars.ready[i], kDecodeWarps);
            mbar_init(&bars.empty[i], 1);
        }
        for (int i = 0; i < kRawRing; ++i) {
            mbar_init(&bars.raw_full[i], 1);
            mbar_init(&bars.raw_empty[i], kDecodeWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars.acc_full[i], 1);
            mbar_init(&bars.acc_empty[i], 4);
        }
        mbar_init(&bars.drain, 1);
        bars.failed = 0;
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars.tmem_base;
    bool ok = true;

    if (warp == 0) {
        // ---- codes and scales, up to kRawRing stages ahead ----
        if (lane == 0) {
            Ring r(kRawRing);
            int filled = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const unsigned quad = (unsigned)(t / g.r_tiles) * kQuads, sf = min((unsigned)kQuads, g.quads - quad) * 512u;
                for (int d = d0; d < d1; ++d, ++filled, r.next()) {
                    if (r.wrapped) ok = mbar_wait_bounded(&bars.raw_empty[r.pos], r.par ^ 1u, status);
                    if (!ok) break;
                    unsigned char *s = raw + (size_t)r.pos * kRawBytes;
                    mbar_expect_tx(&bars.raw_full[r.pos], kCodeBytes + sf);
                    tma_load_2d(s, &map_b, (t / g.r_tiles) * (kTileC / 2), d * kStageD, &bars.raw_full[r.pos]);
                    bulk_g2s(s + kCodeBytes, g.scales + ((size_t)(d >> 1) * g.quads + quad) * 512, sf, &bars.raw_full[r.pos]);
                }
            }
            if (!ok) {                                           // copies in flight must have landed before this CTA's shared memory goes away
                atomicOr(&bars.failed, 1u);
                for (int c = max(0, filled - kRawRing); c < filled; ++c) mbar_wait_bounded(&bars.raw_full[c % kRawRing], (unsigned)(c / kRawRing) & 1u, status);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // BF16 x BF16, FP32 sums, B contiguous along N, A along K or along M, N >> 3, M >> 4
            const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | (g.a_kmajor ? 0u : 1u << 15) | (1u << 16) | ((unsigned)(kTileC >> 3) << 17) | ((128u >> 4) << 24);
            Ring r(kRing), rs(sets);
            for (int t = first; t < tiles && ok; t += step, rs.next()) {
                if (rs.wrapped) ok = mbar_wait_bounded(&bars.acc_empty[rs.pos], rs.par ^ 1u, status);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (int d = d0; d < d1; ++d, r.next()) {
                    ok = mbar_wait_bounded(&bars.a_full[r.pos], r.par, status) && mbar_wait_bounded(&bars.ready[r.pos], r.par, status);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const unsigned s = smem_u32(base + (size_t)r.pos * kOpBytes);
                    const uint64_t da = g.a_kmajor ? smem_desc_sw128(s) : smem_desc_mn_sw128(s), db = smem_desc_mn_sw128(s + kABytes);
                    const uint64_t a_step = g.a_kmajor ? 2u : 128u;
                    const unsigned acc = tmem + (g.halves ? (d >= d_half ? 256u : 0u) : (unsigned)rs.pos * 256u);
                    const bool fresh = d == d0 || (g.halves && d == d_half);
#pragma unroll
                    for (int kk = 0; kk < kStageD / 16; ++kk)
                        mma_f16(acc, da + a_step * (uint64_t)kk, db + (uint64_t)(kk * 128), idesc, !fresh || kk > 0);
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
    } else if (warp == 14) {
        if (lane == 0) {
            Ring r(kRing);
            int filled = 0;
            for (int t = first; t < tiles && ok; t += step) {
                const int row = (t % g.r_tiles) * 128;
                for (int d = d0; d < d1; ++d, ++filled, r.next()) {
                    if (r.wrapped) ok = mbar_wait_bounded(&bars.empty[r.pos], r.par ^ 1u, status);
                    if (!ok) break;
                    unsigned char *s = base + (size_t)r.pos * kOpBytes;
                    mbar_expect_tx(&bars.a_full[r.pos], kABytes);
                    if (g.a_kmajor) {
                        tma_load_2d(s, &map_a, d * kStageD, row, &bars.a_full[r.pos]);
                    } else {
                        tma_load_2d(s, &map_a, row, d * kStageD, &bars.a_full[r.pos]);
                        tma_load_2d(s + kABytes / 2, &map_a, row + 64, d * kStageD, &bars.a_full[r.pos]);
                    }
                }
            }
            if (!ok) {
                atomicOr(&bars.failed, 1u);
                for (int c = max(0, filled - kRing); c < filled; ++c) mbar_wait_bounded(&bars.a_full[c % kRing], (unsigned)(c / kRing) & 1u, status);
            }
        }
    } else if (warp < 2 + kDecodeWarps) {
        // ---- decode: a thread has one row of B and, twice, 32 of its columns; the lanes of a warp have rows beside one another, so that neither the
        // swizzled codes nor the swizzled operand see a bank conflict ----
        const int w = warp - 2, d_in = (w & 1) * 32 + lane;
        Ring r(kRing), rr(kRawRing);
        for (int t = first; t < tiles && ok; t += step) {
            for (int d = d0; d < d1; ++d, r.next(), rr.next()) {
                ok = mbar_wait_bounded(&bars.raw_full[rr.pos], rr.par, status);
                if (ok && r.wrapped) ok = mbar_wait_bounded(&bars.empty[r.pos], r.par ^ 1u, status);
                ok = __all_sync(kFullMask, ok) != 0;
                if (!ok) break;
                const unsigned char *s = raw + (size_t)rr.pos * kRawBytes;
                unsigned char *b = base + (size_t)r.pos * kOpBytes + kABytes + d_in * 128;
                const int row = (d & 1) * 64 + d_in;             // in its scale tile
                const unsigned char *sf = s + kCodeBytes + (row & 31) * 16 + (row >> 5) * 4;
                const bool live = d * kStageD + d_in < g.D;      // (scales behind the last row are anything)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int unit = (w >> 1) + 4 * j;
                    const uint4 c = *reinterpret_cast<const uint4 *>(s + d_in * 128 + ((unit ^ (d_in & 7)) << 4));
                    unsigned s0, s1;
                    if (FMT == kMxFp4) {
                        s0 = s1 = decode_scale<FMT>(live ? sf[(unit >> 2) * 512 + (unit & 3)] : 0u);
                    } else {
                        const unsigned two = live ? *reinterpret_cast<const unsigned short *>(sf + (unit >> 1) * 512 + (unit & 1) * 2) : 0u;
                        s0 = decode_scale<FMT>(two & 0xffu);
                        s1 = decode_scale<FMT>(two >> 8);
                    }
                    unsigned char *dst = b + (unit >> 1) * 8192;
                    const int chunk = (unit & 1) * 4, x = d_in & 7;
                    *reinterpret_cast<uint4 *>(dst + (((chunk + 0) ^ x) << 4)) = decode8<FMT>(c.x, s0);
                    *reinterpret_cast<uint4 *>(dst + (((chunk + 1) ^ x) << 4)) = decode8<FMT>(c.y, s0);
                    *reinterpret_cast<uint4 *>(dst + (((chunk + 2) ^ x) << 4)) = decode8<FMT>(c.z, s1);
                    *reinterpret_cast<uint4 *>(dst + (((chunk + 3) ^ x) << 4)) = decode8<FMT>(c.w, s1);
                }
                fence_proxy_async_smem();                        // stores before the tensor core's reads, reads before the next copy's writes
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bars.ready[r.pos]);
                    mbar_arrive(&bars.raw_empty[rr.pos]);
                }
            }
        }
        if (!ok && lane == 0) atomicOr(&bars.failed, 1u);
    } else {
        const int quarter = warp & 3;                            // the lanes of tensor memory this warp may read
        const float f0 = *g.head, f1 = FMT == kNvFp4 ? kNvHold : 1.0f;
        const int size = g.type == kF32 ? 4 : 2;
        const bool wide = (reinterpret_cast<uintptr_t>(g.out) | (uintptr_t)(g.ld * size)) % 32 == 0;
        Ring rs(sets);
        for (int t = first; t < tiles; t += step, rs.next()) {
            const int row = (t % g.r_tiles) * 128 + quarter * 32 + lane, col = (t / g.r_tiles) * kTileC;
            if (ok) ok = __all_sync(kFullMask, mbar_wait_bounded(&bars.acc_full[rs.pos], rs.par, status)) != 0;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const unsigned taddr = tmem + (unsigned)rs.pos * 256u + ((unsigned)(quarter * 32) << 16);
            for (int c = 0; c < kTileC; c += 16) {
                unsigned p[16], r[16];
                read16(taddr + (unsigned)c, p, ok);
                if (g.halves && d_half < d1) {
                    unsigned q[16];
                    read16(taddr + 256u + (unsigned)c, q, ok);
#pragma unroll
                    for (int j = 0; j < 16; ++j) p[j] = __float_as_uint(__uint_as_float(p[j]) + __uint_as_float(q[j]));
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = p[(j & 8) | ((j & 3) << 1) | ((j & 4) >> 2)];        // decode8's order of columns
                if constexpr (SPLIT) {
                    // operand stages are free: every copy has landed and every MMA has read them
                    float *part = reinterpret_cast<float *>(base) + (quarter * 32 + lane) * (kTileC + 4) + c;
#pragma unroll
                    for (int j = 0; j < 16; j += 4) *reinterpret_cast<uint4 *>(part + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
                } else {
                    if (row < g.R && col + c < g.C) store_run16(g.out, g.type, (long)row * g.ld + col + c, r, f0, f1, min(16, g.C - col - c), wide);
                    __syncwarp();
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.acc_empty[rs.pos]);
        }
        if (!ok && lane == 0) atomicOr(&bars.failed, 1u);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");

    if constexpr (SPLIT) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int rt = first % g.r_tiles, ct = first / g.r_tiles;
        const auto read = [&](int i, int c) { return *cluster.map_shared_rank(reinterpret_cast<const float *>(base) + i, c); };
        add_parts<kGradThreads>(read, rank, kTileC + 4, min(128, g.R - rt * 128), min(kTileC, g.C - ct * kTileC), g.splits, *g.head, FMT == kNvFp4 ? kNvHold : 1.0f, g.out,
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

template <int FMT, bool SPLIT>
cudaError_t launch_grad(const CUtensorMap &map_a, const CUtensorMap &map_b, const Fp4Grad &g, int sm_count, unsigned *status, cudaStream_t stream) {
    constexpr size_t smem = 1024 + kRing * kOpBytes + kRawRing * kRawBytes + sizeof(GradBars) + 64;
    static_assert(smem <= 227 * 1024, "stages do not fit");
    static_assert((size_t)128 * (kTileC + 4) * 4 <= (size_t)kRing * kOpBytes, "partial tile does not fit");
    cudaError_t err = cudaFuncSetAttribute(fp4_grad_kernel<FMT, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return err;
    const int tiles = g.r_tiles * g.c_tiles;
    if (SPLIT) return launch_cluster(fp4_grad_kernel<FMT, SPLIT>, (unsigned)(tiles * g.splits), kGradThreads, g.splits, smem, stream, map_a, map_b, g, status);
    return launch_chained(fp4_grad_kernel<FMT, SPLIT>, (unsigned)(tiles < sm_count ? tiles : sm_count), kGradThreads, smem, stream, map_a, map_b, g, status);
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
    Fp4Grad g = {};
    g.R = (int)R; g.C = (int)C; g.D = (int)D;
    const uint64_t r_tiles = (R + 127) / 128, c_tiles = (C + kTileC - 1) / kTileC;
    if (r_tiles * c_tiles > 0x7fffffffull / 8) return cudaErrorInvalidValue;
    g.r_tiles = (int)r_tiles; g.c_tiles = (int)c_tiles;
    g.d_stages = (int)((D + kStageD - 1) / kStageD);
    g.a_kmajor = a_kmajor;
    g.halves = type == kF32;
    g.quads = (unsigned)fp4_quads(format, C);
    g.scales = b + fp4_scales_at(D, C);
    g.head = reinterpret_cast<const float *>(b);
    g.out = out; g.ld = (long)ld; g.type = type;
    const int tiles = g.r_tiles * g.c_tiles;
    g.splits = 1;
    while (g.splits < 8 && tiles * g.splits * 2 <= sm_count && g.d_stages >= g.splits * 4) g.splits *= 2;
    g.stages_per_split = (g.d_stages + g.splits - 1) / g.splits;
    g.splits = (g.d_stages + g.stages_per_split - 1) / g.stages_per_split;               // no slice is empty
    CUtensorMap map_a, map_b;
    const cuuint64_t dims_a[2] = {N, M}, strides_a[1] = {ld_a * 2}, dims_b[2] = {fp4_ld(C), D}, strides_b[1] = {fp4_ld(C)};
    const cuuint32_t box_a[2] = {64u, a_kmajor ? 128u : 64u}, box_b[2] = {kTileC / 2, kStageD}, estr[2] = {1, 1};
    if (!encode_tiled() ||
        encode_tiled()(&map_a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(dy), dims_a, strides_a, box_a, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
        encode_tiled()(&map_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(b) + kFp4Head, dims_b, strides_b, box_b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    if (format == kNvFp4)
        return g.splits > 1 ? launch_grad<kNvFp4, true>(map_a, map_b, g, sm_count, status, stream) : launch_grad<kNvFp4, false>(map_a, map_b, g, sm_count, status, stream);
    return g.splits > 1 ? launch_grad<kMxFp4, true>(map_a, map_b, g, sm_count, status, stream) : launch_grad<kMxFp4, false>(map_a, map_b, g, sm_count, status, stream);
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
