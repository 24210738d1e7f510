// Gradient of the input for up to 16 rows of dY (a few tokens): out[R x C] = dY[R x D] W[D x C], W packed (bsq_fp4.hpp).
//
// W is read once and bounds it: 0.53 bytes an element from memory, and 3 instructions an element to decode it.  On the path of bsq_fp4_grad.cu every
// decoded element goes through shared memory and three barriers to a tensor core that has next to nothing to do; here it is decoded in the register
// that mma.sync takes it from.  A warp has 128 columns and 32 rows of W at a time; thread (g, t) of it has the 16 columns 16 g.. and the 8 rows 8 t.. .
// The sum may take rows in any order, so the k of an MMA are dealt to fit: B wants pairs of k in a register, and the codes of rows 2 p and
// 2 p + 1, their 16-bit halves put side by side, are decoded to just such pairs by decode8, column after column; A's pairs are neighbours in dY, so that
// eight rows of W make one 16-byte load of dY.  Column i of every thread's 16 is one MMA's n, so a thread ends up with 32 neighbouring
// columns of the result.
//
// Codes and scales come by cp.async, three chunks of 32 rows ahead for each warp on its own (no barrier in the loop).  The warps of a CTA and
// the CTAs of a cluster share the rows; their sums are added in a fixed order.
//
// 16 x 4096 x 14336 MXFP4 18.5 us, one row in NVFP4 16.8 (33 MB, 5 us at the memory's rate): some 5 us are launch, cluster and sums, the loads alone take 5,
// decoding and MMAs 7 to 8 (12 instructions for 4 elements, at 0.6 of the issue rate).
#include "bsq_fp4_decode.cuh"
#include "bsq_fp4_few.hpp"
#include "bsq_fp4_tile.cuh"

#include <algorithm>

namespace bsq {
namespace {

constexpr int kFewStages = 4, kFewCols = 128, kFewRows = 32;
constexpr int kFewChain = 1024 / kFewRows;                       // longest chain of additions in a warp's accumulators where it has more than the result's type hides, in chunks
constexpr unsigned kFewCodes = kFewRows * kFewCols / 2, kFewStage = kFewCodes + 256;

struct Fp4Few {
    int R, C, D, chunks, splits, chunks_per_split;
    const uint8_t *codes, *scales;
    uint64_t ld_codes, quads;
    const float *head;
    const __nv_bfloat16 *dy;
    uint64_t ld_dy;
    void *out;
    long ld;
    int type;
};

// 16 or 4 bytes into shared memory in the background; zeros where `live` is false
__device__ __forceinline__ void copy16(unsigned dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void *src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}

__device__ __forceinline__ void mma_16816(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight neighbouring elements of a row of dY from column d on; zeros behind the last one
__device__ __forceinline__ uint4 load_dy(const __nv_bfloat16 *row, int d, int D, bool live) {
    if (!live || d >= D) return make_uint4(0u, 0u, 0u, 0u);
    if (d + 8 <= D) return *reinterpret_cast<const uint4 *>(row + d);
    unsigned w[4] = {0u, 0u, 0u, 0u};
    const unsigned short *p = reinterpret_cast<const unsigned short *>(row + d);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (d + i < D) w[i >> 1] |= (unsigned)p[i] << (16 * (i & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 32 rows x this thread's 16 columns: decoded and multiplied.  ONE: see decode8.
template <int FMT, bool ONE> __device__ __forceinline__ void few_chunk(const unsigned char *s, int gq, int t, const uint4 &d0, const uint4 &d1, float (&acc)[16][4]) {
#pragma unroll
    for (int step = 0; step < 2; ++step) {
        const unsigned a[4] = {step ? d0.z : d0.x, step ? d1.z : d1.x, step ? d0.w : d0.y, step ? d1.w : d1.y};
        unsigned w[2][2][2], scale[2];                           // [pair][row of the pair][8 columns]
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            unsigned byte[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int place = (step * 4 + p * 2 + e) * 4 + t;
                const uint2 c = *reinterpret_cast<const uint2 *>(s + place * 64 + gq * 8);
                w[p][e][0] = c.x;
                w[p][e][1] = c.y;
                byte[e] = FMT == kNvFp4 ? s[kFewCodes + (place * 2 + (gq >> 2)) * 4 + (gq & 3)] : s[kFewCodes + place * 4 + (gq >> 1)];
            }
            scale[p] = ONE ? decode_scales_one(byte[0], byte[1]) : decode_scales<FMT>(byte[0], byte[1]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {                            // four columns of the 16
            const unsigned sel = q & 1 ? 0x7632u : 0x5410u;
            const uint4 b0 = decode8<FMT, ONE>(__byte_perm(w[0][0][q >> 1], w[0][1][q >> 1], sel), scale[0]);
            const uint4 b1 = decode8<FMT, ONE>(__byte_perm(w[1][0][q >> 1], w[1][1][q >> 1], sel), scale[1]);
            mma_16816(acc[q * 4 + 0], a, b0.x, b1.x);
            mma_16816(acc[q * 4 + 1], a, b0.y, b1.y);
            mma_16816(acc[q * 4 + 2], a, b0.z, b1.z);
            mma_16816(acc[q * 4 + 3], a, b0.w, b1.w);
        }
    }
}

// LONG: every kFewChain chunks the CTA's warps add what they have come to, one behind the other, to a tile in shared memory.  These MMAs cut additions off as well:
// FP32 16 x 14336 from 65536 rows 0.8e-6 off 64 bits in one chain a warp, 0.2e-6 this way; 205 us, 195 without.  (The sums of chains in registers, 8 warps a SM: 249.)
template <int FMT, int WARPS, bool LONG> __global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) fp4_grad_few_kernel(const Fp4Few g) {
    chain_begin();
    extern __shared__ __align__(16) unsigned char smem_few[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, t = lane & 3;
    const int rank = (int)(blockIdx.x % (unsigned)g.splits), col0 = (int)(blockIdx.x / (unsigned)g.splits) * kFewCols;
    const int c_end = min(g.chunks, (rank + 1) * g.chunks_per_split);
    constexpr int kQuads = FMT == kNvFp4 ? 2 : 1;
    unsigned char *mine = smem_few + (unsigned)warp * kFewStages * kFewStage;
    const unsigned mine_u = smem_u32(mine);

    const int first = rank * g.chunks_per_split + warp;
    // What this lane copies of a chunk: 16 bytes of rows lane / 4, + 8, + 16, + 24, and the scales of row `lane`.  Row r lies at place (r & 7) * 4 + (r >> 3): the four
    // threads t that read rows 8 t + j at once read neighbouring places.
    const int quad0 = col0 / (FMT == kNvFp4 ? 64 : 128);
    const bool col_live = (uint64_t)(col0 / 2) + (uint64_t)(lane & 3) * 16 < g.ld_codes;
    const uint8_t *code_at = g.codes + ((uint64_t)first * kFewRows + (lane >> 2)) * g.ld_codes + col0 / 2 + (lane & 3) * 16;
    const uint64_t row8 = 8 * g.ld_codes, code_step = (uint64_t)WARPS * kFewRows * g.ld_codes;
    const unsigned code_to = mine_u + (unsigned)(lane >> 2) * 256u + (unsigned)(lane & 3) * 16u;
    const unsigned scale_to = mine_u + kFewCodes + (unsigned)(((lane & 7) * 4 + (lane >> 3)) * kQuads * 4);
    int ahead = first;                                           // the next chunk to be copied
    const auto fetch = [&](int stage) {
        if (ahead < c_end) {
            const int row0 = ahead * kFewRows;
            const unsigned off = (unsigned)stage * kFewStage;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool live = col_live && row0 + (lane >> 2) + 8 * i < g.D;
                copy16(code_to + off + (unsigned)i * 64u, live ? code_at + i * row8 : g.codes, live);
            }
            const uint8_t *scale_at = g.scales + ((uint64_t)(ahead >> 2) * g.quads + (uint64_t)quad0) * 512 + (unsigned)lane * 16u + (unsigned)(ahead & 3) * 4u;
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                const bool live = row0 + lane < g.D && (uint64_t)(quad0 + q) < g.quads;
                copy4(scale_to + off + (unsigned)q * 4u, live ? scale_at + q * 512 : g.scales, live);
            }
            code_at += code_step;
            ahead += WARPS;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const __nv_bfloat16 *a0 = g.dy + (uint64_t)gq * g.ld_dy, *a1 = g.dy + (uint64_t)(gq + 8) * g.ld_dy;
    const bool live0 = gq < g.R, live1 = gq + 8 < g.R;
    float acc[16][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
#pragma unroll
    for (int s = 0; s < kFewStages - 1; ++s) fetch(s);
    uint4 n0 = load_dy(a0, first * kFewRows + 8 * t, first < c_end ? g.D : 0, live0), n1 = load_dy(a1, first * kFewRows + 8 * t, first < c_end ? g.D : 0, live1);
    constexpr int kWide = 144, kLd = kFewCols + 4, kEach = 16 * kFewCols / 4 / (WARPS * 32);
    float *part = reinterpret_cast<float *>(smem_few), *my = part + warp * 16 * kWide + 36 * t, *total = part + WARPS * 16 * kWide;
    if (LONG)
        for (int i = (int)threadIdx.x; i < 16 * kWide; i += WARPS * 32) total[i] = 0.0f;
    int stage = 0, left = kFewChain;
    // (LONG: all warps of the CTA go round as often)
    for (int chunk = first; (LONG ? chunk - warp : chunk) < c_end; chunk += WARPS) {
        if (LONG && left-- == 0) {
            left = kFewChain - 1;
#pragma unroll 1
            for (int w = 0; w < WARPS; ++w) {
                __syncthreads();
                if (w == warp) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            float4 *to = reinterpret_cast<float4 *>(total + 36 * t + (gq + 8 * (h >> 1)) * kWide + 16 * (h & 1) + i);
                            const float4 o = *to;
                            *to = make_float4(o.x + acc[i][h], o.y + acc[i + 1][h], o.z + acc[i + 2][h], o.w + acc[i + 3][h]);
                            acc[i][h] = acc[i + 1][h] = acc[i + 2][h] = acc[i + 3][h] = 0.0f;
                        }
                }
            }
        }
        if (LONG && chunk >= c_end) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(kFewStages - 2) : "memory");
        __syncwarp();                                            // everybody's copies of this stage are there, and everybody is done with the one before
        fetch((stage + kFewStages - 1) % kFewStages);
        const uint4 d0 = n0, d1 = n1;
        const int next = chunk + WARPS;
        n0 = load_dy(a0, next * kFewRows + 8 * t, next < c_end ? g.D : 0, live0);
        n1 = load_dy(a1, next * kFewRows + 8 * t, next < c_end ? g.D : 0, live1);
        const unsigned char *s = mine + (unsigned)stage * kFewStage;
        if (FMT == kMxFp4) {
            // the words that hold this warp's 128 scale bytes, a lane one of them: none above 128?
            const unsigned four = *reinterpret_cast<const unsigned *>(s + kFewCodes + lane * 4);
            const bool small = __vmaxu4(four, 0x80808080u) == 0x80808080u;
            if (__all_sync(kFullMask, small)) few_chunk<FMT, true>(s, gq, t, d0, d1, acc);
            else few_chunk<FMT, false>(s, gq, t, d0, d1, acc);
        } else {
            few_chunk<FMT, false>(s, gq, t, d0, d1, acc);
        }
        stage = (stage + 1) % kFewStages;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // the warps' sums, 16 rows x 128 columns each, in rows of 144 floats (32 columns of a thread 36 apart: no bank conflicts), added up into rows of 132
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<float4 *>(my + gq * kWide + 16 * h + i) = make_float4(acc[i][h], acc[i + 1][h], acc[i + 2][h], acc[i + 3][h]);
            *reinterpret_cast<float4 *>(my + (gq + 8) * kWide + 16 * h + i) = make_float4(acc[i][2 + h], acc[i + 1][2 + h], acc[i + 2][2 + h], acc[i + 3][2 + h]);
        }
    }
    __syncthreads();
    float4 v[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = (int)threadIdx.x + j * WARPS * 32, row = i / 32, col = (i % 32) * 4;
        const float4 *p = reinterpret_cast<const float4 *>(part + row * kWide + col / 32 * 36 + col % 32);
        v[j] = *p;
#pragma unroll
        for (int w = 1; w < WARPS; ++w) {
            const float4 o = p[w * 16 * kWide / 4];
            v[j] = make_float4(v[j].x + o.x, v[j].y + o.y, v[j].z + o.z, v[j].w + o.w);
        }
        if (LONG) {
            const float4 o = p[WARPS * 16 * kWide / 4];
            v[j] = make_float4(v[j].x + o.x, v[j].y + o.y, v[j].z + o.z, v[j].w + o.w);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int i = (int)threadIdx.x + j * WARPS * 32;
        *reinterpret_cast<float4 *>(part + i / 32 * kLd + (i % 32) * 4) = v[j];
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const auto read = [&](int i, int c) { return *reinterpret_cast<const float4 *>(cluster.map_shared_rank(reinterpret_cast<const float *>(smem_few) + i, c)); };
    add_parts<WARPS * 32>(read, rank, kLd, g.R, min(kFewCols, g.C - col0), g.splits, *g.head, FMT == kNvFp4 ? kNvHold : 1.0f, g.out, g.type, col0, g.ld);
    cluster.sync();                                              // nobody leaves while its shared memory is being read
}

template <int FMT, int WARPS, bool LONG> cudaError_t launch_few(const Fp4Few &g, int blocks, cudaStream_t stream) {
    constexpr size_t stages = (size_t)WARPS * kFewStages * kFewStage, sums = (size_t)WARPS * 16 * 144 * 4, smem = (stages > sums ? stages : sums) + (LONG ? 16 * 144 * 4 : 0);
    static_assert(!LONG || sums >= stages, "the tile of sums lies behind the warps' own");
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = allow_smem(fp4_grad_few_kernel<FMT, WARPS, LONG>, &done);
    if (err != cudaSuccess) return err;
    return launch_cluster(fp4_grad_few_kernel<FMT, WARPS, LONG>, (unsigned)(blocks * g.splits), WARPS * 32, g.splits, smem, stream, g);
}

template <int FMT, int WARPS> cudaError_t launch_warps(bool longer, const Fp4Few &g, int blocks, cudaStream_t stream) {
    return longer ? launch_few<FMT, WARPS, true>(g, blocks, stream) : launch_few<FMT, WARPS, false>(g, blocks, stream);
}

}  // namespace

cudaError_t fp4_grad_few(int format, const void *dy, int R, uint64_t ld_dy, const uint8_t *packed, uint64_t D, uint64_t C, void *out, int type, uint64_t ld,
                         int sm_count, cudaStream_t stream) {
    Fp4Few g;
    g.R = R; g.C = (int)C; g.D = (int)D;
    g.chunks = (int)((D + kFewRows - 1) / kFewRows);
    const int blocks = (int)((C + kFewCols - 1) / kFewCols);
    if (blocks > 0x7fffffff / 8) return cudaErrorInvalidValue;
    // 16 warps a SM, in CTAs of 4 or 8: whichever leaves fewer of them without work, a cluster having at most 8 CTAs and a warp two chunks at least
    const auto splits = [&](int warps) {
        const int most = sm_count * (16 / warps) / blocks, useful = g.chunks / (2 * warps);
        return std::max(1, std::min(8, std::min(most, useful)));
    };
    const int warps = splits(4) * 4 > splits(8) * 8 ? 4 : 8;
    g.splits = splits(warps);
    g.chunks_per_split = (g.chunks + g.splits - 1) / g.splits;
    g.splits = (g.chunks + g.chunks_per_split - 1) / g.chunks_per_split;
    g.codes = packed + kFp4Head;
    g.scales = packed + fp4_scales_at(D, C);
    g.ld_codes = fp4_ld(C);
    g.quads = fp4_quads(format, C);
    g.head = reinterpret_cast<const float *>(packed);
    g.dy = static_cast<const __nv_bfloat16 *>(dy);
    g.ld_dy = ld_dy;
    g.out = out; g.ld = (long)ld; g.type = type;
    // a warp would sum more than 1024 terms of an FP32 result, 65536 of an FP16 one, 524288 of a BF16 one (as in bsq_fp4_grad.cu)
    const bool longer = g.chunks_per_split > (type == kF32 ? 1 : type == kF16 ? 64 : 512) * kFewChain * warps;
    if (format == kNvFp4) return warps == 4 ? launch_warps<kNvFp4, 4>(longer, g, blocks, stream) : launch_warps<kNvFp4, 8>(longer, g, blocks, stream);
    return warps == 4 ? launch_warps<kMxFp4, 4>(longer, g, blocks, stream) : launch_warps<kMxFp4, 8>(longer, g, blocks, stream);
}

}  // namespace bsq
