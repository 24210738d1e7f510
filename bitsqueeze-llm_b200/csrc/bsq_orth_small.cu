// Newton-Schulz steps of matrices with a short side of up to 128, results in BF16 (bsq_orth.hpp).
//
// All the steps are one polynomial in A_0 = X_0 X_0^T:  X_n = Q X_0 with Q_(k+1) = M_k Q_k, A_(k+1) = M_k A_k M_k, M_k = a I + b A_k + c A_k^2.  So the long side is walked
// twice, for A_0 and for Q X_0, and what lies between is products of matrices of 128 x 128 at most, which one CTA does for each matrix without leaving its SM.  (Step by step, with X in memory,
// 24 matrices of 64 x 1024 took 230 us; this way all five take 70.)
//
// Rounding grows with what it meets: an error of A_0 by (a^2)^(n - 1), 2 10^4 for five steps, and where X has one direction Q has 485 for all others and 0.7 there.  So A_0's sums are FP32 in chains of
// at most 256, products are of split operands (22 bits), and the identity's shares stay out of them: M = a I + N, Q = q I + R,  R <- N R + a R + q N,  T = N A + a A,  A <- N T + a T.  (In the products
// a and q are terms of 3.4 and 485 beside others of 1 / s, which the tensor core aligns with them and cuts off: rank one was 2.4e-3 to 3.1e-3 off and up to 2.1e-2 where elements take few values, all
// rounded alike.)  Results are within 4e-4 of those of 64 bits but for their rounding to BF16, 1.7e-3 (where elements take few values one that lies next to the middle of two BF16 numbers may go the
// other way: up to 3.1e-3 in all).  FP32 and FP16 results, and long sides, are bsq_orth.cu's.
//
// Launches: norm (bsq_orth.cu), A_0 in slices of the long side on the FP32 pipes, their sum where there are many, the steps on the tensor core, Q X_0 on the FP32 pipes.
#include "bsq_gemm16.cuh"
#include "bsq_orth_small.hpp"

#include <algorithm>
#include <atomic>

namespace bsq {
namespace {

constexpr int kThreads = 256, kStepThreads = 512;
constexpr int kSliceK = 32;                                      // of the long side at a time
constexpr int kFewSlices = 12;                                   // up to this many are added up by the CTA of the steps

// Elements of a matrix as X has them: the short side is `i`, the long one `k`
template <int TYPE, bool TALL> __device__ __forceinline__ float element(const OrthSmall &g, int z, int i, int k) {
    const size_t at = TALL ? (size_t)k * g.ld[z] + (size_t)i : (size_t)i * g.ld[z] + (size_t)k;
    const unsigned w = TYPE == kF32 ? static_cast<const unsigned *>(g.in[z])[at] : (unsigned)static_cast<const unsigned short *>(g.in[z])[at];
    return word_elem<TYPE>(w, 0);
}
// The sum of squares of a matrix, by each warp for itself
__device__ __forceinline__ double squares_of(const OrthSmall &g, int z) {
    double s = 0.0;
#pragma unroll 4
    for (int i = (int)threadIdx.x & 31; i < g.part_count; i += 32) s += g.parts[(size_t)z * (size_t)g.part_count + (size_t)i];
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(kFullMask, s, d);
    return s;
}
// 2^e that brings the norm, the square root of `squares`, below 2^15, in two factors; e
__device__ __forceinline__ int norm_scale(double squares, float *s0, float *s1) {
    const int of = (int)(((unsigned)__double2hiint(squares) >> 20) & 0x7ffu) - 1023;       // (zero, Inf and NaN: outside of what a sum of FP32's squares has)
    const int e = of < -320 || of > 320 ? 0 : min(max(14 - (of >> 1), -160), 160);
    *s0 = exp2f((float)(e >> 1));
    *s1 = exp2f((float)(e - (e >> 1)));
    return e;
}
// W (2 or 4) neighbouring floats of shared memory
template <int W> __device__ __forceinline__ void load_some(const float *p, float *v) {
    if constexpr (W == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(p);
    else *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(p);
}

// Slice blockIdx.x of A_0 of matrix blockIdx.y: S x S sums over `per` of the long side, 16 x 16 threads with (S / 16)^2 each
template <int TYPE, bool TALL, int S> __global__ void __launch_bounds__(kThreads) small_gram_kernel(const __grid_constant__ OrthSmall g, int per, float *sums) {
    chain_begin();
    constexpr int R = S / 16, W = R % 4 ? 2 : 4;                 // sums of a thread: R rows, R columns in runs of W
    __shared__ float tile[kSliceK][S + 4];
    const int z = blockIdx.y, tid = threadIdx.x, ty = tid / 16, tx = tid % 16, first = (int)blockIdx.x * per, last = min(g.l, first + per);
    float acc[R][R];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) acc[i][j] = 0.0f;
    constexpr int kLoads = S * kSliceK / kThreads;
    float v[kLoads];
    const auto ask = [&](int k0) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int n = tid + j * kThreads, k = TALL ? n / S : n % kSliceK, i = TALL ? n % S : n / kSliceK;
            v[j] = i < g.s && k0 + k < last ? element<TYPE, TALL>(g, z, i, k0 + k) : 0.0f;
        }
    };
    ask(first);                                                  // (before the norm, which is on its way for as long)
    float s0, s1;
    norm_scale(squares_of(g, z), &s0, &s1);
    for (int k0 = first; k0 < last; k0 += kSliceK) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const int n = tid + j * kThreads;
            tile[TALL ? n / S : n % kSliceK][TALL ? n % S : n / kSliceK] = v[j] * s0 * s1;
        }
        __syncthreads();
        if (k0 + kSliceK < last) ask(k0 + kSliceK);              // (on its way while these are summed)
#pragma unroll 4
        for (int k = 0; k < kSliceK; ++k) {
            alignas(16) float a[R], b[R];
#pragma unroll
            for (int j = 0; j < R; j += W) {
                load_some<W>(&tile[k][ty * R + j], a + j);
                load_some<W>(&tile[k][j * 16 + tx * W], b + j);
            }
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < R; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
    }
    float *to = sums + ((size_t)z * gridDim.x + blockIdx.x) * (size_t)(g.s * g.s);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const int r = ty * R + i, c = j / W * 16 * W + tx * W + j % W;
            if (r < g.s && c < g.s) to[r * g.s + c] = acc[i][j];
        }
}
__global__ void __launch_bounds__(kThreads) small_sum_kernel(const float *sums, int slices, int elements, float *to) {
    chain_begin();
    const int i = (int)blockIdx.x * kThreads + (int)threadIdx.x;
    if (i >= elements) return;
    const float *p = sums + (size_t)blockIdx.y * (size_t)slices * (size_t)elements + (size_t)i;
    double v = 0.0;
#pragma unroll 8
    for (int k = 0; k < slices; ++k) v += (double)p[(size_t)k * (size_t)elements];
    to[(size_t)blockIdx.y * (size_t)elements + (size_t)i] = (float)v;
}

// A matrix of 128 x 128 as an operand: high and low parts, each two blocks of 64 columns with rows of 128 bytes (128-byte swizzle)
constexpr unsigned kPart = 128 * 128 * 2, kMatrix = 2 * kPart;
struct CoreBars {
    uint64_t done, drain;
    unsigned tmem_base;
};
// 16 values of the thread's row, from column `col` on (a multiple of 16)
__device__ __forceinline__ void core_put(unsigned char *m, int row, int col, const float (&v)[16]) {
    unsigned p[8], q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const __half2 t = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        const float2 f = __half22float2(t);
        p[j] = *reinterpret_cast<const unsigned *>(&t);
        q[j] = pack_pair<kF16>(v[2 * j] - f.x, v[2 * j + 1] - f.y);
    }
    unsigned char *line = m + (col >> 6) * (kPart / 2) + row * 128;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned at = (unsigned)(((((col & 63) >> 3) + i) ^ (row & 7)) << 4);
        *reinterpret_cast<uint4 *>(line + at) = make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
        *reinterpret_cast<uint4 *>(line + kPart + at) = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
    }
}
__device__ __forceinline__ void core_get(const unsigned char *m, int row, int col, float (&v)[16]) {
    const unsigned char *line = m + (col >> 6) * (kPart / 2) + row * 128;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned at = (unsigned)(((((col & 63) >> 3) + i) ^ (row & 7)) << 4);
        const uint4 a = *reinterpret_cast<const uint4 *>(line + at), b = *reinterpret_cast<const uint4 *>(line + kPart + at);
        const unsigned p[4] = {a.x, a.y, a.z, a.w}, q[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p[j])), e = __half22float2(*reinterpret_cast<const __half2 *>(&q[j]));
            v[8 * i + 2 * j] = f.x + e.x;
            v[8 * i + 2 * j + 1] = f.y + e.y;
        }
    }
}
// ... as the second operand: row k of it is k of the product, columns are contiguous: groups of 64 columns kPart / 2 apart (leading byte offset), of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t core_desc_mn(unsigned addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(kPart / 2 >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// The product a b of two matrices, both parts of each: three walks along K.  The sum comes in two accumulators, the second one 128 columns behind: half of the additions of its size, and with them what
// they cut off.  (The operands are symmetric but for their rounding, and b could be read turned; then what is not symmetric in A grows by a^2 each step and shows at once in the last one: rank one of
// the values 3, 5 and 7, 128 x 1024, 1.1e-2 off.)  One thread.
__device__ __forceinline__ void core_product(unsigned acc, unsigned a, unsigned b, int s) {
    const unsigned n = (unsigned)(s + 15) / 16, half = n / 2;         // (both accumulators are written whatever n is)
    const unsigned idesc = (1u << 4) | (1u << 16) | (n * 16 >> 3 << 17) | (128u >> 4 << 24);          // FP16 x FP16, FP32 sums, b contiguous along N, N >> 3, M >> 4
    for (unsigned w = 0; w < 3; ++w)
        for (unsigned k = 0; k < n; ++k) {
            // (the small products first)
            const unsigned at = a + (w == 0 ? kPart : 0u) + (k >> 2) * (kPart / 2) + (k & 3u) * 32u, bt = b + (w == 1 ? kPart : 0u) + k * 2048u;
            const bool second = w == 2 && k >= half;
            mma_f16(acc + (second ? 128u : 0u), smem_desc_sw128(at), core_desc_mn(bt), idesc, second ? k > half : w + k > 0);
        }
}

// The steps of matrix blockIdx.x: from A_0 (the sum of `slices`) to R and q, times what X_0 is G times and the result's factor.  16 warps: a thread has a row of each result and 16 * NH
// columns, the four warps that may read its lanes of tensor memory the others.
template <int NH>
__global__ void __launch_bounds__(kStepThreads, 1) small_steps_kernel(const __grid_constant__ OrthSmall g, const __grid_constant__ OrthSmallSteps t, const float *sums, int slices,
                                                                      float *r_out, float *identity, unsigned tries, unsigned *status) {
    chain_begin();
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *ma = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u), *mn = ma + kMatrix, *mr = mn + kMatrix;
    CoreBars &bars = *reinterpret_cast<CoreBars *>(mr + kMatrix);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, z = blockIdx.x, s = g.s;
    const int row = (warp & 3) * 32 + lane, col = (warp >> 2) * 16 * NH;
    const bool mine = (warp & 3) * 32 < s && col < s;            // (whole warps)
    if (tid == 0) {
        mbar_init(&bars.done, 1);
        mbar_init(&bars.drain, 1);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc<1>(&bars.tmem_base, 512u);
    for (unsigned i = tid; i < 3 * kMatrix / 16; i += kStepThreads) reinterpret_cast<uint4 *>(ma)[i] = make_uint4(0u, 0u, 0u, 0u);
    const double squares = squares_of(g, z), norm = sqrt(squares);
    float s0, s1;
    const int e = norm_scale(squares, &s0, &s1);
    // X_0 = G 2^e * factor
    const float factor = !(norm < 3.0e38 * 65536.0 * 65536.0) ? __uint_as_float(0x7fffffffu) : norm > 0.0 ? (float)(ldexp(1.0, -e) / (norm + g.eps)) : 1.0f;
    float v[NH][16];
    if (mine) {
        const float x = ldexpf(factor * factor, t.step[0].a);
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h][j] = 0.0f;
        const float *p = sums + (size_t)z * (size_t)slices * (size_t)(s * s) + (size_t)(col * s + row);         // (symmetric: lanes along memory)
        for (int k = 0; k < slices; ++k, p += s * s)
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (row < s && col + 16 * h + j < s) v[h][j] += p[(16 * h + j) * s];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h][j] *= x;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tmem = bars.tmem_base, acc = tmem + ((unsigned)((warp & 3) * 32) << 16) + (unsigned)col;
    unsigned parity = 0;
    bool ok = true;
    // Operands are written: products may read them
    const auto meet = [&] {
        fence_proxy_async_smem();
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncthreads();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    };
    const auto wait = [&] {
        ok = mbar_wait_asleep(&bars.done, parity, status, tries) && ok;
        parity ^= 1u;
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    };
    // The thread's columns of a product times `by`; 0 outside the matrix
    const auto take = [&](unsigned from, float by) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float second[16];
            read16f(acc + from + 16u * (unsigned)h, v[h], true);
            read16f(acc + from + 128u + 16u * (unsigned)h, second, true);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h][j] = row < s && col + 16 * h + j < s ? (v[h][j] + second[j]) * by : 0.0f;
        }
    };
    // ... and an operand times `by`
    const auto add = [&](const unsigned char *m, float by) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float a[16];
            core_get(m, row, col + 16 * h, a);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[h][j] = fmaf(by, a[j], v[h][j]);
        }
    };
    const auto put = [&](unsigned char *m) {
#pragma unroll
        for (int h = 0; h < NH; ++h) core_put(m, row, col + 16 * h, v[h]);
    };
    const auto give = [&](float by) {
        const bool all = __syncthreads_and(ok) != 0;             // (a wait that ran out anywhere: NaN everywhere)
        if (tid == 0) identity[z] = t.identity * factor;
        if (!mine || row >= s) return;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (col + 16 * h + j < s) r_out[(size_t)z * (size_t)(s * s) + (size_t)((col + 16 * h + j) * s + row)] = all ? v[h][j] * by : __uint_as_float(0x7fffffffu);
    };

    if (mine) put(ma);
    for (int k = 0; k < t.steps; ++k) {
        const OrthSmallStep &p = t.step[k];
        const bool last = k + 1 == t.steps;
        // N = b A + c A^2
        meet();
        if (warp == 0 && elect_one()) {
            core_product(tmem, smem_u32(ma), smem_u32(ma), s);
            tc_commit(&bars.done);
        }
        __syncwarp();
        wait();
        if (mine) {
            take(0u, p.square);
            add(ma, p.linear);
        }
        if (k == 0 && last) {
            give(p.first_r * factor);
            break;
        }
        if (mine) {
            put(mn);
            if (k == 0) {
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[h][j] *= p.first_r;
                put(mr);
            }
        }
        // R <- N R + a R + q N, T = N A + a A
        meet();
        if (warp == 0 && elect_one()) {
            if (k > 0) core_product(tmem, smem_u32(mn), smem_u32(mr), s);
            if (!last) core_product(tmem + 256u, smem_u32(mn), smem_u32(ma), s);
            tc_commit(&bars.done);
        }
        __syncwarp();
        wait();
        if (mine && k > 0) {
            take(0u, p.r_product);
            add(mr, p.r_self);
            add(mn, p.r_n);
            if (!last) put(mr);
        }
        if (last) {
            give(factor);
            break;
        }
        if (mine) {
            take(256u, p.t_product);
            add(ma, p.t_self);
            put(ma);
        }
        // A <- N T + a T
        meet();
        if (warp == 0 && elect_one()) {
            core_product(tmem, smem_u32(mn), smem_u32(ma), s);
            tc_commit(&bars.done);
        }
        __syncwarp();
        wait();
        if (mine) {
            take(0u, p.a_product);
            add(ma, p.a_self);
            put(ma);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        if (elect_one()) tc_commit(&bars.drain);                 // products under way, also behind a wait that ran out
        __syncwarp();
        mbar_wait_asleep(&bars.drain, 0, status);
        tmem_free<1>(tmem, 512u);
    }
}

// 64 of the long side of matrix blockIdx.y: out = R G + q G (or G R + q G)
template <int TYPE, bool TALL, int S> __global__ void __launch_bounds__(kThreads) small_apply_kernel(const __grid_constant__ OrthSmall g, const float *r_in, const float *identity) {
    chain_begin();
    constexpr int R = S / 16, W = R % 4 ? 2 : 4;
    extern __shared__ float smem_apply[];
    float *mr = smem_apply, *tile = smem_apply + S * (S + 4);    // R [k][i], G [k][64 of the long side]
    const int z = blockIdx.y, tid = threadIdx.x, ty = tid / 16, tx = tid % 16, first = (int)blockIdx.x * 64;
    // (all of G and the first 16 of R are asked for before anything is waited for)
    constexpr int kLoads = S * 64 / kThreads;
    float v[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int n = tid + j * kThreads, k = TALL ? n % S : n / 64, i = TALL ? n / S : n % 64;
        v[j] = k < g.s && first + i < g.l ? element<TYPE, TALL>(g, z, k, first + i) : 0.0f;
    }
    constexpr int kBatch = S * S / kThreads < 16 ? S * S / kThreads : 16;
#pragma unroll 1
    for (int from = tid; from < S * S; from += kBatch * kThreads) {
        float w[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int n = from + j * kThreads, k = n / S, i = n % S;
            w[j] = k < g.s && i < g.s ? r_in[(size_t)z * (size_t)(g.s * g.s) + (size_t)(k * g.s + i)] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (from + j * kThreads < S * S) mr[(from + j * kThreads) / S * (S + 4) + (from + j * kThreads) % S] = w[j];
    }
    const float q = identity[z];
    float s0, s1;
    norm_scale(squares_of(g, z), &s0, &s1);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int n = tid + j * kThreads;
        tile[(TALL ? n % S : n / 64) * 68 + (TALL ? n / S : n % 64)] = v[j] * s0 * s1;
    }
    __syncthreads();
    // wide: a thread has R rows (ty) x 4 columns (tx); tall: 4 rows (ty) x R columns (tx): neighbouring threads write neighbouring elements
    float acc[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    const int ri = TALL ? tx : ty, gj = TALL ? ty : tx;
#pragma unroll 4
    for (int k = 0; k < g.s; ++k) {
        alignas(16) float a[R];
#pragma unroll
        for (int i = 0; i < R; i += W) load_some<W>(mr + k * (S + 4) + i * 16 + ri * W, a + i);
        const float4 b = *reinterpret_cast<const float4 *>(tile + k * 68 + gj * 4);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            acc[i][0] = fmaf(a[i], b.x, acc[i][0]);
            acc[i][1] = fmaf(a[i], b.y, acc[i][1]);
            acc[i][2] = fmaf(a[i], b.z, acc[i][2]);
            acc[i][3] = fmaf(a[i], b.w, acc[i][3]);
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const float4 b = *reinterpret_cast<const float4 *>(tile + (i / W * 16 * W + ri * W + i % W) * 68 + gj * 4);
        acc[i][0] = fmaf(q, b.x, acc[i][0]);
        acc[i][1] = fmaf(q, b.y, acc[i][1]);
        acc[i][2] = fmaf(q, b.z, acc[i][2]);
        acc[i][3] = fmaf(q, b.w, acc[i][3]);
    }
    // through shared memory, so that neighbouring threads write neighbouring elements whatever the rows' alignment: [S][64], or [64][S] where tall
    __syncthreads();
    unsigned short *box = reinterpret_cast<unsigned short *>(tile);
    const auto bits = [](float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); };
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = i / W * 16 * W + ri * W + i % W;
        if (TALL) {
#pragma unroll
            for (int j = 0; j < 4; ++j) box[(gj * 4 + j) * S + r] = bits(acc[i][j]);
        } else {
            *reinterpret_cast<uint2 *>(box + r * 64 + gj * 4) = make_uint2(pack_pair<kBf16>(acc[i][0], acc[i][1]), pack_pair<kBf16>(acc[i][2], acc[i][3]));
        }
    }
    __syncthreads();
    unsigned short *out = static_cast<unsigned short *>(g.out[z]);
    const size_t ld = (size_t)g.ld_out[z];
    const int rows = TALL ? min(64, g.l - first) : g.s, cols = TALL ? g.s : min(64, g.l - first), width = TALL ? S : 64, at = TALL ? 0 : first, row0 = TALL ? first : 0;
    if ((reinterpret_cast<uintptr_t>(out) | (ld * 2)) % 8 == 0 && cols % 4 == 0) {
        const int per = cols / 4;
        for (int n = tid; n < rows * per; n += kThreads) {
            const int r = n / per, c = (n - r * per) * 4;
            *reinterpret_cast<uint2 *>(out + (size_t)(row0 + r) * ld + (size_t)(at + c)) = *reinterpret_cast<const uint2 *>(box + r * width + c);
        }
    } else {
#pragma unroll 4
        for (int n = tid; n < rows * width; n += kThreads) {
            const int r = n / width, c = n - r * width;
            if (c < cols) out[(size_t)(row0 + r) * ld + (size_t)(at + c)] = box[n];
        }
    }
}

constexpr size_t kStepsSmem = 1024 + 3 * kMatrix + sizeof(CoreBars) + 64;
static_assert(kStepsSmem <= 227 * 1024, "three matrices do not fit");
constexpr size_t apply_smem(int s) { return (size_t)(s * (s + 4) + s * 68) * 4; }

template <int TYPE, bool TALL, int S>
cudaError_t run(const OrthSmall &g, const OrthSmallSteps &t, int count, const OrthSmallRoom &r, unsigned *status, cudaStream_t stream) {
    static std::atomic<uint64_t> done_steps{0}, done_apply{0};
    cudaError_t err = allow_smem(small_steps_kernel<(S + 63) / 64>, &done_steps);
    if (err == cudaSuccess) err = allow_smem(small_apply_kernel<TYPE, TALL, S>, &done_apply);
    if (err != cudaSuccess) return err;
    err = launch_chained(small_gram_kernel<TYPE, TALL, S>, dim3((unsigned)r.slices, (unsigned)count), kThreads, 0, stream, g, r.per, r.sums);
    if (err != cudaSuccess) return err;
    const float *sums = r.sums;
    int slices = r.slices;
    if (slices > kFewSlices) {
        const int n = g.s * g.s;
        err = launch_chained(small_sum_kernel, dim3((unsigned)((n + kThreads - 1) / kThreads), (unsigned)count), kThreads, 0, stream, (const float *)r.sums, slices, n, r.sum);
        if (err != cudaSuccess) return err;
        sums = r.sum;
        slices = 1;
    }
    err = launch_chained(small_steps_kernel<(S + 63) / 64>, (unsigned)count, kStepThreads, kStepsSmem, stream, g, t, sums, slices, r.r, r.identity, epilogue_tries(kWaitTries), status);
    if (err != cudaSuccess) return err;
    return launch_chained(small_apply_kernel<TYPE, TALL, S>, dim3((unsigned)((g.l + 63) / 64), (unsigned)count), kThreads, apply_smem(S), stream, g, (const float *)r.r, (const float *)r.identity);
}
template <int TYPE, bool TALL>
cudaError_t run_side(const OrthSmall &g, const OrthSmallSteps &t, int count, const OrthSmallRoom &r, unsigned *status, cudaStream_t stream) {
    if (g.s <= 32) return run<TYPE, TALL, 32>(g, t, count, r, status, stream);
    if (g.s <= 64) return run<TYPE, TALL, 64>(g, t, count, r, status, stream);
    return g.s <= 96 ? run<TYPE, TALL, 96>(g, t, count, r, status, stream) : run<TYPE, TALL, 128>(g, t, count, r, status, stream);
}
template <int TYPE>
cudaError_t run_type(const OrthSmall &g, bool tall, const OrthSmallSteps &t, int count, const OrthSmallRoom &r, unsigned *status, cudaStream_t stream) {
    return tall ? run_side<TYPE, true>(g, t, count, r, status, stream) : run_side<TYPE, false>(g, t, count, r, status, stream);
}

}  // namespace

// Slices of the long side, which are chains of FP32 sums: of 96 to 256, by the length alone.  (As few as fill the device, they were longer the more matrices went together, and a matrix's result
// was another one: 16384 in a chain left rank one 1.4e-1 off among 64.)
int orth_small_slices(uint64_t l, int *per) {
    const uint64_t want = std::min<uint64_t>(kOrthMaxDim / 256, (l + 95) / 96);
    *per = (int)(((l + want - 1) / want + kSliceK - 1) / kSliceK * kSliceK);
    return (int)((l + (uint64_t)*per - 1) / (uint64_t)*per);
}

cudaError_t orth_small(const OrthSmall &g, bool tall, int type, const OrthSmallSteps &t, int count, const OrthSmallRoom &r, unsigned *status, cudaStream_t stream) {
    if (type == kF32) return run_type<kF32>(g, tall, t, count, r, status, stream);
    if (type == kBf16) return run_type<kBf16>(g, tall, t, count, r, status, stream);
    return run_type<kF16>(g, tall, t, count, r, status, stream);
}

}  // namespace bsq
