// Softmax cross entropy of l = x W^T (x: tokens x cols, W: vocab x cols, FP16 or BF16) and its gradient, without keeping l:
//   loss_t = lse_t - (1 - e) l_t,target - e / vocab sum_v l_tv,   lse_t = log sum_v exp l_tv
//   dl_tv = g_t (exp(l_tv - lse_t) - (1 - e) [v = target] - e / vocab),   dx = dl W,   dW = dl^T x
//
// Loss: one product whose epilogue leaves, for each token and 128 (64) columns of the vocabulary, the largest logit and the sum of exponentials against it, and the target's
// logit; xent_join_kernel joins a token's parts (8 bytes for 128 logits are all that is written of them).
// Gradient: the vocabulary goes by in pieces of some 128 MB of dl (1024 columns at least).  Of a piece the logits are computed again, the epilogue turns them into dl in 16 bits (the
// rounding that a 16-bit gradient of logits has anyway; scaled, see XentScale), then dW of the piece is complete, and dx is summed over the pieces in FP32.
//
// Bound by the tensor core, then by power: the loss of 8192 x 4096 x 32000 1267 us from rest (1695 TFLOP/s, 1.02 of the measured burst rate of a library product; the tensor core is busy 98 %
// of the time), 1510 to 1530 one after the other (1410); loss and gradients of 4096 x 4096 x 32000 3.3 to 3.35 ms (8 T D V: 1280 to 1300 TFLOP/s).  Few tokens by the weight's bytes: 64 x 4096 x
// 131072 193 us (5.6 TB/s), one token 43 us for 262 MB (xent_few_kernel).
//
// Exponents are taken in base 2, and the reference of a tile is the rounded product of its largest logit and log2(e), so that the rounding cancels.
#include "bsq_gemm16.cuh"
#include "bsq_internal.hpp"
#include "bsq_xent.hpp"

namespace bsq {
namespace {

constexpr float kLog2E = 1.4426950408889634f;
constexpr double kLn2 = 1.0 / (double)kLog2E;                    // the way back from exponents that were taken with the rounded log2(e)
constexpr float kLowest = -3.0e38f;                              // below every logit but -Inf, whose exponential is 0 against it
constexpr uint64_t kPieceBytes = 128ull << 20;

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ---- loss ----
struct XentStats {
    int M, N;
    const long long *target;
    float2 *parts;                   // a warp's columns x M: (largest logit) * log2 e, sum of exponentials against it
    float *sums;                     // the same: sum of logits (nullable: no smoothing)
    float *at_target;                // M
    unsigned *joined;                // of XentJoin

    static constexpr bool kChained = true, kBack = false, kTotals = false, kBoxes = false;
    using Ahead = NoAhead;
    __device__ __forceinline__ void begin() const { *joined = 0u; }
    template <int COLS> __device__ __forceinline__ void tile(const TileOut &o, float (&v)[COLS]) const {
        const int row = o.row + o.lane, n = N - o.col;
        const float none = __uint_as_float(0xff800000u);
        if (n < COLS) {
#pragma unroll
            for (int j = 0; j < COLS; ++j)
                if (j >= n) v[j] = none;
        }
        const size_t at = (size_t)(o.col / COLS) * (size_t)M + (size_t)row;
        if (sums) {
            float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < COLS; ++j) total[j & 3] += j < n ? v[j] : 0.0f;
            if (row < M) sums[at] = (total[0] + total[1]) + (total[2] + total[3]);
        }
        float top = v[0];
#pragma unroll
        for (int j = 1; j < COLS; ++j) top = fmaxf(top, v[j]);
        top = fmaxf(top * kLog2E, kLowest);                      // (NaN shows in the sum)
        // The target's logit goes by itself, and out of the sum (XentJoin).  (Chosen for every element: taken out in its place it puts the whole array into memory, and sums taken
        // again in the few warps that have a target spill; 1264 -> 1600 us for 8192 x 4096 x 32000 either way.)
        const long long off = row < M ? target[row] - o.col : -1;
        const bool here = off >= 0 && off < COLS && off < n;
        const int at_j = here ? (int)off : -1;
        float mine = 0.0f, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
            mine = j == at_j ? v[j] : mine;
            s[j & 3] += exp2_fast(fmaf(j == at_j ? none : v[j], kLog2E, -top));
        }
        if (here) at_target[row] = mine;
        if (row < M) parts[at] = make_float2(top, (s[0] + s[1]) + (s[2] + s[3]));
    }
};

// Up to four tokens: the weight's bytes are all there is, and every multiplication fits beside them on the FP32 pipes, with rounded sums.  A warp has a row or two of the weight at a time,
// x lies in shared memory; a CTA leaves one part for each token.  VEC elements to a load, what the rows' alignment allows: 8, 2 or 1, so that nothing is copied first.
// 1 x 4096 x 32000 43 us for 262 MB (6.1 TB/s; on the tensor core, a tile of 128 x 128 with one row, 70); rows off 16 bytes would take three times that with their copy.
constexpr int kFewTokens = 4, kFewThreads = 512;
// Rows that a warp has at a time: two share what is read and unpacked of x; of one token that is little, and the finer division leaves fewer warps without work at the end
__host__ __device__ constexpr int few_rows(int tokens) { return tokens == 1 ? 1 : 2; }
constexpr size_t kFewSmem = 96 << 10;                            // of x: two CTAs to an SM
struct XentFew {
    const unsigned short *x, *w;
    uint64_t ld_x, ld_w;
    int cols;
    long long vocab;
    const long long *target;
    float2 *parts;                   // CTAs x tokens
    float *sums, *at_target;         // (sums nullable)
    unsigned *joined;                // of XentJoin
};
template <int VEC> struct FewWords;
template <> struct FewWords<8> { typedef uint4 type; };
template <> struct FewWords<2> { typedef unsigned type; };
template <> struct FewWords<1> { typedef unsigned short type; };
template <int TYPE, int VEC> __device__ __forceinline__ void few_unpack(const typename FewWords<VEC>::type &w, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        const unsigned a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = word_elem<TYPE>(a[j / 2], j & 1);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[j] = word_elem<TYPE>((unsigned)w, j);
    }
}
template <int TYPE, int VEC, int TOKENS> __global__ void __launch_bounds__(kFewThreads, 2) xent_few_kernel(const XentFew f) {
    chain_begin();
    typedef typename FewWords<VEC>::type Word;
    constexpr int kFewRows = few_rows(TOKENS), kUnroll = VEC == 8 ? 4 / kFewRows : 8;
    extern __shared__ uint4 smem_x[];
    unsigned short *sx = reinterpret_cast<unsigned short *>(smem_x);
    __shared__ float part[3][kFewThreads / 32][TOKENS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, words = f.cols / VEC, ld = (f.cols + 7) / 8 * 8;
    if (blockIdx.x == 0 && tid == 0) *f.joined = 0u;
    for (int t = 0; t < TOKENS; ++t)
        for (int i = tid; i < f.cols; i += kFewThreads) sx[t * ld + i] = f.x[(uint64_t)t * f.ld_x + i];
    long long target[TOKENS];
    float top[TOKENS], s[TOKENS], total[TOKENS];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
        target[t] = f.target[t];
        top[t] = kLowest;
        s[t] = total[t] = 0.0f;
    }
    __syncthreads();
    for (long long r0 = ((long long)blockIdx.x * (kFewThreads / 32) + warp) * kFewRows; r0 < f.vocab; r0 += (long long)gridDim.x * (kFewThreads / 32) * kFewRows) {
        const Word *p[kFewRows];
        float acc[kFewRows][TOKENS];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            p[r] = reinterpret_cast<const Word *>(f.w + (uint64_t)min(r0 + r, f.vocab - 1) * f.ld_w);
#pragma unroll
            for (int t = 0; t < TOKENS; ++t) acc[r][t] = 0.0f;
        }
        for (int i = lane; i < words; i += 32 * kUnroll) {
            Word w[kUnroll][kFewRows];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
                    if (i + 32 * u < words) w[u][r] = p[r][i + 32 * u];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (i + 32 * u >= words) break;
                float a[kFewRows][VEC];
#pragma unroll
                for (int r = 0; r < kFewRows; ++r) few_unpack<TYPE, VEC>(w[u][r], a[r]);
#pragma unroll
                for (int t = 0; t < TOKENS; ++t) {
                    float b[VEC];
                    few_unpack<TYPE, VEC>(reinterpret_cast<const Word *>(sx + t * ld)[i + 32 * u], b);
#pragma unroll
                    for (int r = 0; r < kFewRows; ++r)
#pragma unroll
                        for (int j = 0; j < VEC; ++j) acc[r][t] = fmaf(a[r][j], b[j], acc[r][t]);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < TOKENS; ++t)
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                float l = acc[r][t];
                for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(kFullMask, l, d);
                if (r0 + r >= f.vocab) continue;
                total[t] += l;
                if (r0 + r == target[t]) {                       // (by itself, and out of the sum)
                    if (lane == 0) f.at_target[t] = l;
                    continue;
                }
                const float m = l * kLog2E;
                if (m > top[t]) {
                    s[t] *= exp2_fast(top[t] - m);
                    top[t] = m;
                }
                s[t] += exp2_fast(fmaf(l, kLog2E, -top[t]));
            }
    }
#pragma unroll
    for (int t = 0; t < TOKENS; ++t)
        if (lane == t) {
            part[0][warp][t] = top[t];
            part[1][warp][t] = s[t];
            part[2][warp][t] = total[t];
        }
    __syncthreads();
    if (tid < TOKENS) {
        float m = part[0][0][tid], sum = 0.0f, all = 0.0f;
        for (int i = 1; i < kFewThreads / 32; ++i) m = fmaxf(m, part[0][i][tid]);
        for (int i = 0; i < kFewThreads / 32; ++i) {
            sum += part[1][i][tid] * exp2_fast(part[0][i][tid] - m);
            all += part[2][i][tid];
        }
        const size_t at = (size_t)blockIdx.x * TOKENS + (size_t)tid;
        f.parts[at] = make_float2(m, sum);
        if (f.sums) f.sums[at] = all;
    }
}

struct XentJoin {
    int tokens, tiles;
    long long vocab, ignore;
    double smoothing;
    int reduction;
    const long long *target;
    const float2 *parts;
    const float *sums, *at_target;
    float *loss, *stats;             // stats: log2 of the sum of exponentials of each token, the number of tokens that count, then lse - (logit of the target) of each
    double2 *blocks;                 // loss and tokens of each CTA
    unsigned *joined;                // CTAs that have left theirs; 0 at the start (the kernel in front sees to it)
};

// The sum over a CTA's threads, the same order every time
__device__ __forceinline__ double2 cta_sum(double2 v, double2 *room) {
    for (int d = 16; d; d >>= 1) {
        v.x += __shfl_xor_sync(kFullMask, v.x, d);
        v.y += __shfl_xor_sync(kFullMask, v.y, d);
    }
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    v = room[0];
    for (int i = 1; i < (int)blockDim.x / 32; ++i) {
        v.x += room[i].x;
        v.y += room[i].y;
    }
    return v;
}
__device__ __forceinline__ void write_total(const XentJoin &j, double2 v) {
    j.stats[j.tokens] = (float)v.y;
    if (j.reduction == kXentSum) *j.loss = (float)v.x;
    else if (j.reduction == kXentMean) *j.loss = (float)(v.x / v.y);
}

// 32 tokens a CTA, one for each lane; the warps share the tiles.  The parts are without the target's logit t: the loss is log(1 + sum exp(l_v - t)), and as good where the sum is
// 10^-6 as where it is 10 (with exp(t - t) among the terms, a loss of 10^-3 was 5e-5 off).
__global__ void __launch_bounds__(1024) xent_join_kernel(const XentJoin j) {
    chain_begin();
    __shared__ float2 part[32][32];
    __shared__ float part_sum[32][32];
    __shared__ double2 room[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, token = (int)blockIdx.x * 32 + lane;
    float top = kLowest, s = 0.0f, total = 0.0f;
    if (token < j.tokens) {
#pragma unroll 4
        for (int t = warp; t < j.tiles; t += 32) {
            const float2 p = j.parts[(size_t)t * (size_t)j.tokens + (size_t)token];
            const float m = fmaxf(top, p.x);
            s = s * exp2_fast(top - m) + p.y * exp2_fast(p.x - m);
            top = m;
            if (j.sums) total += j.sums[(size_t)t * (size_t)j.tokens + (size_t)token];
        }
    }
    part[warp][lane] = make_float2(top, s);
    part_sum[warp][lane] = total;
    __syncthreads();
    double2 mine = make_double2(0.0, 0.0);
    if (warp == 0 && token < j.tokens) {
        float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};                // (FP64 additions one behind the other took 3 us)
#pragma unroll
        for (int i = 0; i < 32; ++i) top = fmaxf(top, part[i][lane].x);
#pragma unroll
        for (int i = 0; i < 32; ++i) sums[i & 3] += part[i][lane].y * exp2_fast(part[i][lane].x - top);
        const double sum = (double)((sums[0] + sums[1]) + (sums[2] + sums[3]));
        double all = 0.0;
        if (j.sums)
            for (int i = 0; i < 32; ++i) all += (double)part_sum[i][lane];
        const long long t = j.target[token];
        const bool live = t != j.ignore, in = t >= 0 && t < j.vocab;
        double lse2 = (double)top + log2(sum), apart = 0.0;      // (without its target nobody wants it)
        if (in) {
            const double at = (double)j.at_target[token], at2 = at * (double)kLog2E, other = lse2 - at2;        // (log2 of the others against the target)
            apart = isinf(at) && at > 0.0 ? __longlong_as_double(0x7ff8000000000000ll) : other > 60.0 ? other * kLn2 : log1p(exp2(other));
            lse2 = at2 > (double)top ? at2 + apart / kLn2 : (double)top + log2(sum + exp2(at2 - (double)top));
        }
        double loss = apart;
        if (j.sums) loss += j.smoothing * ((in ? (double)j.at_target[token] : 0.0) - all / (double)j.vocab);
        if (!in) loss = __longlong_as_double(0x7ff8000000000000ll);
        if (!live) loss = 0.0;
        j.stats[token] = (float)lse2;
        j.stats[j.tokens + 1 + token] = (float)apart;
        if (j.reduction == kXentNone) j.loss[token] = (float)loss;
        mine = make_double2(loss, live ? 1.0 : 0.0);
    }
    __syncthreads();
    double2 v = cta_sum(mine, room);
    if (gridDim.x == 1) {
        if (threadIdx.x == 0) write_total(j, v);
        return;
    }
    // the CTA that comes last adds them all up, in their order
    __shared__ bool last;
    if (threadIdx.x == 0) {
        j.blocks[blockIdx.x] = v;
        __threadfence();
        last = atomicAdd(j.joined, 1u) + 1u == gridDim.x;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    v = make_double2(0.0, 0.0);
    for (unsigned i = threadIdx.x; i < gridDim.x; i += 1024) {
        const double2 b = __ldcg(&j.blocks[i]);
        v.x += b.x;
        v.y += b.y;
    }
    v = cta_sum(v, room);
    if (threadIdx.x == 0) write_total(j, v);
}
// No tokens: nothing, 0 or 0 / 0
__global__ void xent_none_kernel(const XentJoin j) {
    chain_begin();
    if (threadIdx.x == 0) write_total(j, make_double2(0.0, 0.0));
}

// ---- gradient ----
// What gradients of logits are multiplied by on the way to 16 bits, and the products by on the way back: what makes the largest |g| (1 - e + e / vocab) 2^13.
// That keeps small gradients within FP16's range (|dl| stays below 2^15), and it makes the element of a target that has next to no probability, the largest of its row and the same in
// all rows where the g are, a number that 16 bits hold: rounded, it was off by the same part of up to 2^-8 in every row, and so were dx and dW (4096 x 4096 x 32000 in BF16 up to
// 2.9e-3 off; 1.7e-3 is what their own rounding takes).
struct XentScale {
    const float *grad, *stats;       // one gradient for all tokens: of the loss, and (the mean's) the number of tokens behind their statistics
    int tokens, reduction;
    float reference;                 // 1 - e + e / vocab, 1 / 4 at least
    const float *coef, *unscale;     // or one for each token: g_t times the scale, and the way back (xent_coef_kernel)

    // (a gradient of 0, Inf or NaN goes through as it is; below 2^-100 the scale stays finite)
    __device__ __forceinline__ float top(float m) const { return m > 0.0f && m < __uint_as_float(0x7f800000u) ? fmaxf(m, 7.888609052e-31f) * reference : 8192.0f; }
    __device__ __forceinline__ float one() const { return reduction == kXentMean ? *grad / stats[tokens] : *grad; }
    __device__ __forceinline__ float back() const { return coef ? *unscale : top(fabsf(one())) * (1.0f / 8192.0f); }
    // ... of a token that counts; NaN for a target that is none
    __device__ __forceinline__ float of(int row, long long target, long long vocab) const {
        if (target < 0 || target >= vocab) return __uint_as_float(0x7fffffffu);
        if (coef) return coef[row];
        const float g = one();
        return g * (8192.0f / top(fabsf(g)));
    }
};
// Each token's own g: the largest of them, and all of them scaled.  One CTA.
__global__ void __launch_bounds__(1024) xent_coef_kernel(const XentScale s, const long long *target, long long ignore, float *coef, float *unscale) {
    chain_begin();
    __shared__ float room[32];
    float m = 0.0f;
    for (int i = threadIdx.x; i < s.tokens; i += 1024) {
        const float a = fabsf(s.grad[i]);
        if (target[i] != ignore && a < __uint_as_float(0x7f800000u)) m = fmaxf(m, a);
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = m;
    __syncthreads();
    const float top = s.top(warp_max(room[threadIdx.x & 31]));
    if (threadIdx.x == 0) *unscale = top * (1.0f / 8192.0f);
    for (int i = threadIdx.x; i < s.tokens; i += 1024) coef[i] = s.grad[i] * (8192.0f / top);
}

template <int TYPE> struct XentGrad {
    CUtensorMap map;                 // the piece: tokens x its columns
    int M, N;                        // N: columns of the vocabulary in the piece; the piece's others are 0
    long long first;                 // of the vocabulary
    long long vocab, ignore;
    const long long *target;
    const float *lse2, *apart;       // apart: lse - (logit of the target)
    XentScale scale;
    float low, rest;                 // e / vocab, e - e / vocab

    static constexpr bool kChained = false, kBack = true, kTotals = false, kBoxes = true;          // (p is exp of these logits less the loss's lse: with 65536 columns in one chain 1.7e-2 too small)
    using Ahead = NoAhead;
    template <int COLS> __device__ void ahead(const TileOut &, Ahead &) const {}
    template <int COLS> __device__ void tile(const TileOut &o, Ahead &) const {
        const int row = o.row + o.lane;
        const long long t = row < M ? target[row] : ignore;
        const bool live = t != ignore;
        const long long off = live ? t - first - o.col : -1;
        const float lse = row < M ? lse2[row] : 0.0f, g = live ? scale.of(row, t, vocab) : 0.0f;
        // The target's element, from the loss: where p is near 1, p - 1 from the logits would be what their last digits leave of it (1 - p = 1e-3: 2 % off)
        const float of_target = !o.ok ? __uint_as_float(0x7fffffffu) : live ? g * (expm1f(-apart[row]) + rest) : 0.0f;
        for (int c = 0; c < COLS; c += 64) {
            unsigned char *box = box_next(o);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float v[16];
                read16f(o.taddr + (unsigned)(c + 16 * h), v, o.ok);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = g * (exp2_fast(fmaf(v[j], kLog2E, -lse)) - low);
                // (chosen, not multiplied: what an ignored token's logits are does not matter)
                if (!live) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = 0.0f;
                }
                if (o.col + c + 16 * h + 16 > N) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (o.col + c + 16 * h + j >= N) v[j] = 0.0f;
                }
                box_put16<TYPE>(box, o.lane, h, v);
            }
            if (off >= c && off < c + 64 && off < COLS) {
                const int col = (int)off - c;
                store_elem<TYPE>(box + o.lane * 128 + (((col >> 3) ^ (o.lane & 7)) << 4), (uint64_t)(col & 7), of_target);
            }
            box_send(o, &map, o.col + c, o.row, box);
        }
    }
};

// A product's tiles out of tensor memory: to 16-bit rows, or into FP32 sums over several launches
enum ProductMode : int { kProductOut = 0, kSumFirst = 1, kSumMore = 2, kSumOut = 3 };
template <int TYPE> struct ProductOut {
    CUtensorMap map, map_sum;
    int M, N, mode;
    bool boxes;                      // the result can be written by TMA
    void *out;
    long ld;
    const float *sum;
    long ld_sum;
    XentScale scale;

    static constexpr bool kChained = false, kBack = true, kTotals = false, kBoxes = true;          // (524288 tokens of one sign in one chain: 3.2e-3 too small)
    using Ahead = NoAhead;
    template <int COLS> __device__ void ahead(const TileOut &, Ahead &) const {}
    template <int COLS> __device__ void tile(const TileOut &o, Ahead &) const {
        if (mode == kSumFirst || mode == kSumMore) {
            for (int c = 0; c < COLS && o.col + c < N; c += 32) {
                unsigned char *box = box_next(o);
                uint4 *line = reinterpret_cast<uint4 *>(box + o.lane * 128);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned r[16];
                    read16(o.taddr + (unsigned)(c + 16 * h), r, o.ok);
#pragma unroll
                    for (int j = 0; j < 4; ++j) line[(4 * h + j) ^ (o.lane & 7)] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                }
                box_send(o, &map_sum, o.col + c, o.row, box, mode == kSumMore);
            }
            return;
        }
        const float f = scale.back();
        const int row = o.row + o.lane;
        for (int c = 0; c < COLS && o.col + c < N; c += 64) {
            unsigned char *box = box_next(o);
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float v[16];
                read16f(o.taddr + (unsigned)(c + 16 * h), v, o.ok);
                if (mode == kSumOut && row < M && o.col + c + 16 * h < N) {
                    // (rows of the sums are padded to a multiple of 16)
                    const float4 *s = reinterpret_cast<const float4 *>(sum + (size_t)row * (size_t)ld_sum + (size_t)(o.col + c + 16 * h));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 a = s[j];
                        v[4 * j] += a.x; v[4 * j + 1] += a.y; v[4 * j + 2] += a.z; v[4 * j + 3] += a.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] *= f;
                box_put16<TYPE>(box, o.lane, h, v);
            }
            if (boxes) box_send(o, &map, o.col + c, o.row, box);
            else box_out_rows(box, o.lane, out, 2, (long)o.row * ld + o.col + c, ld, M - o.row, N - o.col - c);
        }
    }
};

// The slices of a product that was split along K, added up in their order
template <int TYPE>
__global__ void __launch_bounds__(256) sum_slices_kernel(const float *sum, int slices, int rows, int cols, long ld_sum, const XentScale scale, void *out, long ld) {
    chain_begin();
    const float f = scale.back();
    const long all = (long)rows * cols;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        const long r = i / cols, c = i - r * cols;
        float v = 0.0f;
#pragma unroll 4
        for (int s = 0; s < slices; ++s) v += sum[((size_t)s * (size_t)rows + (size_t)r) * (size_t)ld_sum + (size_t)c];
        store_elem<TYPE>(out, (uint64_t)(r * ld + c), v * f);
    }
}

// Rows whose start or distance TMA cannot take, copied to rows on 16 bytes.  A thread writes 16 bytes.
__global__ void __launch_bounds__(256) align_rows_kernel(const unsigned short *in, uint64_t rows, uint64_t cols, uint64_t ld, unsigned short *out, uint64_t ld_out) {
    chain_begin();
    const uint64_t per = ld_out / 8, all = rows * per;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
        const uint64_t r = i / per, c = (i - r * per) * 8;
        const unsigned short *p = in + r * ld + c;
        unsigned w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned lo = c + 2 * j < cols ? p[2 * j] : 0u, hi = c + 2 * j + 1 < cols ? p[2 * j + 1] : 0u;
            w[j] = lo | hi << 16;
        }
        *reinterpret_cast<uint4 *>(out + r * ld_out + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// ---- host ----
bool needs_copy(const void *p, uint64_t rows, uint64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 != 0 || (rows > 1 && ld % 8 != 0); }

struct Operands {
    Stack x, w;
};
// x and W as the products read them, copied where need be
Operands aligned_operands(const XentCall &c, Scratch *s, bool run, cudaError_t *err, int sm_count, cudaStream_t stream) {
    Operands o = {{c.x, c.cols, c.tokens, c.ld_x, 1, 0}, {c.w, c.cols, c.vocab, c.ld_w, 1, 0}};
    for (Stack *m : {&o.x, &o.w}) {
        if (!needs_copy(m->at, m->rows, m->ld)) continue;
        const uint64_t ld = padded(m->cols, 64);                  // (rows of whole lines: boxes of 128 bytes then are a line each, not parts of two)
        unsigned short *to = s->take<unsigned short>(m->rows * ld);
        if (run && *err == cudaSuccess) {
            const uint64_t blocks = (m->rows * (ld / 8) + 255) / 256;
            *err = launch_chained(align_rows_kernel, (unsigned)std::min<uint64_t>(blocks, (uint64_t)sm_count * 16), 256, 0, stream, static_cast<const unsigned short *>(m->at), m->rows,
                                  m->cols, m->ld, to, ld);
        }
        m->at = to;
        m->ld = ld;
    }
    return o;
}

struct LossPlan {
    bool pairs;
    int few;                         // elements to a load of the kernel for up to four tokens, 0: the product
    uint64_t tiles;                  // parts of a token
};
LossPlan loss_plan(const XentCall &c, int sm_count) {
    LossPlan p;
    p.pairs = false;
    p.few = 0;
    if (c.tokens <= (uint64_t)kFewTokens && c.tokens * ((c.cols + 7) / 8 * 8) * 2 <= kFewSmem) {
        const uintptr_t start = reinterpret_cast<uintptr_t>(c.w);
        const uint64_t ld = c.vocab > 1 ? c.ld_w : 0;
        p.few = start % 16 == 0 && (ld | c.cols) % 8 == 0 ? 8 : start % 4 == 0 && (ld | c.cols) % 2 == 0 ? 2 : 1;
        const uint64_t rows = kFewThreads / 32 * (uint64_t)few_rows((int)c.tokens);
        p.tiles = std::min<uint64_t>((uint64_t)std::max(1, 2 * sm_count), (c.vocab + rows - 1) / rows);
        return p;
    }
    p.pairs = g16_pairs(c.tokens, c.vocab, 1, false, sm_count);
    p.tiles = p.pairs ? (c.vocab + 127) / 128 : (c.vocab + 63) / 64;
    return p;
}
struct LossRoom {
    float2 *parts;
    float *sums, *at_target;
    double2 *blocks;
    unsigned *joined;
};
LossRoom loss_room(const XentCall &c, const LossPlan &p, Scratch *s) {
    LossRoom r;
    r.parts = s->take<float2>(p.tiles * c.tokens);
    r.sums = c.smoothing > 0.0 ? s->take<float>(p.tiles * c.tokens) : nullptr;
    r.at_target = s->take<float>(c.tokens);
    r.blocks = s->take<double2>((c.tokens + 31) / 32);
    r.joined = s->take<unsigned>(1);
    return r;
}

template <int TYPE, int VEC, int TOKENS> cudaError_t launch_few_as(const XentFew &f, const LossPlan &p, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t err = allow_smem(xent_few_kernel<TYPE, VEC, TOKENS>, &done, (int)kFewSmem);
    if (err != cudaSuccess) return err;
    return launch_chained(xent_few_kernel<TYPE, VEC, TOKENS>, (unsigned)p.tiles, kFewThreads, (size_t)TOKENS * (size_t)((f.cols + 7) / 8 * 16), stream, f);
}
template <int TYPE, int TOKENS> cudaError_t launch_few_of(const XentFew &f, const LossPlan &p, cudaStream_t stream) {
    return p.few == 8 ? launch_few_as<TYPE, 8, TOKENS>(f, p, stream) : p.few == 2 ? launch_few_as<TYPE, 2, TOKENS>(f, p, stream) : launch_few_as<TYPE, 1, TOKENS>(f, p, stream);
}
template <int TYPE> cudaError_t launch_few(const XentFew &f, const LossPlan &p, int tokens, cudaStream_t stream) {
    return tokens == 1 ? launch_few_of<TYPE, 1>(f, p, stream) : tokens == 2 ? launch_few_of<TYPE, 2>(f, p, stream) : tokens == 3 ? launch_few_of<TYPE, 3>(f, p, stream) : launch_few_of<TYPE, 4>(f, p, stream);
}

struct GradPlan {
    uint64_t piece, pieces;          // columns of the vocabulary at a time
    bool pairs_l, pairs_w, pairs_x;
    int splits;                      // of dx along the vocabulary
    uint64_t ld_sum;
};
GradPlan grad_plan(const XentCall &c, bool dx, int sm_count) {
    GradPlan p;
    const uint64_t whole = padded(c.vocab, 256), most = std::min<uint64_t>(65536, std::max<uint64_t>(1024, kPieceBytes / 2 / c.tokens / 256 * 256));
    p.pieces = (whole + most - 1) / most;
    p.piece = padded((whole + p.pieces - 1) / p.pieces, 256);
    p.pieces = (whole + p.piece - 1) / p.piece;
    p.pairs_l = g16_pairs(c.tokens, p.piece, 1, false, sm_count);
    p.pairs_w = g16_pairs(p.piece, c.cols, 1, false, sm_count);
    p.pairs_x = false;
    p.splits = 1;
    const uint64_t stages = p.piece / kG16K;
    // Few tiles of dx: slices of the vocabulary, added up afterwards.  What takes least by rounds of tiles times their stages (0.35 us for a pair's, 0.3 us for a single CTA's) and some
    // 8 us that a round begins and ends with.  777 x 1031 from 50001: 63 tiles of 128 x 128 in two slices 127 us, 20 of 256 x 256 in seven 84.
    double best = 0.0;
    for (int pairs = c.tokens > 128 ? 1 : 0; dx && pairs >= 0; --pairs) {
        const uint64_t side = pairs ? 256 : 128, tiles = ((c.tokens + side - 1) / side) * ((c.cols + side - 1) / side), units = std::max<uint64_t>(1, (uint64_t)sm_count / (pairs ? 2 : 1));
        for (uint64_t n = 1; n <= 64 && n * 4 <= stages + 3; ++n) {
            const double sums = n > 1 ? 6.0 + (double)(n * c.tokens * c.cols) * (4.0 + 4.0 * (double)p.pieces) / 5e6 : 0.0;                  // (written piece by piece, read once: 5 TB/s)
            const double time = (double)p.pieces * (double)((tiles * n + units - 1) / units) * ((double)((stages + n - 1) / n) * (pairs ? 0.35 : 0.3) + 8.0) + sums;
            if (best != 0.0 && time >= best) continue;
            best = time;
            p.pairs_x = pairs != 0;
            p.splits = (int)n;
        }
    }
    p.ld_sum = padded(c.cols, 16);
    return p;
}
struct GradRoom {
    float *coef, *unscale, *sum;
    unsigned short *piece;
};
GradRoom grad_room(const XentCall &c, const GradPlan &p, bool dx, Scratch *s) {
    GradRoom r;
    r.coef = s->take<float>(c.tokens);
    r.unscale = s->take<float>(1);
    r.piece = s->take<unsigned short>(c.tokens * p.piece);
    r.sum = dx && (p.pieces > 1 || p.splits > 1) ? s->take<float>((uint64_t)p.splits * c.tokens * p.ld_sum) : nullptr;
    return r;
}

Gemm16 product_of(uint64_t M, uint64_t N, bool a_kmajor, bool b_kmajor, bool bf16, int splits = 1) {
    Gemm16 g = {};
    g.M = (int)M;
    g.N = (int)N;
    g.batch = 1;
    g.parts = 1;
    g.splits = splits;
    g.a_kmajor = a_kmajor;
    g.b_kmajor = b_kmajor;
    g.bf16 = bf16;
    return g;
}

// out (or sums): M x N = A B^T
template <int TYPE>
cudaError_t product(const Stack &a, bool a_kmajor, const Stack &b, bool b_kmajor, uint64_t M, uint64_t N, uint64_t K, bool pairs, int splits, int mode, void *out, uint64_t ld,
                    float *sum, uint64_t ld_sum, const XentScale &scale, unsigned *status, int sm_count, cudaStream_t stream) {
    Gemm16Maps maps;
    ProductOut<TYPE> e;
    if (!map_operand(&maps.a[0], a, TYPE == kBf16, a_kmajor) || !map_operand(&maps.b[0], b, TYPE == kBf16, b_kmajor)) return cudaErrorInvalidValue;
    maps.a[1] = maps.a[0];
    maps.b[1] = maps.b[0];
    e.map = e.map_sum = maps.a[0];
    e.M = (int)M;
    e.N = (int)N;
    e.mode = mode;
    e.out = out;
    e.ld = (long)ld;
    e.sum = sum;
    e.ld_sum = (long)ld_sum;
    e.scale = scale;
    e.boxes = out && tma_can_write(out, (M == 1 ? N : ld) * 2, N * 2);
    if (e.boxes && !map_stack(&e.map, {out, N, M, ld, 1, 0}, TYPE, 64, 32)) return cudaErrorInvalidValue;
    if (sum && !map_stack(&e.map_sum, {sum, ld_sum, M, ld_sum, (uint64_t)splits, M * ld_sum}, kF32, 32, 32)) return cudaErrorInvalidValue;
    return launch_gemm16(maps, e, product_of(M, N, a_kmajor, b_kmajor, TYPE == kBf16, splits), K, pairs, status, sm_count, stream);
}

template <int TYPE>
cudaError_t grad_pieces(const XentCall &c, const GradPlan &p, const GradRoom &r, const Operands &o, const float *stats, const XentScale &scale, void *dx, uint64_t ld_dx, void *dw, uint64_t ld_dw,
                        unsigned *status, int sm_count, cudaStream_t stream) {
    cudaError_t err = cudaSuccess;
    for (uint64_t i = 0; i < p.pieces && err == cudaSuccess; ++i) {
        const uint64_t first = i * p.piece, n = std::min(p.piece, c.vocab - first);
        const Stack w = {static_cast<const unsigned short *>(o.w.at) + first * o.w.ld, c.cols, n, o.w.ld, 1, 0};
        const Stack dl = {r.piece, p.piece, c.tokens, p.piece, 1, 0}, dl_valid = {r.piece, n, c.tokens, p.piece, 1, 0};
        Gemm16Maps maps;
        XentGrad<TYPE> e;
        if (!map_operand(&maps.a[0], o.x, TYPE == kBf16, true) || !map_operand(&maps.b[0], w, TYPE == kBf16, true) || !map_stack(&e.map, dl, TYPE, 64, 32)) return cudaErrorInvalidValue;
        maps.a[1] = maps.a[0];
        maps.b[1] = maps.b[0];
        e.M = (int)c.tokens;
        e.N = (int)n;
        e.first = (long long)first;
        e.vocab = (long long)c.vocab;
        e.ignore = c.ignore;
        e.target = c.target;
        e.lse2 = stats;
        e.apart = stats + c.tokens + 1;
        e.scale = scale;
        e.low = (float)(c.smoothing / (double)c.vocab);
        e.rest = (float)(c.smoothing - c.smoothing / (double)c.vocab);
        err = launch_gemm16(maps, e, product_of(c.tokens, n, true, true, TYPE == kBf16), c.cols, p.pairs_l, status, sm_count, stream);
        if (err != cudaSuccess) return err;
        if (dw)
            err = product<TYPE>(dl_valid, false, o.x, false, n, c.cols, c.tokens, p.pairs_w, 1, kProductOut, static_cast<unsigned short *>(dw) + first * ld_dw, ld_dw, nullptr, 0,
                                scale, status, sm_count, stream);
        if (err != cudaSuccess) return err;
        if (dx) {
            const bool last = i + 1 == p.pieces;
            const int mode = !r.sum ? kProductOut : p.splits == 1 && last ? kSumOut : i == 0 ? kSumFirst : kSumMore;
            err = product<TYPE>(dl_valid, true, w, false, c.tokens, c.cols, n, p.pairs_x, p.splits, mode, dx, ld_dx, r.sum, p.ld_sum, scale, status, sm_count, stream);
        }
    }
    if (err == cudaSuccess && dx && p.splits > 1) {
        const uint64_t blocks = (c.tokens * c.cols + 255) / 256;
        err = launch_chained(sum_slices_kernel<TYPE>, (unsigned)std::min<uint64_t>(blocks, (uint64_t)sm_count * 8), 256, 0, stream, (const float *)r.sum, p.splits, (int)c.tokens, (int)c.cols,
                             (long)p.ld_sum, scale, dx, (long)ld_dx);
    }
    return err;
}

}  // namespace

size_t xent_scratch_bytes(const XentCall &c, int sm_count) {
    if (c.tokens == 0) return 0;
    Scratch s = {nullptr};
    cudaError_t err = cudaSuccess;
    const LossPlan p = loss_plan(c, sm_count);
    loss_room(c, p, &s);
    if (!p.few) aligned_operands(c, &s, false, &err, sm_count, nullptr);
    return s.used;
}

size_t xent_grad_scratch_bytes(const XentCall &c, bool dx, int sm_count) {
    if (c.tokens == 0) return 0;
    Scratch s = {nullptr};
    cudaError_t err = cudaSuccess;
    aligned_operands(c, &s, false, &err, sm_count, nullptr);
    grad_room(c, grad_plan(c, dx, sm_count), dx, &s);
    return s.used;
}

cudaError_t xent_loss(const XentCall &c, float *loss, float *stats, void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    Scratch s = {static_cast<unsigned char *>(scratch)};
    cudaError_t err = cudaSuccess;
    if (c.tokens == 0) {
        const XentJoin none = {0, 0, (long long)c.vocab, c.ignore, c.smoothing, c.reduction, nullptr, nullptr, nullptr, nullptr, loss, stats, nullptr, nullptr};
        return launch_chained(xent_none_kernel, 1, 32, 0, stream, none);
    }
    const LossPlan p = loss_plan(c, sm_count);
    const LossRoom r = loss_room(c, p, &s);
    if (p.few) {
        const XentFew f = {static_cast<const unsigned short *>(c.x), static_cast<const unsigned short *>(c.w), c.ld_x, c.ld_w, (int)c.cols, (long long)c.vocab, c.target, r.parts, r.sums, r.at_target, r.joined};
        err = c.type == kBf16 ? launch_few<kBf16>(f, p, (int)c.tokens, stream) : launch_few<kF16>(f, p, (int)c.tokens, stream);
    } else {
        const Operands o = aligned_operands(c, &s, true, &err, sm_count, stream);
        if (err != cudaSuccess) return err;
        Gemm16Maps maps;
        const bool bf16 = c.type == kBf16;
        if (!map_operand(&maps.a[0], o.x, bf16, true) || !map_operand(&maps.b[0], o.w, bf16, true)) return cudaErrorInvalidValue;
        maps.a[1] = maps.a[0];
        maps.b[1] = maps.b[0];
        const XentStats e = {(int)c.tokens, (int)c.vocab, c.target, r.parts, r.sums, r.at_target, r.joined};
        err = launch_gemm16(maps, e, product_of(c.tokens, c.vocab, true, true, bf16), c.cols, p.pairs, status, sm_count, stream);
    }
    if (err != cudaSuccess) return err;
    const XentJoin j = {(int)c.tokens, (int)p.tiles, (long long)c.vocab, c.ignore, c.smoothing, c.reduction, c.target, r.parts, r.sums, r.at_target, loss, stats, r.blocks, r.joined};
    const unsigned blocks = (unsigned)((c.tokens + 31) / 32);
    return launch_chained(xent_join_kernel, blocks, 1024, 0, stream, j);
}

cudaError_t xent_grad(const XentCall &c, const float *stats, const float *grad, void *dx, uint64_t ld_dx, void *dw, uint64_t ld_dw, void *scratch, unsigned *status,
                      int sm_count, cudaStream_t stream) {
    Scratch s = {static_cast<unsigned char *>(scratch)};
    cudaError_t err = cudaSuccess;
    if (c.tokens == 0) return dw ? cudaMemset2DAsync(dw, ld_dw * 2, 0, c.cols * 2, c.vocab, stream) : cudaSuccess;
    const Operands o = aligned_operands(c, &s, true, &err, sm_count, stream);
    if (err != cudaSuccess) return err;
    const GradPlan p = grad_plan(c, dx != nullptr, sm_count);
    const GradRoom r = grad_room(c, p, dx != nullptr, &s);
    const bool each = c.reduction == kXentNone;
    const XentScale scale = {grad, stats, (int)c.tokens, c.reduction, (float)std::max(0.25, 1.0 - c.smoothing + c.smoothing / (double)c.vocab), each ? r.coef : nullptr, each ? r.unscale : nullptr};
    if (each) err = launch_chained(xent_coef_kernel, 1, 1024, 0, stream, scale, c.target, c.ignore, r.coef, r.unscale);
    if (err != cudaSuccess) return err;
    return c.type == kBf16 ? grad_pieces<kBf16>(c, p, r, o, stats, scale, dx, ld_dx, dw, ld_dw, status, sm_count, stream)
                           : grad_pieces<kF16>(c, p, r, o, stats, scale, dx, ld_dx, dw, ld_dw, status, sm_count, stream);
}

}  // namespace bsq
