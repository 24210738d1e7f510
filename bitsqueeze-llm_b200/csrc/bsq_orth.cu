// Newton-Schulz steps that bring a matrix's singular values near 1:  X_0 = G / (|G| + eps),  A = X X^T,  X <- a X + (b A + c A^2) X, on the side of the shorter dimension
// (X^T X and X (b A + c A^2) where G is tall: nothing is transposed, the products read either orientation).  Three launches a step for all matrices of one shape.
//
// What 16-bit operands cost, and what is done about it (the steps pull small singular values up by 3.4 each, and with them whatever rounding has left there):
//   * FP16, not BF16: entries are bounded, a power of two brings them into its range, and it has three bits more at the same rate;
//   * X is kept as high + low, two FP16 words of 22 bits.  Products read the high part (P X both, where the side is short); a X is added up from both in the epilogue.  With one word the
//     large singular values' rounding is what the small ones start from (rank-8 gradients with noise: 4e-3 off after five steps, this way 1e-4);
//   * the diagonals of A and of P = b A + c A^2, of size 1 where everything else is small, are kept in FP32: what rounding takes from them, and what the
//     products leave out of the low part (P_ii X_low), goes back in the epilogues (noise: 1.9e-3 off without, 0.2e-3 to 0.7e-3 with it; a rounding to BF16 is 1.7e-3).
// Results in FP32 or FP16 take both parts of every operand: three products of halves.  BF16 results of matrices with a short side of up to 128, where launches are what a step costs, are
// bsq_orth_small.cu's.
//
// A and P are symmetric: tiles on and below the diagonal are computed, and written twice.  Bound by the tensor core, then by power, and by whole rounds of tiles: 4096 x 4096 in BF16
// 1.34 ms (A 56 us, P 60, X 112 a step: 136 tiles in two rounds of 74, 256 in four), 14336 x 4096 from FP32 3.7 ms (s^2 l + s^3 + 2 s^2 l counted: 1060 TFLOP/s).  Sides of some hundred by
// 15 launches that wait for one another, some 12 us each.
#include "bsq_gemm16.cuh"
#include "bsq_orth_small.hpp"

#include <algorithm>
#include <cmath>
#include <tuple>
#include <vector>

namespace bsq {
namespace {

constexpr uint64_t kOrthRoom = 1ull << 30;                       // scratch that several matrices share at most
// Stages of a chain of sums (4096 of K, of split operands 1024).  What the tensor core cuts off where a sum's terms have one sign is not of X's rank, and each step pulls it up by 3.4: rank one,
// 65536 x 33000, was 8.8e-3 off in BF16 and 3.1e-2 in FP32 with one chain for all of K, and is 2.8e-3 (its rounding to BF16 is 2e-3 of that) and 1.7e-4.  Up to 6100 of K BF16 has one chain still
template <bool SPLIT> constexpr int kOrthChain = (SPLIT ? 1024 : 4096) / kG16K;
// Short sides up to which P goes with X's low part too, in a second walk along K.  Behind it only P's diagonal does: of rank one that is not of X's rank, and each later step pulls it up by a.
// With Gaussian factors it leaves 0.43 / s beside the rounding of 1.7e-3: 129 x 357 3.7e-3 in all (up to 6e-3) without the second walk, 1.7e-3 with it; 1000 x 1000 1.75e-3 without.
// 129 x 129 112 us without, 116 with it; 300 x 2000 some 3 %, 512 x 1024 142 and 153; 1024 x 4096 would take a fifth more.
constexpr uint64_t kOrthLowSide = 512;
constexpr int kNormThreads = 512;
constexpr uint64_t kNormChunk = 16384;                           // elements of a CTA of the pass that finds the norms, at least
constexpr int kNormParts = kNormThreads;

__device__ __forceinline__ float2 pair_of(unsigned w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
// 16 values in two parts of FP16, two to a word
__device__ __forceinline__ void split16(const float (&v)[16], unsigned (&high)[8], unsigned (&low)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        const float2 f = __half22float2(h);
        high[j] = *reinterpret_cast<const unsigned *>(&h);
        low[j] = pack_pair<kF16>(v[2 * j] - f.x, v[2 * j + 1] - f.y);
    }
}
// 64 floats that all rows of a warp share, two to a lane: asked for with whatever else is on its way (16 bytes at a time where they are used they were waited for four times a box)
struct Shared64 {
    float lo, hi;
    __device__ __forceinline__ void load(const float *p, int count, int lane) {
        lo = lane < count ? p[lane] : 0.0f;
        hi = lane + 32 < count ? p[lane + 32] : 0.0f;
    }
    // element 16 h + j; all lanes together
    __device__ __forceinline__ float at(int h, int j) const { return __shfl_sync(kFullMask, h < 2 ? lo : hi, (16 * h + j) & 31); }
};
__device__ __forceinline__ float high_of(float x) { return __half2float(__float2half_rn(x)); }

// ---- G to X_0 ----
struct OrthIn {
    const void *at[kOrthMost];
    uint64_t ld[kOrthMost];
    bool whole[kOrthMost];           // every row starts on 16 bytes
    unsigned rows, cols;
    int type;
};
// Eight neighbouring elements of a row; those behind its end are 0
template <int TYPE> __device__ __forceinline__ void load8(const OrthIn &in, unsigned row, unsigned col, float (&v)[8]) {
    constexpr int kSize = TYPE == kF32 ? 4 : 2, kWords = 8 * kSize / 4;
    const unsigned char *p = static_cast<const unsigned char *>(in.at[blockIdx.y]) + ((size_t)row * in.ld[blockIdx.y] + col) * kSize;
    if (in.whole[blockIdx.y] && col + 8 <= in.cols) {
        unsigned w[kWords];
#pragma unroll
        for (int i = 0; i < kWords; i += 4) {
            const uint4 q = *reinterpret_cast<const uint4 *>(p + 4 * i);
            w[i] = q.x; w[i + 1] = q.y; w[i + 2] = q.z; w[i + 3] = q.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = TYPE == kF32 ? word_elem<TYPE>(w[j * kWords / 8], 0) : word_elem<TYPE>(w[j / 2], j & 1);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        v[j] = col + j >= in.cols ? 0.0f : word_elem<TYPE>(TYPE == kF32 ? reinterpret_cast<const unsigned *>(p)[j] : (unsigned)reinterpret_cast<const unsigned short *>(p)[j], 0);
}
__device__ __forceinline__ double cta_total(double v, double *room) {
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kFullMask, v, d);
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < kNormThreads / 32; ++i) v += room[i];
    return v;
}
// Squares of eight elements: in FP32 where that is good to 24 bits, else in FP64
__device__ __forceinline__ double squares8(const float (&v)[8]) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
    if (s == 0.0f || (s > 1e-30f && s < 1e36f)) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) any |= v[j] != 0.0f;
        if (s != 0.0f || !any) return (double)s;
    }
    double d = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) d = fma((double)v[j], (double)v[j], d);
    return d;
}
// Sums of squares: blockIdx.x a share of a matrix, blockIdx.y the matrix
template <int TYPE> __global__ void __launch_bounds__(kNormThreads) orth_norm_kernel(const __grid_constant__ OrthIn in, double *parts) {
    chain_begin();
    __shared__ double room[kNormThreads / 32];
    const unsigned per = (in.cols + 7) / 8, all = in.rows * per, step = gridDim.x * kNormThreads;
    double s = 0.0;
    for (unsigned i = blockIdx.x * kNormThreads + threadIdx.x; i < all; i += 4 * step) {
        float v[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const unsigned k = i + u * step, r = k / per;
            if (k < all) load8<TYPE>(in, r, (k - r * per) * 8, v[u]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) s += squares8(v[u]);
    }
    s = cta_total(s, room);
    if (threadIdx.x == 0) parts[blockIdx.y * gridDim.x + blockIdx.x] = s;
}

struct OrthX {
    unsigned short *high, *low;
    unsigned ld;
    uint64_t apart;
    float *factor;                   // X = (high + low) * factor, one for each matrix
};
template <int TYPE> __global__ void __launch_bounds__(kNormThreads) orth_begin_kernel(const __grid_constant__ OrthIn in, const double *parts, int count, double eps, const OrthX x) {
    chain_begin();
    __shared__ double room[kNormThreads / 32];
    const double total = cta_total((int)threadIdx.x < count ? parts[blockIdx.y * (unsigned)count + threadIdx.x] : 0.0, room), norm = sqrt(total);
    // 2^e brings the norm, and so every element, below 2^15; a power of two, so that elements of 16 bits stay what they are
    const bool fine = norm < 3.0e38 * 65536.0 * 65536.0;         // (not: Inf or NaN)
    const int e = norm > 0.0 && fine ? min(max(14 - ilogb(norm), -160), 160) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) x.factor[blockIdx.y] = !fine ? __uint_as_float(0x7fffffffu) : norm > 0.0 ? (float)(ldexp(1.0, -e) / (norm + eps)) : 1.0f;
    const float s0 = exp2f((float)(e / 2)), s1 = exp2f((float)(e - e / 2));
    const unsigned per = x.ld / 8, all = in.rows * per, step = gridDim.x * kNormThreads;
    unsigned short *high = x.high + blockIdx.y * x.apart, *low = x.low + blockIdx.y * x.apart;
    for (unsigned i = blockIdx.x * kNormThreads + threadIdx.x; i < all; i += 2 * step) {
        float v[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned k = i + u * step, r = k / per;
            if (k < all) load8<TYPE>(in, r, (k - r * per) * 8, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned k = i + u * step;
            if (k >= all) break;
            unsigned a[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = v[u][2 * j] * s0 * s1, q = v[u][2 * j + 1] * s0 * s1;
                a[j] = pack_pair<kF16>(p, q);
                b[j] = pack_pair<kF16>(p - high_of(p), q - high_of(q));
            }
            *reinterpret_cast<uint4 *>(high + (size_t)k * 8) = make_uint4(a[0], a[1], a[2], a[3]);
            *reinterpret_cast<uint4 *>(low + (size_t)k * 8) = make_uint4(b[0], b[1], b[2], b[3]);
        }
    }
}

// ---- what the epilogues share ----
// The element of v on the diagonal, where the thread's row has one in these 16 columns
__device__ __forceinline__ int diagonal_at(int row, int col) { return (unsigned)(row - col) < 16u ? row - col : -1; }

struct SymmetricOut {
    CUtensorMap map[2], turned[2];   // boxes of 32 rows x 64 columns of the high and low parts, and of 64 rows x 32 columns (64 bytes a row, not swizzled)
    uint64_t ld;                     // distance of the matrices' diagonals
};
// 64 columns of a symmetric result from `fill(h, v)`, which may read what lies in the boxes, and their mirror image too where they lie below the diagonal, in a box that is
// written column by column
template <bool SPLIT, class Fill> __device__ __forceinline__ void put_symmetric(const TileOut &o, const SymmetricOut &m, int c, bool mirror, const Fill &fill) {
    unsigned w[SPLIT ? 2 : 1][4][8];
    const int col = o.col + c;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        float v[16];
        fill(h, v);
        unsigned low[8];
        split16(v, w[0][h], low);
        box_give16(o, 0, h, w[0][h]);
        if constexpr (SPLIT) {
            box_give16(o, 1, h, low);
#pragma unroll
            for (int j = 0; j < 8; ++j) w[1][h][j] = low[j];
        }
    }
    box_send(o, &m.map[0], col, o.row, o.boxes);
    if constexpr (SPLIT) box_send(o, &m.map[1], col, o.row, o.boxes + kG16Box);
    if (!mirror) return;
    if constexpr (SPLIT) boxes_free(o);
#pragma unroll
    for (int p = 0; p < (SPLIT ? 2 : 1); ++p) {
        unsigned char *turned = o.boxes + (SPLIT ? (unsigned)p : 1u) * kG16Box;
#pragma unroll
        for (int j = 0; j < 64; ++j)
            reinterpret_cast<unsigned short *>(turned)[j * 32 + o.lane] = (unsigned short)(w[p][j >> 4][(j >> 1) & 7] >> ((j & 1) * 16));
        box_send(o, &m.turned[p], o.row, col, turned);
    }
}

// ---- A = X X^T (or X^T X), held times 2^e ----
template <bool SPLIT> struct GramOut {
    SymmetricOut to;
    int M;
    const float *factor;             // of X, one for each matrix, or null
    float constant;                  // ... for all
    float scale;                     // 2^e
    float *rest;                     // what rounding to FP16 takes from the diagonal

    static constexpr bool kChained = false, kBack = false, kTotals = true, kBoxes = true;
    using Ahead = NoAhead;
    template <int COLS> __device__ void ahead(const TileOut &, Ahead &) const {}
    template <int COLS> __device__ void tile(const TileOut &o, Ahead &) const {
        const float x = factor ? factor[o.z] : constant;
        const int row = o.row + o.lane;
        for (int c = 0; c < COLS && o.col + c < M; c += 64) {
            const int col = o.col + c;
            if (col > o.row + 31) continue;                      // above the diagonal: the mirror image of what another warp has
            boxes_free(o);
            put_symmetric<SPLIT>(o, to, c, col + 63 < o.row, [&](int h, float (&v)[16]) {
                read16f(o.taddr + (unsigned)(c + 16 * h), v, o.ok);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = v[j] * x * x * scale;
                if (SPLIT) return;
                const int d = diagonal_at(row, col + 16 * h);
                if (d >= 0 && row < M) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j == d) rest[(size_t)o.z * to.ld + (size_t)row] = v[j] - high_of(v[j]);
                }
            });
        }
    }
};

// ---- P = b A + c A^2, held times 2^e ----
template <bool SPLIT> struct PolyOut {
    SymmetricOut to;
    int M;
    CUtensorMap map[2];              // A's high and low parts
    float b, c;                      // b 2^(e - e_A), c 2^(e - 2 e_A)
    const float *rest;               // of A
    float a, back;                   // 2^-e
    float *of_high, *of_low;         // what the parts of X are multiplied by beside the product: a + what rounding takes from the diagonal of P, a + the diagonal

    static constexpr bool kChained = false, kBack = false, kTotals = true, kBoxes = true;
    struct Ahead {
        float mine;                  // of A's diagonal: the row's, the columns'
        Shared64 theirs;
    };
    __device__ __forceinline__ bool wanted(const TileOut &o, int c) const { return o.col + c < M && o.col + c <= o.row + 31; }
    __device__ __forceinline__ void ask(const TileOut &o, int c, Ahead &n) const {
        boxes_ask(o, &map[0], SPLIT ? &map[1] : nullptr, o.col + c);
        if (!SPLIT) n.theirs.load(rest + (size_t)o.z * to.ld + (size_t)(o.col + c), M - o.col - c, o.lane);
    }
    template <int COLS> __device__ __forceinline__ void ahead(const TileOut &o, Ahead &n) const {
        if (!wanted(o, 0)) return;
        ask(o, 0, n);
        n.mine = !SPLIT && o.row + o.lane < M ? rest[(size_t)o.z * to.ld + (size_t)(o.row + o.lane)] : 0.0f;
    }
    template <int COLS> __device__ __forceinline__ void tile(const TileOut &o, Ahead &n) const {
        const int row = o.row + o.lane;
        const float mine = n.mine;
        for (int at = 0; at < COLS && wanted(o, at); at += 64) {
            const int col = o.col + at;
            if (at) ask(o, at, n);
            const TileOut t = boxes_wait(o);
            put_symmetric<SPLIT>(o, to, at, col + 63 < o.row, [&](int h, float (&v)[16]) {
                const int c0 = col + 16 * h;
                unsigned wp[8], wq[8];
                box_take16(o, 0, h, wp);
                if (SPLIT) box_take16(o, 1, h, wq);
                read16f(o.taddr + (unsigned)(at + 16 * h), v, t.ok);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // A_ij = p + [i = j] rest_i, of which the product has p only
                    const float2 p = pair_of(wp[j]);
                    if (SPLIT) {
                        const float2 q = pair_of(wq[j]);
                        v[2 * j] = fmaf(c, v[2 * j], b * (p.x + q.x));
                        v[2 * j + 1] = fmaf(c, v[2 * j + 1], b * (p.y + q.y));
                    } else {
                        v[2 * j] = fmaf(c, fmaf(p.x, mine + n.theirs.at(h, 2 * j), v[2 * j]), b * p.x);
                        v[2 * j + 1] = fmaf(c, fmaf(p.y, mine + n.theirs.at(h, 2 * j + 1), v[2 * j + 1]), b * p.y);
                    }
                }
                const int d = SPLIT ? -1 : diagonal_at(row, c0);
                if (d >= 0 && row < M) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j == d) {
                            v[j] += mine * fmaf(c, mine, b);
                            of_high[(size_t)o.z * to.ld + (size_t)row] = fmaf(v[j] - high_of(v[j]), back, a);
                            of_low[(size_t)o.z * to.ld + (size_t)row] = fmaf(v[j], back, a);
                        }
                }
            });
        }
    }
};

// ---- X <- a X + P X (or X P) ----
struct OrthOut {
    void *at[kOrthMost];
    uint64_t ld[kOrthMost];
};
template <bool SPLIT> struct StepOut {
    CUtensorMap map[2], next[2];     // X and the next X, high and low
    int M, N;
    bool tall;                       // the diagonal of P goes with the columns
    bool last;
    int type;                        // of the result
    const float *factor;             // of X, one for each matrix, or null
    float constant;                  // ... for all
    float a, back, scale;            // P is held times 1 / back; the next X is held times `scale` (or the result is multiplied by it)
    const float *of_high, *of_low;   // (SPLIT: a)
    uint64_t ld_p;                   // of P: distance of the matrices' diagonals
    OrthOut out;                     // (last)

    static constexpr bool kChained = false, kBack = false, kTotals = true, kBoxes = true;
    struct Ahead {
        float of_sum, of_p, of_q;
        Shared64 e, d;               // (tall: the columns')
    };
    __device__ __forceinline__ void ask(const TileOut &o, int c, Ahead &n) const {
        boxes_ask(o, &map[0], &map[1], o.col + c);
        if (!SPLIT && tall) {
            const size_t k = (size_t)o.z * ld_p + (size_t)(o.col + c);
            n.e.load(of_high + k, N - o.col - c, o.lane);
            n.d.load(of_low + k, N - o.col - c, o.lane);
        }
    }
    template <int COLS> __device__ __forceinline__ void ahead(const TileOut &o, Ahead &n) const {
        ask(o, 0, n);
        const float x = (factor ? factor[o.z] : constant) * scale;
        const int row = o.row + o.lane;
        n.of_sum = x * back;
        n.of_p = n.of_q = SPLIT ? a * x : x;
        if (!SPLIT && !tall && row < M) {
            n.of_p = x * of_high[(size_t)o.z * ld_p + (size_t)row];
            n.of_q = x * of_low[(size_t)o.z * ld_p + (size_t)row];
        }
    }
    // 16 columns of the next X
    __device__ __forceinline__ void values(const TileOut &o, const Ahead &n, int c, int h, float (&v)[16]) const {
        unsigned wp[8], wq[8];
        box_take16(o, 0, h, wp);
        box_take16(o, 1, h, wq);
        read16f(o.taddr + (unsigned)(c + 16 * h), v, o.ok);
        if (!SPLIT && tall) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 p = pair_of(wp[j]), q = pair_of(wq[j]);
                v[2 * j] = fmaf(n.of_p, fmaf(n.e.at(h, 2 * j), p.x, n.d.at(h, 2 * j) * q.x), n.of_sum * v[2 * j]);
                v[2 * j + 1] = fmaf(n.of_p, fmaf(n.e.at(h, 2 * j + 1), p.y, n.d.at(h, 2 * j + 1) * q.y), n.of_sum * v[2 * j + 1]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 p = pair_of(wp[j]), q = pair_of(wq[j]);
                v[2 * j] = fmaf(n.of_p, p.x, fmaf(n.of_q, q.x, n.of_sum * v[2 * j]));
                v[2 * j + 1] = fmaf(n.of_p, p.y, fmaf(n.of_q, q.y, n.of_sum * v[2 * j + 1]));
            }
        }
    }

    template <int COLS> __device__ __forceinline__ void tile(const TileOut &o, Ahead &n) const {
        for (int c = 0; c < COLS && o.col + c < N; c += 64) {
            const int col = o.col + c;
            if (c) ask(o, c, n);
            const TileOut t = boxes_wait(o);
            if (!last) {
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    float v[16];
                    unsigned p[8], q[8];
                    values(t, n, c, h, v);
                    split16(v, p, q);
                    box_give16(o, 0, h, p);
                    box_give16(o, 1, h, q);
                }
                box_send(o, &next[0], col, o.row, o.boxes);
                box_send(o, &next[1], col, o.row, o.boxes + kG16Box);
                continue;
            }
            const long ld_out = (long)out.ld[o.z];
            if (type == kF32) {
                // (32 columns to a box: both are read before one is written)
                float v[4][16];
#pragma unroll
                for (int h = 0; h < 4; ++h) values(t, n, c, h, v[h]);
#pragma unroll
                for (int h = 0; h < 4; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *box_piece(o, h >> 1, 4 * (h & 1) + j) =
                            make_uint4(__float_as_uint(v[h][4 * j]), __float_as_uint(v[h][4 * j + 1]), __float_as_uint(v[h][4 * j + 2]), __float_as_uint(v[h][4 * j + 3]));
                box_out_rows(o.boxes, o.lane, out.at[o.z], 4, (long)o.row * ld_out + col, ld_out, M - o.row, N - col);
                if (col + 32 < N) box_out_rows(o.boxes + kG16Box, o.lane, out.at[o.z], 4, (long)o.row * ld_out + col + 32, ld_out, M - o.row, N - col - 32);
                continue;
            }
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float v[16];
                values(t, n, c, h, v);
                if (type == kBf16) box_put16<kBf16>(o.boxes, o.lane, h, v);
                else box_put16<kF16>(o.boxes, o.lane, h, v);
            }
            box_out_rows(o.boxes, o.lane, out.at[o.z], 2, (long)o.row * ld_out + col, ld_out, M - o.row, N - col);
        }
    }
};

// ---- host ----
// Powers of two that X, A and P of a step are held times: largest magnitudes below 2^15
struct StepScale {
    int x, a, p;
    double most;                     // the largest singular value that X may have
};
int below_2_15(double most) { return std::min(24, std::max(-14, most > 0.0 ? (int)std::floor(std::log2(32768.0 / most)) : 14)); }
// Largest singular value that each step may meet, from 0 .. 1 at the start; false: it grows beyond 1000
// (the polynomials are smooth: 256 points are within 1e-4 of their largest values, for which the scales leave a factor of two)
constexpr int kPoints = 256;
bool scales_of(const float *k, int steps, std::vector<StepScale> *out) {
    double most = 1.0;
    for (int i = 0; i < steps; ++i, k += 3) {
        const double a = k[0], b = k[1], c = k[2];
        if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
        double next = 0.0, p = 0.0;
        const double top = most * 1.02;                          // (room for what rounding adds)
        for (int j = 0; j <= kPoints; ++j) {
            const double s = top * j / kPoints, l = s * s, y = b * l + c * l * l;
            p = std::max(p, std::fabs(y));
            next = std::max(next, std::fabs((a + y) * s));
        }
        if (!(next < 1000.0) || !(p < 1e6)) return false;
        out->push_back({below_2_15(top), below_2_15(top * top), below_2_15(p), top});
        most = std::max(next, 1e-30);
    }
    return true;
}

struct Group {
    int begin, count;                // in the order of `order`
};
// Matrices of one shape and type, as many as share a launch
struct Plan {
    std::vector<int> order;
    std::vector<Group> groups;
};
enum Way { kHigh, kSplit, kSmall };                              // products of the high parts, of both parts; few rows or columns
// tame: the steps' polynomial stays within what its coefficients may grow by (small_steps)
Way way_of(const OrthMatrix &m, int out_type, bool tame) {
    if (out_type != kBf16) return kSplit;
    return std::min(m.rows, m.cols) > (uint64_t)kOrthSmallSide ? kHigh : tame ? kSmall : kSplit;
}

struct Room {
    unsigned short *high[2], *low[2], *a[2], *p[2];
    float *factor, *rest, *of_high, *of_low;
    double *parts;
    OrthSmallRoom small;
    uint64_t ld_x, apart_x, ld_a, apart_a;
    size_t bytes;
};
Room room_of(const OrthMatrix &m, Way way, int count, void *scratch) {
    Room r = {};
    Scratch room = {static_cast<unsigned char *>(scratch)};
    const uint64_t s = std::min(m.rows, m.cols), n = (uint64_t)count;
    r.parts = room.take<double>(n * kNormParts);
    if (way == kSmall) {
        r.small.slices = orth_small_slices(std::max(m.rows, m.cols), &r.small.per);
        r.small.sums = room.take<float>(n * (uint64_t)r.small.slices * s * s);
        r.small.sum = room.take<float>(n * s * s);
        r.small.r = room.take<float>(n * s * s);
        r.small.identity = room.take<float>(n);
        r.bytes = room.used;
        return r;
    }
    r.ld_x = padded(m.cols, 16);
    r.apart_x = m.rows * r.ld_x;
    r.ld_a = padded(s, 16);
    r.apart_a = s * r.ld_a;
    for (int i = 0; i < 2; ++i) {
        r.high[i] = room.take<unsigned short>(n * r.apart_x);
        r.low[i] = room.take<unsigned short>(n * r.apart_x);
    }
    for (int i = 0; i < (way == kSplit ? 2 : 1); ++i) {
        r.a[i] = room.take<unsigned short>(n * r.apart_a);
        r.p[i] = room.take<unsigned short>(n * r.apart_a);
    }
    r.factor = room.take<float>(n);
    r.rest = room.take<float>(n * r.ld_a);
    r.of_high = room.take<float>(n * r.ld_a);
    r.of_low = room.take<float>(n * r.ld_a);
    r.bytes = room.used;
    return r;
}

// Scratch of matrices whatever the steps are
size_t room_for(const OrthMatrix &m, int out_type, int count) {
    return std::max(room_of(m, way_of(m, out_type, true), count, nullptr).bytes, room_of(m, way_of(m, out_type, false), count, nullptr).bytes);
}

Plan plan_of(const OrthCall &c) {
    Plan p;
    for (int i = 0; i < c.n; ++i)
        if (c.m[i].rows && c.m[i].cols) p.order.push_back(i);
    const auto key = [&](int i) { return std::make_tuple(c.m[i].rows, c.m[i].cols, c.m[i].type); };
    std::stable_sort(p.order.begin(), p.order.end(), [&](int i, int j) { return key(i) < key(j); });
    for (int i = 0; i < (int)p.order.size();) {
        const OrthMatrix &m = c.m[p.order[i]];
        const uint64_t one = room_for(m, c.out_type, 1);
        const int most = (int)std::min<uint64_t>(kOrthMost, std::max<uint64_t>(1, kOrthRoom / one));
        int n = 1;
        while (n < most && i + n < (int)p.order.size() && key(p.order[i + n]) == key(p.order[i])) ++n;
        p.groups.push_back({i, n});
        i += n;
    }
    return p;
}

// (boxes are of whole rows of `ld`: a store never ends inside 16 bytes; what lies behind the last column is not read by a product)
bool box_maps(CUtensorMap (&map)[2], unsigned short *high, unsigned short *low, uint64_t rows, uint64_t ld, uint64_t count, uint64_t apart) {
    return map_stack(&map[0], {high, ld, rows, ld, count, apart}, kF16, 64, 32) && map_stack(&map[1], {low, ld, rows, ld, count, apart}, kF16, 64, 32);
}
bool symmetric_out(SymmetricOut *m, unsigned short *high, unsigned short *low, uint64_t s, uint64_t ld, uint64_t count, uint64_t apart) {
    m->ld = ld;
    return box_maps(m->map, high, low, s, ld, count, apart) && map_stack(&m->turned[0], {high, ld, s, ld, count, apart}, kF16, 32, 64, CU_TENSOR_MAP_SWIZZLE_NONE) &&
           map_stack(&m->turned[1], {low, ld, s, ld, count, apart}, kF16, 32, 64, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// The norms of a group's matrices, as parts of their sums of squares
cudaError_t norms_of(const OrthMatrix *const *m, int count, OrthIn *in, double *sums, unsigned *parts, cudaStream_t stream) {
    *in = {};
    in->rows = (unsigned)m[0]->rows;
    in->cols = (unsigned)m[0]->cols;
    in->type = m[0]->type;
    const uint64_t size = (uint64_t)op_bytes(in->type);
    for (int i = 0; i < count; ++i) {
        in->at[i] = m[i]->in;
        in->ld[i] = m[i]->ld_in;
        in->whole[i] = (reinterpret_cast<uintptr_t>(in->at[i]) | (in->rows > 1 ? in->ld[i] * size : 0)) % 16 == 0;
    }
    *parts = (unsigned)std::min<uint64_t>(kNormParts, (m[0]->rows * m[0]->cols + kNormChunk - 1) / kNormChunk);      // (by the matrix alone: its sum is the same whatever goes with it)
    const dim3 grid(*parts, (unsigned)count);
    return in->type == kF32    ? launch_chained(orth_norm_kernel<kF32>, grid, kNormThreads, 0, stream, *in, sums)
           : in->type == kBf16 ? launch_chained(orth_norm_kernel<kBf16>, grid, kNormThreads, 0, stream, *in, sums)
                               : launch_chained(orth_norm_kernel<kF16>, grid, kNormThreads, 0, stream, *in, sums);
}

// A step's operands and what they are held times, from bounds of A, N, M = a I + N and the Q = q I + R that has come together; false where Q may grow beyond 1024: rounding grows with its
// square, and where X has nothing Q still grows (five steps of the usual coefficients: 485)
bool small_steps(const OrthCall &c, const std::vector<StepScale> &scales, OrthSmallSteps *out) {
    out->steps = c.steps;
    double most = 1.0, q = 1.0;                                  // of Q
    int of_r = 0;                                                // R is held times 2^of_r
    for (int i = 0; i < c.steps; ++i) {
        const double a = c.coefficients[3 * i], b = c.coefficients[3 * i + 1], k = c.coefficients[3 * i + 2], top = scales[(size_t)i].most;
        const bool last = i + 1 == c.steps;
        double m = 0.0, n = 0.0;
        for (int j = 0; j <= kPoints; ++j) {
            const double l = top * top * j / kPoints, y = b * l + k * l * l;
            m = std::max(m, std::fabs(a + y));
            n = std::max(n, std::fabs(y));
        }
        const int at = below_2_15(top * top), an = below_2_15(n), t = below_2_15(m * top * top);
        const int next_a = last ? 0 : below_2_15(scales[(size_t)i + 1].most * scales[(size_t)i + 1].most);
        most *= m;
        if (!(most <= 1024.0)) return false;
        const int next_r = last ? 0 : below_2_15(most + std::fabs(q * a));
        const float scale = last ? c.scale : 1.0f;
        OrthSmallStep &s = out->step[i];
        s.a = at;
        s.square = std::ldexp((float)k, an - 2 * at);
        s.linear = std::ldexp((float)b, an - at);
        s.first_r = std::ldexp(scale, next_r - an);
        s.r_product = std::ldexp(scale, next_r - an - of_r);
        s.r_self = std::ldexp(scale * (float)a, next_r - of_r);
        s.r_n = std::ldexp(scale * (float)q, next_r - an);
        s.t_product = std::ldexp(1.0f, t - an - at);
        s.t_self = std::ldexp((float)a, t - at);
        s.a_product = std::ldexp(1.0f, next_a - an - t);
        s.a_self = std::ldexp((float)a, next_a - t);
        of_r = next_r;
        q *= a;
    }
    out->identity = (float)(c.scale * q);
    return true;
}

cudaError_t run_small(const OrthCall &c, const OrthSmallSteps &steps, const OrthMatrix *const *m, int count, void *scratch, unsigned *status, cudaStream_t stream) {
    const uint64_t rows = m[0]->rows, cols = m[0]->cols;
    const Room r = room_of(*m[0], kSmall, count, scratch);
    OrthIn in;
    unsigned parts;
    const cudaError_t err = norms_of(m, count, &in, r.parts, &parts, stream);
    if (err != cudaSuccess) return err;
    OrthSmall g = {};
    for (int i = 0; i < count; ++i) {
        g.in[i] = m[i]->in;
        g.out[i] = m[i]->out;
        g.ld[i] = m[i]->ld_in;
        g.ld_out[i] = m[i]->ld_out;
    }
    g.s = (int)std::min(rows, cols);
    g.l = (int)std::max(rows, cols);
    g.parts = r.parts;
    g.part_count = (int)parts;
    g.eps = c.eps;
    return orth_small(g, rows > cols, in.type, steps, count, r.small, status, stream);
}

template <bool SPLIT>
cudaError_t run_group(const OrthCall &c, const std::vector<StepScale> &scales, const OrthMatrix *const *m, int count, void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    const uint64_t rows = m[0]->rows, cols = m[0]->cols, s = std::min(rows, cols);
    const bool tall = rows > cols, low = !SPLIT && s <= kOrthLowSide;
    const Room r = room_of(*m[0], SPLIT ? kSplit : kHigh, count, scratch);
    OrthIn in;
    OrthOut out = {};
    for (int i = 0; i < count; ++i) {
        out.at[i] = m[i]->out;
        out.ld[i] = m[i]->ld_out;
    }
    unsigned parts;
    cudaError_t err = norms_of(m, count, &in, r.parts, &parts, stream);
    if (err != cudaSuccess) return err;
    const unsigned blocks = (unsigned)std::min<uint64_t>((uint64_t)std::max(1, sm_count * 4 / count), (rows * r.ld_x / 8 + kNormThreads * 2 - 1) / (kNormThreads * 2));
    const OrthX x0 = {r.high[0], r.low[0], (unsigned)r.ld_x, r.apart_x, r.factor};
    const dim3 grid(blocks, (unsigned)count);
    err = in.type == kF32    ? launch_chained(orth_begin_kernel<kF32>, grid, kNormThreads, 0, stream, in, (const double *)r.parts, (int)parts, c.eps, x0)
          : in.type == kBf16 ? launch_chained(orth_begin_kernel<kBf16>, grid, kNormThreads, 0, stream, in, (const double *)r.parts, (int)parts, c.eps, x0)
                             : launch_chained(orth_begin_kernel<kF16>, grid, kNormThreads, 0, stream, in, (const double *)r.parts, (int)parts, c.eps, x0);
    if (err != cudaSuccess) return err;

    SymmetricOut to_a, to_p;
    if (!symmetric_out(&to_a, r.a[0], r.a[SPLIT], s, r.ld_a, (uint64_t)count, r.apart_a) || !symmetric_out(&to_p, r.p[0], r.p[SPLIT], s, r.ld_a, (uint64_t)count, r.apart_a))
        return cudaErrorInvalidValue;
    Gemm16 g = {};
    g.batch = count;
    g.splits = 1;
    g.parts = SPLIT ? 3 : 1;
    g.chain = kOrthChain<SPLIT>;
    const bool pairs_s = g16_pairs(s, s, (uint64_t)count, true, sm_count), pairs_x = g16_pairs(rows, cols, (uint64_t)count, false, sm_count);
    for (int step = 0; step < c.steps; ++step) {
        const int now = step & 1;
        const bool last = step + 1 == c.steps;
        const StepScale &k = scales[(size_t)step];
        const float *co = c.coefficients + 3 * step;
        const float *factor = step == 0 ? r.factor : nullptr;
        const float constant = std::ldexp(1.0f, -k.x);
        Gemm16Maps ops;
        // A
        for (int i = 0; i < 2; ++i) {
            const Stack x = {i && SPLIT ? r.low[now] : r.high[now], cols, rows, r.ld_x, (uint64_t)count, r.apart_x};
            if (!map_operand(&ops.a[i], x, false, !tall)) return cudaErrorInvalidValue;
            ops.b[i] = ops.a[i];
        }
        g.M = g.N = (int)s;
        g.lower = true;
        g.a_kmajor = g.b_kmajor = !tall;
        GramOut<SPLIT> gram = {to_a, (int)s, factor, constant, std::ldexp(1.0f, k.a), r.rest};
        if ((err = launch_gemm16(ops, gram, g, std::max(rows, cols), pairs_s, status, sm_count, stream)) != cudaSuccess) return err;
        // P
        for (int i = 0; i < 2; ++i) {
            const Stack a = {r.a[SPLIT ? i : 0], s, s, r.ld_a, (uint64_t)count, r.apart_a};
            if (!map_operand(&ops.a[i], a, false, true)) return cudaErrorInvalidValue;
            ops.b[i] = ops.a[i];
        }
        g.a_kmajor = g.b_kmajor = true;
        PolyOut<SPLIT> poly = {to_p, (int)s, {to_a.map[0], to_a.map[1]}, std::ldexp(co[1], k.p - k.a), std::ldexp(co[2], k.p - 2 * k.a), r.rest,
                               co[0], std::ldexp(1.0f, -k.p), r.of_high, r.of_low};
        if ((err = launch_gemm16(ops, poly, g, s, pairs_s, status, sm_count, stream)) != cudaSuccess) return err;
        // X
        for (int i = 0; i < 2; ++i) {
            const Stack p = {r.p[SPLIT ? i : 0], s, s, r.ld_a, (uint64_t)count, r.apart_a}, x = {i && (SPLIT || low) ? r.low[now] : r.high[now], cols, rows, r.ld_x, (uint64_t)count, r.apart_x};
            if (!map_operand(tall ? &ops.b[i] : &ops.a[i], p, false, true) || !map_operand(tall ? &ops.a[i] : &ops.b[i], x, false, tall)) return cudaErrorInvalidValue;
        }
        const Gemm16 one = g;
        if (low) {
            g.parts = 2;
            g.low_a = tall;
        }
        g.M = (int)rows;
        g.N = (int)cols;
        g.lower = false;
        g.a_kmajor = true;
        g.b_kmajor = tall;
        StepOut<SPLIT> e = {};
        if (!box_maps(e.map, r.high[now], r.low[now], rows, r.ld_x, (uint64_t)count, r.apart_x) ||
            !box_maps(e.next, r.high[now ^ 1], r.low[now ^ 1], rows, r.ld_x, (uint64_t)count, r.apart_x))
            return cudaErrorInvalidValue;
        e.M = (int)rows;
        e.N = (int)cols;
        e.tall = tall;
        e.last = last;
        e.type = c.out_type;
        e.factor = factor;
        e.constant = constant;
        e.a = co[0];
        e.back = std::ldexp(1.0f, -k.p);
        e.scale = last ? c.scale : std::ldexp(1.0f, scales[(size_t)step + 1].x);
        e.of_high = r.of_high;
        e.of_low = low ? r.of_high : r.of_low;
        e.ld_p = r.ld_a;
        e.out = out;
        if ((err = launch_gemm16(ops, e, g, s, pairs_x, status, sm_count, stream)) != cudaSuccess) return err;
        g = one;
    }
    return cudaSuccess;
}

}  // namespace

bool orth_steps_ok(const float *coefficients, int steps) {
    std::vector<StepScale> scales;
    return scales_of(coefficients, steps, &scales);
}

size_t orth_scratch_bytes(const OrthCall &c) {
    size_t most = 0;
    const Plan p = plan_of(c);
    for (const Group &g : p.groups) {
        const OrthMatrix &m = c.m[p.order[(size_t)g.begin]];
        most = std::max(most, room_for(m, c.out_type, g.count));
    }
    return most;
}

cudaError_t orthogonalize(const OrthCall &c, void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    std::vector<StepScale> scales;
    if (!scales_of(c.coefficients, c.steps, &scales)) return cudaErrorInvalidValue;
    OrthSmallSteps steps;
    const bool tame = small_steps(c, scales, &steps);
    const Plan p = plan_of(c);
    for (const Group &g : p.groups) {
        const OrthMatrix *m[kOrthMost];
        for (int i = 0; i < g.count; ++i) m[i] = &c.m[p.order[(size_t)(g.begin + i)]];
        const Way way = way_of(*m[0], c.out_type, tame);
        const cudaError_t err = way == kSmall   ? run_small(c, steps, m, g.count, scratch, status, stream)
                                : way == kSplit ? run_group<true>(c, scales, m, g.count, scratch, status, sm_count, stream)
                                                : run_group<false>(c, scales, m, g.count, scratch, status, sm_count, stream);
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace bsq
