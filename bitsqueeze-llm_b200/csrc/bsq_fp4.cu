// Quantisation to and from microscaled 4-bit matrices (bsq_fp4.hpp has the formats and the packed form).
//
// quantise:  block b of a row: m = max |x|.  MXFP4: s = 2^(floor(log2 m) - 2), at least 2^-127.  NVFP4: s = e4m3((m / g) fl(1/6)) g with the
// matrix scale g = 2^t, t from the largest magnitude of the matrix, and fl(1/6) the FP32 number nearest to 1/6.  Codes: x / s to the nearest e2m1, ties to even, saturated at 6.
// A block with an Inf or NaN gets the scale NaN and codes 0, so that whatever reads it says so; the matrix scale goes by the finite elements.
//
// x / s: MXFP4 multiplies by a power of two, exact.  NVFP4 takes q0 = x * (1/s), r = q0 s - x (exact in the fma), q = q0 - r * (1/s), which is
// x / s correctly rounded; a correctly rounded quotient lies on the same side of a halfway point of e2m1 as the quotient itself
// (halfway point times s has 7 bits: an x beside it is at least 2^-24 of itself away, more than half a step of the quotient there).
// q0 alone is one step off for some s (15 * 0.125 against 5: 5.0000005), and a tie then goes the wrong way.  The block scale is defined by the FP32 product instead: for
// 16-bit elements that is the nearest E4M3 to m / (6 g) all the same (a tie, m / g = 6 h with a halfway point h, gives h (1 + 2^-25), which rounds to h, and
// the next m is 2^-11 away); an FP32 m beside a tie may go with it, to a scale that is as near to 2^-24.
//
// Bound by memory: 4096 x 14336 in BF16 is read once for the matrix scale and once for the codes (MXFP4: once).  A thread
// takes 32 columns (16 bytes of codes); a warp's lanes are 8 such units of 4 rows that lie 32 apart, because those are the
// rows whose scales are neighbours in the packed form.  4096 x 14336 BF16: MXFP4 24.3 us (154 MB, 6.3 TB/s), NVFP4 43.4 (two passes over 117 MB), back to BF16
// 27 (5.6 TB/s).  The NVFP4 quantiser executes 10 instructions an element and issues in 0.68 of the clocks, so it is not far from that bound either.
#include "bsq_fp4.cuh"
#include "bsq_internal.hpp"

#include <atomic>

namespace bsq {
namespace {

constexpr int kThreads = 256, kUnits = 8;                        // threads of a CTA; units of 32 columns in a warp's tile
enum : int { kNoAmax = 0, kGivenAmax, kPartialAmax, kOwnAmax };  // where the largest magnitude of the matrix comes from

// Largest finite magnitude of `n` consecutive elements, as a word of magnitudes: this thread's share of `threads`.
template <int TYPE> __device__ unsigned absmax_span(const unsigned char *p, uint64_t n, uint64_t me, uint64_t threads) {
    using W = Words<TYPE>;
    constexpr int kSize = TYPE == kF32 ? 4 : 2, kVec = 16 / kSize;
    unsigned acc = 0;
    auto one = [&](uint64_t i) {
        const unsigned w = TYPE == kF32 ? reinterpret_cast<const unsigned *>(p)[i] : reinterpret_cast<const unsigned short *>(p)[i];
        acc = W::larger(acc, W::drop(w));
    };
    uint64_t head = ((16u - (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / kSize;
    if (head > n) head = n;
    if (me < head) one(me);
    const uint4 *v = reinterpret_cast<const uint4 *>(p + head * kSize);
    const uint64_t vecs = (n - head) / kVec;
    for (uint64_t i = me; i < vecs; i += 4 * threads) {          // (four loads in flight, also at the end)
        unsigned w[16], m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint4 a = i + j * threads < vecs ? v[i + j * threads] : make_uint4(0u, 0u, 0u, 0u);
            w[4 * j] = a.x; w[4 * j + 1] = a.y; w[4 * j + 2] = a.z; w[4 * j + 3] = a.w;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) m = W::larger(m, w[j]);
        if (not_finite<TYPE>(m)) {                               // without what is not finite
            m = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) m = W::larger(m, W::drop(w[j]));
        }
        acc = W::larger(acc, m);
    }
    for (uint64_t t = head + vecs * kVec + me; t < n; t += threads) one(t);
    return acc;
}

// ... of a matrix: contiguous ones as one span, others a row per warp
template <int TYPE> __device__ float absmax_share(const unsigned char *x, uint64_t rows, uint64_t cols, uint64_t ld, uint64_t cta, uint64_t ctas) {
    constexpr int kSize = TYPE == kF32 ? 4 : 2;
    unsigned acc = 0;
    if (ld == cols || rows == 1) {
        acc = absmax_span<TYPE>(x, rows * cols, cta * blockDim.x + threadIdx.x, ctas * blockDim.x);
    } else {
        const unsigned warps = blockDim.x >> 5;
        for (uint64_t r = cta * warps + (threadIdx.x >> 5); r < rows; r += ctas * warps)
            acc = Words<TYPE>::larger(acc, absmax_span<TYPE>(x + r * ld * kSize, cols, threadIdx.x & 31, 32));
    }
    return Words<TYPE>::top(acc);
}

__device__ __forceinline__ float cta_max(float v) {
    __shared__ float part[32];
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = part[0];
    for (unsigned i = 1; i < (blockDim.x >> 5); ++i) m = fmaxf(m, part[i]);
    return m;
}

template <int TYPE>
__global__ void __launch_bounds__(512) fp4_absmax_kernel(const unsigned char *x, uint64_t rows, uint64_t cols, uint64_t ld, float *partials) {
    chain_begin();
    const float m = cta_max(absmax_share<TYPE>(x, rows, cols, ld, blockIdx.x, gridDim.x));
    if (threadIdx.x == 0) partials[blockIdx.x] = m;
}

struct QuantArgs {
    const unsigned char *x;
    uint64_t rows, cols, ld;             // ld in elements
    uint8_t *packed;
    const float *amax;                   // given, or partial maxima
    int partials;
    unsigned chunks, blocks;             // tasks: column chunks (kUnits x unit_run units of 32), row blocks (32 rows: 8 by 4 that lie 32 apart)
};
// Units of 32 columns that a thread has in a task: two where a row is read straight into registers and they are 16 words, for more loads in flight and
// less arithmetic on addresses
__host__ __device__ constexpr int unit_run(int type, int word) { return word == 32 && type != kF32 ? 2 : 1; }

// x / d correctly rounded from r, 1 / d correctly rounded: the residual of x r is exact in the fma, and one step with it rounds as the quotient does (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", IBM J. Res. Dev. 34 (1990), theorem 8.3)
__device__ __forceinline__ float divide_by(float x, float d, float r) {
    const float q0 = x * r, e = __fmaf_rn(q0, d, -x);
    return __fmaf_rn(-e, r, q0);                                 // (signs this way round: -0 stays -0)
}
// 32 columns in words -> codes and scale bytes (MXFP4: one, NVFP4: two, the first in the low byte).
// table (NVFP4): the value of every E4M3 byte and its reciprocal (0 for 0), correctly rounded
template <int FMT, int TYPE, bool CLAMP>
__device__ __forceinline__ void quantise_unit(const unsigned *w, float g, float ginv, const float2 *table, uint4 *codes, unsigned *bytes) {
    using W = Words<TYPE>;
    constexpr int kBlocks = FMT == kMxFp4 ? 1 : 2, kElems = 32 / kBlocks, kWordsPer = kElems / W::kPer;
    unsigned out[4];
    *bytes = 0;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < kWordsPer; ++i) top = W::larger(top, w[b * kWordsPer + i]);
        const bool bad = not_finite<TYPE>(top);
        const float amax = W::top(top);
        unsigned byte;
        float s, inv, lim = 3.402823466e+38f;
        if (FMT == kMxFp4) {
            byte = (unsigned)max((int)(__float_as_uint(amax) >> 23) - 2, 0);
            s = 0.0f;
            inv = __uint_as_float((254u - byte) << 23);
        } else {
            const float u = CLAMP ? fminf(amax * ginv, 65536.0f) : amax * ginv;
            byte = ue4m3_byte(u * (1.0f / 6.0f));
            const float2 e = table[byte];
            s = e.x * g;
            inv = e.y * ginv;
            if (CLAMP && u > 2688.0f) lim = 2688.0f * g;         // above the given largest magnitude: saturates (and 1/s times x may not overflow)
        }
        if (bad) {
            byte = FMT == kMxFp4 ? 255u : 127u;
            inv = 0.0f;
        }
        *bytes |= byte << (8 * b);
#pragma unroll
        for (int o = 0; o < kElems / 8; ++o) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = o * 8 + e;
                float x = word_elem<TYPE>(w[b * kWordsPer + at / W::kPer], at % W::kPer);
                if (FMT == kMxFp4) {
                    v[e] = x * inv;
                } else {
                    if (CLAMP) x = fminf(fmaxf(x, -lim), lim);
                    v[e] = divide_by(x, s, inv);
                }
            }
            out[b * (kElems / 8) + o] = bad ? 0u : e2m1_pack8(v);
        }
    }
    *codes = make_uint4(out[0], out[1], out[2], out[3]);
}

template <int WORD> struct Piece { typedef unsigned type; };
template <> struct Piece<8> { typedef uint2 type; };
template <> struct Piece<2> { typedef unsigned short type; };
// Piece p of a row, of which `live` elements from its start on are there; zeros behind them
template <int WORD, int SIZE> __device__ __forceinline__ typename Piece<WORD>::type load_piece(const unsigned char *src, int p, int live) {
    constexpr int kElems = WORD / SIZE;
    typename Piece<WORD>::type v = {};
    if (live >= kElems) return reinterpret_cast<const typename Piece<WORD>::type *>(src)[p];
    if constexpr (kElems > 1) {
        unsigned char *b = reinterpret_cast<unsigned char *>(&v);
#pragma unroll
        for (int i = 0; i < kElems; ++i)
            if (i < live) {
                if (SIZE == 4) *reinterpret_cast<unsigned *>(b + 4 * i) = reinterpret_cast<const unsigned *>(src + (size_t)p * WORD)[i];
                else *reinterpret_cast<unsigned short *>(b + 2 * i) = reinterpret_cast<const unsigned short *>(src + (size_t)p * WORD)[i];
            }
    }
    return v;
}
template <int WORD, int SIZE> __device__ __forceinline__ void store_piece(unsigned char *dst, int p, int live, const typename Piece<WORD>::type &v) {
    constexpr int kElems = WORD / SIZE;
    if (live >= kElems) {
        reinterpret_cast<typename Piece<WORD>::type *>(dst)[p] = v;
    } else if constexpr (kElems > 1) {
        const unsigned char *b = reinterpret_cast<const unsigned char *>(&v);
#pragma unroll
        for (int i = 0; i < kElems; ++i)
            if (i < live) {
                if (SIZE == 4) reinterpret_cast<unsigned *>(dst + (size_t)p * WORD)[i] = *reinterpret_cast<const unsigned *>(b + 4 * i);
                else reinterpret_cast<unsigned short *>(dst + (size_t)p * WORD)[i] = *reinterpret_cast<const unsigned short *>(b + 2 * i);
            }
    }
}

// WORD: bytes of the pieces that rows are read in: 32 where every row starts on 32 bytes (straight into the thread's registers), else 8, 4 or 2,
// neighbouring lanes neighbouring pieces, handed out through shared memory (unit stride + 16 bytes: no bank conflicts).
template <int FMT, int TYPE, int WORD, int AMAX>
__global__ void __launch_bounds__(kThreads) fp4_quantize_kernel(const QuantArgs g) {
    chain_begin();
    constexpr int kSize = TYPE == kF32 ? 4 : 2, kWords = 32 * kSize / 4, kUnitStride = 32 * kSize + 16;
    extern __shared__ __align__(16) unsigned char stage[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, unit = lane & 7;
    float scale = 1.0f, inv = 1.0f;
    __shared__ float2 table[FMT == kNvFp4 ? 128 : 1];
    if (FMT == kNvFp4) {
        if (threadIdx.x < 128) {
            const float s = e4m3_decode(threadIdx.x);
            table[threadIdx.x] = make_float2(s, threadIdx.x ? __fdiv_rn(1.0f, s) : 0.0f);
        }
        __syncthreads();
    }
    if (AMAX != kNoAmax) {
        float m;
        if (AMAX == kGivenAmax) {
            m = *g.amax;
        } else if (AMAX == kPartialAmax) {
            m = 0.0f;
            for (int i = threadIdx.x; i < g.partials; i += kThreads) m = fmaxf(m, g.amax[i]);
            m = cta_max(m);
        } else {
            m = cta_max(absmax_share<TYPE>(g.x, g.rows, g.cols, g.ld, 0, 1));
        }
        const int t = nvfp4_matrix_exp(m);
        scale = pow2f(t);
        inv = pow2f(-t);
    }
    if (blockIdx.x == 0 && threadIdx.x < kFp4Head / 4) reinterpret_cast<float *>(g.packed)[threadIdx.x] = threadIdx.x == 0 ? scale : 0.0f;
    const uint64_t ldc = fp4_ld(g.cols), quads = fp4_quads(FMT, g.cols), units = quads * (FMT == kMxFp4 ? 4 : 2);
    uint8_t *codes = g.packed + kFp4Head, *scales = g.packed + fp4_scales_at(g.rows, g.cols);
    constexpr int kRun = unit_run(TYPE, WORD), kTile = kUnits * kRun;                     // units of a thread; of a row of a warp's tile
    const unsigned by = gridDim.x / g.chunks, on = gridDim.x - by * g.chunks;            // from one task to the next: row blocks, chunks
    unsigned nb = blockIdx.x / g.chunks, nc = blockIdx.x - nb * g.chunks;
    for (; nb < g.blocks; nb += by, nc += on) {
        if (nc >= g.chunks) {
            nc -= g.chunks;
            if (++nb >= g.blocks) break;
        }
        // behind a pass that has just read the matrix from its start to its end: the other way round, what was read last comes from the L2
        const unsigned block = AMAX == kPartialAmax ? g.blocks - 1 - nb : nb;
        const uint64_t first = (uint64_t)(AMAX == kPartialAmax ? g.chunks - 1 - nc : nc) * kTile;
        const unsigned r0 = (block & 3) * 8 + warp;                                       // row in its group, first of four
        const uint64_t group = block >> 2, row = group * 128 + r0 + 32 * sub;
        unsigned w[kRun][kWords];
        if constexpr (WORD == 32) {
            const unsigned char *src = g.x + (row * g.ld + (first + unit) * 32) * kSize;
#pragma unroll
            for (int j = 0; j < kRun; ++j, src += 256 * kSize) {
                const uint64_t col = (first + unit + 8 * j) * 32;
                const int have = row < g.rows && col < g.cols ? (int)min((uint64_t)32, g.cols - col) : 0;   // columns of this thread
                if (have == 32) {
#pragma unroll
                    for (int i = 0; i < kWords; i += 8) ld_words8(src + i * 4, *reinterpret_cast<unsigned(*)[8]>(&w[j][i]));
                } else {
#pragma unroll
                    for (int i = 0; i < kWords; ++i) {
                        w[j][i] = 0;
                        if (TYPE == kF32) {
                            if (i < have) w[j][i] = reinterpret_cast<const unsigned *>(src)[i];
                        } else {
                            if (2 * i < have) w[j][i] = reinterpret_cast<const unsigned short *>(src)[2 * i];
                            if (2 * i + 1 < have) w[j][i] |= (unsigned)reinterpret_cast<const unsigned short *>(src)[2 * i + 1] << 16;
                        }
                    }
                }
            }
        } else {
            unsigned char *mine = stage + warp * 4 * kUnits * kUnitStride;
            constexpr int kPieces = kUnits * 32 * kSize / WORD, kPerUnit = 32 * kSize / WORD, kElems = WORD / kSize, kEach = kPieces / 32;   // pieces of a row of the tile
            typename Piece<WORD>::type piece[4][kEach];          // (all loads of the tile before the first store)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint64_t rq = group * 128 + r0 + 32 * q;
                const unsigned char *src = g.x + (rq * g.ld + first * 32) * kSize;
                const int live = rq < g.rows && first * 32 < g.cols ? (int)min((uint64_t)kUnits * 32, g.cols - first * 32) : 0;
#pragma unroll
                for (int i = 0; i < kEach; ++i) piece[q][i] = load_piece<WORD, kSize>(src, lane + 32 * i, live - (lane + 32 * i) * kElems);
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int p = lane + 32 * i;
                    *reinterpret_cast<typename Piece<WORD>::type *>(mine + (q * kUnits + p / kPerUnit) * kUnitStride + (p % kPerUnit) * WORD) = piece[q][i];
                }
            __syncwarp();
            const uint4 *from = reinterpret_cast<const uint4 *>(mine + (sub * kUnits + unit) * kUnitStride);
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = from[i];
                w[0][4 * i] = v.x; w[0][4 * i + 1] = v.y; w[0][4 * i + 2] = v.z; w[0][4 * i + 3] = v.w;
            }
        }
        if (row < g.rows) {
            uint8_t *to = codes + row * ldc + (first + unit) * 16;
            uint8_t *tile = scales + (group * quads + (FMT == kMxFp4 ? first / 4 + (unit >> 2) : first / 2 + (unit >> 1))) * kFp4ScaleTile + r0 * 16 + sub * 4;
#pragma unroll
            for (int j = 0; j < kRun; ++j, to += 128, tile += (FMT == kMxFp4 ? 2 : 4) * kFp4ScaleTile) {
                const uint64_t u = first + unit + 8 * j;
                if (u >= units) break;
                uint4 c;
                unsigned bytes;
                quantise_unit<FMT, TYPE, AMAX == kGivenAmax>(w[j], scale, inv, table, &c, &bytes);
                if (u * 16 < ldc) *reinterpret_cast<uint4 *>(to) = c;
                if (FMT == kMxFp4) tile[unit & 3] = (uint8_t)bytes;
                else *reinterpret_cast<unsigned short *>(tile + 2 * (unit & 1)) = (unsigned short)bytes;
            }
        }
    }
}

struct DequantArgs {
    const uint8_t *packed;
    uint64_t rows, cols, ld;
    unsigned char *out;
    unsigned chunks, tasks;
};

template <int FMT, int TYPE, int WORD>
__global__ void __launch_bounds__(kThreads) fp4_dequantize_kernel(const DequantArgs g) {
    chain_begin();
    constexpr int kSize = TYPE == kF32 ? 4 : 2, kWords = 32 * kSize / 4, kUnitStride = 32 * kSize + 16;
    extern __shared__ __align__(16) unsigned char stage[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, unit = lane & 7;
    const float scale = *reinterpret_cast<const float *>(g.packed);
    const uint64_t ldc = fp4_ld(g.cols), quads = fp4_quads(FMT, g.cols);
    const uint8_t *codes = g.packed + kFp4Head, *scales = g.packed + fp4_scales_at(g.rows, g.cols);
    for (unsigned task = blockIdx.x; task < g.tasks; task += gridDim.x) {
        const unsigned block = task / g.chunks;
        const uint64_t first = (uint64_t)(task - block * g.chunks) * kUnits;
        const unsigned r0 = (block & 3) * 8 + warp;
        const uint64_t group = block >> 2, row = group * 128 + r0 + 32 * sub, u = first + unit, col = u * 32;
        const int have = row < g.rows && col < g.cols ? (int)min((uint64_t)32, g.cols - col) : 0;
        unsigned w[kWords];
        if (have) {
            const uint4 c = *reinterpret_cast<const uint4 *>(codes + row * ldc + u * 16);
            const uint8_t *tile = scales + (group * quads + (FMT == kMxFp4 ? u >> 2 : u >> 1)) * kFp4ScaleTile + r0 * 16 + sub * 4;
            const unsigned bytes = FMT == kMxFp4 ? tile[u & 3] : *reinterpret_cast<const unsigned short *>(tile + 2 * (u & 1));
            const float s0 = fp4_scale_value<FMT>(bytes & 0xffu), s1 = FMT == kMxFp4 ? s0 : fp4_scale_value<FMT>(bytes >> 8);
            const unsigned words[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int o = 0; o < 4; ++o) {
                unsigned h[4];
                e2m1_unpack8(words[o], h);
                const float s = o < 2 ? s0 : s1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
                    // code times block scale is exact (6 bits); one rounding where the matrix scale is not a power of two
                    const float a = (f.x * s) * scale, b = (f.y * s) * scale;
                    if (TYPE == kF32) {
                        w[(o * 8 + 2 * i) % kWords] = __float_as_uint(a);
                        w[(o * 8 + 2 * i + 1) % kWords] = __float_as_uint(b);
                    } else {
                        w[o * 4 + i] = pack_pair<TYPE>(a, b);
                    }
                }
            }
        }
        if constexpr (WORD == 32) {
            unsigned char *dst = g.out + (row * g.ld + col) * kSize;
            if (have == 32) {
#pragma unroll
                for (int i = 0; i < kWords; i += 8) st_words8(dst + i * 4, *reinterpret_cast<unsigned(*)[8]>(&w[i]));
            } else if (have) {
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    if (TYPE == kF32) {
                        if (i < have) reinterpret_cast<unsigned *>(dst)[i] = w[i];
                    } else {
                        if (2 * i < have) reinterpret_cast<unsigned short *>(dst)[2 * i] = (unsigned short)w[i];
                        if (2 * i + 1 < have) reinterpret_cast<unsigned short *>(dst)[2 * i + 1] = (unsigned short)(w[i] >> 16);
                    }
                }
            }
        } else {
            unsigned char *mine = stage + warp * 4 * kUnits * kUnitStride;
            constexpr int kPieces = kUnits * 32 * kSize / WORD, kPerUnit = 32 * kSize / WORD, kElems = WORD / kSize;
            __syncwarp();
            if (have) {
                uint4 *to = reinterpret_cast<uint4 *>(mine + (sub * kUnits + unit) * kUnitStride);
#pragma unroll
                for (int i = 0; i < kWords / 4; ++i) to[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint64_t rq = group * 128 + r0 + 32 * q;
                unsigned char *dst = g.out + (rq * g.ld + first * 32) * kSize;
                const int live = rq < g.rows && first * 32 < g.cols ? (int)min((uint64_t)kUnits * 32, g.cols - first * 32) : 0;
#pragma unroll
                for (int i = 0; i < kPieces / 32; ++i) {
                    const int p = lane + 32 * i;
                    store_piece<WORD, kSize>(dst, p, live - p * kElems,
                                             *reinterpret_cast<const typename Piece<WORD>::type *>(mine + (q * kUnits + p / kPerUnit) * kUnitStride + (p % kPerUnit) * WORD));
                }
            }
        }
    }
}

// tiles of 32 rows (8 by 4) x 256 columns; the blocks of 8 rows of the last group that lie behind the matrix are left out
unsigned row_blocks(uint64_t rows) {
    const uint64_t last = rows % 128;
    return (unsigned)(rows / 128 * 4 + (last >= 32 ? 4 : (last + 7) / 8));
}
// the widest pieces that rows of this stride, from this address on, can be moved in
int piece_bytes(const void *p, uint64_t row_bytes, uint64_t rows, int size) {
    const uint64_t a = reinterpret_cast<uintptr_t>(p) | (rows > 1 ? row_bytes : 0);
    return a % 32 == 0 ? 32 : a % 8 == 0 ? 8 : (a % 4 == 0 || size == 4) ? 4 : 2;
}

template <int FMT, int TYPE, int WORD>
cudaError_t launch_quantize(const QuantArgs &g, int amax, unsigned grid, cudaStream_t stream) {
    const size_t smem = WORD == 32 ? 0 : (size_t)kThreads * (32 * (TYPE == kF32 ? 4 : 2) + 16);
    if (FMT == kMxFp4) return launch_chained(fp4_quantize_kernel<FMT, TYPE, WORD, kNoAmax>, grid, kThreads, smem, stream, g);
    if (amax == kGivenAmax) return launch_chained(fp4_quantize_kernel<kNvFp4, TYPE, WORD, kGivenAmax>, grid, kThreads, smem, stream, g);
    if (amax == kOwnAmax) return launch_chained(fp4_quantize_kernel<kNvFp4, TYPE, WORD, kOwnAmax>, grid, kThreads, smem, stream, g);
    return launch_chained(fp4_quantize_kernel<kNvFp4, TYPE, WORD, kPartialAmax>, grid, kThreads, smem, stream, g);
}
template <int FMT, int TYPE>
cudaError_t quantize_typed(const QuantArgs &g, int amax, int word, unsigned grid, cudaStream_t stream) {
    if (word == 32) return launch_quantize<FMT, TYPE, 32>(g, amax, grid, stream);
    if (word == 8) return launch_quantize<FMT, TYPE, 8>(g, amax, grid, stream);
    if (word == 4 || TYPE == kF32) return launch_quantize<FMT, TYPE, 4>(g, amax, grid, stream);
    return launch_quantize<FMT, TYPE == kF32 ? kF16 : TYPE, 2>(g, amax, grid, stream);
}
template <int FMT>
cudaError_t quantize_format(const QuantArgs &g, int type, int amax, int word, unsigned grid, cudaStream_t stream) {
    if (type == kF32) return quantize_typed<FMT, kF32>(g, amax, word, grid, stream);
    if (type == kF16) return quantize_typed<FMT, kF16>(g, amax, word, grid, stream);
    return quantize_typed<FMT, kBf16>(g, amax, word, grid, stream);
}

template <int FMT, int TYPE, int WORD> cudaError_t launch_dequantize(const DequantArgs &g, unsigned grid, cudaStream_t stream) {
    const size_t smem = WORD == 32 ? 0 : (size_t)kThreads * (32 * (TYPE == kF32 ? 4 : 2) + 16);
    return launch_chained(fp4_dequantize_kernel<FMT, TYPE, WORD>, grid, kThreads, smem, stream, g);
}
template <int FMT, int TYPE> cudaError_t dequantize_typed(const DequantArgs &g, int word, unsigned grid, cudaStream_t stream) {
    if (word == 32) return launch_dequantize<FMT, TYPE, 32>(g, grid, stream);
    if (word == 8) return launch_dequantize<FMT, TYPE, 8>(g, grid, stream);
    if (word == 4 || TYPE == kF32) return launch_dequantize<FMT, TYPE, 4>(g, grid, stream);
    return launch_dequantize<FMT, TYPE == kF32 ? kF16 : TYPE, 2>(g, grid, stream);
}
template <int FMT> cudaError_t dequantize_format(const DequantArgs &g, int type, int word, unsigned grid, cudaStream_t stream) {
    if (type == kF32) return dequantize_typed<FMT, kF32>(g, word, grid, stream);
    if (type == kF16) return dequantize_typed<FMT, kF16>(g, word, grid, stream);
    return dequantize_typed<FMT, kBf16>(g, word, grid, stream);
}

std::atomic<unsigned> g_tries{~0u};

}  // namespace

void limit_epilogue_tries(unsigned tries) { g_tries.store(tries, std::memory_order_relaxed); }
unsigned epilogue_tries(unsigned usual) {
    const unsigned tries = g_tries.load(std::memory_order_relaxed);
    return tries < usual ? tries : usual;
}

cudaError_t fp4_quantize(int format, const void *x, int type, uint64_t rows, uint64_t cols, uint64_t ld, const float *amax, void *packed,
                         void *scratch, int sm_count, cudaStream_t stream) {
    if (rows == 0) return cudaMemsetAsync(packed, 0, kFp4Head, stream);
    QuantArgs g;
    g.x = static_cast<const unsigned char *>(x);
    g.rows = rows; g.cols = cols; g.ld = ld;
    g.packed = static_cast<uint8_t *>(packed);
    g.amax = amax;
    g.partials = 0;
    const int size = op_bytes(type);
    const int word = piece_bytes(x, ld * size, rows, size), tile = kUnits * unit_run(type, word);
    const uint64_t units = fp4_quads(format, cols) * (format == kMxFp4 ? 4 : 2);
    g.chunks = (unsigned)((units + tile - 1) / tile);
    g.blocks = row_blocks(rows);
    const uint64_t tasks = (uint64_t)g.chunks * g.blocks;
    if (tasks > 0xf0000000ull) return cudaErrorInvalidValue;
    int mode = format == kMxFp4 ? kNoAmax : amax ? kGivenAmax : fp4_quantize_scratch(format, type, rows, cols) == 0 ? kOwnAmax : kPartialAmax;
    if (mode == kPartialAmax) {
        const uint64_t want = (rows * cols * size + 32767) / 32768;                      // four 16-byte loads of 512 threads each
        const unsigned grid = (unsigned)(want < (uint64_t)sm_count * 2 ? want : (uint64_t)sm_count * 2);
        g.partials = (int)(grid < (unsigned)kFp4Partials ? grid : (unsigned)kFp4Partials);
        float *part = static_cast<float *>(scratch);
        g.amax = part;
        const cudaError_t err = type == kF32 ? launch_chained(fp4_absmax_kernel<kF32>, g.partials, 512, 0, stream, g.x, rows, cols, ld, part)
                              : type == kF16 ? launch_chained(fp4_absmax_kernel<kF16>, g.partials, 512, 0, stream, g.x, rows, cols, ld, part)
                                             : launch_chained(fp4_absmax_kernel<kBf16>, g.partials, 512, 0, stream, g.x, rows, cols, ld, part);
        if (err != cudaSuccess) return err;
    }
    const unsigned most = (unsigned)sm_count * 8, grid = tasks < most ? (unsigned)tasks : most;
    return format == kMxFp4 ? quantize_format<kMxFp4>(g, type, mode, word, grid, stream) : quantize_format<kNvFp4>(g, type, mode, word, grid, stream);
}

cudaError_t fp4_dequantize(int format, const void *packed, uint64_t rows, uint64_t cols, void *out, int type, uint64_t ld, int sm_count,
                           cudaStream_t stream) {
    if (rows == 0) return cudaSuccess;
    DequantArgs g;
    g.packed = static_cast<const uint8_t *>(packed);
    g.rows = rows; g.cols = cols; g.ld = ld;
    g.out = static_cast<unsigned char *>(out);
    g.chunks = (unsigned)((cols + 32 * kUnits - 1) / (32 * kUnits));
    const uint64_t tasks = (uint64_t)g.chunks * row_blocks(rows);
    if (tasks > 0xf0000000ull) return cudaErrorInvalidValue;
    g.tasks = (unsigned)tasks;
    const unsigned most = (unsigned)sm_count * 8, grid = g.tasks < most ? g.tasks : most;
    const int word = piece_bytes(out, ld * op_bytes(type), rows, op_bytes(type));
    return format == kMxFp4 ? dequantize_format<kMxFp4>(g, type, word, grid, stream) : dequantize_format<kNvFp4>(g, type, word, grid, stream);
}

}  // namespace bsq
