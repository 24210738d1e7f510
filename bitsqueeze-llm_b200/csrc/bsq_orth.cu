// Newton-Schulz steps that bring a matrix's singular values near 1:  X_0 = G / (|G| + eps),  A = X X^T,  X <- a X + (b A + c A^2) X, on the side of the shorter dimension
// (X^T X and X (b A + c A^2) where G is tall: nothing is transposed, the products read either orientation).  Three launches a step for all matrices of one shape.
//
// What 16-bit operands cost, and what is done about it (the steps pull small singular values up by 3.4 each, and with them whatever rounding has left there):
//   * FP16, not BF16: entries are bounded, a power of two brings them into its range, and it has three bits more at the same rate;
//   * X is kept as high + low, two FP16 words of 22 bits.  Products read the high part; a X is added up from both in the epilogue.  With one word the
//     large singular values' rounding is what the small ones start from (rank-8 gradients with noise: 4e-3 off after five steps, this way 1e-4);
//   * the diagonals of A and of P = b A + c A^2, of size 1 where everything else is small, are kept in FP32: what rounding takes from them, and what the
//     products leave out of the low part (P_ii X_low), goes back in the epilogues (noise: 1.9e-3 off without, 0.2e-3 to 0.7e-3 with it; a rounding to BF16 is 1.7e-3).
// Results in FP32 or FP16, and matrices with a short side of up to 128 (where launches are what a step costs), take both parts of every operand: three products of halves.
//
// A and P are symmetric: tiles on and below the diagonal are computed, and written twice.  Bound by the tensor core, then by power.
#include "bsq_gemm16.cuh"
#include "bsq_orth.hpp"

#include <algorithm>
#include <cmath>
#include <tuple>
#include <vector>

namespace bsq {
namespace {

constexpr int kOrthMost = 64;                                    // matrices of a launch
constexpr uint64_t kOrthRoom = 1ull << 30;                       // scratch that several matrices share at most
constexpr uint64_t kSplitShort = 128;                            // short sides up to this: split operands
constexpr int kNormThreads = 512;
constexpr uint64_t kNormChunk = 32768;                           // elements of a CTA of the pass that finds the norms, 64 CTAs at most
constexpr int kNormParts = 64;

__device__ __forceinline__ float half_bits(unsigned short b) { return __half2float(__ushort_as_half(b)); }
// 16 FP16 elements on a 32-byte boundary
__device__ __forceinline__ void load16h(const unsigned short *p, float (&v)[16]) {
    unsigned w[8];
    ld_words8(p, w);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = half_bits((unsigned short)(w[j >> 1] >> ((j & 1) * 16)));
}
__device__ __forceinline__ float high_of(float x) { return __half2float(__float2half_rn(x)); }

// ---- G to X_0 ----
struct OrthIn {
    const void *at[kOrthMost];
    uint64_t ld[kOrthMost];
    uint64_t rows, cols;
    int type;
};
__device__ __forceinline__ float elem(const void *p, int type, uint64_t i) {
    if (type == kF32) return static_cast<const float *>(p)[i];
    if (type == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ double cta_total(double v, double *room) {
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kFullMask, v, d);
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) v += room[i];
    return v;
}
// Sums of squares, in FP64: blockIdx.x a part of a matrix's rows, blockIdx.y the matrix
__global__ void __launch_bounds__(kNormThreads) orth_norm_kernel(const __grid_constant__ OrthIn in, double *parts) {
    chain_begin();
    __shared__ double room[kNormThreads / 32];
    const void *p = in.at[blockIdx.y];
    const uint64_t ld = in.ld[blockIdx.y], all = in.rows * in.cols;
    double s = 0.0;
    for (uint64_t i = (uint64_t)blockIdx.x * kNormThreads + threadIdx.x; i < all; i += (uint64_t)gridDim.x * kNormThreads) {
        const uint64_t r = i / in.cols;
        const double x = (double)elem(p, in.type, r * ld + (i - r * in.cols));
        s = fma(x, x, s);
    }
    s = cta_total(s, room);
    if (threadIdx.x == 0) parts[blockIdx.y * gridDim.x + blockIdx.x] = s;
}

struct OrthX {
    unsigned short *high, *low;
    uint64_t ld, apart;
    float *factor;                   // X = (high + low) * factor, one for each matrix
};
__global__ void __launch_bounds__(kNormThreads) orth_begin_kernel(const __grid_constant__ OrthIn in, const double *parts, int count, double eps, const OrthX x) {
    chain_begin();
    __shared__ double room[kNormThreads / 32];
    const void *p = in.at[blockIdx.y];
    const double total = cta_total((int)threadIdx.x < count ? parts[blockIdx.y * (unsigned)count + threadIdx.x] : 0.0, room), norm = sqrt(total);
    // 2^e brings the norm, and so every element, below 2^15; a power of two, so that elements of 16 bits stay what they are
    const bool fine = norm < 3.0e38 * 65536.0 * 65536.0;         // (not: Inf or NaN)
    const int e = norm > 0.0 && fine ? min(max(14 - ilogb(norm), -160), 160) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) x.factor[blockIdx.y] = !fine ? __uint_as_float(0x7fffffffu) : norm > 0.0 ? (float)(ldexp(1.0, -e) / (norm + eps)) : 1.0f;
    const float s0 = exp2f((float)(e / 2)), s1 = exp2f((float)(e - e / 2));
    const uint64_t ld = in.ld[blockIdx.y], all = in.rows * x.ld;
    unsigned short *high = x.high + blockIdx.y * x.apart, *low = x.low + blockIdx.y * x.apart;
    for (uint64_t i = (uint64_t)blockIdx.x * kNormThreads + threadIdx.x; i < all; i += (uint64_t)gridDim.x * kNormThreads) {
        const uint64_t r = i / x.ld, c = i - r * x.ld;
        const float v = c < in.cols ? elem(p, in.type, r * ld + c) * s0 * s1 : 0.0f;
        const float h = high_of(v);
        high[i] = __half_as_ushort(__float2half_rn(h));
        low[i] = __half_as_ushort(__float2half_rn(v - h));
    }
}

// ---- what the epilogues share ----
// 16 values to a box of 16-bit elements: high parts, and low parts to another one
__device__ __forceinline__ void put_parts(unsigned char *high, unsigned char *low, int lane, int h, const float (&v)[16]) {
    float a[16], b[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        a[j] = high_of(v[j]);
        b[j] = v[j] - a[j];
    }
    box_put16<kF16>(high, lane, h, a);
    if (low) box_put16<kF16>(low, lane, h, b);
}
// A box of 32 rows x 64 columns turned into one of 64 rows x 32 (64 bytes a row, not swizzled)
__device__ __forceinline__ void turn_box(const unsigned char *box, unsigned char *turned, int lane) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint4 q = *reinterpret_cast<const uint4 *>(box + lane * 128 + ((i ^ (lane & 7)) << 4));
        const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) reinterpret_cast<unsigned short *>(turned)[(i * 8 + j) * 32 + lane] = (unsigned short)(w[j >> 1] >> ((j & 1) * 16));
    }
}
// The element of v on the diagonal, where the thread's row has one in these 16 columns
__device__ __forceinline__ int diagonal_at(int row, int col) { return (unsigned)(row - col) < 16u ? row - col : -1; }

struct SymmetricMaps {
    CUtensorMap map[2], turned[2];   // high, low
};
// 64 columns of a symmetric result from `fill(h, v)`, their mirror image too where the tile is below the diagonal
template <bool SPLIT, class Fill> __device__ __forceinline__ void put_symmetric(const TileOut &o, const SymmetricMaps &m, int c, bool mirror, const Fill &fill) {
    float keep[SPLIT ? 64 : 1];
    unsigned char *box = box_next(o);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        float v[16];
        fill(h, v);
        if constexpr (SPLIT) {
#pragma unroll
            for (int j = 0; j < 16; ++j) keep[16 * h + j] = v[j] - high_of(v[j]);
        }
        put_parts(box, nullptr, o.lane, h, v);
    }
    box_send(o, &m.map[0], o.col + c, o.row, box);
    if (mirror) {
        unsigned char *turned = box_next(o);
        turn_box(box, turned, o.lane);
        box_send(o, &m.turned[0], o.row, o.col + c, turned);
    }
    if constexpr (SPLIT) {
        box = box_next(o);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = keep[16 * h + j];
            box_put16<kF16>(box, o.lane, h, v);
        }
        box_send(o, &m.map[1], o.col + c, o.row, box);
        if (mirror) {
            unsigned char *turned = box_next(o);
            turn_box(box, turned, o.lane);
            box_send(o, &m.turned[1], o.row, o.col + c, turned);
        }
    }
}

// ---- A = X X^T (or X^T X), held times 2^e ----
template <bool SPLIT> struct GramOut {
    SymmetricMaps maps;
    int M;
    const float *factor;             // of X, one for each matrix, or null
    float constant;                  // ... for all
    float scale;                     // 2^e
    float *rest;                     // what rounding to FP16 takes from the diagonal

    template <int COLS> __device__ void tile(const TileOut &o) const {
        const float x = factor ? factor[o.z] : constant;
        const int row = o.row + o.lane;
        for (int c = 0; c < COLS && o.col + c < M; c += 64) {
            const int col = o.col + c;
            if (col > o.row + 31) continue;                      // above the diagonal: the mirror image of what another warp has
            put_symmetric<SPLIT>(o, maps, c, col + 63 < o.row, [&](int h, float (&v)[16]) {
                read16f(o.taddr + (unsigned)(c + 16 * h), v, o.ok);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = v[j] * x * x * scale;
                if (SPLIT) return;
                const int d = diagonal_at(row, col + 16 * h);
                if (d >= 0 && row < M) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j == d) rest[(size_t)o.z * (size_t)M + (size_t)row] = v[j] - high_of(v[j]);
                }
            });
        }
    }
};

// ---- P = b A + c A^2, held times 2^e ----
template <bool SPLIT> struct PolyOut {
    SymmetricMaps maps;
    int M;
    const unsigned short *high, *low;
    uint64_t ld, apart;
    float b, c;                      // b 2^(e - e_A), c 2^(e - 2 e_A)
    const float *rest_a;
    float *whole, *rest;             // the diagonal, and what rounding takes from it

    template <int COLS> __device__ void tile(const TileOut &o) const {
        const int row = o.row + o.lane;
        const float *ra = rest_a + (size_t)o.z * (size_t)M;
        const float mine = !SPLIT && row < M ? ra[row] : 0.0f;
        for (int at = 0; at < COLS && o.col + at < M; at += 64) {
            const int col = o.col + at;
            if (col > o.row + 31) continue;
            put_symmetric<SPLIT>(o, maps, at, col + 63 < o.row, [&](int h, float (&v)[16]) {
                const int c0 = col + 16 * h;
                float p[16], q[16], r[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) p[j] = q[j] = r[j] = 0.0f;
                if (row < M && c0 < M) {
                    const size_t i = (size_t)o.z * apart + (size_t)row * ld + (size_t)c0;
                    load16h(high + i, p);
                    if (SPLIT) load16h(low + i, q);
                    else {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c0 + j < M) r[j] = ra[c0 + j];
                    }
                }
                read16f(o.taddr + (unsigned)(at + 16 * h), v, o.ok);
                const int d = SPLIT ? -1 : diagonal_at(row, c0);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    // A_ij = p + [i = j] rest_i, of which the product has p only
                    const float a = SPLIT ? p[j] + q[j] : j == d ? p[j] + mine : p[j];
                    const float squares = SPLIT ? v[j] : fmaf(p[j], mine + r[j], v[j]) + (j == d ? mine * mine : 0.0f);
                    v[j] = fmaf(c, squares, b * a);
                }
                if (d >= 0 && row < M) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (j == d) {
                            whole[(size_t)o.z * (size_t)M + (size_t)row] = v[j];
                            rest[(size_t)o.z * (size_t)M + (size_t)row] = v[j] - high_of(v[j]);
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
    CUtensorMap map[2];              // of the next X, high and low
    int M, N;
    bool tall;                       // the diagonal of P goes with the columns
    bool last;
    int type;                        // of the result
    const unsigned short *high, *low;
    uint64_t ld, apart;
    const float *factor;             // of X, one for each matrix, or null
    float constant;                  // ... for all
    float a, back, scale;            // P is held times 1 / back; the next X is held times `scale` (or the result is multiplied by it)
    const float *whole, *rest;
    int side;                        // of P
    OrthOut out;                     // (last)

    __device__ __forceinline__ void values(const TileOut &o, int row, int c, float x, float mine, float mine_low, float (&v)[16]) const {
        const int c0 = o.col + c;
        float p[16], q[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) p[j] = q[j] = 0.0f;
        if (row < M && c0 < N) {
            const size_t i = (size_t)o.z * apart + (size_t)row * ld + (size_t)c0;
            load16h(high + i, p);
            load16h(low + i, q);
        }
        read16f(o.taddr + (unsigned)c, v, o.ok);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float s;
            if (SPLIT) {
                s = fmaf(a, p[j], fmaf(a, q[j], v[j] * back));
            } else {
                float e = mine, d = mine_low;
                if (tall) {
                    const size_t k = (size_t)o.z * (size_t)side + (size_t)min(c0 + j, side - 1);
                    e = rest[k];
                    d = whole[k];
                }
                s = fmaf(fmaf(e, back, a), p[j], fmaf(fmaf(d, back, a), q[j], v[j] * back));
            }
            v[j] = s * x * scale;
        }
    }

    template <int COLS> __device__ void tile(const TileOut &o) const {
        const int row = o.row + o.lane;
        const float x = factor ? factor[o.z] : constant;
        const bool wide = !SPLIT && !tall && row < M;
        const float mine = wide ? rest[(size_t)o.z * (size_t)side + (size_t)row] : 0.0f, mine_low = wide ? whole[(size_t)o.z * (size_t)side + (size_t)row] : 0.0f;
        if (!last) {
            for (int c = 0; c < COLS && o.col + c < N; c += 64) {
                unsigned char *box = box_next(o);
                if (o.lane == 0) bulk_wait_read_all();           // (both boxes: high and low)
                __syncwarp();
                unsigned char *other = o.boxes + (unsigned)*o.which * kG16Box;
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    float v[16];
                    values(o, row, c + 16 * h, x, mine, mine_low, v);
                    put_parts(box, other, o.lane, h, v);
                }
                box_send(o, &map[0], o.col + c, o.row, box);
                *o.which ^= 1;
                box_send(o, &map[1], o.col + c, o.row, other);
            }
            return;
        }
        void *to = out.at[o.z];
        const long ld_out = (long)out.ld[o.z];
        const int per = type == kF32 ? 32 : 64;
        for (int c = 0; c < COLS && o.col + c < N; c += per) {
            unsigned char *box = box_next(o);
#pragma unroll 1
            for (int h = 0; h < per / 16; ++h) {
                float v[16];
                values(o, row, c + 16 * h, x, mine, mine_low, v);
                if (type == kF32) {
                    uint4 *line = reinterpret_cast<uint4 *>(box + o.lane * 128);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        line[(4 * h + j) ^ (o.lane & 7)] = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
                } else if (type == kBf16) {
                    box_put16<kBf16>(box, o.lane, h, v);
                } else {
                    box_put16<kF16>(box, o.lane, h, v);
                }
            }
            box_out(box, o.lane, to, type == kF32 ? 4 : 2, (long)o.row * ld_out + o.col + c, ld_out, M - o.row, N - o.col - c);
        }
    }
};

// ---- host ----
uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// Powers of two that X, A and P of a step are held times: largest magnitudes below 2^15
struct StepScale {
    int x, a, p;
};
int below_2_15(double most) { return std::min(24, std::max(-14, most > 0.0 ? (int)std::floor(std::log2(32768.0 / most)) : 14)); }
// Largest singular value that each step may meet, from 0 .. 1 at the start; false: it grows beyond 1000
bool scales_of(const float *k, int steps, std::vector<StepScale> *out) {
    double most = 1.0;
    for (int i = 0; i < steps; ++i, k += 3) {
        const double a = k[0], b = k[1], c = k[2];
        if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
        double next = 0.0, p = 0.0;
        const double top = most * 1.02;                          // (room for what rounding adds)
        for (int j = 0; j <= 4096; ++j) {
            const double s = top * j / 4096, l = s * s, y = b * l + c * l * l;
            p = std::max(p, std::fabs(y));
            next = std::max(next, std::fabs((a + y) * s));
        }
        if (!(next < 1000.0) || !(p < 1e6)) return false;
        if (out) out->push_back({below_2_15(top), below_2_15(top * top), below_2_15(p)});
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
bool split_of(const OrthMatrix &m, int out_type) { return out_type != kBf16 || std::min(m.rows, m.cols) <= kSplitShort; }

struct Room {
    unsigned short *high[2], *low[2], *a[2], *p[2];
    float *factor, *rest_a, *whole, *rest;
    double *parts;
    uint64_t ld_x, apart_x, ld_a, apart_a;
    size_t bytes;
};
Room room_of(const OrthMatrix &m, bool split, int count, void *scratch) {
    Room r = {};
    const uint64_t s = std::min(m.rows, m.cols), n = (uint64_t)count;
    unsigned char *base = static_cast<unsigned char *>(scratch);
    const auto take = [&](uint64_t bytes) {
        unsigned char *p = base + r.bytes;
        r.bytes += up(bytes, 128);
        return p;
    };
    r.ld_x = up(m.cols, 16);
    r.apart_x = m.rows * r.ld_x;
    r.ld_a = up(s, 16);
    r.apart_a = s * r.ld_a;
    for (int i = 0; i < 2; ++i) {
        r.high[i] = reinterpret_cast<unsigned short *>(take(n * r.apart_x * 2));
        r.low[i] = reinterpret_cast<unsigned short *>(take(n * r.apart_x * 2));
    }
    for (int i = 0; i < (split ? 2 : 1); ++i) {
        r.a[i] = reinterpret_cast<unsigned short *>(take(n * r.apart_a * 2));
        r.p[i] = reinterpret_cast<unsigned short *>(take(n * r.apart_a * 2));
    }
    r.factor = reinterpret_cast<float *>(take(n * 4));
    r.rest_a = reinterpret_cast<float *>(take(n * s * 4));
    r.whole = reinterpret_cast<float *>(take(n * s * 4));
    r.rest = reinterpret_cast<float *>(take(n * s * 4));
    r.parts = reinterpret_cast<double *>(take(n * kNormParts * 8));
    return r;
}

Plan plan_of(const OrthCall &c) {
    Plan p;
    for (int i = 0; i < c.n; ++i)
        if (c.m[i].rows && c.m[i].cols) p.order.push_back(i);
    const auto key = [&](int i) { return std::make_tuple(c.m[i].rows, c.m[i].cols, c.m[i].type); };
    std::stable_sort(p.order.begin(), p.order.end(), [&](int i, int j) { return key(i) < key(j); });
    for (int i = 0; i < (int)p.order.size();) {
        const OrthMatrix &m = c.m[p.order[i]];
        const uint64_t one = room_of(m, split_of(m, c.out_type), 1, nullptr).bytes;
        const int most = (int)std::min<uint64_t>(kOrthMost, std::max<uint64_t>(1, kOrthRoom / one));
        int n = 1;
        while (n < most && i + n < (int)p.order.size() && key(p.order[i + n]) == key(p.order[i])) ++n;
        p.groups.push_back({i, n});
        i += n;
    }
    return p;
}

bool symmetric_maps(SymmetricMaps *m, unsigned short *const (&to)[2], bool split, uint64_t s, uint64_t ld, uint64_t count, uint64_t apart) {
    for (int i = 0; i < 2; ++i) {
        // (whole rows of `ld`: a store never ends inside 16 bytes; what lies behind the last column is not read)
        const Stack st = {to[split ? i : 0], ld, s, ld, count, apart};
        if (!map_stack(&m->map[i], st, kF16, 64, 32) || !map_stack(&m->turned[i], st, kF16, 32, 64, CU_TENSOR_MAP_SWIZZLE_NONE)) return false;
    }
    return true;
}

template <bool SPLIT>
cudaError_t run_group(const OrthCall &c, const std::vector<StepScale> &scales, const OrthMatrix *const *m, int count, void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    const uint64_t rows = m[0]->rows, cols = m[0]->cols, s = std::min(rows, cols);
    const bool tall = rows > cols;
    const Room r = room_of(*m[0], SPLIT, count, scratch);
    OrthIn in = {};
    OrthOut out = {};
    for (int i = 0; i < count; ++i) {
        in.at[i] = m[i]->in;
        in.ld[i] = m[i]->ld_in;
        out.at[i] = m[i]->out;
        out.ld[i] = m[i]->ld_out;
    }
    in.rows = rows;
    in.cols = cols;
    in.type = m[0]->type;
    const unsigned parts = (unsigned)std::min<uint64_t>(kNormParts, (rows * cols + kNormChunk - 1) / kNormChunk);
    cudaError_t err = launch_chained(orth_norm_kernel, dim3(parts, (unsigned)count), kNormThreads, 0, stream, in, r.parts);
    if (err != cudaSuccess) return err;
    const OrthX x0 = {r.high[0], r.low[0], r.ld_x, r.apart_x, r.factor};
    const unsigned blocks = (unsigned)std::min<uint64_t>((rows * r.ld_x + kNormThreads * 4 - 1) / (kNormThreads * 4), std::max(1, sm_count * 8 / count));
    err = launch_chained(orth_begin_kernel, dim3(blocks, (unsigned)count), kNormThreads, 0, stream, in, (const double *)r.parts, (int)parts, c.eps, x0);
    if (err != cudaSuccess) return err;

    SymmetricMaps maps_a, maps_p;
    if (!symmetric_maps(&maps_a, r.a, SPLIT, s, r.ld_a, (uint64_t)count, r.apart_a) || !symmetric_maps(&maps_p, r.p, SPLIT, s, r.ld_a, (uint64_t)count, r.apart_a)) return cudaErrorInvalidValue;
    Gemm16 g = {};
    g.batch = count;
    g.splits = 1;
    g.parts = SPLIT ? 3 : 1;
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
        GramOut<SPLIT> gram = {maps_a, (int)s, factor, constant, std::ldexp(1.0f, k.a), r.rest_a};
        if ((err = launch_gemm16(ops, gram, g, std::max(rows, cols), pairs_s, status, sm_count, stream)) != cudaSuccess) return err;
        // P
        for (int i = 0; i < 2; ++i) {
            const Stack a = {r.a[SPLIT ? i : 0], s, s, r.ld_a, (uint64_t)count, r.apart_a};
            if (!map_operand(&ops.a[i], a, false, true)) return cudaErrorInvalidValue;
            ops.b[i] = ops.a[i];
        }
        g.a_kmajor = g.b_kmajor = true;
        PolyOut<SPLIT> poly = {maps_p, (int)s, r.a[0], r.a[1], r.ld_a, r.apart_a, std::ldexp(co[1], k.p - k.a), std::ldexp(co[2], k.p - 2 * k.a), r.rest_a, r.whole, r.rest};
        if ((err = launch_gemm16(ops, poly, g, s, pairs_s, status, sm_count, stream)) != cudaSuccess) return err;
        // X
        for (int i = 0; i < 2; ++i) {
            const Stack p = {r.p[SPLIT ? i : 0], s, s, r.ld_a, (uint64_t)count, r.apart_a}, x = {i && SPLIT ? r.low[now] : r.high[now], cols, rows, r.ld_x, (uint64_t)count, r.apart_x};
            if (!map_operand(tall ? &ops.b[i] : &ops.a[i], p, false, true) || !map_operand(tall ? &ops.a[i] : &ops.b[i], x, false, tall)) return cudaErrorInvalidValue;
        }
        g.M = (int)rows;
        g.N = (int)cols;
        g.lower = false;
        g.a_kmajor = true;
        g.b_kmajor = tall;
        StepOut<SPLIT> e = {};
        for (int i = 0; i < 2; ++i)
            if (!map_stack(&e.map[i], {i ? r.low[now ^ 1] : r.high[now ^ 1], r.ld_x, rows, r.ld_x, (uint64_t)count, r.apart_x}, kF16, 64, 32)) return cudaErrorInvalidValue;
        e.M = (int)rows;
        e.N = (int)cols;
        e.tall = tall;
        e.last = last;
        e.type = c.out_type;
        e.high = r.high[now];
        e.low = r.low[now];
        e.ld = r.ld_x;
        e.apart = r.apart_x;
        e.factor = factor;
        e.constant = constant;
        e.a = co[0];
        e.back = std::ldexp(1.0f, -k.p);
        e.scale = last ? c.scale : std::ldexp(1.0f, scales[(size_t)step + 1].x);
        e.whole = r.whole;
        e.rest = r.rest;
        e.side = (int)s;
        e.out = out;
        if ((err = launch_gemm16(ops, e, g, s, pairs_x, status, sm_count, stream)) != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace

bool orth_steps_ok(const float *coefficients, int steps) { return scales_of(coefficients, steps, nullptr); }

size_t orth_scratch_bytes(const OrthCall &c) {
    size_t most = 0;
    const Plan p = plan_of(c);
    for (const Group &g : p.groups) {
        const OrthMatrix &m = c.m[p.order[(size_t)g.begin]];
        most = std::max(most, room_of(m, split_of(m, c.out_type), g.count, nullptr).bytes);
    }
    return most;
}

cudaError_t orthogonalize(const OrthCall &c, void *scratch, unsigned *status, int sm_count, cudaStream_t stream) {
    std::vector<StepScale> scales;
    if (!scales_of(c.coefficients, c.steps, &scales)) return cudaErrorInvalidValue;
    const Plan p = plan_of(c);
    for (const Group &g : p.groups) {
        const OrthMatrix *m[kOrthMost];
        for (int i = 0; i < g.count; ++i) m[i] = &c.m[p.order[(size_t)(g.begin + i)]];
        const cudaError_t err = split_of(*m[0], c.out_type) ? run_group<true>(c, scales, m, g.count, scratch, status, sm_count, stream)
                                                             : run_group<false>(c, scales, m, g.count, scratch, status, sm_count, stream);
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace bsq
