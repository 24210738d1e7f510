// The norm of many tensors taken as one vector, and the tensors times min(1, max_norm / (norm + 1e-6)).
//
// Two passes, each one launch for up to 640 tensors: a pass over the data that leaves a partial sum per CTA, and one in which every CTA adds those up
// in the same order (so the result does not depend on timing), works out the factor and scales.  The list of tensors travels as a kernel
// parameter: nothing is staged in device memory, and a captured call replays with the pointers it was captured with.  Tensors are cut into chunks
// of 16384 elements which CTAs take in turn; a chunk finds its tensor by bisection.
//
// Bound by memory: in, in again, out.  The second pass walks the chunks from the last to the first, so that what the first pass read last comes
// from the L2.  Where the factor is 1 and the result goes where the input is, the second pass ends at once.  403 MB of BF16 in 14 tensors: the norm 66 us (6.1
// TB/s), with the scaled copies 196 us (1209 MB, 6.2 TB/s); 50 MB 21 to 24 us.
//
// Squares are summed in FP32 over at most 32 elements of a thread and in FP64 from there on.  Where such a sum leaves the range in which FP32 squares are
// good to 24 bits (gradients beyond 10^18 or below 10^-15), the thread takes the same elements in FP64: the norm is right wherever it is itself
// representable.  A NaN or Inf anywhere shows in the norm.
#include <algorithm>
#include <vector>

#include "bsq_fp4.cuh"
#include "bsq_grad_norm.hpp"

namespace bsq {
namespace {

constexpr int kNormThreads = 512;
constexpr unsigned kChunk = 16384;                               // elements
constexpr int kPartialMax = kNormScratchBytes / sizeof(double);

struct NormEntry {
    const unsigned char *in;
    unsigned char *out;
    uint64_t count;
    unsigned first;                      // number of the tensor's first chunk
    int type;
};
template <int N> struct NormTable {
    NormEntry e[N];
    int tensors;
    unsigned chunks;
};

template <int N> __device__ __forceinline__ const NormEntry &entry_of(const NormTable<N> &t, unsigned chunk) {
    int lo = 0, hi = t.tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.e[mid].first <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return t.e[lo];
}

// Words of up to 64 bytes of elements, summed as squares
template <int TYPE, int COUNT> __device__ __forceinline__ double squares(const unsigned (&w)[COUNT]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
#pragma unroll
        for (int j = 0; j < Words<TYPE>::kPer; ++j) {
            const float x = word_elem<TYPE>(w[i], j);
            s = fmaf(x, x, s);
        }
    if (TYPE == kF16 || (s > 1e-30f && s < 1e36f)) return (double)s;
    unsigned any = 0;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) any |= w[i] & Words<TYPE>::kAbs;
    if (any == 0) return 0.0;
    double d = 0.0;
#pragma unroll 1
    for (int j = 0; j < Words<TYPE>::kPer; ++j)
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const double x = (double)word_elem<TYPE>(w[i], j);
            d = fma(x, x, d);
        }
    return d;
}

template <int TYPE> __device__ void chunk_norm(const unsigned char *p, unsigned n, bool largest, double *sum, unsigned *top) {
    using W = Words<TYPE>;
    constexpr int kSize = TYPE == kF32 ? 4 : 2, kVec = 16 / kSize;
    const unsigned me = threadIdx.x;
    unsigned head = ((16u - (unsigned)(reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / kSize;
    if (head > n) head = n;
    const unsigned vecs = (n - head) / kVec, tail = head + vecs * kVec;
    const uint4 *v = reinterpret_cast<const uint4 *>(p + head * kSize);
    for (unsigned i = me; i < vecs; i += 4 * kNormThreads) {
        unsigned w[16];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint4 a = i + u * kNormThreads < vecs ? v[i + u * kNormThreads] : make_uint4(0u, 0u, 0u, 0u);
            w[4 * u] = a.x; w[4 * u + 1] = a.y; w[4 * u + 2] = a.z; w[4 * u + 3] = a.w;
        }
        if (largest) {
#pragma unroll
            for (int u = 0; u < 16; ++u) *top = W::larger(*top, w[u]);
        } else {
            *sum += squares<TYPE>(w);
        }
    }
    // elements in front of the first 16-byte boundary and behind the last one: at most 14 of them
    const unsigned edge = me < head ? me : me - head + tail;
    if (edge < n) {
        const unsigned w[1] = {TYPE == kF32 ? reinterpret_cast<const unsigned *>(p)[edge] : (unsigned)reinterpret_cast<const unsigned short *>(p)[edge]};
        if (largest) *top = W::larger(*top, w[0]);
        else *sum += squares<TYPE>(w);
    }
}

__device__ __forceinline__ double cta_reduce(double v, bool largest) {
    __shared__ double part[kNormThreads / 32];
    for (int d = 16; d; d >>= 1) {
        const double o = __shfl_xor_sync(kFullMask, v, d);
        v = largest ? (v > o || v != v ? v : o) : v + o;
    }
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kNormThreads / 32; ++i) v = largest ? (v > part[i] || v != v ? v : part[i]) : v + part[i];
    return v;
}

template <int N> __global__ void __launch_bounds__(kNormThreads) norm_pass_kernel(const __grid_constant__ NormTable<N> t, bool largest, double *partials) {
    chain_begin();
    double sum = 0.0;
    float best = 0.0f;
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const NormEntry &e = entry_of(t, c);
        const uint64_t at = (uint64_t)(c - e.first) * kChunk;
        const unsigned n = (unsigned)min((uint64_t)kChunk, e.count - at);
        unsigned top = 0;
        float m;
        if (e.type == kF32) {
            chunk_norm<kF32>(e.in + at * 4, n, largest, &sum, &top);
            m = Words<kF32>::top(top);
        } else if (e.type == kBf16) {
            chunk_norm<kBf16>(e.in + at * 2, n, largest, &sum, &top);
            m = Words<kBf16>::top(top);
        } else {
            chunk_norm<kF16>(e.in + at * 2, n, largest, &sum, &top);
            m = Words<kF16>::top(top);
        }
        best = best > m || best != best ? best : m;              // (a NaN stays)
    }
    const double v = cta_reduce(largest ? (double)best : sum, largest);
    if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

template <int TYPE> __device__ void chunk_scale(const unsigned char *in, unsigned char *out, unsigned n, float f) {
    constexpr int kSize = TYPE == kF32 ? 4 : 2, kVec = 16 / kSize;
    const unsigned me = threadIdx.x;
    auto word = [&](unsigned w) {
        if (TYPE == kF32) return __float_as_uint(__uint_as_float(w) * f);
        return pack_pair<TYPE>(word_elem<TYPE>(w, 0) * f, word_elem<TYPE>(w, 1) * f);
    };
    auto one = [&](unsigned i) { store_elem<TYPE>(out, i, word_elem<TYPE>(TYPE == kF32 ? reinterpret_cast<const unsigned *>(in)[i] : (unsigned)reinterpret_cast<const unsigned short *>(in)[i], 0) * f); };
    if ((reinterpret_cast<uintptr_t>(in) ^ reinterpret_cast<uintptr_t>(out)) & 15u) {                     // never both on a boundary
        for (unsigned i = me; i < n; i += kNormThreads) one(i);
        return;
    }
    unsigned head = ((16u - (unsigned)(reinterpret_cast<uintptr_t>(in) & 15u)) & 15u) / kSize;
    if (head > n) head = n;
    const unsigned vecs = (n - head) / kVec, tail = head + vecs * kVec;
    const uint4 *v = reinterpret_cast<const uint4 *>(in + head * kSize);
    uint4 *o = reinterpret_cast<uint4 *>(out + head * kSize);
    for (unsigned i = me; i < vecs; i += 4 * kNormThreads) {
        uint4 a[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * kNormThreads < vecs) a[u] = v[i + u * kNormThreads];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * kNormThreads < vecs) o[i + u * kNormThreads] = make_uint4(word(a[u].x), word(a[u].y), word(a[u].z), word(a[u].w));
    }
    const unsigned edge = me < head ? me : me - head + tail;
    if (edge < n) one(edge);
}

// partials: of all launches of the first pass
template <int N>
__global__ void __launch_bounds__(kNormThreads) norm_scale_kernel(const __grid_constant__ NormTable<N> t, bool largest, const double *partials, int count, double max_norm,
                                                                  bool in_place, bool scale, float *norm) {
    chain_begin();
    double v = 0.0;
    for (int i = threadIdx.x; i < count; i += kNormThreads) {
        const double p = partials[i];
        v = largest ? (v > p || v != v ? v : p) : v + p;
    }
    v = cta_reduce(v, largest);
    const double total = largest ? v : sqrt(v);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    const double coef = max_norm / (total + 1e-6);
    const float f = coef > 1.0 ? 1.0f : (float)coef;             // (NaN stays NaN)
    if (!scale || (in_place && f == 1.0f)) return;
    for (unsigned i = blockIdx.x; i < t.chunks; i += gridDim.x) {
        const unsigned c = t.chunks - 1 - i;
        const NormEntry &e = entry_of(t, c);
        const uint64_t at = (uint64_t)(c - e.first) * kChunk;
        const unsigned n = (unsigned)min((uint64_t)kChunk, e.count - at);
        if (e.type == kF32) chunk_scale<kF32>(e.in + at * 4, e.out + at * 4, n, f);
        else if (e.type == kBf16) chunk_scale<kBf16>(e.in + at * 2, e.out + at * 2, n, f);
        else chunk_scale<kF16>(e.in + at * 2, e.out + at * 2, n, f);
    }
}

struct Part {
    int begin, end;                      // tensors of one launch
};

template <int N> NormTable<N> table_of(const Part &p, const void *const *ins, const uint64_t *counts, const int *types, void *const *outs) {
    NormTable<N> t;
    t.tensors = 0;
    t.chunks = 0;
    for (int i = p.begin; i < p.end; ++i) {
        if (counts[i] == 0) continue;
        NormEntry &e = t.e[t.tensors++];
        e.in = static_cast<const unsigned char *>(ins[i]);
        e.out = outs ? static_cast<unsigned char *>(outs[i]) : nullptr;
        e.count = counts[i];
        e.first = t.chunks;
        e.type = types[i];
        t.chunks += (unsigned)((counts[i] + kChunk - 1) / kChunk);
    }
    return t;
}

template <int N>
cudaError_t run_parts(const std::vector<Part> &parts, const void *const *ins, const uint64_t *counts, const int *types, void *const *outs, double max_norm, bool largest,
                      float *norm, double *partials, unsigned most, cudaStream_t stream) {
    int used = 0;
    bool in_place = true;
    for (size_t i = 0; i < parts.size(); ++i) {
        const NormTable<N> t = table_of<N>(parts[i], ins, counts, types, outs);
        const unsigned room = (unsigned)(kPartialMax - used) / (unsigned)(parts.size() - i);
        const unsigned grid = std::max(1u, std::min(std::min(t.chunks, most), room));
        const cudaError_t err = launch_chained(norm_pass_kernel<N>, grid, kNormThreads, 0, stream, t, largest, partials + used);
        if (err != cudaSuccess) return err;
        used += (int)grid;
    }
    if (outs)
        for (const Part &p : parts)
            for (int i = p.begin; i < p.end; ++i) in_place = in_place && (counts[i] == 0 || outs[i] == ins[i]);
    for (size_t i = parts.size(); i-- > 0;) {
        const bool last = i == 0;
        if (!outs && !last) continue;                            // the norm alone: one launch
        const NormTable<N> t = table_of<N>(parts[i], ins, counts, types, outs);
        const unsigned grid = outs ? std::max(1u, std::min(t.chunks, most)) : 1u;
        const cudaError_t err = launch_chained(norm_scale_kernel<N>, grid, kNormThreads, 0, stream, t, largest, (const double *)partials, used, max_norm, in_place, outs != nullptr,
                                               last ? norm : nullptr);
        if (err != cudaSuccess) return err;
    }
    return cudaSuccess;
}

}  // namespace

bool norm_layout_ok(const void *const *ins, const uint64_t *counts, const int *types, int n, void *const *outs) {
    if (!outs) return true;
    struct Span {
        uintptr_t begin, end;
        bool out;
    };
    std::vector<Span> spans;
    spans.reserve(2 * (size_t)n);
    for (int i = 0; i < n; ++i) {
        if (counts[i] == 0) continue;
        const uint64_t bytes = counts[i] * (uint64_t)op_bytes(types[i]);
        const uintptr_t a = reinterpret_cast<uintptr_t>(ins[i]), b = reinterpret_cast<uintptr_t>(outs[i]);
        if (a != b) spans.push_back({a, a + bytes, false});
        spans.push_back({b, b + bytes, true});
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
    uintptr_t any = 0, out = 0;                                  // where what came before ends
    for (const Span &s : spans) {
        if (s.begin < (s.out ? any : out)) return false;
        any = std::max(any, s.end);
        if (s.out) out = std::max(out, s.end);
    }
    return true;
}

cudaError_t grad_norm_clip(const void *const *ins, const uint64_t *counts, const int *types, int n, void *const *outs, double max_norm, int norm_kind, float *norm,
                           void *scratch, int sm_count, cudaStream_t stream) {
    constexpr int kFew = 64, kMany = 640;
    std::vector<Part> parts;
    Part p = {0, 0};
    int held = 0;
    uint64_t chunks = 0;
    for (int i = 0; i < n; ++i) {
        const uint64_t c = (counts[i] + kChunk - 1) / kChunk;
        if (c > 0x7fffffffull) return cudaErrorInvalidValue;
        if (held == kMany || chunks + c > 0x7fffffffull) {
            parts.push_back(p);
            p.begin = i;
            held = 0;
            chunks = 0;
        }
        held += counts[i] != 0;
        chunks += c;
        p.end = i + 1;
    }
    parts.push_back(p);
    if (parts.size() > (size_t)kPartialMax) return cudaErrorInvalidValue;
    const bool few = parts.size() == 1 && held <= kFew;
    const unsigned most = (unsigned)sm_count * 4;
    double *partials = static_cast<double *>(scratch);
    return few ? run_parts<kFew>(parts, ins, counts, types, outs, max_norm, norm_kind == 0, norm, partials, most, stream)
               : run_parts<kMany>(parts, ins, counts, types, outs, max_norm, norm_kind == 0, norm, partials, most, stream);
}

}  // namespace bsq
