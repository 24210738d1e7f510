// extern "C" surface of the library (include/bitsqz_llm_c.h): thin forwards onto the C++
// interface and onto the stage launchers.  No logic lives here beyond argument translation.
#include <bitsqz_llm.hpp>
#include <bitsqz_llm_c.h>

#include "bsq_fp4.hpp"
#include "bsq_grad_norm.hpp"
#include "bsq_internal.hpp"
#include "bsq_orth.hpp"
#include "bsq_xent.hpp"

#include <algorithm>
#include <cmath>
#include <vector>

using namespace bsq;

static inline cudaStream_t as_stream(void *s) { return static_cast<cudaStream_t>(s); }
static inline int rc(cudaError_t e) {
    if (e != cudaSuccess) cudaGetLastError();
    return e == cudaSuccess ? 0 : 1;
}

extern "C" {

int bsq_compress_initialize(uint16_t num_rows, uint16_t num_columns, float outlier_topk_ratio,
                            float error_correction_topk_ratio, int svd_ranks, int svd_niters, int svd_uv_format,
                            int svd_s_format, int quantization_only_format, int input_location) {
    return bitsqz_llm_compress_initialize(num_rows, num_columns, outlier_topk_ratio, error_correction_topk_ratio,
                                          svd_ranks, svd_niters, (quantization_method_t)svd_uv_format,
                                          (quantization_method_t)svd_s_format,
                                          (quantization_method_t)quantization_only_format,
                                          (bitsqz_llm_input_location_t)input_location);
}
void bsq_compress_release(void) { bitsqz_llm_compress_release(); }
int bsq_decompress_initialize(uint16_t num_rows, uint16_t num_columns, float outlier_topk_ratio,
                              float error_correction_topk_ratio, int svd_ranks, int svd_uv_format, int svd_s_format,
                              int quantization_only_format) {
    return bitsqz_llm_decompress_initialize(num_rows, num_columns, outlier_topk_ratio, error_correction_topk_ratio,
                                            svd_ranks, (quantization_method_t)svd_uv_format,
                                            (quantization_method_t)svd_s_format,
                                            (quantization_method_t)quantization_only_format);
}
void bsq_decompress_release(void) { bitsqz_llm_decompress_release(); }
int bsq_compress(const float *row_major_matrix, struct bitsqz_llm_array **out, void *profile) {
    return bitsqz_llm_compress(row_major_matrix, out, static_cast<bitsqz_llm_compress_profile_t *>(profile));
}
int bsq_decompress(const struct bitsqz_llm_array *compressed, float *d_dst, uint32_t dst_num_elements) {
    return bitsqz_llm_decompress(compressed, d_dst, dst_num_elements);
}
uint64_t bsq_get_packed_size(const struct bitsqz_llm_array *compressed) { return bitsqz_llm_get_packed_size(compressed); }
struct bitsqz_llm_array *bsq_load_from_buffer(const void *buffer, uint64_t buffer_size) {
    return load_bitsqz_llm_from_buffer(buffer, buffer_size);
}
void bsq_free(struct bitsqz_llm_array *compressed) { bitsqz_llm_free(compressed); }

int bsq_topk_num_columns(uint16_t num_columns, float topk_ratio) { return topk_num_columns(num_columns, topk_ratio); }
int bsq_topk_rows(const float *d_in, float *d_residual, uint32_t rows, uint32_t cols, uint32_t k, uint16_t *d_idx,
                  float *d_val, uint32_t *d_status, void *stream) {
    return rc(topk_rows(d_in, d_residual, rows, cols, k, d_idx, d_val, d_status, device_sm_count(), as_stream(stream)));
}
int bsq_topk_apply(const uint16_t *d_idx, const float *d_val, uint32_t rows, uint32_t cols, uint32_t k, float *d_dense,
                   uint32_t *d_status, void *stream) {
    return rc(topk_apply(d_idx, d_val, rows, cols, k, d_dense, d_status, as_stream(stream)));
}

int bsq_nf4_quantize(const float *d_x, uint64_t n, float *d_scales, uint8_t *d_data, float *d_deq_out, void *stream) {
    if (!d_x || !n || !d_scales || !d_data) return 1;
    return rc(nf4_quantize(d_x, n, d_scales, d_data, d_deq_out, device_sm_count(), as_stream(stream)));
}
size_t bsq_nf4dq_scratch_bytes(uint64_t n) { return nf4dq_scratch_bytes(n); }
int bsq_nf4dq_quantize(const float *d_x, uint64_t n, float *d_dq, uint8_t *d_scale_codes, uint8_t *d_data,
                       float *d_deq_out, void *d_scratch, void *stream) {
    if (!d_x || !n || !d_dq || !d_scale_codes || !d_data || !d_scratch) return 1;
    return rc(nf4dq_quantize(d_x, n, d_dq, d_scale_codes, d_data, d_deq_out, d_scratch, device_sm_count(), as_stream(stream)));
}
uint64_t bsq_nf4dq_quantize_static_max_elements(void) { return nf4dq_static_max_elements(); }
int bsq_nf4dq_quantize_static(const float *d_x, uint64_t n, float *d_dq, uint8_t *d_scale_codes, uint8_t *d_data,
                              void *stream) {
    if (!d_x || !d_dq || !d_scale_codes || !d_data) return 1;
    if (n == 0 || n > nf4dq_static_max_elements()) return 1;      // beyond the built-in scratch: use bsq_nf4dq_quantize
    return rc(nf4dq_quantize_static(d_x, n, d_dq, d_scale_codes, d_data, device_sm_count(), as_stream(stream)));
}
int bsq_nf4_dequantize(const float *d_scales, const uint8_t *d_data, uint64_t n, float *d_out, void *stream) {
    if (!d_scales || !d_data || !n || !d_out) return 1;
    return rc(nf4_dequantize(d_scales, d_data, n, d_out, device_sm_count(), as_stream(stream)));
}
int bsq_nf4dq_dequantize(const float *d_dq, const uint8_t *d_scale_codes, const uint8_t *d_data, uint64_t n,
                         float *d_out, void *stream) {
    if (!d_dq || !d_scale_codes || !d_data || !n || !d_out) return 1;
    return rc(nf4dq_dequantize(d_dq, d_scale_codes, d_data, n, d_out, device_sm_count(), as_stream(stream)));
}

int bsq_dequantize_add_topk(int method, const float *d_scales_f32, const float *d_dq, const uint8_t *d_scale_codes,
                            const uint8_t *d_data, uint32_t rows, uint32_t cols, const uint16_t *d_idx, const float *d_val,
                            uint32_t k, float *d_out, uint32_t *d_status, void *stream) {
    if (method != 10 && method != 11) return 1;
    return rc(nf4_dequantize_add_topk(method == 11 ? d_scales_f32 : nullptr, method == 10 ? d_dq : nullptr,
                                      method == 10 ? d_scale_codes : nullptr, d_data, rows, cols, d_idx, d_val, k, d_out, d_status,
                                      device_sm_count(), as_stream(stream)));
}

int bsq_frontend_supported(uint32_t rows, uint32_t cols, uint32_t k) { return frontend_supported(rows, cols, k) ? 1 : 0; }
size_t bsq_frontend_scratch_bytes(uint32_t rows, uint32_t cols) { return frontend_scratch_bytes(rows, cols); }
int bsq_frontend_quantize(int method, const float *d_in, uint32_t rows, uint32_t cols, uint32_t k, uint16_t *d_idx,
                          float *d_val, float *d_scales_f32, float *d_dq, uint8_t *d_scale_codes, uint8_t *d_data,
                          void *d_scratch, uint32_t *d_status, void *stream) {
    return rc(frontend_quantize(method, d_in, rows, cols, k, d_idx, d_val, d_scales_f32, d_dq, d_scale_codes, d_data,
                                d_scratch, d_status, device_sm_count(), as_stream(stream)));
}

int bsq_frontend_quantize_timed(int method, const float *d_in, uint32_t rows, uint32_t cols, uint32_t k, uint16_t *d_idx,
                                float *d_val, float *d_scales_f32, float *d_dq, uint8_t *d_scale_codes, uint8_t *d_data,
                                void *d_scratch, uint32_t *d_status, void *stream, float *ms_pass) {
    if (!ms_pass) return 1;
    cudaEvent_t ev[3] = {nullptr, nullptr, nullptr};
    for (auto &e : ev)
        if (cudaEventCreate(&e) != cudaSuccess) return 1;
    int r = rc(frontend_quantize(method, d_in, rows, cols, k, d_idx, d_val, d_scales_f32, d_dq, d_scale_codes, d_data,
                                 d_scratch, d_status, device_sm_count(), as_stream(stream), ev));
    r |= rc(cudaEventSynchronize(ev[2]));
    if (r == 0) {
        r |= rc(cudaEventElapsedTime(&ms_pass[0], ev[0], ev[1]));
        r |= rc(cudaEventElapsedTime(&ms_pass[1], ev[1], ev[2]));
    }
    for (auto &e : ev) cudaEventDestroy(e);
    return r;
}

int bsq_residual_error(const float *d_a, const float *d_b, uint64_t n, float *d_e, uint32_t *d_flag, void *stream) {
    return rc(residual_error(d_a, d_b, n, d_e, d_flag, device_sm_count(), as_stream(stream)));
}

static int svd_once(const float *d_A, int m, int n, int k, int niter, unsigned long long seed, unsigned long long offset, bool coded_factors,
                    float *d_U, float *d_S, float *d_V, void *stream) {
    if (!d_A || !d_U || !d_S || !d_V || m <= 0 || n <= 0 || k <= 0 || niter < 0) return 1;
    SvdWorkspace *ws = svd_workspace_create(m, n, k, niter, device_sm_count(), coded_factors);
    if (!ws) return 1;
    const cudaError_t e = svd_lowrank(ws, d_A, d_U, d_S, d_V, seed, nullptr, as_stream(stream), offset);
    const cudaError_t s = svd_workspace_finish(ws, as_stream(stream));  // the workspace dies with this call
    svd_workspace_destroy(ws);
    return rc(e) | rc(s);
}
int bsq_svd_lowrank(const float *d_A, int m, int n, int k, int niter, unsigned long long seed, float *d_U, float *d_S,
                    float *d_V, void *stream) {
    return svd_once(d_A, m, n, k, niter, seed, 0, false, d_U, d_S, d_V, stream);
}
int bsq_svd_lowrank_at(const float *d_A, int m, int n, int k, int niter, unsigned long long seed, unsigned long long offset,
                       float *d_U, float *d_S, float *d_V, void *stream) {
    return svd_once(d_A, m, n, k, niter, seed, offset, false, d_U, d_S, d_V, stream);
}
int bsq_svd_lowrank_coded(const float *d_A, int m, int n, int k, int niter, unsigned long long seed, float *d_U, float *d_S,
                          float *d_V, void *stream) {
    return svd_once(d_A, m, n, k, niter, seed, 0, true, d_U, d_S, d_V, stream);
}
int bsq_gemm(int a_kmajor, int b_kmajor, const float *d_A, long lda, const float *d_B, long ldb, float *d_C, long ldc, int M,
             int N, int K, float *d_workspace, size_t workspace_bytes, int allow_tensor_cores, uint32_t *d_status, void *stream) {
    if (!d_A || !d_B || !d_C || M <= 0 || N <= 0 || K <= 0) return 1;
    return rc(gemm_select(allow_tensor_cores != 0, a_kmajor != 0, b_kmajor != 0, d_A, lda, d_B, ldb, d_C, ldc, M, N, K, nullptr,
                          nullptr, 0, nullptr, d_status, d_workspace, workspace_bytes, device_sm_count(), as_stream(stream)));
}
int bsq_gemm_bounded(int a_kmajor, int b_kmajor, const float *d_A, long lda, const float *d_B, long ldb, float *d_C, long ldc, int M,
                     int N, int K, float *d_workspace, size_t workspace_bytes, const uint32_t *d_a_absmax_bits, uint32_t *d_status,
                     void *stream) {
    if (!d_A || !d_B || !d_C || !d_a_absmax_bits || M <= 0 || N <= 0 || K <= 0) return 1;
    return rc(gemm_select(true, a_kmajor != 0, b_kmajor != 0, d_A, lda, d_B, ldb, d_C, ldc, M, N, K, nullptr, nullptr, 0, nullptr,
                          d_status, d_workspace, workspace_bytes, device_sm_count(), as_stream(stream), d_a_absmax_bits));
}
int bsq_reconstruct(const float *d_U, const float *d_S, const float *d_V, int m, int n, int k, const float *d_minuend,
                    float *d_out, uint32_t *d_flag, uint32_t *d_status, void *stream) {
    if (!d_U || !d_S || !d_V || !d_out || m <= 0 || n <= 0 || k <= 0) return 1;
    if (d_minuend && !d_flag) return 1;
    return rc(reconstruct_lowrank(d_U, d_S, d_V, m, n, k, d_minuend, d_out, d_flag, d_status, nullptr, 0, device_sm_count(), as_stream(stream)));
}

// ---- microscaled 4-bit matrices ----
static inline bool fp4_aligned(const void *packed) { return packed && reinterpret_cast<uintptr_t>(packed) % 16 == 0; }
static inline bool op_rows_ok(const void *p, int type, uint64_t rows, uint64_t cols, uint64_t ld) {
    const int size = op_bytes(type);
    return size && p && reinterpret_cast<uintptr_t>(p) % size == 0 && (rows <= 1 || (ld >= cols && ld < (1ull << 38)));
}

uint64_t bsq_fp4_packed_bytes(int format, uint64_t rows, uint64_t cols) { return fp4_shape_ok(format, rows, cols) ? fp4_packed_bytes(format, rows, cols) : 0; }
size_t bsq_fp4_scratch_bytes(int format, int type, uint64_t rows, uint64_t cols) { return fp4_shape_ok(format, rows, cols) ? fp4_quantize_scratch(format, type, rows, cols) : 0; }
int bsq_fp4_quantize(int format, const void *d_x, int type, uint64_t rows, uint64_t cols, uint64_t ld, const float *d_amax, void *d_packed, void *d_scratch,
                     void *stream) {
    if (!fp4_shape_ok(format, rows, cols) || !op_bytes(type) || !fp4_aligned(d_packed) || (rows && !op_rows_ok(d_x, type, rows, cols, ld))) return 1;
    if (!d_amax && fp4_quantize_scratch(format, type, rows, cols) && (!d_scratch || reinterpret_cast<uintptr_t>(d_scratch) % 4 != 0)) return 1;
    return rc(fp4_quantize(format, d_x, type, rows, cols, rows > 1 ? ld : cols, d_amax, d_packed, d_scratch, device_sm_count(), as_stream(stream)));
}
int bsq_fp4_dequantize(int format, const void *d_packed, uint64_t rows, uint64_t cols, void *d_out, int type, uint64_t ld, void *stream) {
    if (!fp4_shape_ok(format, rows, cols) || !op_bytes(type) || !fp4_aligned(d_packed) || (rows && !op_rows_ok(d_out, type, rows, cols, ld))) return 1;
    return rc(fp4_dequantize(format, d_packed, rows, cols, d_out, type, rows > 1 ? ld : cols, device_sm_count(), as_stream(stream)));
}
int bsq_fp4_matmul(int format, const void *d_a, uint64_t M, const void *d_b, uint64_t N, uint64_t K, void *d_out, int type, uint64_t ld, uint32_t *d_status,
                   void *stream) {
    if (!fp4_shape_ok(format, M, K) || !fp4_shape_ok(format, N, K) || !op_bytes(type) || !fp4_aligned(d_a) || !fp4_aligned(d_b)) return 1;
    if (M && N && !op_rows_ok(d_out, type, M, N, ld)) return 1;
    return rc(fp4_matmul(format, d_a, M, d_b, N, K, d_out, type, M > 1 ? ld : N, d_status, device_sm_count(), as_stream(stream)));
}
size_t bsq_fp4_grad_scratch_bytes(const void *d_dy, uint64_t M, uint64_t N, uint64_t ld_dy) { return fp4_grad_scratch_bytes(M, N, d_dy, ld_dy); }
static inline bool fp4_grad_ok(int format, const void *d_dy, uint64_t M, uint64_t N, uint64_t ld_dy, uint64_t packed_rows, uint64_t K, const void *packed,
                               const void *d_out, uint64_t out_rows, int type, uint64_t ld, const void *d_scratch) {
    if (!fp4_shape_ok(format, packed_rows, K) || M > kFp4MaxDim || N > kFp4MaxDim || !op_bytes(type) || !fp4_aligned(packed)) return false;
    if (M && N && !op_rows_ok(d_dy, kBf16, M, N, ld_dy)) return false;
    if (out_rows && !op_rows_ok(d_out, type, out_rows, K, ld)) return false;
    return fp4_grad_scratch_bytes(M, N, d_dy, ld_dy) == 0 || (d_scratch && reinterpret_cast<uintptr_t>(d_scratch) % 16 == 0);
}
int bsq_fp4_grad_input(int format, const void *d_dy, uint64_t M, uint64_t ld_dy, const void *d_w, uint64_t N, uint64_t K, void *d_out, int type, uint64_t ld,
                       void *d_scratch, uint32_t *d_status, void *stream) {
    if (!fp4_grad_ok(format, d_dy, M, N, ld_dy, N, K, d_w, d_out, M, type, ld, d_scratch)) return 1;
    return rc(fp4_grad_input(format, d_dy, M, ld_dy, d_w, N, K, d_out, type, M > 1 ? ld : K, d_scratch, d_status, device_sm_count(), as_stream(stream)));
}
int bsq_fp4_grad_weight(int format, const void *d_dy, uint64_t M, uint64_t N, uint64_t ld_dy, const void *d_x, uint64_t K, void *d_out, int type, uint64_t ld,
                        void *d_scratch, uint32_t *d_status, void *stream) {
    if (!fp4_grad_ok(format, d_dy, M, N, ld_dy, M, K, d_x, d_out, N, type, ld, d_scratch)) return 1;
    return rc(fp4_grad_weight(format, d_dy, M, N, ld_dy, d_x, K, d_out, type, N > 1 ? ld : K, d_scratch, d_status, device_sm_count(), as_stream(stream)));
}

// ---- gradients of many tensors ----
size_t bsq_grad_norm_scratch_bytes(void) { return kNormScratchBytes; }
int bsq_grad_norm_clip(const void *const *d_grads, const uint64_t *counts, const int *types, int n, void *const *d_outs, double max_norm, int norm_kind, float *d_norm,
                       void *d_scratch, void *stream) {
    if (n < 0 || (n && (!d_grads || !counts || !types)) || (norm_kind != 0 && norm_kind != 2) || (d_outs && !(max_norm >= 0.0))) return 1;
    if (!d_scratch || reinterpret_cast<uintptr_t>(d_scratch) % 8 != 0 || reinterpret_cast<uintptr_t>(d_norm) % 4 != 0 || (!d_outs && !d_norm)) return 1;
    for (int i = 0; i < n; ++i) {
        const int size = op_bytes(types[i]);
        if (!size || counts[i] > (1ull << 44)) return 1;
        if (counts[i] && (!d_grads[i] || reinterpret_cast<uintptr_t>(d_grads[i]) % size != 0)) return 1;
        if (counts[i] && d_outs && (!d_outs[i] || reinterpret_cast<uintptr_t>(d_outs[i]) % size != 0)) return 1;
    }
    try {
        if (!norm_layout_ok(d_grads, counts, types, n, d_outs)) return 1;
        return rc(grad_norm_clip(d_grads, counts, types, n, d_outs, max_norm, norm_kind, d_norm, d_scratch, device_sm_count(), as_stream(stream)));
    } catch (...) {
        return 1;
    }
}

// ---- loss over a vocabulary ----
static inline bool xent_call(XentCall *c, int type, const void *d_x, uint64_t tokens, uint64_t cols, uint64_t ld_x, const void *d_w, uint64_t vocab, uint64_t ld_w,
                             const int64_t *d_target, int64_t ignore, double smoothing, int reduction) {
    if ((type != kF16 && type != kBf16) || cols < 1 || cols > kXentMaxCols || vocab < 1 || vocab > kFp4MaxDim || tokens > xent_max_tokens(type)) return false;
    if ((tokens && !op_rows_ok(d_x, type, tokens, cols, ld_x)) || !op_rows_ok(d_w, type, vocab, cols, ld_w)) return false;
    if (!(smoothing >= 0.0 && smoothing <= 1.0) || reduction < kXentNone || reduction > kXentMean) return false;
    *c = {type, d_x, d_w, tokens, cols, vocab, tokens > 1 ? ld_x : cols, vocab > 1 ? ld_w : cols, reinterpret_cast<const long long *>(d_target), ignore, smoothing, reduction};
    return true;
}
static inline bool on_bytes(const void *p, unsigned n) { return p && reinterpret_cast<uintptr_t>(p) % n == 0; }

size_t bsq_linear_xent_scratch_bytes(int type, const void *d_x, uint64_t tokens, uint64_t cols, uint64_t ld_x, const void *d_w, uint64_t vocab, uint64_t ld_w, double smoothing) {
    XentCall c;
    return xent_call(&c, type, d_x, tokens, cols, ld_x, d_w, vocab, ld_w, nullptr, 0, smoothing, kXentNone) ? xent_scratch_bytes(c, device_sm_count()) : 0;
}
int bsq_linear_xent(int type, const void *d_x, uint64_t tokens, uint64_t cols, uint64_t ld_x, const void *d_w, uint64_t vocab, uint64_t ld_w, const int64_t *d_target,
                    int64_t ignore, double smoothing, int reduction, float *d_loss, float *d_stats, void *d_scratch, uint32_t *d_status, void *stream) {
    XentCall c;
    if (!xent_call(&c, type, d_x, tokens, cols, ld_x, d_w, vocab, ld_w, d_target, ignore, smoothing, reduction) || !on_bytes(d_stats, 4)) return 1;
    if ((tokens || reduction != kXentNone) && !on_bytes(d_loss, 4)) return 1;
    if (tokens && (!on_bytes(d_target, 8) || !on_bytes(d_scratch, 128))) return 1;
    return rc(xent_loss(c, d_loss, d_stats, d_scratch, d_status, device_sm_count(), as_stream(stream)));
}
size_t bsq_linear_xent_grad_scratch_bytes(int type, const void *d_x, uint64_t tokens, uint64_t cols, uint64_t ld_x, const void *d_w, uint64_t vocab, uint64_t ld_w, int with_dx) {
    XentCall c;
    return xent_call(&c, type, d_x, tokens, cols, ld_x, d_w, vocab, ld_w, nullptr, 0, 0.0, kXentNone) ? xent_grad_scratch_bytes(c, with_dx != 0, device_sm_count()) : 0;
}
int bsq_linear_xent_grad(int type, const void *d_x, uint64_t tokens, uint64_t cols, uint64_t ld_x, const void *d_w, uint64_t vocab, uint64_t ld_w, const int64_t *d_target,
                         int64_t ignore, double smoothing, int reduction, const float *d_stats, const float *d_grad, void *d_dx, uint64_t ld_dx, void *d_dw, uint64_t ld_dw,
                         void *d_scratch, uint32_t *d_status, void *stream) {
    XentCall c;
    if (!xent_call(&c, type, d_x, tokens, cols, ld_x, d_w, vocab, ld_w, d_target, ignore, smoothing, reduction)) return 1;
    if ((tokens && d_dx && !op_rows_ok(d_dx, type, tokens, cols, ld_dx)) || (d_dw && !op_rows_ok(d_dw, type, vocab, cols, ld_dw))) return 1;
    if (tokens && (!on_bytes(d_target, 8) || !on_bytes(d_scratch, 128) || !on_bytes(d_stats, 4) || !on_bytes(d_grad, 4))) return 1;
    if (!d_dx && !d_dw) return 0;
    return rc(xent_grad(c, d_stats, d_grad, d_dx, tokens > 1 ? ld_dx : cols, d_dw, vocab > 1 ? ld_dw : cols, d_scratch, d_status, device_sm_count(), as_stream(stream)));
}

// ---- orthogonalised updates ----
size_t bsq_orthogonalize_scratch_bytes(const uint64_t *rows, const uint64_t *cols, const int *types, int n, int out_type) {
    if (n < 1 || !rows || !cols || !types || !op_bytes(out_type)) return 0;
    try {
        std::vector<OrthMatrix> m((size_t)n);
        for (int i = 0; i < n; ++i) {
            if (!op_bytes(types[i]) || rows[i] > kOrthMaxDim || cols[i] > kOrthMaxDim) return 0;
            m[(size_t)i] = {nullptr, nullptr, rows[i], cols[i], cols[i], cols[i], types[i]};
        }
        return orth_scratch_bytes({m.data(), n, out_type, 0, nullptr, 0.0, 0.0f});
    } catch (...) {
        return 0;
    }
}
namespace {
// Where a matrix lies, in bytes: `rows` rows of `width`, `pitch` apart
struct Lies {
    uintptr_t begin, end;
    uint64_t pitch, width, rows;
    bool out;
};
// Whether two matrices share a byte.  Where one begins before the other ends they do not if their rows are equally far apart and their columns lie beside one another (or one is a single row that lies
// beside the other's columns); rows at other distances that pass one another count as sharing.
bool share(const Lies &a, const Lies &b) {
    if (a.end <= b.begin || b.end <= a.begin) return false;
    if (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) return true;
    const uint64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
    if (a.rows == 1 && b.rows == 1) return true;
    const uint64_t at = a.begin <= b.begin ? (b.begin - a.begin) % pitch : (pitch - (a.begin - b.begin) % pitch) % pitch;          // b's columns, from a's first
    return at < a.width || at + b.width > pitch;
}
// Whether a matrix that is written shares a byte with another one
bool written_shared(std::vector<Lies> &all) {
    std::sort(all.begin(), all.end(), [](const Lies &a, const Lies &b) { return a.begin < b.begin; });
    std::vector<const Lies *> open[2];                            // of what came before: what has not ended yet, inputs and outputs
    for (const Lies &m : all) {
        for (int out = 0; out < 2; ++out) {
            std::vector<const Lies *> &o = open[out];
            if (!m.out && !out) continue;
            o.erase(std::remove_if(o.begin(), o.end(), [&](const Lies *p) { return p->end <= m.begin; }), o.end());
            for (const Lies *p : o)
                if (share(*p, m)) return true;
        }
        open[m.out].push_back(&m);
    }
    return false;
}
enum { kFine = 0, kRefused = 1, kSteps = 2, kShared = 3 };
int orth_call(const void *const *d_in, const uint64_t *rows, const uint64_t *cols, const uint64_t *lds, const int *types, int n, void *const *d_out, const uint64_t *ld_outs, int out_type, int steps,
              const float *coefficients, double eps, float scale, std::vector<OrthMatrix> *m) {
    if (n < 0 || (n && (!d_in || !rows || !cols || !lds || !types || !d_out || !ld_outs)) || !op_bytes(out_type)) return kRefused;
    if (steps < 1 || steps > kOrthMaxSteps || !coefficients || !(eps >= 0.0) || std::isinf(eps) || !std::isfinite(scale)) return kRefused;
    m->resize((size_t)n);
    std::vector<Lies> all;
    for (int i = 0; i < n; ++i) {
        const uint64_t r = rows[i], c = cols[i], in = r > 1 ? lds[i] : c, out = r > 1 ? ld_outs[i] : c;
        if (!op_bytes(types[i]) || r > kOrthMaxDim || c > kOrthMaxDim) return kRefused;
        if (r && c && (!op_rows_ok(d_in[i], types[i], r, c, in) || !op_rows_ok(d_out[i], out_type, r, c, out))) return kRefused;
        (*m)[(size_t)i] = {d_in[i], d_out[i], r, c, in, out, types[i]};
        if (!r || !c) continue;
        const auto lies = [&](const void *p, uint64_t ld, int type, bool written) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(p);
            const uint64_t size = (uint64_t)op_bytes(type);
            all.push_back({at, at + ((r - 1) * ld + c) * size, ld * size, c * size, r, written});
        };
        lies(d_in[i], in, types[i], false);
        lies(d_out[i], out, out_type, true);
    }
    return written_shared(all) ? kShared : kFine;
}
}  // namespace

int bsq_orthogonalize_check(const void *const *d_in, const uint64_t *rows, const uint64_t *cols, const uint64_t *lds, const int *types, int n, void *const *d_out, const uint64_t *ld_outs,
                            int out_type, int steps, const float *coefficients, double eps, float scale) {
    try {
        std::vector<OrthMatrix> m;
        const int why = orth_call(d_in, rows, cols, lds, types, n, d_out, ld_outs, out_type, steps, coefficients, eps, scale, &m);
        return why != kRefused && !orth_steps_ok(coefficients, steps) ? kSteps : why;
    } catch (...) {
        return kRefused;
    }
}
int bsq_orthogonalize(const void *const *d_in, const uint64_t *rows, const uint64_t *cols, const uint64_t *lds, const int *types, int n, void *const *d_out, const uint64_t *ld_outs,
                      int out_type, int steps, const float *coefficients, double eps, float scale, void *d_scratch, uint32_t *d_status, void *stream) {
    try {
        std::vector<OrthMatrix> m;
        if (orth_call(d_in, rows, cols, lds, types, n, d_out, ld_outs, out_type, steps, coefficients, eps, scale, &m) != kFine) return 1;
        if (std::none_of(m.begin(), m.end(), [](const OrthMatrix &a) { return a.rows && a.cols; })) return 0;
        if (!on_bytes(d_scratch, 128)) return 1;
        return rc(orthogonalize({m.data(), n, out_type, steps, coefficients, eps, scale}, d_scratch, d_status, device_sm_count(), as_stream(stream)));
    } catch (...) {
        return 1;
    }
}

void bsq_test_limit_waits(uint32_t tries) { limit_epilogue_tries(tries); }

const char *bsq_build_info(void) { return "bitsqz_llm sm_100a " __DATE__; }

}  // extern "C"
