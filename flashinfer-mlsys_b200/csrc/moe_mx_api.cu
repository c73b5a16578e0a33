// moe_mx_api.cu — C ABI of the microscaled operators and of the balance loss
// (include/moe_fp8_ds.h): argument checks, tensor maps, launches.
#include "moe_fp8_ds.h"
#include "moe_kernels.h"
#include "moe_mx.cuh"

using namespace moe;

namespace {

constexpr int64_t kMaxRows = int64_t(1) << 24;
constexpr int64_t kMaxCols = int64_t(1) << 20;
constexpr int64_t kMaxN = int64_t(1) << 18;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool valid_fmt(int fmt) { return fmt == MOE_MX_NVFP4 || fmt == MOE_MX_MXFP4 || fmt == MOE_MX_MXFP8; }
bool valid_dt(int dt) { return dt == MOE_DT_BF16 || dt == MOE_DT_FP16 || dt == MOE_DT_FP32; }
int64_t dt_size(int dt) { return dt == MOE_DT_FP32 ? 4 : 2; }

int rows_cols(int64_t rows, int64_t cols, int fmt, int dt) {
  if (rows < 0 || rows > kMaxRows || cols <= 0 || cols > kMaxCols || cols % kMxCols || !valid_fmt(fmt) || !valid_dt(dt))
    return MOE_ERR_INVALID_ARG;
  return MOE_OK;
}

// Rows of `cols` elements, `ld` apart: 16-byte aligned and not overlapping.
int strided(const void* p, int64_t ld, int64_t rows, int64_t cols, int dt) {
  if (!p || (rows > 1 && ld < cols) || ld < 0 || ld > (int64_t(1) << 40)) return MOE_ERR_INVALID_ARG;
  if (!aligned(p, 16) || (rows > 1 && (ld * dt_size(dt)) % 16)) return MOE_ERR_ALIGNMENT;
  return MOE_OK;
}

int packed(const void* q, const void* scale) {
  if (!q || !scale) return MOE_ERR_INVALID_ARG;
  return aligned(q, 16) ? MOE_OK : MOE_ERR_ALIGNMENT;
}

int tensor_scale(const float* g, int fmt) {
  if (g && fmt != MOE_MX_NVFP4) return MOE_ERR_INVALID_ARG;
  return aligned(g, 4) ? MOE_OK : MOE_ERR_ALIGNMENT;
}

#define MOE_TRY(e)                 \
  do {                             \
    const int rc_ = (e);           \
    if (rc_ != MOE_OK) return rc_; \
  } while (0)

int cuda_rc(cudaError_t e) {
  if (e == cudaSuccess) return MOE_OK;
  cudaGetLastError();
  return MOE_ERR_CUDA;
}

int matmul(const void* a, const void* a_scale, const void* b, const void* b_scale, const int32_t* off, int64_t experts,
           int64_t M, int64_t N, int64_t K, int fmt, const float* alpha, void* out, int out_dt, int64_t out_ld,
           void* stream) {
  if (M < 0 || M > kMaxRows || N <= 0 || N > kMaxN || K <= 0 || K > kMaxCols || K % 32 || experts < 1 ||
      experts > kMxGemmMaxExperts || !valid_fmt(fmt) || !valid_dt(out_dt))
    return MOE_ERR_INVALID_ARG;
  if (M == 0) return check_device_sm100();  // empty tensors may carry null data pointers
  if (!a || !a_scale || !b || !b_scale || !out || out_ld < 0 || (M > 1 && out_ld < N) || out_ld > (int64_t(1) << 40))
    return MOE_ERR_INVALID_ARG;
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(alpha, 4) || !aligned(off, 4) || !aligned(out, dt_size(out_dt)))
    return MOE_ERR_ALIGNMENT;
  MOE_TRY(check_device_sm100());
  const uint64_t row_bytes = static_cast<uint64_t>(fmt == MOE_MX_MXFP8 ? K : K / 2);
  const MxPlan pl = mx_gemm_plan(M, N, static_cast<int>(experts), mx_gemm_stages(K, fmt), off != nullptr);
  CUtensorMap mw, ma;
  if (!encode_map_3d(&mw, b, row_bytes, static_cast<uint64_t>(N), static_cast<uint64_t>(experts), 128) ||
      !encode_map_3d(&ma, a, row_bytes, static_cast<uint64_t>(M), 1, static_cast<uint32_t>(pl.box_rows)))
    return MOE_ERR_CUDA;
  MxGemmCall c{};
  c.a_scale = a_scale;
  c.b_scale = b_scale;
  c.off = off;
  c.alpha = alpha;
  c.out = out;
  c.out_ld = out_ld;
  c.out_dt = out_dt;
  c.experts = static_cast<int>(experts);
  c.rows = M;
  c.N = N;
  c.K = K;
  c.fmt = fmt;
  return cuda_rc(launch_mx_gemm(mw, ma, c, pl, static_cast<cudaStream_t>(stream)));
}

int balance(BalanceCall* c, const void* logits, int dtype, int64_t ld, const int32_t* ids, const int32_t* off,
            int64_t tokens, int64_t experts, int64_t topk, int64_t seqs, int score, float coeff) {
  if (tokens < 0 || tokens > kMaxRows || experts < 1 || experts > MOE_BALANCE_MAX_EXPERTS || topk < 1 || topk > experts ||
      seqs < 1 || seqs > kMaxRows || !valid_dt(dtype) || (score != MOE_SCORE_SIGMOID && score != MOE_SCORE_SOFTMAX) ||
      ld < 0 || (tokens > 1 && ld < experts) || ld > (int64_t(1) << 40) || (!off && seqs != 1))
    return MOE_ERR_INVALID_ARG;
  if (tokens > 0 && (!logits || !ids)) return MOE_ERR_INVALID_ARG;
  if (!aligned(logits, dt_size(dtype)) || !aligned(ids, 4) || !aligned(off, 4)) return MOE_ERR_ALIGNMENT;
  *c = BalanceCall{logits, dtype, ld, ids, off, tokens, static_cast<int>(experts), static_cast<int>(topk),
                   static_cast<int>(seqs), score == MOE_SCORE_SOFTMAX ? 1 : 0, coeff};
  return MOE_OK;
}

}  // namespace

extern "C" {

int moe_fp8_ds_quantize_mx(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_ld, int fmt,
                           const float* global_scale, void* q_out, void* scale_out, void* stream) {
  MOE_TRY(rows_cols(rows, cols, fmt, dtype));
  MOE_TRY(tensor_scale(global_scale, fmt));
  if (rows == 0) return check_device_sm100();
  MOE_TRY(strided(x, x_ld, rows, cols, dtype));
  MOE_TRY(packed(q_out, scale_out));
  MOE_TRY(check_device_sm100());
  return cuda_rc(launch_mx_quant(x, dtype, x_ld, rows, cols, fmt, global_scale, q_out, scale_out,
                                 static_cast<cudaStream_t>(stream)));
}

int moe_fp8_ds_dequantize_mx(const void* q, const void* scale, int64_t rows, int64_t cols, int fmt,
                             const float* global_scale, int dtype, void* x_out, int64_t x_ld, void* stream) {
  MOE_TRY(rows_cols(rows, cols, fmt, dtype));
  MOE_TRY(tensor_scale(global_scale, fmt));
  if (rows == 0) return check_device_sm100();
  MOE_TRY(strided(x_out, x_ld, rows, cols, dtype));
  MOE_TRY(packed(q, scale));
  MOE_TRY(check_device_sm100());
  return cuda_rc(launch_mx_dequant(q, scale, rows, cols, fmt, global_scale, dtype, x_out, x_ld,
                                   static_cast<cudaStream_t>(stream)));
}

int moe_fp8_ds_add_norm_quantize_mx(const void* x, int64_t x_ld, void* residual, int64_t residual_ld,
                                    const void* norm_weight, float eps, int dtype, int64_t rows, int64_t cols, int fmt,
                                    const float* global_scale, void* q_out, void* scale_out, void* stream) {
  MOE_TRY(rows_cols(rows, cols, fmt, dtype));
  MOE_TRY(tensor_scale(global_scale, fmt));
  if (cols > kMxNormMaxCols || !(eps >= 0.f)) return MOE_ERR_INVALID_ARG;
  if (rows == 0) return check_device_sm100();
  MOE_TRY(strided(x, x_ld, rows, cols, dtype));
  if (residual) MOE_TRY(strided(residual, residual_ld, rows, cols, dtype));
  if (!aligned(norm_weight, 16)) return MOE_ERR_ALIGNMENT;
  MOE_TRY(packed(q_out, scale_out));
  MOE_TRY(check_device_sm100());
  const MxNormCall c{x, x_ld, residual, residual_ld, norm_weight, eps, rows, cols, global_scale, q_out, scale_out};
  return cuda_rc(launch_mx_norm(c, fmt, dtype, static_cast<cudaStream_t>(stream)));
}

int moe_fp8_ds_matmul_mx(const void* a, const void* a_scale, const void* b, const void* b_scale, int64_t m, int64_t n,
                         int64_t k, int fmt, const float* alpha, void* out, int out_dtype, int64_t out_ld,
                         void* stream) {
  return matmul(a, a_scale, b, b_scale, nullptr, 1, m, n, k, fmt, alpha, out, out_dtype, out_ld, stream);
}

int moe_fp8_ds_experts_matmul_mx(const void* a, const void* a_scale, const void* b, const void* b_scale,
                                 const int32_t* expert_offsets, int64_t num_experts, int64_t m, int64_t n, int64_t k,
                                 int fmt, const float* alpha, void* out, int out_dtype, int64_t out_ld, void* stream) {
  if (!expert_offsets) return MOE_ERR_INVALID_ARG;
  return matmul(a, a_scale, b, b_scale, expert_offsets, num_experts, m, n, k, fmt, alpha, out, out_dtype, out_ld,
                stream);
}

size_t moe_fp8_ds_balance_loss_work_bytes(int64_t tokens, int64_t experts, int64_t seqs) {
  if (tokens < 0 || tokens > kMaxRows || experts < 1 || experts > MOE_BALANCE_MAX_EXPERTS || seqs < 1 || seqs > kMaxRows)
    return 0;
  return static_cast<size_t>(balance_slots(tokens, seqs)) * experts * 8;
}

int moe_fp8_ds_balance_loss(const void* routing_logits, int dtype, int64_t logits_ld, const int32_t* topk_ids,
                            const int32_t* seq_offsets, int64_t tokens, int64_t experts, int64_t topk, int64_t seqs,
                            int score, float coeff, void* work, float* loss_out, int32_t* counts_out, void* stream) {
  BalanceCall c;
  MOE_TRY(balance(&c, routing_logits, dtype, logits_ld, topk_ids, seq_offsets, tokens, experts, topk, seqs, score, coeff));
  if (!work || !loss_out || !counts_out) return MOE_ERR_INVALID_ARG;
  if (!aligned(work, 8) || !aligned(loss_out, 4) || !aligned(counts_out, 4)) return MOE_ERR_ALIGNMENT;
  MOE_TRY(check_device_sm100());
  return cuda_rc(launch_balance(c, work, loss_out, counts_out, static_cast<cudaStream_t>(stream)));
}

int moe_fp8_ds_balance_loss_backward(const void* routing_logits, int dtype, int64_t logits_ld, const int32_t* topk_ids,
                                     const int32_t* seq_offsets, int64_t tokens, int64_t experts, int64_t topk,
                                     int64_t seqs, int score, float coeff, const int32_t* counts,
                                     const float* grad_loss, void* grad_logits_out, void* stream) {
  BalanceCall c;
  MOE_TRY(balance(&c, routing_logits, dtype, logits_ld, topk_ids, seq_offsets, tokens, experts, topk, seqs, score, coeff));
  if (tokens == 0) return check_device_sm100();
  if (!counts || !grad_loss || !grad_logits_out) return MOE_ERR_INVALID_ARG;
  if (!aligned(counts, 4) || !aligned(grad_loss, 4) || !aligned(grad_logits_out, dt_size(dtype))) return MOE_ERR_ALIGNMENT;
  MOE_TRY(check_device_sm100());
  return cuda_rc(launch_balance_backward(c, counts, grad_loss, grad_logits_out, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
