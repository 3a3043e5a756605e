// Layer norm of residual + dropout(x) over the last axis: the C entries (kernels and launches: egnn_norm.h).
#include "egnn_norm.h"

using namespace egnn::norm;

extern "C" {

int32_t egnn_norm_drop_fwd(const EgnnNormDims* d, const EgnnDropout* drop, const void* x, int64_t ldx, const void* residual,
                           int64_t ldr, const void* weight, const void* bias, void* y, void* sum, void* low, float* mean,
                           float* rstd, void* stream) {
  if (!d || !drop) return EGNN_ERR_NULL;
  if (!dims_ok(d) || !egnn::drop_ok(drop) || (low && d->dtype != EGNN_BF16)) return EGNN_ERR_DIMS;
  if (!drop->rng || !mean != !rstd || (d->N && (!x || !residual || !y || !sum))) return EGNN_ERR_NULL;
  if (ldx < 0 || ldr < 0) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e;
  if ((uintptr_t)drop->rng % 8 || (uintptr_t)x % e || (uintptr_t)residual % e || (uintptr_t)weight % ep || (uintptr_t)bias % ep ||
      (uintptr_t)y % e || (uintptr_t)sum % e || (uintptr_t)low % (d->f32_params ? 2 : 1) || (uintptr_t)mean % 4 || (uintptr_t)rstd % 4)
    return EGNN_ERR_ALIGN;
  Args a{};
  a.x = x; a.ldx = ldx; a.r = residual; a.ldr = ldr; a.w = weight; a.b = bias; a.y = y; a.s = sum;
  a.mean = mean; a.rstd = rstd; a.N = d->N; a.C = d->C; a.eps = d->eps; a.f32_params = d->f32_params != 0;
  a.d = egnn::drop_args(drop);
  a.low = (void*)low;
  if (d->dtype == EGNN_F32) return launch<float, kDrop>(a, false, (hipStream_t)stream);
  if (!low) return launch<egnn::bf16, kDrop>(a, false, (hipStream_t)stream);
  return a.f32_params ? launch<egnn::bf16, kDropLow>(a, false, (hipStream_t)stream) : launch<egnn::bf16, kDropByte>(a, false, (hipStream_t)stream);
}

int32_t egnn_norm_drop_bwd(const EgnnNormDims* d, const EgnnDropout* drop, const void* grad_y, int64_t ldg, const void* sum,
                           int64_t lds, const void* low, const void* weight, const float* mean, const float* rstd, const void* grad_sum,
                           int64_t ldgs, void* grad_x, void* grad_residual, void* grad_weight, void* grad_bias, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (!d || !drop) return EGNN_ERR_NULL;
  if (!dims_ok(d) || !egnn::drop_ok(drop) || (low && d->dtype != EGNN_BF16)) return EGNN_ERR_DIMS;
  if (!drop->rng || (d->N && (!grad_y || !sum || !mean || !rstd || !grad_x || !grad_residual))) return EGNN_ERR_NULL;
  if (ldg < 0 || lds < 0 || (grad_sum && ldgs < 0)) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e;
  if ((uintptr_t)drop->rng % 8 || (uintptr_t)grad_y % e || (uintptr_t)sum % e || (uintptr_t)low % (d->f32_params ? 2 : 1) || (uintptr_t)weight % ep || (uintptr_t)grad_sum % e ||
      (uintptr_t)grad_x % e || (uintptr_t)grad_residual % e || (uintptr_t)grad_weight % ep || (uintptr_t)grad_bias % ep ||
      (uintptr_t)mean % 4 || (uintptr_t)rstd % 4 || (uintptr_t)workspace % 16)
    return EGNN_ERR_ALIGN;
  const bool weights = grad_weight || grad_bias;
  if (weights && (!workspace || workspace_bytes < egnn_norm_bwd_workspace_bytes(d))) return EGNN_ERR_WORKSPACE;
  Args a{};
  a.gy = grad_y; a.ldg = ldg; a.x = sum; a.ldx = lds; a.w = weight; a.mean = (float*)mean; a.rstd = (float*)rstd;
  a.gsum = grad_sum; a.ldgs = ldgs; a.gx = grad_x; a.gr = grad_residual; a.gw = grad_weight; a.gb = grad_bias;
  a.part = weights ? (float*)workspace : nullptr; a.N = d->N; a.C = d->C; a.eps = d->eps; a.f32_params = d->f32_params != 0;
  a.d = egnn::drop_args(drop);
  a.low = (void*)low;
  if (d->dtype == EGNN_F32) return launch<float, kDrop>(a, true, (hipStream_t)stream);
  if (!low) return launch<egnn::bf16, kDrop>(a, true, (hipStream_t)stream);
  return a.f32_params ? launch<egnn::bf16, kDropLow>(a, true, (hipStream_t)stream) : launch<egnn::bf16, kDropByte>(a, true, (hipStream_t)stream);
}

}  // extern "C"
