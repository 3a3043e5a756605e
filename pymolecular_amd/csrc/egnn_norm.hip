// Layer norm over the last axis: the C entries without dropout (kernels and launches: egnn_norm.h).
#include "egnn_norm.h"

using namespace egnn::norm;

extern "C" {

size_t egnn_norm_bwd_workspace_bytes(const EgnnNormDims* d) {
  return d && dims_ok(d) ? (size_t)part_rows(d->N) * 2 * d->C * 4 : 0;
}

int32_t egnn_norm_fwd(const EgnnNormDims* d, const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                      const void* bias, void* y, void* sum, float* mean, float* rstd, void* stream) {
  if (!d) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (!mean != !rstd || (residual && !sum) || (d->N && (!x || !y))) return EGNN_ERR_NULL;
  if (ldx < 0 || (residual && ldr < 0)) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e;
  if ((uintptr_t)x % e || (uintptr_t)residual % e || (uintptr_t)weight % ep || (uintptr_t)bias % ep || (uintptr_t)y % e ||
      (uintptr_t)sum % e || (uintptr_t)mean % 4 || (uintptr_t)rstd % 4)
    return EGNN_ERR_ALIGN;
  Args a{};
  a.x = x; a.ldx = ldx; a.r = residual; a.ldr = ldr; a.w = weight; a.b = bias; a.y = y; a.s = residual ? sum : nullptr;
  a.mean = mean; a.rstd = rstd; a.N = d->N; a.C = d->C; a.eps = d->eps; a.f32_params = d->f32_params != 0;
  return d->dtype == EGNN_BF16 ? launch<egnn::bf16, kPlain>(a, false, (hipStream_t)stream) : launch<float, kPlain>(a, false, (hipStream_t)stream);
}

int32_t egnn_norm_bwd(const EgnnNormDims* d, const void* grad_y, int64_t ldg, const void* sum, int64_t lds, const void* weight,
                      const float* mean, const float* rstd, const void* grad_sum, int64_t ldgs, void* grad_x, void* grad_weight,
                      void* grad_bias, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  if (d->N && (!grad_y || !sum || !mean || !rstd || !grad_x)) return EGNN_ERR_NULL;
  if (ldg < 0 || lds < 0 || (grad_sum && ldgs < 0)) return EGNN_ERR_STRIDE;
  const uintptr_t e = d->dtype == EGNN_F32 ? 4 : 2, ep = d->f32_params ? 4 : e;
  if ((uintptr_t)grad_y % e || (uintptr_t)sum % e || (uintptr_t)weight % ep || (uintptr_t)grad_sum % e || (uintptr_t)grad_x % e ||
      (uintptr_t)grad_weight % ep || (uintptr_t)grad_bias % ep || (uintptr_t)mean % 4 || (uintptr_t)rstd % 4 || (uintptr_t)workspace % 16)
    return EGNN_ERR_ALIGN;
  const bool weights = grad_weight || grad_bias;
  if (weights && (!workspace || workspace_bytes < egnn_norm_bwd_workspace_bytes(d))) return EGNN_ERR_WORKSPACE;
  Args a{};
  a.gy = grad_y; a.ldg = ldg; a.x = sum; a.ldx = lds; a.w = weight; a.mean = (float*)mean; a.rstd = (float*)rstd;
  a.gsum = grad_sum; a.ldgs = ldgs; a.gx = grad_x; a.gw = grad_weight; a.gb = grad_bias;
  a.part = weights ? (float*)workspace : nullptr; a.N = d->N; a.C = d->C; a.eps = d->eps; a.f32_params = d->f32_params != 0;
  return d->dtype == EGNN_BF16 ? launch<egnn::bf16, kPlain>(a, true, (hipStream_t)stream) : launch<float, kPlain>(a, true, (hipStream_t)stream);
}

}  // extern "C"
