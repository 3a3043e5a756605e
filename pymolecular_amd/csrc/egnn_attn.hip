// C entries of the segment attention: checks, how the axes are cut, workspaces.
#include "egnn_attn.h"

namespace egnn {
namespace attn {
namespace {

bool dims_ok(const EgnnAttnDims* d) {
  const int64_t top = INT32_MAX - (1 << 18);   // room for a step of every split past the end
  return d && d->Nq >= 0 && d->Nk >= 0 && d->n_seg >= 0 && d->Hq >= 1 && d->Hkv >= 1 && d->Hq % d->Hkv == 0 && d->D >= 8 &&
         d->D <= 128 && d->D % 8 == 0 && (d->dtype == EGNN_F32 || d->dtype == EGNN_BF16) && d->scale - d->scale == 0.f &&
         d->scale != 0.f && d->Nk <= top && d->n_seg <= top && d->Nq <= top && d->Nq * d->Hq <= top;
}

// own: (virtual) rows of the axis that is cut into tiles, other: rows of the axis a tile walks
Plan make_plan(int64_t own, int64_t other, int64_t n_seg, int heads, int widest, bool f32, int D) {
  const int64_t segs = n_seg > 0 ? n_seg : 1, mean = own / segs, len = other / segs;
  auto items_of = [&](int64_t rows) {
    const int64_t tiles = cdiv(own, rows) > n_seg ? cdiv(own, rows) : n_seg;
    return (tiles > 0 ? tiles : 1) * heads;
  };
  Plan p;
  // Measured on both sides, forward and backward in us, bf16 unless stated.  A wave a tile, and a whole small segment
  // (form 0), against 64 rows a workgroup (1): 15 .. 32 rows a segment, D = 64: 33.5 and 44.7; 9 .. 40, D = 16: 35 and 51;
  // 25 .. 45, D = 64: 59 and 41; 20 .. 40, fp32, D = 32: 61 and 37.  64 rows against 128 (2), 4 heads: 80 rows, D = 64, 54 and
  // 61; 100 .. 260, D = 32, 45 and 46; 256 61 and 56 at D = 32, 87 and 86 at 64; 512 94 and 75, 135 and 120.  128 rows only
  // where they fill the device, or splits will: 37 chains of 301 in fp32, 8 heads on 2, 135 and 156; 12,289 rows 1,252 and 881.
  p.form = mean <= kShortMean ? 0 : mean >= 256 && (items_of(128) >= 1024 || len >= 2048) ? 2 : 1;
  if (widest < 0) p.form = 1;
  else if (p.form > widest) p.form = widest;
  const int64_t BQ = p.rows();
  p.slots = own / BQ + n_seg + 2;
  const int64_t items = items_of(BQ);
  p.nsplit = 1;
  if (p.form == 0) {
    if (items < 2048 && len >= 512) p.nsplit = (int)cdiv(4096, items);
  } else if (items < 512 && len >= 512) {
    // Somewhat more workgroups a CU than it holds (four of heads up to 32 wide) and up to six, as evenly on the 256 CUs as
    // may be; a part more costs its share of the joining, per tile about the time of 256 rows in bf16 and 48 in fp32.
    // (Measured with parts of dq half as wide as bf16 has them now.  As against 1,024 workgroups or the next number above, forward and backward: one graph of 2,500 rows, 8 heads, 164
    // and 135 us; of 20,000, 2 heads on 1, 1,096 and 1,044.  Fewer for heads up to 32 wide: 8,000 rows, 8 heads on 2, dk
    // and dv 182 us in 9 parts and 200 in 8.)
    const int64_t most = len / 128, hi = cdiv(1536, items) < most ? cdiv(1536, items) : most;
    const int64_t want = cdiv(D <= 32 ? 1100 : 640, items), lo = want < hi ? want : hi;
    double best = 0.;
    for (int64_t n = lo; n <= hi; n += 1 + lo / 64) {   // at most some hundred
      const double x = (double)(items * n) / 256., cost = (double)cdiv(items * n, 256) / x + (double)(n * (f32 ? 48 : 256)) / (double)len;
      if (n == lo || cost < best) { best = cost; p.nsplit = (int)n; }
    }
  }
  if (p.nsplit > len / 128) p.nsplit = (int)(len / 128 > 0 ? len / 128 : 1);
  if (p.nsplit > 2048) p.nsplit = 2048;
  return p;
}
// The widest form whose registers hold the tile; -1: form 1 alone.  (Spills are left where the next smaller form is slower
// or there is none: of dk and dv, 2 registers at bf16 D = 32 and 3 at fp32 D = 32 with 128 rows, 19 at fp32 above 64.)  dq in
// bf16 above 64 with 128 rows would spill 95.
int widest_q(const EgnnAttnDims* d) { return d->dtype == EGNN_F32 && d->D > 64 ? -1 : 2; }
int widest_dq(const EgnnAttnDims* d) { return d->dtype == EGNN_BF16 && d->D > 64 ? 1 : widest_q(d); }
int widest_k(const EgnnAttnDims* d) {
  return d->dtype == EGNN_F32 && d->D > 64 ? -1 : d->D > (d->dtype == EGNN_F32 ? 32 : 64) ? 1 : 2;
}
Plan plan_q(const EgnnAttnDims* d) { return make_plan(d->Nq * (d->Hq / d->Hkv), d->Nk, d->n_seg, d->Hkv, widest_q(d), d->dtype == EGNN_F32, d->D); }
Plan plan_dq(const EgnnAttnDims* d) { return make_plan(d->Nq * (d->Hq / d->Hkv), d->Nk, d->n_seg, d->Hkv, widest_dq(d), d->dtype == EGNN_F32, d->D); }
Plan plan_k(const EgnnAttnDims* d) { return make_plan(d->Nk, d->Nq * (d->Hq / d->Hkv), d->n_seg, d->Hkv, widest_k(d), d->dtype == EGNN_F32, d->D); }

size_t fwd_bytes(const EgnnAttnDims* d) {
  const Plan p = plan_q(d);
  return p.nsplit == 1 ? 0 : (size_t)p.nsplit * d->Nq * d->Hq * (padded(d->D) + 2) * 4;   // sums, then (m, l)
}
size_t delta_bytes(const EgnnAttnDims* d) { return align_up((size_t)d->Nq * d->Hq * 4); }
size_t bwd_bytes(const EgnnAttnDims* d) {
  const Plan pq = plan_dq(d), pk = plan_k(d);
  // sums of ds k; of bf16 also of p k and of ds
  const size_t q = pq.nsplit == 1 ? 0 : (size_t)pq.nsplit * d->Nq * d->Hq * (d->dtype == EGNN_BF16 ? 2 * padded(d->D) + 1 : padded(d->D)) * 4;
  const size_t k = pk.nsplit == 1 ? 0 : (size_t)pk.nsplit * d->Nk * d->Hkv * 2 * padded(d->D) * 4;
  return delta_bytes(d) + (q > k ? q : k);
}

bool grid_ok(const EgnnAttnDims* d, const Plan& p) { return p.slots * d->Hkv * p.nsplit <= INT32_MAX; }

// rows and heads 16-byte aligned; rows apart from each other or, of an input, all the same one (stride 0); a row at most
// 2^24 bytes and a group's heads at most 2^29 from each other (the kernels' buffer offsets); an output's heads apart too
int check_view(const void* p, int64_t rows, int heads, int D, int64_t rs, int64_t hs, int group, int esz, bool output) {
  if (rows == 0) return EGNN_OK;
  if (!p) return EGNN_ERR_NULL;
  if (rs < 0 || hs < 0 || (rs * esz) % 16 || (hs * esz) % 16 || (rs && rs < D) || rs > (1 << 24) / esz) return EGNN_ERR_STRIDE;
  if (group > 1 && hs > (1 << 29) / esz / (group - 1)) return EGNN_ERR_STRIDE;
  if (output && ((heads > 1 && hs < D) || (rows > 1 && rs < D))) return EGNN_ERR_STRIDE;
  return (uintptr_t)p % 16 ? EGNN_ERR_ALIGN : EGNN_OK;
}

Args make_args(const EgnnAttnDims* d, const EgnnAttnStrides* s) {
  Args a{};
  a.q_r = s->q_row; a.q_h = s->q_head; a.k_r = s->k_row; a.k_h = s->k_head; a.v_r = s->v_row; a.v_h = s->v_head;
  a.o_r = s->out_row; a.o_h = s->out_head; a.go_r = s->grad_out_row; a.go_h = s->grad_out_head;
  a.gq_r = s->grad_q_row; a.gq_h = s->grad_q_head; a.gk_r = s->grad_k_row; a.gk_h = s->grad_k_head;
  a.gv_r = s->grad_v_row; a.gv_h = s->grad_v_head;
  a.Nq = (int32_t)d->Nq; a.Nk = (int32_t)d->Nk; a.B = d->n_seg; a.Hq = d->Hq; a.Hkv = d->Hkv; a.G = d->Hq / d->Hkv; a.D = d->D;
  a.scale = d->scale < 0 ? -d->scale : d->scale;
  a.c2 = a.scale * kLog2e;
  a.flip = d->scale < 0 ? 0x80000000u : 0u;
  a.by_g = Div::of(a.G);
  a.by_heads = Div::of(a.Hkv);
  return a;
}

}  // namespace
}  // namespace attn
}  // namespace egnn

using namespace egnn::attn;

extern "C" {

size_t egnn_attn_fwd_workspace_bytes(const EgnnAttnDims* d) { return dims_ok(d) ? fwd_bytes(d) : 0; }
size_t egnn_attn_bwd_workspace_bytes(const EgnnAttnDims* d) { return dims_ok(d) ? bwd_bytes(d) : 0; }

#define EGNN_TRY(x) do { const int rc_ = (x); if (rc_ != EGNN_OK) return rc_; } while (0)

int32_t egnn_attn_fwd(const EgnnAttnDims* d, const EgnnAttnStrides* s, const void* q, const void* k, const void* v,
                      const int32_t* q_ptr, const int32_t* kv_ptr, const uint8_t* key_mask, void* out, float* lse, void* workspace,
                      size_t workspace_bytes, void* stream) {
  if (!d || !s) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  const int esz = d->dtype == EGNN_F32 ? 4 : 2;
  if (!q_ptr || !kv_ptr) return EGNN_ERR_NULL;
  EGNN_TRY(check_view(q, d->Nq, d->Hq, d->D, s->q_row, s->q_head, d->Hq / d->Hkv, esz, false));
  EGNN_TRY(check_view(k, d->Nk, d->Hkv, d->D, s->k_row, s->k_head, 1, esz, false));
  EGNN_TRY(check_view(v, d->Nk, d->Hkv, d->D, s->v_row, s->v_head, 1, esz, false));
  EGNN_TRY(check_view(out, d->Nq, d->Hq, d->D, s->out_row, s->out_head, d->Hq / d->Hkv, esz, true));
  const Plan p = plan_q(d);
  if (!grid_ok(d, p)) return EGNN_ERR_DIMS;
  const size_t need = fwd_bytes(d);
  if (need && (!workspace || workspace_bytes < need)) return EGNN_ERR_WORKSPACE;
  if (need && (uintptr_t)workspace % 16) return EGNN_ERR_ALIGN;
  if (d->Nq == 0) return EGNN_OK;
  Args a = make_args(d, s);
  a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse; a.q_ptr = q_ptr; a.kv_ptr = kv_ptr; a.mask = key_mask;
  a.same = q_ptr == kv_ptr && a.Nq == a.Nk;
  a.nsplit = p.nsplit;
  a.slots = (uint32_t)p.slots;
  a.guess = (float)(a.B + 2) / (float)a.slots;
  a.by_slots = Div::of(a.slots);
  a.part = (float*)workspace;
  return launch_fwd(a, d->dtype == EGNN_BF16, p, (hipStream_t)stream) ? EGNN_ERR_HIP : EGNN_OK;
}

int32_t egnn_attn_bwd(const EgnnAttnDims* d, const EgnnAttnStrides* s, const void* q, const void* k, const void* v, const void* out,
                      const float* lse, const void* grad_out, const int32_t* q_ptr, const int32_t* kv_ptr, const uint8_t* key_mask,
                      void* grad_q, void* grad_k, void* grad_v, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d || !s) return EGNN_ERR_NULL;
  if (!dims_ok(d)) return EGNN_ERR_DIMS;
  const int esz = d->dtype == EGNN_F32 ? 4 : 2;
  if (!q_ptr || !kv_ptr || (d->Nq && !lse)) return EGNN_ERR_NULL;
  EGNN_TRY(check_view(q, d->Nq, d->Hq, d->D, s->q_row, s->q_head, d->Hq / d->Hkv, esz, false));
  EGNN_TRY(check_view(k, d->Nk, d->Hkv, d->D, s->k_row, s->k_head, 1, esz, false));
  EGNN_TRY(check_view(v, d->Nk, d->Hkv, d->D, s->v_row, s->v_head, 1, esz, false));
  EGNN_TRY(check_view(out, d->Nq, d->Hq, d->D, s->out_row, s->out_head, d->Hq / d->Hkv, esz, false));
  EGNN_TRY(check_view(grad_out, d->Nq, d->Hq, d->D, s->grad_out_row, s->grad_out_head, d->Hq / d->Hkv, esz, false));
  EGNN_TRY(check_view(grad_q, d->Nq, d->Hq, d->D, s->grad_q_row, s->grad_q_head, d->Hq / d->Hkv, esz, true));
  EGNN_TRY(check_view(grad_k, d->Nk, d->Hkv, d->D, s->grad_k_row, s->grad_k_head, 1, esz, true));
  EGNN_TRY(check_view(grad_v, d->Nk, d->Hkv, d->D, s->grad_v_row, s->grad_v_head, 1, esz, true));
  const Plan pq = plan_dq(d), pk = plan_k(d);
  if (!grid_ok(d, pq) || !grid_ok(d, pk)) return EGNN_ERR_DIMS;
  const size_t need = bwd_bytes(d);
  if (need && (!workspace || workspace_bytes < need)) return EGNN_ERR_WORKSPACE;
  if (need && (uintptr_t)workspace % 16) return EGNN_ERR_ALIGN;
  if (d->Nq == 0 && d->Nk == 0) return EGNN_OK;
  Args a = make_args(d, s);
  a.q = q; a.k = k; a.v = v; a.o = out; a.lse = (float*)lse; a.go = grad_out; a.gq = grad_q; a.gk = grad_k; a.gv = grad_v;
  a.q_ptr = q_ptr; a.kv_ptr = kv_ptr; a.mask = key_mask;
  a.same = q_ptr == kv_ptr && a.Nq == a.Nk;
  a.delta = (float*)workspace;
  a.part = (float*)((char*)workspace + delta_bytes(d));
  return launch_bwd(a, d->dtype == EGNN_BF16, pq, pk, (hipStream_t)stream) ? EGNN_ERR_HIP : EGNN_OK;
}

}  // extern "C"
