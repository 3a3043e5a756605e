// One message-passing layer (GCLLayerFn of layer_fn.py) as a native autograd node.
//
// The kernels of a layer over a few graphs take less time than the Python around them (molecule-sized calls:
// 45 us of kernels behind 75 us of host work forward, 300 us behind 450 us forward and backward), most of it tensor
// allocations, argument conversion and the autograd engine's calls back into Python.  This is the same sequence of
// C-ABI calls with the allocations and the backward in C++.  It takes only calls whose tensors need no conversion
// (gcl_layer returns None for any other, and the Python node, which converts and reports errors, runs instead):
// plain device tensors of one dtype and device, contiguous, shapes that fit together.
#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/hip/HIPStream.h>
#include <c10/core/DeviceGuard.h>
#include <cmath>
#include "../../include/egnn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Opt;

// the status as the Python bindings report it (EgnnError); any thread
void check(const char* fn, int32_t status) {
  if (status == EGNN_OK) return;
  pybind11::gil_scoped_acquire gil;
  pybind11::module_::import("pymolecular_amd._capi").attr("check")(fn, status);
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
Tensor get(const Opt& t) { return t.has_value() ? *t : Tensor(); }
bool aligned16(const Tensor& t) { return ((uintptr_t)t.data_ptr() & 15) == 0; }
// unit-stride rows that start 16-byte aligned and do not overlap (an expanded gradient's have stride 0), else a copy
Tensor rowmajor(const Tensor& t) {
  return t.stride(1) == 1 && t.stride(0) >= t.size(1) && (t.stride(0) * t.element_size()) % 16 == 0 && aligned16(t)
             ? t : t.clone(at::MemoryFormat::Contiguous);
}

// no tensor subclass, functorch wrapper or functionalised tensor, on h's device
bool plain(const Tensor& t, const Tensor& h) {
  const auto ks = t.key_set();
  return t.is_cuda() && t.device() == h.device() && t.layout() == c10::kStrided && !t.is_conj() && !t.is_neg() &&
         !ks.has(c10::DispatchKey::Python) && !ks.has(c10::DispatchKey::FuncTorchBatched) &&
         !ks.has(c10::DispatchKey::FuncTorchGradWrapper) && !ks.has(c10::DispatchKey::Functionalize) &&
         !t._fw_grad(0).defined();
}
bool fits(const Tensor& t, const Tensor& h, at::ScalarType dt, std::initializer_list<int64_t> shape) {
  return plain(t, h) && t.scalar_type() == dt && t.sizes() == c10::IntArrayRef(shape) && t.is_contiguous();
}
bool fits_opt(const Opt& t, const Tensor& h, at::ScalarType dt, int64_t n) { return !t || fits(*t, h, dt, {n}); }

// the layer's tensors in the order they are saved
enum { kH, kX, kE, kRow, kCol, kPerm, kW1, kW2, kM1, kM2, kB1, kB2, kBx, kN0, kN2, kSched, kPQ, kAgg, kPre, kAct, kCount };

struct Layer {
  variable_list t;
  bool mean, residual, eq, nb0, nb2;
  EgnnDims dims() const {
    EgnnDims d{};
    const Tensor &h = t[kH], &w1 = t[kW1];
    d.N = h.size(0); d.E = t[kCol].numel(); d.F = (int32_t)h.size(1);
    d.FE = t[kE].defined() ? (int32_t)t[kE].size(1) : 0;
    d.H = (int32_t)w1.size(0); d.O = (int32_t)t[kW2].size(0); d.M = eq ? (int32_t)t[kM1].size(0) : d.O;
    d.equivariant = eq; d.mean_agg = mean;
    d.dtype = h.scalar_type() == at::kFloat ? EGNN_F32 : EGNN_BF16;
    d.weight_layout = EGNN_WEIGHTS_LINEAR;
    d.flags = eq ? EGNN_FLAG_COORD_RESIDUAL : 0;
    return d;
  }
  EgnnNodeDims node_dims() const {
    EgnnNodeDims d{};
    d.N = t[kH].size(0); d.K1 = (int32_t)t[kH].size(1); d.K2 = (int32_t)t[kW2].size(0);
    d.Hn = (int32_t)t[kN0].size(0); d.Fo = (int32_t)t[kN2].size(0);
    d.residual = residual; d.dtype = t[kH].scalar_type() == at::kFloat ? EGNN_F32 : EGNN_BF16;
    return d;
  }
};

class GclLayer : public torch::autograd::Function<GclLayer> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& h, const Opt& x, const Opt& ef, const Tensor& row,
                               const Tensor& col, const Opt& perm, const Tensor& e0w, const Opt& e0b, const Tensor& e2w,
                               const Opt& e2b, const Opt& c0w, const Opt& c0b, const Opt& c2w, const Tensor& n0w,
                               const Opt& n0b, const Tensor& n2w, const Opt& n2b, const Tensor& sched, bool mean,
                               bool residual, bool eq) {
    Layer a{{h, get(x), get(ef), row, col, get(perm), e0w, e2w, get(c0w), get(c2w), get(e0b), get(e2b), get(c0b), n0w,
             n2w, sched, {}, {}, {}, {}}, mean, residual, eq, n0b.has_value(), n2b.has_value()};
    const EgnnDims d = a.dims();
    const EgnnNodeDims nd = a.node_dims();
    const auto act = h.options(), bytes = act.dtype(at::kByte), f32 = act.dtype(at::kFloat);
    void* st = stream_of(h);
    a.t[kPQ] = at::empty({(int64_t)std::max<size_t>(egnn_node_proj_bytes(&d), 16)}, bytes);
    a.t[kAgg] = at::empty({d.N, d.O}, act);
    Tensor x_new = eq ? at::empty({d.N, 3}, f32) : Tensor();
    {
      const size_t nb = egnn_fwd_workspace_bytes(&d);
      const Tensor ws = at::empty({(int64_t)nb}, bytes);
      EgnnStrides s{};
      s.h = h.stride(0); s.coord = eq ? 3 : 4; s.edge = ef ? ef->stride(0) : 0; s.msg = d.O; s.mov = 3;
      check("egnn_fwd", egnn_fwd(&d, &s, ptr(h), ptr<float>(a.t[kX]), ptr(a.t[kE]), ptr<int32_t>(row), ptr<int32_t>(col),
                                 ptr<int32_t>(a.t[kPerm]), ptr(e0w), ptr(e2w), ptr(a.t[kM1]), ptr(a.t[kM2]), ptr(a.t[kB1]),
                                 ptr(a.t[kB2]), ptr(a.t[kBx]), ptr(a.t[kAgg]), ptr<float>(x_new), ptr(a.t[kPQ]), ptr(sched),
                                 ptr(ws), nb, st));
    }
    a.t[kPre] = at::empty({d.N, nd.Hn}, act);
    if (egnn_node_act_required(&nd)) a.t[kAct] = at::empty({d.N, nd.Hn}, act);
    Tensor out = at::empty({d.N, nd.Fo}, act);
    check("egnn_node_fwd", egnn_node_fwd(&nd, ptr(h), h.stride(0), ptr(a.t[kAgg]), d.O, ptr(n0w), ptr(get(n0b)), ptr(n2w),
                                         ptr(get(n2b)), ptr(a.t[kPre]), ptr(a.t[kAct]), ptr(out), nd.Fo, st));
    ctx->save_for_backward(a.t);
    ctx->saved_data["flags"] = (int64_t)(mean | residual << 1 | eq << 2 | a.nb0 << 3 | a.nb2 << 4);
    return eq ? variable_list{out, x_new} : variable_list{out};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t f = ctx->saved_data["flags"].toInt();
    Layer a{ctx->get_saved_variables(), bool(f & 1), bool(f & 2), bool(f & 4), bool(f & 8), bool(f & 16)};
    const Tensor &h = a.t[kH], &x = a.t[kX], &ef = a.t[kE], &w1 = a.t[kW1], &w2 = a.t[kW2];
    EgnnDims d = a.dims();
    const EgnnNodeDims nd = a.node_dims();
    const auto act = h.options(), bytes = act.dtype(at::kByte), f32 = act.dtype(at::kFloat);
    void* st = stream_of(h);
    // the node update's backward: grad_x = [dL/dh | dL/dagg]
    const Tensor gout = grads[0].defined() ? rowmajor(grads[0].to(h.scalar_type())) : at::zeros({d.N, nd.Fo}, act);
    const int64_t K = nd.K1 + nd.K2;
    const Tensor grad_x = at::empty({d.N, K}, act);
    const Tensor gn0 = at::empty_like(a.t[kN0]), gn2 = at::empty_like(a.t[kN2]);
    const Tensor gnb0 = a.nb0 ? at::empty({nd.Hn}, act) : Tensor(), gnb2 = a.nb2 ? at::empty({nd.Fo}, act) : Tensor();
    {
      const size_t nb = egnn_node_bwd_workspace_bytes(&nd);
      const Tensor ws = at::empty({(int64_t)std::max<size_t>(nb, 16)}, bytes);
      check("egnn_node_bwd", egnn_node_bwd(&nd, ptr(h), h.stride(0), ptr(a.t[kAgg]), d.O, ptr(a.t[kN0]), ptr(a.t[kN2]),
                                           ptr(a.t[kPre]), ptr(a.t[kAct]), ptr(gout), gout.stride(0), ptr(grad_x), ptr(gn0),
                                           ptr(gnb0), ptr(gn2), ptr(gnb2), ptr(ws), nb, st));
    }
    // the messages' backward, its gradient of h added to the node update's
    const Tensor grad_h = grad_x.narrow(1, 0, nd.K1);
    const Tensor gm = rowmajor(grad_x.narrow(1, nd.K1, nd.K2));
    Tensor gx, grad_c;
    if (a.eq) {
      gx = grads.size() > 1 && grads[1].defined() ? grads[1].to(at::kFloat).contiguous() : at::zeros({d.N, 3}, f32);
      grad_c = at::empty({d.N, 3}, f32);
    }
    auto like = [](const Tensor& t) { return t.defined() ? at::empty_like(t) : Tensor(); };
    const Tensor g1 = like(w1), g2 = like(w2), gm1 = like(a.t[kM1]), gm2 = like(a.t[kM2]);
    const Tensor gb1 = like(a.t[kB1]), gb2 = like(a.t[kB2]), gbx = like(a.t[kBx]);
    {
      d.flags |= EGNN_FLAG_ACCUMULATE_GRAD_H;
      const size_t nb = egnn_bwd_workspace_bytes(&d);
      const Tensor ws = at::empty({(int64_t)nb}, bytes);
      EgnnStrides s{};
      s.h = h.stride(0); s.coord = 3; s.edge = ef.defined() ? ef.stride(0) : 0; s.msg = gm.stride(0);
      s.mov = 3; s.grad_h = grad_h.stride(0);
      check("egnn_bwd", egnn_bwd(&d, &s, ptr(h), ptr<float>(x), ptr(ef), ptr<int32_t>(a.t[kRow]), ptr<int32_t>(a.t[kCol]),
                                 ptr<int32_t>(a.t[kPerm]), ptr(w1), ptr(w2), ptr(a.t[kM1]), ptr(a.t[kM2]), ptr(a.t[kB1]),
                                 ptr(a.t[kB2]), ptr(a.t[kBx]), ptr(gm), ptr<float>(gx), ptr(grad_h), ptr<float>(grad_c),
                                 ptr(g1), ptr(g2), ptr(gm1), ptr(gm2), ptr(gb1), ptr(gb2), ptr(gbx), ptr(a.t[kPQ]),
                                 ptr(a.t[kSched]), ptr(ws), nb, st));
    }
    return {grad_h, grad_c, {}, {}, {}, {}, g1, gb1, g2, gb2, gm1, gbx, gm2, gn0, gnb0, gn2, gnb2, {}, {}, {}, {}};
  }
};

// The layer, or None when a tensor would need a conversion or the dimensions are not supported
pybind11::object gcl_layer(const Tensor& h, const Opt& x, const Opt& ef, const Tensor& row, const Tensor& col,
                           const Opt& perm, const Tensor& e0w, const Opt& e0b, const Tensor& e2w, const Opt& e2b,
                           const Opt& c0w, const Opt& c0b, const Opt& c2w, const Tensor& n0w, const Opt& n0b,
                           const Tensor& n2w, const Opt& n2b, const Tensor& sched, bool mean, bool residual, bool eq) {
  const pybind11::object none = pybind11::none();
  if (torch::jit::tracer::isTracing() || h.dim() != 2 || h.size(0) < 1 || e0w.dim() != 2 || e2w.dim() != 2 ||
      n0w.dim() != 2 || n2w.dim() != 2 || col.dim() != 1)
    return none;
  const auto dt = h.scalar_type();
  if (dt != at::kFloat && dt != at::kBFloat16) return none;
  const int64_t N = h.size(0), F = h.size(1), H = e0w.size(0), O = e2w.size(0), Hn = n0w.size(0), Fo = n2w.size(0);
  const int64_t g = eq ? 1 : 0, FE = ef ? (ef->dim() == 2 ? ef->size(1) : -1) : 0;
  if (FE < 0 || (ef && (ef->size(0) < 1 || FE < 1)) || F % 16 || Hn % 8 || Fo % 8 || O % 8 || (residual && Fo != F)) return none;
  if (!fits(h, h, dt, {N, F}) || !aligned16(h) || !fits(e0w, h, dt, {H, 2 * F + g + FE}) || !fits(e2w, h, dt, {O, H}) ||
      !fits(n0w, h, dt, {Hn, F + O}) || !fits(n2w, h, dt, {Fo, Hn}) || !fits_opt(e0b, h, dt, H) ||
      !fits_opt(e2b, h, dt, O) || !fits_opt(n0b, h, dt, Hn) || !fits_opt(n2b, h, dt, Fo))
    return none;
  if (ef && !fits(*ef, h, dt, {ef->size(0), FE})) return none;
  if (!fits(row, h, at::kInt, {N + 1}) || !fits(col, h, at::kInt, {col.numel()}) ||
      (perm && !fits(*perm, h, at::kInt, {col.numel()})) || !plain(sched, h))
    return none;
  if (eq) {
    if (!x || !c0w || !c2w || c0w->dim() != 2 || !fits(*x, h, at::kFloat, {N, 3})) return none;
    const int64_t M = c0w->size(0);
    if (!fits(*c0w, h, dt, {M, O}) || !fits_opt(c0b, h, dt, M) || !plain(*c2w, h) || c2w->scalar_type() != dt ||
        c2w->numel() != M || !c2w->is_contiguous())
      return none;
  } else if (x || c0w || c0b || c2w) {
    return none;
  }
  {   // dimensions the library refuses are reported by the Python path
    Layer a{{h, get(x), get(ef), row, col, get(perm), e0w, e2w, get(c0w), get(c2w), {}, {}, {}, n0w, n2w, sched, {}, {}, {}, {}},
            mean, residual, eq, false, false};
    const EgnnDims d = a.dims();
    if (egnn_fwd_workspace_bytes(&d) == 0) return none;
  }
  variable_list r;
  {
    pybind11::gil_scoped_release nogil;
    r = GclLayer::apply(h, x, ef, row, col, perm, e0w, e0b, e2w, e2b, c0w, c0b, c2w, n0w, n0b, n2w, n2b, sched, mean,
                        residual, eq);
  }
  if (eq) return pybind11::make_tuple(r[0], r[1]);
  return pybind11::cast(r[0]);
}

// ---- segment attention and layer norm ---------------------------------------------
// The functions of segment_attention.py and layer_norm.py for tensors that need no conversion: checks, allocations and
// the library call without returning to Python (a forward and backward over a small batch of molecules: 46 us of host
// work in Python for 24 us of kernels).  None, before anything is allocated, for every other call: the Python path
// converts, or reports the error.
bool heads_ok(const Tensor& t, const Tensor& h, int64_t n, int64_t heads, int64_t d, int64_t group = 1) {
  const int64_t e = t.element_size(), per = 16 / e;
  return plain(t, h) && t.scalar_type() == h.scalar_type() && t.dim() == 3 && t.size(0) == n && t.size(1) == heads &&
         t.size(2) == d && t.stride(2) == 1 && t.stride(0) % per == 0 && t.stride(1) % per == 0 && aligned16(t) &&
         (t.stride(0) == 0 || (t.stride(0) >= d && t.stride(0) * e <= 1 << 24)) && (group - 1) * t.stride(1) * e <= 1 << 29;
}
bool attn_ok(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr, const Opt& kv_ptr, const Opt& mask,
             double scale) {
  if (torch::jit::tracer::isTracing() || q.dim() != 3 || k.dim() != 3) return false;
  const auto dt = q.scalar_type();
  const int64_t d = q.size(2), hk = k.size(1);
  if ((dt != at::kFloat && dt != at::kBFloat16) || d < 8 || d > 128 || d % 8 || hk < 1 || q.size(1) < 1 || q.size(1) % hk ||
      q.size(1) > INT32_MAX || q_ptr.numel() - 1 > INT32_MAX || !std::isfinite(scale) || scale == 0.0 ||
      (!kv_ptr && q.size(0) != k.size(0)))
    return false;
  if (q_ptr.dim() != 1 || q_ptr.numel() < 1 || !fits(q_ptr, q, at::kInt, {q_ptr.numel()}) ||
      (kv_ptr && !fits(*kv_ptr, q, at::kInt, {q_ptr.numel()})))
    return false;
  if (mask && !fits(*mask, q, at::kBool, {k.size(0)}) && !fits(*mask, q, at::kByte, {k.size(0)})) return false;
  return heads_ok(q, q, q.size(0), q.size(1), d, q.size(1) / hk) && heads_ok(k, q, k.size(0), hk, d) && heads_ok(v, q, k.size(0), hk, d);
}
EgnnAttnDims attn_dims(const Tensor& q, const Tensor& k, const Tensor& q_ptr, double scale) {
  EgnnAttnDims d{};
  d.Nq = q.size(0); d.Nk = k.size(0); d.n_seg = (int32_t)(q_ptr.numel() - 1);
  d.Hq = (int32_t)q.size(1); d.Hkv = (int32_t)k.size(1); d.D = (int32_t)q.size(2);
  d.dtype = q.scalar_type() == at::kFloat ? EGNN_F32 : EGNN_BF16;
  d.scale = (float)scale;
  return d;
}
Tensor workspace(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

pybind11::object attn_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr, const Opt& kv_ptr,
                              const Opt& mask, double scale, bool need_lse) {
  if (!attn_ok(q, k, v, q_ptr, kv_ptr, mask, scale)) return pybind11::none();
  const EgnnAttnDims d = attn_dims(q, k, q_ptr, scale);
  Tensor out = at::empty({d.Nq, d.Hq, d.D}, q.options());
  Tensor lse = need_lse ? at::empty({d.Hq, d.Nq}, q.options().dtype(at::kFloat)) : Tensor();
  const size_t nb = egnn_attn_fwd_workspace_bytes(&d);
  const Tensor ws = workspace(nb, q);
  EgnnAttnStrides s{};
  s.q_row = q.stride(0); s.q_head = q.stride(1); s.k_row = k.stride(0); s.k_head = k.stride(1);
  s.v_row = v.stride(0); s.v_head = v.stride(1); s.out_row = out.stride(0); s.out_head = out.stride(1);
  check("egnn_attn_fwd", egnn_attn_fwd(&d, &s, ptr(q), ptr(k), ptr(v), ptr<int32_t>(q_ptr), ptr<int32_t>(kv_ptr ? *kv_ptr : q_ptr),
                                       ptr<uint8_t>(get(mask)), ptr(out), ptr<float>(lse), ptr(ws), nb, stream_of(q)));
  return pybind11::make_tuple(out, need_lse ? pybind11::cast(lse) : pybind11::none());
}

pybind11::object attn_backward(const Tensor& go, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out,
                               const Tensor& lse, const Tensor& q_ptr, const Opt& kv_ptr, const Opt& mask, double scale,
                               const std::optional<std::vector<Tensor>>& into) {
  if (!attn_ok(q, k, v, q_ptr, kv_ptr, mask, scale) || !heads_ok(go, q, q.size(0), q.size(1), q.size(2), q.size(1) / k.size(1)) ||
      !heads_ok(out, q, q.size(0), q.size(1), q.size(2), q.size(1) / k.size(1)) || !fits(lse, q, at::kFloat, {q.size(1), q.size(0)}))
    return pybind11::none();
  const EgnnAttnDims d = attn_dims(q, k, q_ptr, scale);
  if (into && (into->size() != 3 || !heads_ok((*into)[0], q, d.Nq, d.Hq, d.D) || !heads_ok((*into)[1], q, d.Nk, d.Hkv, d.D) ||
               !heads_ok((*into)[2], q, d.Nk, d.Hkv, d.D)))
    return pybind11::none();
  const Tensor gq = into ? (*into)[0] : at::empty({d.Nq, d.Hq, d.D}, q.options()),
               gk = into ? (*into)[1] : at::empty({d.Nk, d.Hkv, d.D}, q.options()),
               gv = into ? (*into)[2] : at::empty({d.Nk, d.Hkv, d.D}, q.options());
  const size_t nb = egnn_attn_bwd_workspace_bytes(&d);
  const Tensor ws = workspace(nb, q);
  EgnnAttnStrides s{};
  s.q_row = q.stride(0); s.q_head = q.stride(1); s.k_row = k.stride(0); s.k_head = k.stride(1);
  s.v_row = v.stride(0); s.v_head = v.stride(1); s.out_row = out.stride(0); s.out_head = out.stride(1);
  s.grad_out_row = go.stride(0); s.grad_out_head = go.stride(1); s.grad_q_row = gq.stride(0); s.grad_q_head = gq.stride(1);
  s.grad_k_row = gk.stride(0); s.grad_k_head = gk.stride(1); s.grad_v_row = gv.stride(0); s.grad_v_head = gv.stride(1);
  check("egnn_attn_bwd", egnn_attn_bwd(&d, &s, ptr(q), ptr(k), ptr(v), ptr(out), ptr<float>(lse), ptr(go), ptr<int32_t>(q_ptr),
                                       ptr<int32_t>(kv_ptr ? *kv_ptr : q_ptr), ptr<uint8_t>(get(mask)), ptr(gq), ptr(gk), ptr(gv),
                                       ptr(ws), nb, stream_of(q)));
  return pybind11::make_tuple(gq, gk, gv);
}

// contiguous rows of one dtype; the parameters of that one too, or (f32) of fp32
bool norm_ok(const Tensor& x, const Opt& w, const Opt& b, double eps, bool f32) {
  const auto dt = x.scalar_type();
  return !torch::jit::tracer::isTracing() && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 1 << 20 && (dt == at::kFloat || dt == at::kBFloat16) &&
         plain(x, x) && x.is_contiguous() && fits_opt(w, x, f32 ? at::kFloat : dt, x.size(-1)) &&
         fits_opt(b, x, f32 ? at::kFloat : dt, x.size(-1)) && eps >= 0 && std::isfinite(eps);
}
bool same_rows(const Tensor& t, const Tensor& x) {
  return plain(t, x) && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes() && t.is_contiguous();
}
EgnnNormDims norm_dims(const Tensor& x, double eps, bool f32) {
  EgnnNormDims d{};
  d.C = (int32_t)x.size(-1); d.N = x.numel() / x.size(-1);
  d.dtype = x.scalar_type() == at::kFloat ? EGNN_F32 : EGNN_BF16;
  d.eps = (float)eps;
  d.f32_params = f32 && d.dtype == EGNN_BF16;
  return d;
}

pybind11::object norm_forward(const Tensor& x, const Opt& w, const Opt& b, double eps, const Opt& res, bool need_stats) {
  const bool f32 = (w && w->scalar_type() == at::kFloat) || (b && b->scalar_type() == at::kFloat);
  if (!norm_ok(x, w, b, eps, f32) || (res && !same_rows(*res, x))) return pybind11::none();
  const EgnnNormDims d = norm_dims(x, eps, f32);
  const auto stat = x.options().dtype(at::kFloat);
  const Tensor y = at::empty(x.sizes(), x.options()), s = res ? at::empty(x.sizes(), x.options()) : x;
  const Tensor mean = need_stats ? at::empty({d.N}, stat) : Tensor(), rstd = need_stats ? at::empty({d.N}, stat) : Tensor();
  check("egnn_norm_fwd", egnn_norm_fwd(&d, ptr(x), d.C, ptr(get(res)), d.C, ptr(get(w)), ptr(get(b)), ptr(y),
                                       res ? ptr(s) : nullptr, ptr<float>(mean), ptr<float>(rstd), stream_of(x)));
  if (!need_stats) return pybind11::make_tuple(y, s, pybind11::none(), pybind11::none());
  return pybind11::make_tuple(y, s, mean, rstd);
}

// f32: the weight is, and the gradients of weight and bias are wanted in, fp32
pybind11::object norm_backward(const Tensor& gy, const Tensor& s, const Opt& w, const Tensor& mean, const Tensor& rstd,
                               const Opt& gsum, bool need_w, bool need_b, bool f32) {
  if (!norm_ok(s, w, Opt(), 0.0, f32) || !same_rows(gy, s) || (gsum && !same_rows(*gsum, s))) return pybind11::none();
  const EgnnNormDims d = norm_dims(s, 0.0, f32);
  if (!fits(mean, s, at::kFloat, {d.N}) || !fits(rstd, s, at::kFloat, {d.N})) return pybind11::none();
  const Tensor gx = at::empty(s.sizes(), s.options());
  const auto param = s.options().dtype(f32 ? at::kFloat : s.scalar_type());
  const Tensor gw = need_w ? at::empty({d.C}, param) : Tensor(), gb = need_b ? at::empty({d.C}, param) : Tensor();
  const size_t nb = need_w || need_b ? egnn_norm_bwd_workspace_bytes(&d) : 0;
  const Tensor ws = workspace(nb, s);
  check("egnn_norm_bwd", egnn_norm_bwd(&d, ptr(gy), d.C, ptr(s), d.C, ptr(get(w)), ptr<float>(mean), ptr<float>(rstd),
                                       ptr(get(gsum)), d.C, ptr(gx), ptr(gw), ptr(gb), ptr(ws), nb, stream_of(s)));
  auto out = [](const Tensor& t) -> pybind11::object { return t.defined() ? pybind11::cast(t) : pybind11::none(); };
  return pybind11::make_tuple(gx, out(gw), out(gb));
}

// ---- dropout ------------------------------------------------------------------------
bool drop_ok(const Tensor& x, double p, const Tensor& rng) { return p >= 0.0 && p <= 1.0 && fits(rng, x, at::kLong, {2}); }

pybind11::object dropout(const Tensor& x, double p, const Tensor& rng, int64_t site, const Opt& res) {
  if (!norm_ok(x, Opt(), Opt(), 0.0, false) || !drop_ok(x, p, rng) || (res && !same_rows(*res, x))) return pybind11::none();
  const c10::DeviceGuard device(x.device());
  const Tensor y = at::empty(x.sizes(), x.options());
  const int64_t C = x.size(-1);
  const EgnnDropout d{ptr<const int64_t>(rng), site, p};
  check("egnn_dropout", egnn_dropout(&d, x.scalar_type() == at::kFloat ? EGNN_F32 : EGNN_BF16, x.numel() / C, (int32_t)C, ptr(x), C,
                                     ptr(get(res)), C, ptr(y), stream_of(x)));
  return pybind11::cast(y);
}

pybind11::object norm_drop_forward(const Tensor& x, const Opt& res, double p, const Tensor& rng, int64_t site, const Opt& w,
                                   const Opt& b, double eps, bool need_stats) {
  const bool f32 = (w && w->scalar_type() == at::kFloat) || (b && b->scalar_type() == at::kFloat);
  if (!norm_ok(x, w, b, eps, f32) || !res || !same_rows(*res, x) || !drop_ok(x, p, rng)) return pybind11::none();
  const EgnnNormDims d = norm_dims(x, eps, f32);
  const EgnnDropout dr{ptr<const int64_t>(rng), site, p};
  const auto stat = x.options().dtype(at::kFloat);
  const c10::DeviceGuard device(x.device());
  const Tensor y = at::empty(x.sizes(), x.options()), s = at::empty(x.sizes(), x.options());
  const Tensor mean = need_stats ? at::empty({d.N}, stat) : Tensor(), rstd = need_stats ? at::empty({d.N}, stat) : Tensor();
  const Tensor low = need_stats && d.dtype == EGNN_BF16 ? at::empty(x.sizes(), x.options().dtype(d.f32_params ? at::kShort : at::kChar)) : Tensor();
  check("egnn_norm_drop_fwd", egnn_norm_drop_fwd(&d, &dr, ptr(x), d.C, ptr(*res), d.C, ptr(get(w)), ptr(get(b)), ptr(y), ptr(s),
                                                 ptr(low), ptr<float>(mean), ptr<float>(rstd), stream_of(x)));
  if (!need_stats) return pybind11::make_tuple(y, s, pybind11::none(), pybind11::none());
  if (low.defined()) return pybind11::make_tuple(y, s, mean, pybind11::make_tuple(rstd, low));
  return pybind11::make_tuple(y, s, mean, rstd);
}

pybind11::object norm_drop_backward(const Tensor& gy, const Tensor& s, double p, const Tensor& rng, int64_t site, const Opt& w,
                                    const Tensor& mean, const Tensor& rstd, const Opt& low, const Opt& gsum, bool need_w, bool need_b, bool f32) {
  if (!norm_ok(s, w, Opt(), 0.0, f32) || !same_rows(gy, s) || (gsum && !same_rows(*gsum, s)) || !drop_ok(s, p, rng) ||
      (low && (s.scalar_type() != at::kBFloat16 || !plain(*low, s) || low->scalar_type() != (f32 ? at::kShort : at::kChar) || low->sizes() != s.sizes() ||
               !low->is_contiguous())))
    return pybind11::none();
  const EgnnNormDims d = norm_dims(s, 0.0, f32);
  if (!fits(mean, s, at::kFloat, {d.N}) || !fits(rstd, s, at::kFloat, {d.N})) return pybind11::none();
  const EgnnDropout dr{ptr<const int64_t>(rng), site, p};
  const c10::DeviceGuard device(s.device());
  const Tensor gx = at::empty(s.sizes(), s.options()), gr = at::empty(s.sizes(), s.options());
  const auto param = s.options().dtype(f32 ? at::kFloat : s.scalar_type());
  const Tensor gw = need_w ? at::empty({d.C}, param) : Tensor(), gb = need_b ? at::empty({d.C}, param) : Tensor();
  const size_t nb = need_w || need_b ? egnn_norm_bwd_workspace_bytes(&d) : 0;
  const Tensor ws = workspace(nb, s);
  check("egnn_norm_drop_bwd", egnn_norm_drop_bwd(&d, &dr, ptr(gy), d.C, ptr(s), d.C, ptr(get(low)), ptr(get(w)), ptr<float>(mean), ptr<float>(rstd),
                                                 ptr(get(gsum)), d.C, ptr(gx), ptr(gr), ptr(gw), ptr(gb), ptr(ws), nb, stream_of(s)));
  auto out = [](const Tensor& t) -> pybind11::object { return t.defined() ? pybind11::cast(t) : pybind11::none(); };
  return pybind11::make_tuple(gx, gr, out(gw), out(gb));
}

// ---- rows of a table -------------------------------------------------------------------
// tokens of any shape, contiguous; rows of dtype dt and a table of that one, or of fp32 beside bf16 rows
bool embed_ok(const Tensor& tokens, int64_t V, int64_t C, at::ScalarType dt, at::ScalarType table) {
  const auto it = tokens.scalar_type();
  return !torch::jit::tracer::isTracing() && plain(tokens, tokens) && tokens.is_contiguous() && (it == at::kInt || it == at::kLong) &&
         (dt == at::kFloat || dt == at::kBFloat16) && (table == dt || table == at::kFloat) && V >= 1 && V <= INT32_MAX && C >= 1 &&
         C <= 1 << 20 && tokens.numel() <= INT32_MAX;
}
EgnnEmbedDims embed_dims(const Tensor& tokens, int64_t V, int64_t C, double scale, at::ScalarType dt, at::ScalarType table) {
  EgnnEmbedDims d{};
  d.N = tokens.numel(); d.V = (int32_t)V; d.C = (int32_t)C;
  d.dtype = dt == at::kFloat ? EGNN_F32 : EGNN_BF16;
  d.f32_table = table != dt;
  d.index64 = tokens.scalar_type() == at::kLong;
  d.scale = (float)scale;
  return d;
}

pybind11::object embed_forward(const Tensor& tokens, const Tensor& w, double scale, at::ScalarType dt) {
  if (w.dim() != 2 || !plain(w, tokens) || w.stride(1) != 1 || w.stride(0) < w.size(1) || !std::isfinite(scale) ||
      !embed_ok(tokens, w.size(0), w.size(1), dt, w.scalar_type()))
    return pybind11::none();
  const EgnnEmbedDims d = embed_dims(tokens, w.size(0), w.size(1), scale, dt, w.scalar_type());
  auto shape = tokens.sizes().vec();
  shape.push_back(d.C);
  const c10::DeviceGuard device(w.device());
  const Tensor out = at::empty(shape, w.options().dtype(dt));
  check("egnn_embed_fwd", egnn_embed_fwd(&d, ptr(tokens), ptr(w), w.stride(0), ptr(out), stream_of(w)));
  return pybind11::cast(out);
}

pybind11::object embed_backward(const Tensor& go, const Tensor& tokens, int64_t V, double scale, int64_t padding, at::ScalarType table) {
  const auto dt = go.scalar_type();
  if (go.dim() != tokens.dim() + 1 || !plain(go, tokens) || !go.is_contiguous() || !std::isfinite(scale) ||
      !embed_ok(tokens, V, go.size(-1), dt, table) || go.sizes().slice(0, tokens.dim()) != tokens.sizes() || padding < -1 || padding >= V)
    return pybind11::none();
  const EgnnEmbedDims d = embed_dims(tokens, V, go.size(-1), scale, dt, table);
  const c10::DeviceGuard device(go.device());
  const Tensor gw = at::empty({V, d.C}, go.options().dtype(table));
  const size_t nb = egnn_embed_bwd_workspace_bytes(&d);
  const Tensor ws = workspace(nb, go);
  check("egnn_embed_bwd", egnn_embed_bwd(&d, padding, ptr(go), d.C, ptr(tokens), ptr(gw), ptr(ws), nb, stream_of(go)));
  return pybind11::cast(gw);
}

// ---- norm and rotation of queries and keys ---------------------------------------------
bool heads_of(const Tensor& t, const Tensor& q, int64_t n, int64_t heads, int64_t d) {
  return plain(t, q) && t.scalar_type() == q.scalar_type() && t.dim() == 3 && t.size(0) == n && t.size(1) == heads && t.size(2) == d &&
         t.stride(2) == 1;
}
// a gradient's buffer: rows apart, heads apart
bool room_of(const Tensor& t, const Tensor& q, int64_t n, int64_t heads, int64_t d) {
  return heads_of(t, q, n, heads, d) && t.stride(1) >= d && t.stride(0) >= heads * d;
}
struct Qk {
  bool ok;
  EgnnQkDims d;
};
Qk qk_of(const Tensor& q, const Tensor& k, const Opt& qw, const Opt& kw, const Opt& pos, double base, int64_t rotary, bool il,
         double eps) {
  Qk r{};
  if (torch::jit::tracer::isTracing() || q.dim() != 3 || k.dim() != 3) return r;
  const auto dt = q.scalar_type();
  const int64_t n = q.size(0), D = q.size(2);
  if ((dt != at::kFloat && dt != at::kBFloat16) || D < 2 || D > 128 || D % 2 || q.size(1) < 1 || q.size(1) > 4096 || k.size(1) < 1 ||
      k.size(1) > 4096 || n > INT32_MAX || rotary < 0 || rotary > D || rotary % 2 || !(base >= 1.0) || !std::isfinite(base) ||
      !(eps >= 0.0) || !std::isfinite(eps) || !heads_of(q, q, n, q.size(1), D) || !heads_of(k, q, n, k.size(1), D))
    return r;
  const bool f32 = (qw && qw->scalar_type() == at::kFloat) || (kw && kw->scalar_type() == at::kFloat);
  const auto pt = f32 ? at::kFloat : dt;
  if (!fits_opt(qw, q, pt, D) || !fits_opt(kw, q, pt, D)) return r;
  if (!pos ? rotary != 0 : !fits(*pos, q, at::kInt, {n}) && !fits(*pos, q, at::kLong, {n})) return r;
  EgnnQkDims& d = r.d;
  d.N = n; d.Hq = (int32_t)q.size(1); d.Hk = (int32_t)k.size(1); d.D = (int32_t)D; d.rotary = (int32_t)rotary; d.interleaved = il;
  d.dtype = dt == at::kFloat ? EGNN_F32 : EGNN_BF16;
  d.f32_params = f32 && d.dtype == EGNN_BF16;
  d.index64 = pos && pos->scalar_type() == at::kLong;
  d.eps = (float)eps; d.base = base;
  r.ok = true;
  return r;
}

pybind11::object qk_forward(const Tensor& q, const Tensor& k, const Opt& qw, const Opt& kw, const Opt& pos, double base, int64_t rotary,
                            bool il, double eps) {
  const Qk r = qk_of(q, k, qw, kw, pos, base, rotary, il, eps);
  if (!r.ok) return pybind11::none();
  const c10::DeviceGuard device(q.device());
  const Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), q.options());
  EgnnQkStrides s{};
  s.q_row = q.stride(0); s.q_head = q.stride(1); s.k_row = k.stride(0); s.k_head = k.stride(1);
  s.q_out_row = qo.stride(0); s.q_out_head = qo.stride(1); s.k_out_row = ko.stride(0); s.k_out_head = ko.stride(1);
  check("egnn_qk_fwd", egnn_qk_fwd(&r.d, &s, ptr(q), ptr(k), ptr(get(qw)), ptr(get(kw)), ptr(get(pos)), ptr(qo), ptr(ko), stream_of(q)));
  return pybind11::make_tuple(qo, ko);
}

pybind11::object qk_backward(const Tensor& gqo, const Tensor& gko, const Tensor& q, const Tensor& k, const Opt& qw, const Opt& kw,
                             const Opt& pos, double base, int64_t rotary, bool il, double eps,
                             const std::optional<std::vector<Tensor>>& into) {
  const Qk r = qk_of(q, k, qw, kw, pos, base, rotary, il, eps);
  const EgnnQkDims& d = r.d;
  if (!r.ok || !heads_of(gqo, q, d.N, d.Hq, d.D) || !heads_of(gko, q, d.N, d.Hk, d.D)) return pybind11::none();
  if (into && (into->size() != 2 || !room_of((*into)[0], q, d.N, d.Hq, d.D) || !room_of((*into)[1], q, d.N, d.Hk, d.D)))
    return pybind11::none();
  const c10::DeviceGuard device(q.device());
  const Tensor gq = into ? (*into)[0] : at::empty(q.sizes(), q.options()), gk = into ? (*into)[1] : at::empty(k.sizes(), q.options());
  const auto param = q.options().dtype(d.f32_params ? at::kFloat : q.scalar_type());
  const Tensor gqw = qw ? at::empty({d.D}, param) : Tensor(), gkw = kw ? at::empty({d.D}, param) : Tensor();
  const size_t nb = qw || kw ? egnn_qk_bwd_workspace_bytes(&d) : 0;
  const Tensor ws = workspace(nb, q);
  EgnnQkStrides s{};
  s.q_row = q.stride(0); s.q_head = q.stride(1); s.k_row = k.stride(0); s.k_head = k.stride(1);
  s.grad_q_out_row = gqo.stride(0); s.grad_q_out_head = gqo.stride(1); s.grad_k_out_row = gko.stride(0); s.grad_k_out_head = gko.stride(1);
  s.grad_q_row = gq.stride(0); s.grad_q_head = gq.stride(1); s.grad_k_row = gk.stride(0); s.grad_k_head = gk.stride(1);
  check("egnn_qk_bwd", egnn_qk_bwd(&d, &s, ptr(gqo), ptr(gko), ptr(q), ptr(k), ptr(get(qw)), ptr(get(kw)), ptr(get(pos)), ptr(gq), ptr(gk),
                                   ptr(gqw), ptr(gkw), ptr(ws), nb, stream_of(q)));
  auto out = [](const Tensor& t) -> pybind11::object { return t.defined() ? pybind11::cast(t) : pybind11::none(); };
  return pybind11::make_tuple(gq, gk, out(gqw), out(gkw));
}

}  // namespace

PYBIND11_MODULE(_egnn_torch, m) {
  m.def("gcl_layer", &gcl_layer);
  m.def("attn_forward", &attn_forward);
  m.def("attn_backward", &attn_backward);
  m.def("norm_forward", &norm_forward);
  m.def("norm_backward", &norm_backward);
  m.def("dropout", &dropout);
  m.def("norm_drop_forward", &norm_drop_forward);
  m.def("norm_drop_backward", &norm_drop_backward);
  m.def("embed_forward", &embed_forward);
  m.def("embed_backward", &embed_backward);
  m.def("qk_forward", &qk_forward);
  m.def("qk_backward", &qk_backward);
}
