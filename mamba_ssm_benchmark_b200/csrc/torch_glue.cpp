// torch_glue.cpp — torch tensors and autograd for the operators whose host time counts: the gated delta rule, the group
// norm and the operators around the mixers (embedding, RMS norm, 8-bit products, sampling).  The module _C/_glue.so, which
// calls the C entry points of libssm_b200.so (include/ssm_b200.h).
//
// These operators are small enough in training and decoding that the host decides: as Python autograd functions
// over ctypes a head norm of 8192 x 512 took 135 us forward and backward, 33 of them on the GPU; through here 85.  Arguments
// of the delta rule and the group norm are checked by the Python layer (delta.py, norm.py); what arrives here has the right
// shapes, one device and unit inner strides, except gradients, which autograd hands over as they are.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <initializer_list>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <type_traits>
#include <variant>
#include <vector>

#include "ssm_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

void check(int rc, const char* what) {
  if (rc == SSM_OK) return;
  const std::string msg = std::string(what) + ": " + ssm_last_error_message();
  TORCH_CHECK_VALUE(rc != SSM_ERR_INVALID && rc != SSM_ERR_DTYPE, msg);
  TORCH_CHECK(false, msg + " (status " + std::to_string(rc) + ")");
}
// Messages are put together as strings: numbers written to a stream here end the process where the compiler's libstdc++ is
// newer than the one that is loaded (its streams are then linked in, without the loaded one's locale).
std::string text(at::IntArrayRef sizes) {
  std::string s = "(";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i > 0 ? ", " : "") + std::to_string(sizes[i]);
  return s + (sizes.size() == 1 ? ",)" : ")");
}
std::string text(const Tensor& t) { return t.defined() ? text(t.sizes()) : std::string("none"); }
std::string text(at::ScalarType t) { return c10::toString(t); }

int32_t code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? SSM_BF16 : SSM_F32; }
const void* data(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
float* f32(const Tensor& t) { return t.defined() ? static_cast<float*>(t.mutable_data_ptr()) : nullptr; }
Tensor value(const Maybe& t) { return t.has_value() ? *t : Tensor(); }

// (samples, C) or (samples, positions, C)
ssm_view view(const Tensor& t) {
  if (!t.defined()) return ssm_view{nullptr, 0, 0, 0, 0};
  return ssm_view{t.const_data_ptr(), code(t), 0, t.stride(0), t.dim() == 3 ? t.stride(1) : 0};
}
// (B, L, H, width), or one token's (B, H, width)
ssm_heads heads(const Tensor& t) {
  if (t.dim() == 3) return ssm_heads{t.const_data_ptr(), code(t), 0, t.stride(0), 0, t.stride(1)};
  return ssm_heads{t.const_data_ptr(), code(t), 0, t.stride(0), t.stride(1), t.stride(2)};
}
// a gradient in the kernels' type with unit inner stride
Tensor dense(const Tensor& t, at::ScalarType type) {
  Tensor r = t.scalar_type() == type ? t : t.to(type);
  return r.stride(-1) == 1 || r.size(-1) == 1 ? r : r.contiguous();
}
// Results are dense whatever the layout of the input: torch's *_like follow its strides, and for rows that overlap
// (sliding windows) choose some that are not unit along the channels.
Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor bytes(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }
void* stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The kernels write gradients that have no history of their own.
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: create_graph=True is not supported");
}

// What a call would drop without a word: the tangent of a forward-mode derivative, which the kernels do not form, and the
// launch itself under torch.jit.trace, which records the allocation of a result and not what fills it.
void plain(const char* what, std::initializer_list<Tensor> inputs) {
  for (const Tensor& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode derivative");
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced by torch.jit.trace");
}

// ---- group norm -------------------------------------------------------------------------------
struct NormArgs {
  int64_t groups;
  double eps;
  bool silu, center;
};
struct NormDims {
  int64_t n, p, c;
  explicit NormDims(const Tensor& x) : n(x.size(0)), p(x.dim() == 3 ? x.size(1) : 1), c(x.size(-1)) {}
};

// (y, statistics): the statistics are kept for a backward where more than one position makes them costly.
std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& z,
                                        const NormArgs& a, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  const NormDims d(x);
  const Tensor y = dense_like(x);
  Tensor stats, ws;
  if (keep && d.p > 1) stats = at::empty({d.n, a.groups, 2}, x.options().dtype(at::kFloat));
  size_t need = 0;
  check(ssm_group_norm_workspace_size(d.n, d.p, d.c, a.groups, 0, &need), "ssm_group_norm_workspace_size");
  if (need > 0) ws = bytes(need, x);
  check(ssm_group_norm_fwd(d.n, d.p, d.c, a.groups, view(x), f32(weight), f32(bias), (float)a.eps, a.center, a.silu, view(z),
                           view(y), f32(stats), const_cast<void*>(data(ws)), need, stream(x)),
        "ssm_group_norm_fwd");
  return {y, stats};
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, const Maybe& z,
                        int64_t groups, double eps, bool silu, bool center) {
    const auto [y, stats] = norm_forward(x, value(weight), value(bias), value(z), NormArgs{groups, eps, silu, center}, true);
    ctx->save_for_backward({x, value(weight), value(bias), value(z), stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["form"] = (int64_t)silu | (int64_t)center << 1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("group_norm");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &z = saved[3], &stats = saved[4];
    const int64_t groups = ctx->saved_data["groups"].toInt(), form = ctx->saved_data["form"].toInt();
    const double eps = ctx->saved_data["eps"].toDouble();
    const c10::cuda::CUDAGuard guard(x.device());
    const NormDims d(x);
    const Tensor dy = dense(grads[0], x.scalar_type()), dx = dense_like(x);
    Tensor dz, dw, db;
    if (z.defined()) dz = dense_like(z);
    if (weight.defined()) dw = dense_like(weight);
    if (bias.defined()) db = dense_like(bias);
    size_t need = 0;
    check(ssm_group_norm_workspace_size(d.n, d.p, d.c, groups, 1, &need), "ssm_group_norm_workspace_size");
    const Tensor ws = bytes(need, x);
    check(ssm_group_norm_bwd(d.n, d.p, d.c, groups, view(x), f32(weight), f32(bias), (float)eps, form >> 1 & 1, form & 1, view(z),
                             f32(stats), view(dy), view(dx), f32(dw), f32(db), view(dz), ws.mutable_data_ptr(), need,
                             stream(x)),
          "ssm_group_norm_bwd");
    return {dx, dw, db, dz, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const Maybe& t) { return t.has_value() && t->requires_grad(); }

Tensor group_norm(const Tensor& x, int64_t groups, const Maybe& weight, const Maybe& bias, const Maybe& z, double eps,
                  bool silu, bool center) {
  plain("group_norm", {x, value(weight), value(bias), value(z)});
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias) || wants(z)))
    return GroupNorm::apply(x, weight, bias, z, groups, eps, silu, center);
  return std::get<0>(norm_forward(x, value(weight), value(bias), value(z), NormArgs{groups, eps, silu, center}, false));
}

// ---- gated delta rule ---------------------------------------------------------------------------
struct DeltaDims {
  int64_t B, L, Hk, Hv, dk, dv;
  DeltaDims(const Tensor& q, const Tensor& v)
      : B(q.size(0)), L(q.size(1)), Hk(q.size(2)), Hv(v.size(2)), dk(q.size(3)), dv(v.size(3)) {}
};

// (o, last, what the backward needs)
std::tuple<Tensor, Tensor, Tensor> delta_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                                 const Tensor& beta, const Tensor& h0, double scale, bool keep) {
  const c10::cuda::CUDAGuard guard(q.device());
  const DeltaDims d(q, v);
  const Tensor o = at::empty({d.B, d.L, d.Hv, d.dv}, v.options()), last = at::empty({d.B, d.Hv, d.dk, d.dv}, g.options());
  Tensor saved, ws;
  size_t need = 0;
  if (keep) {
    check(ssm_gated_delta_saved_size(d.B, d.L, d.Hk, d.Hv, d.dk, d.dv, code(q), &need), "ssm_gated_delta_saved_size");
    saved = bytes(need, q);
    need = 0;
  } else {
    check(ssm_gated_delta_workspace_size(d.B, d.L, d.Hk, d.Hv, d.dk, d.dv, code(q), 0, &need),
          "ssm_gated_delta_workspace_size");
    ws = bytes(need, q);
  }
  check(ssm_gated_delta_fwd(d.B, d.L, d.Hk, d.Hv, d.dk, d.dv, heads(q), heads(k), heads(v), view(g), view(beta), f32(h0),
                            (float)scale, heads(o), f32(last), const_cast<void*>(data(saved)), const_cast<void*>(data(ws)),
                            need, stream(q)),
        "ssm_gated_delta_fwd");
  return {o, last, saved};
}

struct GatedDelta : torch::autograd::Function<GatedDelta> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                               const Tensor& beta, const Maybe& h0, double scale) {
    const auto [o, last, saved] = delta_forward(q, k, v, g, beta, value(h0), scale, true);
    ctx->save_for_backward({q, k, v, g, beta, saved});      // the first state is in `saved`: h0 may be updated in place
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["h0"] = h0.has_value();
    ctx->set_materialize_grads(false);
    return {o, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("gated_delta_rule");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &g = saved[3], &beta = saved[4], &tiles = saved[5];
    const c10::cuda::CUDAGuard guard(q.device());
    const DeltaDims d(q, v);
    const Tensor d_o = grads[0].defined() ? dense(grads[0], v.scalar_type())
                                          : at::zeros({d.B, d.L, d.Hv, d.dv}, v.options());
    Tensor dlast, dh0;
    if (grads[1].defined()) dlast = grads[1].to(at::kFloat).contiguous();
    if (ctx->saved_data["h0"].toBool()) dh0 = at::empty({d.B, d.Hv, d.dk, d.dv}, g.options());
    const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
                 dv = at::empty(v.sizes(), v.options()), dg = at::empty(g.sizes(), g.options()),
                 dbeta = at::empty(g.sizes(), g.options());
    size_t need = 0;
    check(ssm_gated_delta_workspace_size(d.B, d.L, d.Hk, d.Hv, d.dk, d.dv, code(q), 1, &need),
          "ssm_gated_delta_workspace_size");
    const Tensor ws = bytes(need, q);
    check(ssm_gated_delta_bwd(d.B, d.L, d.Hk, d.Hv, d.dk, d.dv, heads(q), heads(k), heads(v), view(g), view(beta),
                              (float)ctx->saved_data["scale"].toDouble(), tiles.const_data_ptr(), heads(d_o), f32(dlast),
                              heads(dq), heads(dk), heads(dv), f32(dg), f32(dbeta), f32(dh0), ws.mutable_data_ptr(), need,
                              stream(q)),
          "ssm_gated_delta_bwd");
    return {dq, dk, dv, dg, dbeta, dh0, Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_delta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                                       const Maybe& h0, double scale) {
  plain("gated_delta_rule", {q, k, v, g, beta, value(h0)});
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(g) || wants(beta) || wants(h0))) {
    const variable_list r = GatedDelta::apply(q, k, v, g, beta, h0, scale);
    return {r[0], r[1]};
  }
  const auto [o, last, saved] = delta_forward(q, k, v, g, beta, value(h0), scale, false);
  return {o, last};
}

// One token: q, k (B, Hk, dk), v (B, Hv, dv), g, beta (B, Hv); the state in place.
Tensor gated_delta_step(const Tensor& state, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                        const Tensor& beta, double scale, const Maybe& out) {
  plain("gated_delta_state_update", {state, q, k, v, g, beta});
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor o = out.has_value() ? *out : at::empty(v.sizes(), v.options());
  check(ssm_gated_delta_state_update(q.size(0), q.size(1), v.size(1), q.size(2), v.size(2), f32(state), heads(q), heads(k),
                                     heads(v), view(g), view(beta), (float)scale, heads(o), stream(q)),
        "ssm_gated_delta_state_update");
  return o;
}

// ---- the operators around the mixers ------------------------------------------------------------------
// Their arguments are checked here: in Python the checks of an 8-bit norm took longer than everything else (18 us a call for
// a token, 10 this way).
bool kernel_type(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
Tensor kernel_typed(const Tensor& t) { return kernel_type(t) ? t : t.to(at::kFloat); }
// unit stride along the last axis
Tensor unit(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }
Tensor as_rows(const Tensor& t) { return unit(t.dim() == 2 ? t : t.reshape({-1, t.size(-1)})); }
// a layout that is (rows, C) without a copy
Tensor row_layout(const Tensor& t) {
  bool fits = t.stride(-1) == 1 || t.size(-1) == 1;
  int64_t next = -1;                          // the stride that the axis before needs
  for (int64_t i = t.dim() - 2; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    fits = fits && (next < 0 || t.stride(i) == next);
    next = t.stride(i) * t.size(i);
  }
  return fits ? t : t.contiguous();
}
Tensor shaped(const Tensor& t, at::IntArrayRef shape) { return t.sizes() == shape ? t : t.reshape(shape); }

void needs_cuda(const char* what, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "the sm_100a ", what, " needs CUDA tensors (this package has no CPU path)");
}
void one_device(const Tensor& a, std::initializer_list<Tensor> others) {
  for (const Tensor& t : others) TORCH_CHECK_VALUE(!t.defined() || t.device() == a.device(), "all tensors must be on one device");
}
void no_gradient(const char* what, std::initializer_list<Tensor> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor& t : inputs)
    TORCH_CHECK(!t.defined() || !t.requires_grad(), what, " has no gradient: call it under torch.no_grad()");
}

// ---- embedding ------------------------------------------------------------------------------------
// idx: T dense ids; the result is (T, C).
Tensor embedding_forward(const Tensor& idx, const Tensor& weight, double scale) {
  const c10::cuda::CUDAGuard guard(weight.device());
  const Tensor y = at::empty({idx.numel(), weight.size(1)}, weight.options());
  check(ssm_embedding_fwd(idx.numel(), weight.size(0), weight.size(1), idx.const_data_ptr(), (int)idx.element_size(),
                          view(weight), (float)scale, view(y), stream(weight)),
        "ssm_embedding_fwd");
  return y;
}

// idx: T dense ids, dy: (T, C); the result is (V, C).
Tensor embedding_backward(const Tensor& idx, const Tensor& dy0, int64_t V, double scale) {
  const c10::cuda::CUDAGuard guard(dy0.device());
  const Tensor dy = dense(dy0, dy0.scalar_type()), dw = at::empty({V, dy.size(1)}, dy.options());
  size_t need = 0;
  check(ssm_embedding_bwd_workspace_size(dy.size(0), V, dy.size(1), &need), "ssm_embedding_bwd_workspace_size");
  const Tensor ws = bytes(need, dy);
  check(ssm_embedding_bwd(dy.size(0), V, dy.size(1), idx.const_data_ptr(), (int)idx.element_size(), (float)scale, view(dy), view(dw),
                          ws.mutable_data_ptr(), need, stream(dy)),
        "ssm_embedding_bwd");
  return dw;
}

// again: the gradient can be differentiated once more, and so on; both directions are linear, and each is the other's.
struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& idx, double scale, bool again) {
    ctx->save_for_backward({idx});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["again"] = again;
    return embedding_forward(idx, unit(weight), scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};
struct EmbeddingGrad : torch::autograd::Function<EmbeddingGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& dy, const Tensor& idx, int64_t V, double scale) {
    ctx->save_for_backward({idx});
    ctx->saved_data["scale"] = scale;
    return embedding_backward(idx, dy, V, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor idx = ctx->get_saved_variables()[0];
    return {Embedding::apply(grads[0], idx, ctx->saved_data["scale"].toDouble(), true), Tensor(), Tensor(), Tensor()};
  }
};
variable_list Embedding::backward(AutogradContext* ctx, variable_list grads) {
  const bool again = ctx->saved_data["again"].toBool();
  if (!again) once("embedding");
  const Tensor idx = ctx->get_saved_variables()[0];
  const int64_t V = ctx->saved_data["vocab"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  const Tensor dw = at::GradMode::is_enabled() ? EmbeddingGrad::apply(grads[0], idx, V, scale)
                                               : embedding_backward(idx, grads[0], V, scale);
  return {dw, Tensor(), Tensor(), Tensor()};
}

Tensor embedding(const Tensor& idx, const Tensor& weight, double scale, bool again) {
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.numel() > 0,
                    "weight must be (vocabulary, channels) with no empty axis, got " + text(weight));
  TORCH_CHECK_TYPE(idx.scalar_type() == at::kLong || idx.scalar_type() == at::kInt,
                   "idx must be int64 or int32, got " + text(idx.scalar_type()));
  TORCH_CHECK_VALUE(idx.numel() > 0, "idx must have no empty axis, got " + text(idx));
  TORCH_CHECK_TYPE(kernel_type(weight), "weight must be float32 or bfloat16, got " + text(weight.scalar_type()));
  needs_cuda("embedding", weight);
  one_device(weight, {idx});
  plain("embedding", {weight});
  const Tensor ids = idx.dim() == 1 && idx.is_contiguous() ? idx : idx.reshape({-1}).contiguous(), w = unit(weight);
  const Tensor y = at::GradMode::is_enabled() && wants(w) ? Embedding::apply(w, ids, scale, again)
                                                              : embedding_forward(ids, w, scale);
  if (idx.dim() == 1) return y;
  std::vector<int64_t> shape = idx.sizes().vec();
  shape.push_back(weight.size(1));
  return y.reshape(shape);
}

// ---- root-mean-square norm --------------------------------------------------------------------------
// The arguments as the kernels take them, but in the caller's shape: x and residual are (rows, C) without a copy, the residual is
// float32 or like x.  They become rows inside the autograd function: a reshape in front of it would hand x and residual
// two views of their one gradient, which leaves would both keep and add the next one to, each to the memory of the other.
struct RmsArgs {
  Tensor x, residual, weight;
  at::ScalarType y_type, total_type;          // what the caller gets
  RmsArgs(const char* what, const Tensor& x0, const Maybe& w0, const Maybe& r0, double eps) {
    TORCH_CHECK_VALUE(x0.dim() >= 1 && x0.numel() > 0, "x must be (..., C) with no empty axis, got " + text(x0));
    const int64_t C = x0.size(-1);
    residual = value(r0);
    weight = value(w0);
    TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == x0.sizes(),
                      "residual must be shaped like x " + text(x0) + ", got " + text(residual));
    TORCH_CHECK_VALUE(!weight.defined() || (weight.dim() == 1 && weight.size(0) == C),
                      "weight must be (" + std::to_string(C) + ",), got " + text(weight));
    TORCH_CHECK_VALUE(eps >= 0.0, "eps must not be negative, got " + std::to_string(eps));
    for (const Tensor& t : {x0, residual, weight})
      TORCH_CHECK_TYPE(!t.defined() || (t.is_floating_point() && t.scalar_type() != at::kDouble && t.element_size() > 1),
                       "float64, 8-bit and integer tensors are not supported by the sm_100a kernels; use float32 or bfloat16");
    needs_cuda(what, x0);
    one_device(x0, {residual, weight});
    y_type = total_type = x0.scalar_type();
    x = row_layout(kernel_typed(x0));
    if (residual.defined()) {
      total_type = at::promote_types(y_type, residual.scalar_type());
      if (residual.scalar_type() != at::kFloat && residual.scalar_type() != x.scalar_type()) residual = residual.to(at::kFloat);
      residual = row_layout(residual);
    }
    if (weight.defined()) weight = kernel_typed(weight).contiguous();
  }
  static Tensor as(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }
};

// of what row_layout gives: never a copy, whose memory would be free before the launch
ssm_view rows_view(const Tensor& t) { return view(!t.defined() || t.dim() == 2 ? t : t.view({-1, t.size(-1)})); }

// (y, total), total undefined without a residual.
std::tuple<Tensor, Tensor> rms_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor y = dense_like(x);
  Tensor total;
  if (residual.defined()) total = dense_like(residual);
  const int64_t C = x.size(-1);
  check(ssm_rms_norm_fwd(x.numel() / C, C, rows_view(x), rows_view(residual), data(weight),
                         weight.defined() ? code(weight) : SSM_F32, (float)eps, rows_view(y), rows_view(total), stream(x)),
        "ssm_rms_norm_fwd");
  return {y, total};
}

// The gradients by torch's operators, which can be differentiated again: what the kernels do of the same tensors.
variable_list rms_gradients(const Tensor& total, const Tensor& weight, const Tensor& dy, const Tensor& dtotal, double eps,
                            at::ScalarType type, bool residual) {
  const Tensor t = total.to(at::kFloat), g0 = dy.to(at::kFloat), rstd = (t.square().mean(-1, true) + eps).rsqrt(), n = t * rstd;
  const Tensor g = weight.defined() ? g0 * weight.to(at::kFloat) : g0;
  Tensor d = rstd * (g - n * (g * n).mean(-1, true)), dw;
  if (dtotal.defined()) d = d + dtotal.to(at::kFloat);
  if (weight.defined()) dw = (g0 * n).reshape({-1, t.size(-1)}).sum(0).to(weight.scalar_type());
  return {d.to(type), residual ? d.to(total.scalar_type()) : Tensor(), dw, Tensor(), Tensor()};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, const Maybe& weight, double eps,
                               bool again) {
    const auto [y, total] = rms_forward(x, value(residual), value(weight), eps);
    ctx->save_for_backward({total.defined() ? total : x, value(weight)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["again"] = again;
    ctx->saved_data["bf16"] = x.scalar_type() == at::kBFloat16;
    ctx->saved_data["residual"] = total.defined();
    ctx->set_materialize_grads(false);
    return total.defined() ? variable_list{y, total} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!ctx->saved_data["again"].toBool()) once("rms_norm");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &total = saved[0], &weight = saved[1];
    const bool residual = ctx->saved_data["residual"].toBool();
    const at::ScalarType type = ctx->saved_data["bf16"].toBool() ? at::kBFloat16 : at::kFloat;
    const c10::cuda::CUDAGuard guard(total.device());
    Tensor dtotal;
    if (residual && grads[1].defined()) dtotal = dense(grads[1], total.scalar_type());
    if (!grads[0].defined()) {                       // only the sum was used
      Tensor dw;
      if (weight.defined()) dw = at::zeros(weight.sizes(), weight.options());
      return {dtotal.defined() ? dtotal.to(type) : Tensor(), dtotal, dw, Tensor(), Tensor()};
    }
    if (at::GradMode::is_enabled())
      return rms_gradients(total, weight, grads[0], dtotal, ctx->saved_data["eps"].toDouble(), type, residual);
    const Tensor dy = row_layout(dense(grads[0], type)), dx = at::empty(total.sizes(), total.options().dtype(type));
    if (dtotal.defined()) dtotal = row_layout(dtotal);
    Tensor dr, dw;
    if (residual && total.scalar_type() != type) dr = dense_like(total);
    if (weight.defined()) dw = dense_like(weight);
    const int64_t C = dy.size(-1), rows = dy.numel() / C;
    size_t need = 0;
    check(ssm_rms_norm_bwd_workspace_size(rows, C, &need), "ssm_rms_norm_bwd_workspace_size");
    const Tensor ws = bytes(need, dy);
    check(ssm_rms_norm_bwd(rows, C, rows_view(total), data(weight), weight.defined() ? code(weight) : SSM_F32,
                           (float)ctx->saved_data["eps"].toDouble(), rows_view(dy), rows_view(dtotal), rows_view(dx), rows_view(dr),
                           dw.defined() ? dw.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), need, stream(dy)),
          "ssm_rms_norm_bwd");
    // in one type the two inputs' gradients are one tensor, as those of a sum of two tensors are; leaves then keep a copy and it
    return {dx, !residual ? Tensor() : dr.defined() ? dr : dx, dw, Tensor(), Tensor()};
  }
};

// (y) or (y, total)
variable_list rms_norm(const Tensor& x, const Maybe& weight, const Maybe& residual, double eps, bool again) {
  const RmsArgs a("RMS norm", x, weight, residual, eps);
  plain("rms_norm", {x, value(residual), value(weight)});
  variable_list out;
  const bool wanted = wants(a.x) || (a.residual.defined() && wants(a.residual)) || (a.weight.defined() && wants(a.weight));
  if (at::GradMode::is_enabled() && wanted) {
    auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
    out = RmsNorm::apply(a.x, maybe(a.residual), maybe(a.weight), eps, again);
  } else {
    const auto [y, total] = rms_forward(a.x, a.residual, a.weight, eps);
    out = total.defined() ? variable_list{y, total} : variable_list{y};
  }
  out[0] = RmsArgs::as(out[0], a.y_type);
  if (out.size() > 1) out[1] = RmsArgs::as(out[1], a.total_type);
  return out;
}

// Rows of 8 bits start at multiples of 16 bytes, as ssm_linear_fp8 reads them.
Tensor rows8(int64_t rows, int64_t C, const Tensor& like) {
  const Tensor t = at::empty({rows, (C + 15) / 16 * 16}, like.options().dtype(at::kFloat8_e4m3fn));
  return t.size(1) == C ? t : t.narrow(1, 0, C);
}

// (y8, scale) or (y8, scale, total)
variable_list rms_norm_fp8(const Tensor& x, const Maybe& weight, const Maybe& residual, double eps, bool norm) {
  const char* what = norm ? "rms_norm_fp8" : "quantize_fp8";
  no_gradient(what, {x, value(weight), value(residual)});
  const RmsArgs a(what, x, weight, residual, eps);
  plain(what, {x, a.residual, a.weight});
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t C = x.size(-1), rows = x.numel() / C;
  Tensor y8 = rows8(rows, C, a.x), scale = at::empty({rows}, a.x.options().dtype(at::kFloat)), total;
  if (a.residual.defined()) total = dense_like(a.residual);
  check(ssm_rms_norm_fp8(rows, C, rows_view(a.x), rows_view(a.residual), data(a.weight), a.weight.defined() ? code(a.weight) : SSM_F32,
                         (float)eps, norm, y8.mutable_data_ptr(), y8.stride(0), f32(scale), rows_view(total), stream(a.x)),
        "ssm_rms_norm_fp8");
  if (x.dim() != 2) {
    const std::vector<int64_t> outer(x.sizes().begin(), x.sizes().end() - 1);
    y8 = outer.empty() ? y8.select(0, 0) : y8.unflatten(0, outer);
    scale = scale.reshape(outer);
  }
  if (!total.defined()) return {y8, scale};
  return {y8, scale, RmsArgs::as(total, a.total_type)};
}

// ---- 8-bit products -----------------------------------------------------------------------------------
Tensor linear_fp8(const Tensor& x8, const Tensor& x_scale, const Tensor& w8, const Tensor& w_scale, const Maybe& bias0, bool silu,
                  const Maybe& residual0, std::optional<at::ScalarType> dtype) {
  TORCH_CHECK_TYPE(x8.scalar_type() == at::kFloat8_e4m3fn && w8.scalar_type() == at::kFloat8_e4m3fn,
                   "x8 and weight8 must be float8_e4m3fn, got " + text(x8.scalar_type()) + " and " + text(w8.scalar_type()));
  TORCH_CHECK_VALUE(w8.dim() == 2 && x8.dim() >= 1 && x8.numel() > 0 && w8.numel() > 0,
                    "x8 must be (..., K) and weight8 (N, K) with no empty axis, got " + text(x8) + " and " + text(w8));
  const int64_t N = w8.size(0), K = w8.size(1);
  TORCH_CHECK_VALUE(x8.size(-1) == K, "x8 must have weight8's " + std::to_string(K) + " columns, got " + text(x8));
  const at::IntArrayRef outer = x8.sizes().slice(0, x8.dim() - 1);
  TORCH_CHECK_VALUE(x_scale.sizes() == outer && w_scale.dim() == 1 && w_scale.size(0) == N,
                    "the scales must be " + text(outer) + " and (" + std::to_string(N) + ",), got " + text(x_scale) + " and " +
                        text(w_scale));
  TORCH_CHECK_TYPE(x_scale.scalar_type() == at::kFloat && w_scale.scalar_type() == at::kFloat, "the scales must be float32");
  Tensor bias = value(bias0), residual = value(residual0);
  TORCH_CHECK_VALUE(!bias.defined() || (bias.dim() == 1 && bias.size(0) == N),
                    "bias must be (" + std::to_string(N) + ",), got " + text(bias));
  const at::ScalarType type = dtype.has_value() ? *dtype : residual.defined() ? residual.scalar_type() : at::kBFloat16;
  TORCH_CHECK_TYPE(type == at::kFloat || type == at::kBFloat16, "dtype must be float32 or bfloat16, got " + text(type));
  std::vector<int64_t> shape = outer.vec();
  shape.push_back(N);
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == at::IntArrayRef(shape) && residual.scalar_type() == type),
                    "residual must be " + text(shape) + " in " + text(type) + ", got " + text(residual));
  no_gradient("linear_fp8", {x_scale, w_scale, bias, residual});
  needs_cuda("products", x8);
  one_device(x8, {x_scale, w8, w_scale, bias, residual});
  plain("linear_fp8", {x8, x_scale, w8, w_scale, bias, residual});
  const c10::cuda::CUDAGuard guard(x8.device());
  auto rows = [](const Tensor& t) {                  // rows that start at multiples of 16 bytes
    const bool fits = (t.stride(1) == 1 || t.size(1) == 1) && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
    if (fits && (t.size(0) == 1 || (t.stride(0) % 16 == 0 && t.stride(0) >= t.size(1)))) return t;
    const Tensor u = rows8(t.size(0), t.size(1), t);
    u.copy_(t);
    return u;
  };
  auto stride = [](const Tensor& t) { return t.size(0) == 1 ? (t.size(1) + 15) / 16 * 16 : t.stride(0); };
  const Tensor x = rows(x8.dim() == 2 ? x8 : x8.reshape({-1, K})), w = rows(w8);
  const Tensor xs = x_scale.contiguous(), ws = w_scale.contiguous();
  if (bias.defined()) bias = bias.to(at::kFloat).contiguous();
  if (residual.defined()) residual = as_rows(residual);
  const Tensor y = at::empty({x.size(0), N}, x_scale.options().dtype(type));
  check(ssm_linear_fp8(x.size(0), N, K, x.const_data_ptr(), stride(x), f32(xs), w.const_data_ptr(), stride(w), f32(ws), f32(bias),
                       silu, view(residual), view(y), stream(x)),
        "ssm_linear_fp8");
  return shaped(y, shape);
}

// ---- sampling -------------------------------------------------------------------------------------
// A setting: none, a number, or a tensor with one for every row.
template <typename N>
using Setting = std::optional<std::variant<Tensor, N>>;
template <typename N>
struct Given {
  Tensor rows;
  N one;
  Given(const char* name, const Setting<N>& s, const Tensor& logits, N none, N lo, N hi) : one(none) {
    if (!s.has_value()) return;
    if (const Tensor* t = std::get_if<Tensor>(&*s)) {
      TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == logits.size(0),
                        std::string(name) + " must be a number or a (" + std::to_string(logits.size(0)) + ",) tensor, got " + text(*t));
      one_device(logits, {*t});
      rows = t->detach().to(std::is_same_v<N, double> ? at::kDouble : at::kLong).contiguous();
    } else {
      one = std::get<N>(*s);
      TORCH_CHECK_VALUE(one >= lo && one <= hi, std::string(name) + " must be in " + std::to_string(lo) + " .. " + std::to_string(hi) +
                                                    ", got " + std::to_string(one));
    }
  }
  const N* by_row() const { return rows.defined() ? static_cast<const N*>(rows.const_data_ptr()) : nullptr; }
};

Tensor sample_tokens(const Tensor& logits0, const Tensor& uniforms, const Setting<double>& temperature,
                     const Setting<int64_t>& top_k, const Setting<double>& top_p, const Setting<double>& min_p) {
  TORCH_CHECK_VALUE(logits0.dim() == 2 && logits0.numel() > 0, "logits must be (B, V) with no empty axis, got " + text(logits0));
  const int64_t B = logits0.size(0), V = logits0.size(1), most = 1 << 20;
  TORCH_CHECK_VALUE(V <= most, "the vocabulary must be at most " + std::to_string(most) + ", got " + std::to_string(V));
  TORCH_CHECK_VALUE(uniforms.dim() == 1 && uniforms.size(0) == B,
                    "uniforms must be (" + std::to_string(B) + ",), got " + text(uniforms));
  TORCH_CHECK_TYPE(logits0.is_floating_point() && logits0.scalar_type() != at::kDouble && logits0.element_size() > 1 &&
                       uniforms.scalar_type() == at::kFloat,
                   "logits must be float32 or bfloat16 and uniforms float32, got " + text(logits0.scalar_type()) + " and " +
                       text(uniforms.scalar_type()));
  const double inf = std::numeric_limits<double>::infinity();
  const Given<double> t("temperature", temperature, logits0, 1.0, 0.0, inf), p("top_p", top_p, logits0, 1.0, 0.0, 1.0),
      m("min_p", min_p, logits0, 0.0, 0.0, 1.0);
  const Given<int64_t> k("top_k", top_k, logits0, 0, 0, (int64_t)1 << 62);
  needs_cuda("sampling", logits0);
  one_device(logits0, {uniforms});
  plain("sample_tokens", {logits0, uniforms});
  const c10::cuda::CUDAGuard guard(logits0.device());
  const Tensor logits = unit(kernel_typed(logits0.detach())), u = uniforms.contiguous();
  const Tensor tokens = at::empty({B}, logits.options().dtype(at::kLong));
  check(ssm_sample_tokens(B, V, view(logits), u.const_data_ptr<float>(), t.by_row(), t.one, k.by_row(), k.one, p.by_row(), p.one,
                          m.by_row(), m.one, tokens.mutable_data_ptr<int64_t>(), stream(logits)),
        "ssm_sample_tokens");
  return tokens;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi_version", [] { return SSM_B200_ABI_VERSION; });
  m.def("group_norm", &group_norm, py::call_guard<py::gil_scoped_release>());
  m.def("gated_delta", &gated_delta, py::call_guard<py::gil_scoped_release>());
  m.def("gated_delta_step", &gated_delta_step, py::call_guard<py::gil_scoped_release>());
  m.def("embedding", &embedding, py::call_guard<py::gil_scoped_release>());
  m.def("rms_norm", &rms_norm, py::call_guard<py::gil_scoped_release>());
  m.def("rms_norm_fp8", &rms_norm_fp8, py::call_guard<py::gil_scoped_release>());
  m.def("linear_fp8", &linear_fp8, py::call_guard<py::gil_scoped_release>());
  m.def("sample_tokens", &sample_tokens, py::call_guard<py::gil_scoped_release>());
}
