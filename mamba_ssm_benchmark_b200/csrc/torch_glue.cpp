// torch_glue.cpp — torch tensors and autograd for the gated delta rule and the group norm: the module _C/_glue.so,
// which calls the C entry points of libssm_b200.so (include/ssm_b200.h).
//
// These operators are small enough in training and decoding that the host decides: as Python autograd functions
// over ctypes a head norm of 8192 x 512 took 135 us forward and backward, 33 of them on the GPU; through here 85.  Arguments are
// checked by the Python layer (delta.py, norm.py); what arrives here has the right shapes, one device and unit
// inner strides, except gradients, which autograd hands over as they are.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>

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
  TORCH_CHECK(false, msg, " (status ", rc, ")");
}

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

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("abi_version", [] { return SSM_B200_ABI_VERSION; });
  m.def("group_norm", &group_norm, py::call_guard<py::gil_scoped_release>());
  m.def("gated_delta", &gated_delta, py::call_guard<py::gil_scoped_release>());
  m.def("gated_delta_step", &gated_delta_step, py::call_guard<py::gil_scoped_release>());
}
