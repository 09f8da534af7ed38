// Native autograd of the apb200 operators for CUDA tensors.
//
// The formulas are those that ops/library.py and ops/moe_ops.py register for every device; here they are registered
// again, for the AutogradCUDA key only, so that a call on CUDA tensors passes through no Python on its way to the CUDA
// kernel's entry and its gradient node is a C++ one.  What that costs on the host per call (forward alone / forward that
// records a gradient): 18 -> 8 us / 38 -> 10 us, the CUDA entry apart.
// CPU, meta and fake CPU tensors (planning) keep the Python registration.  Everything below autograd - dispatch modes, fake
// tensors, functionalisation, the CUDA entries at the end of binding.cpp - is reached as before, by redispatch; functorch
// transforms and forward-mode differentiation of a recorded call are refused by the C++ function itself as they are by the Python
// one; a dual tensor in a call that records nothing loses its tangent, as it does there.
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <algorithm>
#include <tuple>

bool apb_mx4_matmul_ours();  // binding.cpp

namespace {

using at::ScalarType;
using at::Tensor;
using c10::DispatchKeySet;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A typed operator of this namespace, looked up once.  ``below`` runs what is under the autograd layer.
template <typename Sig>
struct Op;
template <typename R, typename... Args>
struct Op<R(Args...)> {
  c10::TypedOperatorHandle<R(Args...)> h;
  explicit Op(const char* name) : h(c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<R(Args...)>()) {}
  R operator()(Args... args) const { return h.call(args...); }
  R below(DispatchKeySet ks, Args... args) const {
    at::AutoDispatchBelowAutograd guard;
    return h.redispatch(ks & c10::after_autograd_keyset, args...);
  }
};

template <typename... Ts>
bool records(const Ts&... ts) {
  return at::GradMode::is_enabled() && (ts.requires_grad() || ...);
}

#define APB_OP(var, name, ...) static const Op<__VA_ARGS__> var("apb200::" name)
using Pair = std::tuple<Tensor, Tensor>;
using Triple = std::tuple<Tensor, Tensor, Tensor>;

using CastSig = Tensor(const Tensor&, ScalarType);
using MmNdSig = Tensor(const Tensor&, const Tensor&, bool, ScalarType);
using WgradSig = Tensor(const Tensor&, const Tensor&, ScalarType);
using GemmSig = Tensor(const Tensor&, const Tensor&, bool, bool, ScalarType);
using RmsSig = Pair(const Tensor&, const Tensor&, double);
using RmsBwdSig = Pair(const Tensor&, const Tensor&, const Tensor&, const Tensor&);
using RopeSig = Tensor(const Tensor&, const Tensor&, const Tensor&, bool);
using SwigluSig = Tensor(const Tensor&, const Tensor&);
using SwigluBwdSig = Pair(const Tensor&, const Tensor&, const Tensor&);
using AttnSig = Pair(const Tensor&, const Tensor&, const Tensor&, bool, double);
using AttnBwdSig = Triple(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, bool, double);
using XentSig = Pair(const Tensor&, const Tensor&);
using XentBwdSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&);
using EmbSig = Tensor(const Tensor&, const Tensor&);
using EmbBwdSig = Tensor(const Tensor&, const Tensor&, int64_t);
using ScatterSig = Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t, int64_t, int64_t);
using GatherSig = Tensor(const Tensor&, const Tensor&, const Tensor&);

// Gradient of the first output of an operator whose second one (1 / rms, log-sum-exp) is seldom used.  The engine would fill a tensor of zeros for
// the second one's gradient, which no formula reads: a launch, an allocation and 8 us of host time per call (RMSNorm of 2047 x 2048 fp32, forward
// and backward, 81 -> 73 us).  So these operators take gradients as they come; where only the second output was used, the first one's is zeros.
Tensor first_grad(const variable_list& g, const Tensor& like) { return g[0].defined() ? g[0] : at::zeros_like(like); }

// Gradients that cannot be differentiated again: where a second derivative could be asked for (create_graph) they come with a node that refuses, on every way
// to an input of the forward call and to the gradient that came in.  Without it they would count as constants, and the second derivative would be
// wrong without a word.
template <typename F>
variable_list once(const char* what, const variable_list& g, F gradients) {
  if (!at::GradMode::is_enabled()) return gradients();
  auto edges = torch::autograd::get_current_node()->next_edges();
  for (auto& e : torch::autograd::collect_next_edges(g)) edges.push_back(std::move(e));
  variable_list out;
  {
    at::AutoGradMode off(false);
    out = gradients();
  }
  auto refuse = std::make_shared<torch::autograd::Error>(std::string(what) + ": no second derivatives on CUDA", std::move(edges));
  for (Tensor& t : out)
    if (t.defined()) torch::autograd::set_history(t, refuse);
  return out;
}

// The dispatch keys of the call travel to ``forward`` in a wrapper, so that they are not taken for an input.
struct Keys {
  DispatchKeySet ks;
};

// ---------------------------------------------------------------------------------------------- dtype_cast
const Op<CastSig>& op_cast() { APB_OP(o, "dtype_cast", CastSig); return o; }
struct Cast : torch::autograd::Function<Cast> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, ScalarType dtype, Keys k) {
    ctx->saved_data["dtype"] = x.scalar_type();
    return op_cast().below(k.ks, x, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    return {op_cast()(g[0], ctx->saved_data["dtype"].toScalarType()), Tensor(), Tensor()};
  }
};
Tensor cast(DispatchKeySet ks, const Tensor& x, ScalarType dtype) {
  return records(x) ? Cast::apply(x, dtype, Keys{ks}) : op_cast().below(ks, x, dtype);
}

// ---------------------------------------------------------------------------------------------- projections
const Op<MmNdSig>& op_mm_nd() { APB_OP(o, "mm_nd", MmNdSig); return o; }
const Op<WgradSig>& op_mm_wgrad() { APB_OP(o, "mm_wgrad", WgradSig); return o; }
struct MmNd : torch::autograd::Function<MmNd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, bool tb, ScalarType dtype, Keys k) {
    ctx->save_for_backward({a, b});
    ctx->saved_data["tb"] = tb;
    return op_mm_nd().below(k.ks, a, b, tb, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &a = s[0], &b = s[1], &dc = g[0];
    const bool tb = ctx->saved_data["tb"].toBool();
    Tensor da, db;
    if (ctx->needs_input_grad(0)) da = op_mm_nd()(dc, b, !tb, a.scalar_type());
    if (ctx->needs_input_grad(1)) db = tb ? op_mm_wgrad()(dc, a, b.scalar_type()) : op_mm_wgrad()(a, dc, b.scalar_type());
    return {da, db, Tensor(), Tensor(), Tensor()};
  }
};
Tensor mm_nd(DispatchKeySet ks, const Tensor& a, const Tensor& b, bool tb, ScalarType dtype) {
  return records(a, b) ? MmNd::apply(a, b, tb, dtype, Keys{ks}) : op_mm_nd().below(ks, a, b, tb, dtype);
}

const Op<GemmSig>& op_gemm() { APB_OP(o, "gemm", GemmSig); return o; }
struct Gemm : torch::autograd::Function<Gemm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, bool ta, bool tb, ScalarType dtype, Keys k) {
    ctx->save_for_backward({a, b});
    ctx->saved_data["ta"] = ta;
    ctx->saved_data["tb"] = tb;
    return op_gemm().below(k.ks, a, b, ta, tb, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &a = s[0], &b = s[1], &dc = g[0];
    const bool ta = ctx->saved_data["ta"].toBool(), tb = ctx->saved_data["tb"].toBool();
    // C = op(A) op(B): dA_op = dC op(B)^T, dB_op = op(A)^T dC, then the storage transpose is undone
    Tensor da, db;
    if (ctx->needs_input_grad(0)) da = ta ? op_gemm()(b, dc, tb, true, a.scalar_type()) : op_gemm()(dc, b, false, !tb, a.scalar_type());
    if (ctx->needs_input_grad(1)) db = tb ? op_gemm()(dc, a, true, ta, b.scalar_type()) : op_gemm()(a, dc, !ta, false, b.scalar_type());
    return {da, db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor gemm(DispatchKeySet ks, const Tensor& a, const Tensor& b, bool ta, bool tb, ScalarType dtype) {
  return records(a, b) ? Gemm::apply(a, b, ta, tb, dtype, Keys{ks}) : op_gemm().below(ks, a, b, ta, tb, dtype);
}

const Op<MmNdSig>& op_grouped_mm() { APB_OP(o, "grouped_mm", MmNdSig); return o; }
const Op<WgradSig>& op_grouped_wgrad() { APB_OP(o, "grouped_mm_wgrad", WgradSig); return o; }
struct GroupedMm : torch::autograd::Function<GroupedMm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, bool tb, ScalarType dtype, Keys k) {
    ctx->save_for_backward({a, b});
    ctx->saved_data["tb"] = tb;
    return op_grouped_mm().below(k.ks, a, b, tb, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &a = s[0], &b = s[1], &dc = g[0];
    const bool tb = ctx->saved_data["tb"].toBool();
    Tensor da, db;
    if (ctx->needs_input_grad(0)) da = op_grouped_mm()(dc, b, !tb, a.scalar_type());
    if (ctx->needs_input_grad(1)) db = tb ? op_grouped_wgrad()(dc, a, b.scalar_type()) : op_grouped_wgrad()(a, dc, b.scalar_type());
    return {da, db, Tensor(), Tensor(), Tensor()};
  }
};
Tensor grouped_mm(DispatchKeySet ks, const Tensor& a, const Tensor& b, bool tb, ScalarType dtype) {
  return records(a, b) ? GroupedMm::apply(a, b, tb, dtype, Keys{ks}) : op_grouped_mm().below(ks, a, b, tb, dtype);
}

// ---------------------------------------------------------------------------------------------- norm, rotary, SwiGLU
const Op<RmsSig>& op_rms() { APB_OP(o, "rms_norm", RmsSig); return o; }
const Op<RmsBwdSig>& op_rms_bwd() { APB_OP(o, "rms_norm_bwd", RmsBwdSig); return o; }
struct Rms : torch::autograd::Function<Rms> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, double eps, Keys k) {
    auto [y, rstd] = op_rms().below(k.ks, x, w, eps);
    ctx->save_for_backward({x, w, rstd});
    ctx->set_materialize_grads(false);
    return {y, rstd};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    auto [dx, dw] = op_rms_bwd()(first_grad(g, s[0]), s[0], s[1], s[2]);
    return {dx, dw, Tensor(), Tensor()};
  }
};
Pair rms_norm(DispatchKeySet ks, const Tensor& x, const Tensor& w, double eps) {
  if (!records(x, w)) return op_rms().below(ks, x, w, eps);
  auto o = Rms::apply(x, w, eps, Keys{ks});
  return {o[0], o[1]};
}

const Op<RopeSig>& op_rope() { APB_OP(o, "rope", RopeSig); return o; }
struct Rope : torch::autograd::Function<Rope> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& cos, const Tensor& sin, bool conj, Keys k) {
    ctx->save_for_backward({cos, sin});
    ctx->saved_data["conj"] = conj;
    return op_rope().below(k.ks, x, cos, sin, conj);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    return {op_rope()(g[0], s[0], s[1], !ctx->saved_data["conj"].toBool()), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor rope(DispatchKeySet ks, const Tensor& x, const Tensor& cos, const Tensor& sin, bool conj) {
  return records(x, cos, sin) ? Rope::apply(x, cos, sin, conj, Keys{ks}) : op_rope().below(ks, x, cos, sin, conj);
}

const Op<SwigluSig>& op_swiglu() { APB_OP(o, "swiglu", SwigluSig); return o; }
const Op<SwigluBwdSig>& op_swiglu_bwd() { APB_OP(o, "swiglu_bwd", SwigluBwdSig); return o; }
struct Swiglu : torch::autograd::Function<Swiglu> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& b, Keys k) {
    ctx->save_for_backward({a, b});
    return op_swiglu().below(k.ks, a, b);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    auto [da, db] = op_swiglu_bwd()(g[0], s[0], s[1]);
    return {da, db, Tensor()};
  }
};
Tensor swiglu(DispatchKeySet ks, const Tensor& a, const Tensor& b) {
  return records(a, b) ? Swiglu::apply(a, b, Keys{ks}) : op_swiglu().below(ks, a, b);
}

// ---------------------------------------------------------------------------------------------- attention, loss, embedding
const Op<AttnSig>& op_attn() { APB_OP(o, "attention", AttnSig); return o; }
const Op<AttnBwdSig>& op_attn_bwd() { APB_OP(o, "attention_bwd", AttnBwdSig); return o; }
struct Attn : torch::autograd::Function<Attn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale, Keys key) {
    auto [out, lse] = op_attn().below(key.ks, q, k, v, causal, scale);
    ctx->save_for_backward({q, k, v, out, lse});
    ctx->set_materialize_grads(false);
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dv] =
        op_attn_bwd()(first_grad(g, s[3]), s[0], s[1], s[2], s[3], s[4], ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
  }
};
Pair attention(DispatchKeySet ks, const Tensor& q, const Tensor& k, const Tensor& v, bool causal, double scale) {
  if (!records(q, k, v)) return op_attn().below(ks, q, k, v, causal, scale);
  auto o = Attn::apply(q, k, v, causal, scale, Keys{ks});
  return {o[0], o[1]};
}

const Op<XentSig>& op_xent() { APB_OP(o, "cross_entropy", XentSig); return o; }
const Op<XentBwdSig>& op_xent_bwd() { APB_OP(o, "cross_entropy_bwd", XentBwdSig); return o; }
struct Xent : torch::autograd::Function<Xent> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, Keys k) {
    auto [loss, lse] = op_xent().below(k.ks, logits, labels);
    ctx->save_for_backward({logits, labels, lse});
    ctx->set_materialize_grads(false);
    return {loss, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    return {op_xent_bwd()(first_grad(g, s[2]), s[0], s[1], s[2]), Tensor(), Tensor()};
  }
};
Pair cross_entropy(DispatchKeySet ks, const Tensor& logits, const Tensor& labels) {
  if (!records(logits)) return op_xent().below(ks, logits, labels);
  auto o = Xent::apply(logits, labels, Keys{ks});
  return {o[0], o[1]};
}

const Op<EmbSig>& op_emb() { APB_OP(o, "embedding", EmbSig); return o; }
const Op<EmbBwdSig>& op_emb_bwd() { APB_OP(o, "embedding_bwd", EmbBwdSig); return o; }
struct Emb : torch::autograd::Function<Emb> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& ids, Keys k) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = weight.sym_size(0).guard_int(__FILE__, __LINE__);
    return op_emb().below(k.ks, weight, ids);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    return {op_emb_bwd()(g[0], s[0], ctx->saved_data["rows"].toInt()), Tensor(), Tensor()};
  }
};
Tensor embedding(DispatchKeySet ks, const Tensor& weight, const Tensor& ids) {
  return records(weight) ? Emb::apply(weight, ids, Keys{ks}) : op_emb().below(ks, weight, ids);
}

// ---------------------------------------------------------------------------------------------- mixture-of-experts dispatch
const Op<ScatterSig>& op_scatter() { APB_OP(o, "moe_scatter", ScatterSig); return o; }
const Op<GatherSig>& op_gather() { APB_OP(o, "moe_gather", GatherSig); return o; }
const Op<GatherSig>& op_gate_grad() { APB_OP(o, "moe_gate_grad", GatherSig); return o; }
struct Scatter : torch::autograd::Function<Scatter> {
  static Tensor forward(AutogradContext* ctx, const Tensor& src, const Tensor& slot, const Tensor& w, int64_t E, int64_t C, int64_t nb, Keys k) {
    ctx->save_for_backward({src, slot, w});
    return op_scatter().below(k.ks, src, slot, w, E, C, nb);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    Tensor dsrc, dw;
    if (ctx->needs_input_grad(0)) dsrc = op_gather()(g[0], s[1], s[2]);
    if (ctx->needs_input_grad(2)) dw = op_gate_grad()(g[0], s[1], s[0]).to(s[2].scalar_type());
    return {dsrc, Tensor(), dw, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor moe_scatter(DispatchKeySet ks, const Tensor& src, const Tensor& slot, const Tensor& w, int64_t E, int64_t C, int64_t nb) {
  return records(src, w) ? Scatter::apply(src, slot, w, E, C, nb, Keys{ks}) : op_scatter().below(ks, src, slot, w, E, C, nb);
}
struct Gather : torch::autograd::Function<Gather> {
  static Tensor forward(AutogradContext* ctx, const Tensor& buf, const Tensor& slot, const Tensor& w, Keys k) {
    ctx->save_for_backward({buf, slot, w});
    return op_gather().below(k.ks, buf, slot, w);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &buf = s[0], &slot = s[1], &w = s[2];
    Tensor dbuf, dw;
    if (ctx->needs_input_grad(0))
      dbuf = op_scatter()(g[0], slot, w, buf.sym_size(0).guard_int(__FILE__, __LINE__), buf.sym_size(2).guard_int(__FILE__, __LINE__),
                          buf.sym_size(1).guard_int(__FILE__, __LINE__));
    if (ctx->needs_input_grad(2)) dw = op_gate_grad()(buf, slot, g[0]).to(w.scalar_type());
    return {dbuf, Tensor(), dw, Tensor()};
  }
};
Tensor moe_gather(DispatchKeySet ks, const Tensor& buf, const Tensor& slot, const Tensor& w) {
  return records(buf, w) ? Gather::apply(buf, slot, w, Keys{ks}) : op_gather().below(ks, buf, slot, w);
}

// ---------------------------------------------------------------------------------------------- routing
using RouteSig = Pair(const Tensor&, const c10::optional<Tensor>&, int64_t, bool, int64_t, int64_t, bool, double);
using RouteBwdSig = Tensor(const Tensor&, const Tensor&, const Tensor&, bool, bool, double);
const Op<RouteSig>& op_route() { APB_OP(o, "moe_route", RouteSig); return o; }
const Op<RouteBwdSig>& op_route_bwd() { APB_OP(o, "moe_route_bwd", RouteBwdSig); return o; }
struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& bias, int64_t k, bool sigmoid, int64_t groups,
                               int64_t top_groups, bool renorm, double scale, Keys key) {
    auto [w, idx] = op_route().below(key.ks, x, bias, k, sigmoid, groups, top_groups, renorm, scale);
    ctx->save_for_backward({x, idx});
    ctx->mark_non_differentiable({idx});
    ctx->set_materialize_grads(false);
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->saved_data["renorm"] = renorm;
    ctx->saved_data["scale"] = scale;
    return {w, idx};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    return once("moe_route", g, [&]() -> variable_list {
      const auto s = ctx->get_saved_variables();
      Tensor dx;
      if (g[0].defined())
        dx = op_route_bwd()(g[0], s[0], s[1], ctx->saved_data["sigmoid"].toBool(), ctx->saved_data["renorm"].toBool(), ctx->saved_data["scale"].toDouble());
      return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};
Pair moe_route(DispatchKeySet ks, const Tensor& x, const c10::optional<Tensor>& bias, int64_t k, bool sigmoid, int64_t groups, int64_t top_groups,
               bool renorm, double scale) {
  if (!records(x)) return op_route().below(ks, x, bias, k, sigmoid, groups, top_groups, renorm, scale);
  auto o = Route::apply(x, bias, k, sigmoid, groups, top_groups, renorm, scale, Keys{ks});
  return {o[0], o[1]};
}

// ---------------------------------------------------------------------------------------------- MXFP4 (straight through the rounding)
using MxRoundSig = Tensor(const Tensor&, int64_t);
using MxValuesSig = Tensor(const Tensor&, const Tensor&, int64_t, ScalarType);
using MxLinearSig = Tensor(const Tensor&, const Tensor&, const Tensor&, ScalarType);
const Op<MxRoundSig>& op_mx_round() { APB_OP(o, "mx4_round", MxRoundSig); return o; }
const Op<MxValuesSig>& op_mx_values() { APB_OP(o, "mx4_dequantize", MxValuesSig); return o; }
using MxMmValuesSig = Tensor(const Tensor&, const Tensor&, const Tensor&, int64_t, ScalarType);
const Op<MxMmValuesSig>& op_mx_mm_values() { APB_OP(o, "mx4_mm_values", MxMmValuesSig); return o; }
const Op<MxLinearSig>& op_mx_linear() { APB_OP(o, "mx4_linear", MxLinearSig); return o; }
const Op<MmNdSig>& op_mx_matmul() { APB_OP(o, "mx4_matmul", MmNdSig); return o; }

// Zeros up to multiples of 8 in the last dim and, if asked for, in the one before: the 16-bit products address rows of whole 16 bytes.
Tensor pad8(const Tensor& t, bool rows, bool columns) {
  const int64_t c = columns ? (8 - t.size(-1) % 8) % 8 : 0, r = rows ? (8 - t.size(-2) % 8) % 8 : 0;
  return c == 0 && r == 0 ? t : at::constant_pad_nd(t, {0, c, 0, r}, 0);
}
Tensor times(const Tensor& a, const Tensor& b, bool trans_b, ScalarType dtype) {
  return b.dim() == 3 ? op_grouped_mm()(a, b, trans_b, dtype) : op_mm_nd()(a, b, trans_b, dtype);
}
Tensor pad_last(const Tensor& t) { return t.size(-1) % 8 == 0 ? t : at::constant_pad_nd(t, {0, 8 - t.size(-1) % 8}, 0); }
Tensor cut(const Tensor& t, int64_t dim, int64_t size) { return t.size(dim) == size ? t : t.narrow(dim, 0, size); }

struct MxRound : torch::autograd::Function<MxRound> {
  static Tensor forward(AutogradContext*, const Tensor& x, int64_t dim, Keys k) { return op_mx_round().below(k.ks, x, dim); }
  static variable_list backward(AutogradContext*, const variable_list& g) { return {g[0], Tensor(), Tensor()}; }
};
Tensor mx4_round(DispatchKeySet ks, const Tensor& x, int64_t dim) {
  return records(x) ? MxRound::apply(x, dim, Keys{ks}) : op_mx_round().below(ks, x, dim);
}
struct MxMmValues : torch::autograd::Function<MxMmValues> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& codes, const Tensor& scales, int64_t k, ScalarType dtype, Keys ks) {
    ctx->save_for_backward({codes, scales});
    ctx->saved_data["k"] = k;
    ctx->saved_data["dtype"] = a.scalar_type();
    return op_mx_mm_values().below(ks.ks, a, codes, scales, k, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const Tensor& dc = g[0];
    const int64_t n = s[0].size(-2), k8 = (ctx->saved_data["k"].toInt() + 7) / 8 * 8;
    const ScalarType dtype = ctx->saved_data["dtype"].toScalarType();
    Tensor da;
    if (n == 0 || k8 == 0) {
      auto shape = dc.sizes().vec();
      shape.back() = n;
      da = at::zeros(shape, dc.options().dtype(dtype));
    } else {
      da = cut(times(pad_last(dc), pad8(op_mx_values()(s[0], s[1], k8, dc.scalar_type()), true, false), true, dtype), -1, n);
    }
    return {da, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor mx4_mm_values(DispatchKeySet ks, const Tensor& a, const Tensor& codes, const Tensor& scales, int64_t k, ScalarType dtype) {
  return records(a) ? MxMmValues::apply(a, codes, scales, k, dtype, Keys{ks}) : op_mx_mm_values().below(ks, a, codes, scales, k, dtype);
}
struct MxLinear : torch::autograd::Function<MxLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales, ScalarType dtype, Keys k) {
    ctx->save_for_backward({codes, scales});
    ctx->saved_data["k"] = x.size(-1);
    ctx->saved_data["dtype"] = x.scalar_type();
    return op_mx_linear().below(k.ks, x, codes, scales, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    return {op_mx_mm_values()(g[0], s[0], s[1], ctx->saved_data["k"].toInt(), ctx->saved_data["dtype"].toScalarType()), Tensor(), Tensor(), Tensor(),
            Tensor()};
  }
};
Tensor mx4_linear(DispatchKeySet ks, const Tensor& x, const Tensor& codes, const Tensor& scales, ScalarType dtype) {
  return records(x) ? MxLinear::apply(x, codes, scales, dtype, Keys{ks}) : op_mx_linear().below(ks, x, codes, scales, dtype);
}
// Saves the operands in 4 bits, which the product needs anyway, and takes the values of the gradients' products from them: less memory held, and less
// to read than the 16-bit operands.
using MxQuantSig = Pair(const Tensor&);
using MxMmSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, ScalarType);
const Op<MxQuantSig>& op_mx_quantize() { APB_OP(o, "mx4_quantize", MxQuantSig); return o; }
const Op<MxMmSig>& op_mx_mm() { APB_OP(o, "mx4_mm", MxMmSig); return o; }
struct MxMatmul : torch::autograd::Function<MxMatmul> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, bool trans_b, ScalarType dtype) {
    at::AutoDispatchBelowAutograd guard;
    const bool flat = w.dim() == 2 && x.dim() != 2;
    auto [a, sa] = op_mx_quantize()(flat ? x.reshape({c10::multiply_integers(x.sizes().slice(0, x.dim() - 1)), x.size(-1)}) : x);
    auto [b, sb] = op_mx_quantize()(trans_b ? w : w.transpose(-1, -2));
    Tensor y = op_mx_mm()(a, sa, b, sb, dtype);
    const bool of_x = x.requires_grad(), of_w = w.requires_grad();
    ctx->save_for_backward({of_w ? a : Tensor(), of_w ? sa : Tensor(), of_x ? b : Tensor(), of_x ? sb : Tensor()});
    ctx->saved_data["tb"] = trans_b;
    ctx->saved_data["k"] = x.size(-1);
    ctx->saved_data["n"] = y.size(-1);
    ctx->saved_data["x"] = x.scalar_type();
    ctx->saved_data["w"] = w.scalar_type();
    if (!flat) return y;
    auto shape = x.sizes().vec();
    shape.back() = y.size(-1);
    return y.view(shape);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    return once("mx4_matmul", g, [&] { return gradients(ctx, g); });  // (the operands themselves are not kept)
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const bool tb = ctx->saved_data["tb"].toBool();
    const int64_t k = ctx->saved_data["k"].toInt(), kp = (k + 31) / 32 * 32, n = ctx->saved_data["n"].toInt();
    Tensor dx, dw;
    if (ctx->needs_input_grad(0)) dx = op_mx_mm_values()(g[0], s[2], s[3], k, ctx->saved_data["x"].toScalarType());
    if (ctx->needs_input_grad(1)) {
      const ScalarType type = ctx->saved_data["w"].toScalarType();
      if (k == 0 || n == 0) {  // (the products take no matrices without columns)
        std::vector<int64_t> shape{tb ? n : k, tb ? k : n};
        if (s[0].dim() == 3) shape.insert(shape.begin(), s[0].size(0));
        return {dx, at::zeros(shape, g[0].options().dtype(type)), Tensor(), Tensor()};
      }
      const Tensor dy = pad_last(g[0]);
      const Tensor xq = op_mx_values()(s[0], s[1], kp, dy.scalar_type());  // [rows, kp], or [E, rows, kp]
      const Tensor d = xq.dim() == 3 ? dy : dy.reshape({xq.size(0), dy.size(-1)});
      const Op<WgradSig>& wgrad = xq.dim() == 3 ? op_grouped_wgrad() : op_mm_wgrad();
      dw = tb ? cut(cut(wgrad(d, xq, type), -1, k), -2, n) : cut(cut(wgrad(xq, d, type), -1, n), -2, k);
    }
    return {dx, dw, Tensor(), Tensor()};
  }
};
// What a tracer, another mode or an installed function sees is the one operator, and the formula of ops/mx4_ops.py.
struct MxMatmulTraced : torch::autograd::Function<MxMatmulTraced> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, bool trans_b, ScalarType dtype, Keys k) {
    ctx->save_for_backward({x, w});
    ctx->saved_data["tb"] = trans_b;
    return op_mx_matmul().below(k.ks, x, w, trans_b, dtype);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], dy = pad_last(g[0]);
    const bool tb = ctx->saved_data["tb"].toBool();
    if (x.size(-1) == 0 || dy.size(-1) == 0) return {at::zeros_like(x), at::zeros_like(w), Tensor(), Tensor(), Tensor()};
    Tensor dx, dw;
    if (ctx->needs_input_grad(0))
      dx = cut(times(dy, pad8(op_mx_round()(w, tb ? -1 : -2).to(dy.scalar_type()), true, true), !tb, x.scalar_type()), -1, x.size(-1));
    if (ctx->needs_input_grad(1)) {
      const Tensor xq = pad_last(op_mx_round()(x, -1).to(dy.scalar_type()));
      const Op<WgradSig>& wgrad = w.dim() == 3 ? op_grouped_wgrad() : op_mm_wgrad();
      dw = cut(cut(tb ? wgrad(dy, xq, w.scalar_type()) : wgrad(xq, dy, w.scalar_type()), -1, w.size(-1)), -2, w.size(-2));
    }
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};
Tensor mx4_matmul(DispatchKeySet ks, const Tensor& x, const Tensor& w, bool trans_b, ScalarType dtype) {
  if (!records(x, w)) return op_mx_matmul().below(ks, x, w, trans_b, dtype);
  if (!apb_mx4_matmul_ours() || c10::impl::dispatch_mode_enabled() || x.unsafeGetTensorImpl()->is_python_dispatch() || w.unsafeGetTensorImpl()->is_python_dispatch())
    return MxMatmulTraced::apply(x, w, trans_b, dtype, Keys{ks});
  return MxMatmul::apply(x, w, trans_b, dtype);
}

}  // namespace

TORCH_LIBRARY_IMPL(apb200, AutogradCUDA, m) {
  m.impl("dtype_cast", cast);
  m.impl("mm_nd", mm_nd);
  m.impl("gemm", gemm);
  m.impl("grouped_mm", grouped_mm);
  m.impl("rms_norm", rms_norm);
  m.impl("rope", rope);
  m.impl("swiglu", swiglu);
  m.impl("attention", attention);
  m.impl("cross_entropy", cross_entropy);
  m.impl("embedding", embedding);
  m.impl("moe_scatter", moe_scatter);
  m.impl("moe_gather", moe_gather);
  m.impl("moe_route", moe_route);
  m.impl("mx4_round", mx4_round);
  m.impl("mx4_mm_values", mx4_mm_values);
  m.impl("mx4_linear", mx4_linear);
  m.impl("mx4_matmul", mx4_matmul);
}
