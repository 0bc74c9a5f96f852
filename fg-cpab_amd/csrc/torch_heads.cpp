// The operators over heads as torch functions over the C ABI: what
// cpab/pytorch/heads.py calls.
#include "torch_common.hpp"

#include <cmath>

namespace {

using namespace cpab_torch;

// [.., H, D] with its last dimension contiguous, detached; no copy where it is already.
Tensor heads_of(const Tensor& t) {
  const Tensor d = t.detach();
  return d.size(-1) <= 1 || d.stride(-1) == 1 ? d : d.contiguous();
}
void strides_to(const Tensor& t, int64_t* to, int count) {
  for (int k = 0; k < count; ++k) to[k] = t.size(k) > 1 ? t.stride(k) : 0;
}

// ---- norms of queries and keys -------------------------------------------------

struct QkNorm : torch::autograd::Function<QkNorm> {
  static cpab_qk_norm describe(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                               const Tensor& freqs, const Tensor& positions, bool neighbours,
                               double eps) {
    cpab_qk_norm n{};
    n.dtype = type_of(q);
    n.weight_dtype = type_of(qw);
    n.neighbours = neighbours;
    n.B = q.size(0), n.T = q.size(1), n.heads = q.size(2), n.key_heads = k.size(2);
    n.width = q.size(3);
    n.turned = freqs.defined() ? 2 * freqs.size(0) : 0;
    n.q = ptr(q), n.k = ptr(k);
    strides_to(q, n.q_strides, 3);
    strides_to(k, n.k_strides, 3);
    n.q_weight = ptr(qw), n.k_weight = ptr(kw);
    n.freqs = in(freqs);
    if (positions.defined()) {
      n.positions = ptr(positions);
      n.position_type = positions.scalar_type() == at::kInt    ? CPAB_POSITION_I32
                        : positions.scalar_type() == at::kLong ? CPAB_POSITION_I64
                                                               : CPAB_POSITION_F32;
      strides_to(positions, n.position_strides, 2);
    }
    n.eps = (float)eps;
    return n;
  }

  static variable_list forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_,
                               const Tensor& qw_, const Tensor& kw_, const Maybe& freqs_,
                               const Maybe& positions_, bool neighbours, double eps, bool keep) {
    const c10::OptionalDeviceGuard guard(q_.device());
    const Tensor q = heads_of(q_), k = heads_of(k_), qw = plain(qw_), kw = plain(kw_);
    const Tensor freqs = freqs_ ? plain(*freqs_) : Tensor(), positions = of(positions_);
    Tensor qo = at::empty(q_.sizes(), q.options()), ko = at::empty(k_.sizes(), k.options());
    const cpab_qk_norm n = describe(q, k, qw, kw, freqs, positions, neighbours, eps);
    check(cpab_qk_norm_forward(&n, ptr(qo), ptr(ko), stream_of(q)), "cpab_qk_norm_forward");
    ctx->set_materialize_grads(false);
    if (keep) {
      ctx->save_for_backward({q, k, qw, kw, freqs, positions});
      ctx->saved_data["neighbours"] = neighbours;
      ctx->saved_data["eps"] = eps;
    }
    return {qo, ko};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (!any_defined(grads)) return variable_list(9);
    Tensor d[2], dw[2];
    {
      const at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const c10::OptionalDeviceGuard guard(saved[0].device());
      const cpab_qk_norm n =
          describe(saved[0], saved[1], saved[2], saved[3], saved[4], saved[5],
                   ctx->saved_data["neighbours"].toBool(), ctx->saved_data["eps"].toDouble());
      Tensor up[2];
      int64_t strides[6];
      const void* in_ptr[2];
      void *out_ptr[2], *weight_ptr[2];
      for (int k = 0; k < 2; ++k) {
        const Tensor& x = saved[k];
        up[k] = grads[k].defined() ? heads_of(grad_of(grads[k], x.scalar_type()))
                                   : at::zeros(x.sizes(), x.options());
        strides_to(up[k], strides + 3 * k, 3);
        if (ctx->needs_input_grad(k)) d[k] = at::empty(x.sizes(), x.options());
        if (ctx->needs_input_grad(2 + k)) dw[k] = at::empty(saved[2 + k].sizes(), saved[2 + k].options());
        in_ptr[k] = ptr(up[k]);
        out_ptr[k] = ptr(d[k]);
        weight_ptr[k] = ptr(dw[k]);
      }
      const int64_t bytes = cpab_qk_norm_backward_workspace_size(&n);
      const at::DataPtr ws = scratch(bytes);
      check(cpab_qk_norm_backward(&n, in_ptr, strides, out_ptr, weight_ptr, ws.get(), bytes,
                                  stream_of(saved[0])),
            "cpab_qk_norm_backward");
    }
    variable_list out(9);
    out[0] = d[0], out[1] = d[1], out[2] = dw[0], out[3] = dw[1];
    return once_any(std::move(out));
  }
};

variable_list qk_norm(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                      const Maybe& freqs_, const Maybe& positions_, bool neighbours, double eps) {
  const Tensor freqs = of(freqs_), positions = of(positions_);
  if (!q.is_cuda()) fail("qk_norm: only GPU tensors are supported");
  if (!has_type(q)) fail("qk_norm: expected float32 or bfloat16, got " + dtype_of(q));
  if (q.dim() != 4) fail("qk_norm: q must be [B, T, heads, width], got " + shape_of(q));
  if (k.device() != q.device() || k.scalar_type() != q.scalar_type() || k.dim() != 4 ||
      k.size(0) != q.size(0) || k.size(1) != q.size(1) || k.size(3) != q.size(3))
    fail("qk_norm: k must be [" + std::to_string(q.size(0)) + ", " + std::to_string(q.size(1)) +
         ", heads, " + std::to_string(q.size(3)) + "] of q's type and device, got " + shape_of(k) +
         " " + dtype_of(k));
  const int64_t D = q.size(3);
  for (const auto& [w, name] : {std::make_pair(&qw, "q_weight"), std::make_pair(&kw, "k_weight")})
    if (w->device() != q.device() || !has_type(*w) || w->scalar_type() != qw.scalar_type() ||
        w->dim() != 1 || w->size(0) != D)
      fail(std::string("qk_norm: ") + name + " must be float32 or bfloat16 (both weights of one type) [" +
           std::to_string(D) + "] on q's device, got " + shape_of(*w) + " " + dtype_of(*w));
  if (freqs.defined()) {
    if (freqs.device() != q.device() || freqs.scalar_type() != at::kFloat || freqs.dim() != 1 ||
        2 * freqs.size(0) > D)
      fail("qk_norm: freqs must be float32 of at most " + std::to_string(D / 2) +
           " values on q's device, got " + shape_of(freqs) + " " + dtype_of(freqs));
    if (at::GradMode::is_enabled() && freqs.requires_grad())
      fail("qk_norm: freqs have no gradient");
  }
  Maybe places;
  if (positions.defined()) {
    if (!freqs.defined()) fail("qk_norm: positions without freqs (give freqs of no values where nothing turns)");
    const auto type = positions.scalar_type();
    const int64_t dims = positions.dim();
    if (positions.device() != q.device() ||
        (type != at::kInt && type != at::kLong && type != at::kFloat) || dims < 1 || dims > 2 ||
        (positions.size(-1) != q.size(1) && positions.size(-1) != 1) ||
        (dims == 2 && positions.size(0) != q.size(0) && positions.size(0) != 1))
      fail("qk_norm: positions must be int32, int64 or float32 [" + std::to_string(q.size(0)) + ", " +
           std::to_string(q.size(1)) + "] (or broadcast to it) on q's device, got " +
           shape_of(positions) + " " + dtype_of(positions));
    if (at::GradMode::is_enabled() && positions.requires_grad())
      fail("qk_norm: positions have no gradient");
    places = positions.detach().expand({q.size(0), q.size(1)});
  }
  if (!(eps >= 0)) fail("qk_norm: eps must not be negative");
  const bool keep = any_grad({q, k, qw, kw});
  py::gil_scoped_release nogil;
  if (D == 0) fail("qk_norm: heads of no values");
  return QkNorm::apply(q, k, qw, kw, freqs_, places, neighbours, eps, keep);
}

// ---- gated delta rule ------------------------------------------------------------

struct DeltaRule : torch::autograd::Function<DeltaRule> {
  static cpab_delta_rule describe(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay,
                                  const Tensor& beta, const Tensor& h0, const Tensor& lengths,
                                  double scale) {
    cpab_delta_rule r{};
    r.dtype = type_of(q);
    r.gate_dtype = type_of(decay);
    r.B = v.size(0), r.T = v.size(1), r.heads = v.size(2), r.key_heads = q.size(2);
    r.dk = q.size(3), r.dv = v.size(3);
    r.q = ptr(q), r.k = ptr(k), r.v = ptr(v), r.decay = ptr(decay), r.beta = ptr(beta);
    strides_to(q, r.q_strides, 3);
    strides_to(k, r.k_strides, 3);
    strides_to(v, r.v_strides, 3);
    strides_to(decay, r.decay_strides, 3);
    strides_to(beta, r.beta_strides, 3);
    r.h0 = in(h0);
    r.lengths = ptr(lengths);
    r.lengths64 = lengths.defined() && lengths.scalar_type() == at::kLong;
    r.scale = (float)scale;
    return r;
  }

  static variable_list forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_,
                               const Tensor& decay_, const Tensor& beta_, const Maybe& maybe_h0,
                               const Maybe& maybe_lengths, double scale, bool keep) {
    const c10::OptionalDeviceGuard guard(v_.device());
    const auto near = [](const Tensor& t) {   // samples no further apart than the kernels reach
      const Tensor n = heads_of(t);
      return n.size(1) <= 1 || n.stride(1) <= CPAB_DELTA_MOST_STRIDE ? n : n.contiguous();
    };
    const Tensor q = near(q_), k = near(k_), v = near(v_), decay = decay_.detach(),
                 beta = beta_.detach(), h0_ = of(maybe_h0), lengths = of(maybe_lengths);
    const Tensor h0 = h0_.defined() ? plain(h0_) : Tensor();
    const cpab_delta_rule r = describe(q, k, v, decay, beta, h0, lengths, scale);
    Tensor o = at::empty(v.sizes(), v.options()), h = empty({r.B, r.heads, r.dk, r.dv}, v), kept;
    if (keep) kept = empty({cpab_delta_rule_kept(&r)}, v);
    const int64_t bytes = cpab_delta_rule_workspace_size(&r, keep, 0);
    at::DataPtr ws;
    if (bytes > 0) ws = scratch(bytes);
    check(cpab_delta_rule_forward(&r, ptr(o), out(h), out(kept), ws.get(), bytes, stream_of(v)),
          "cpab_delta_rule_forward");
    ctx->set_materialize_grads(false);
    if (keep) {
      ctx->save_for_backward({q, k, v, decay, beta, h0, lengths, kept});
      ctx->saved_data["scale"] = scale;
    }
    return {o, h};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (!any_defined(grads)) return variable_list(9);
    variable_list d(9);
    {
      const at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const Tensor &v = saved[2], &h0 = saved[5], &kept = saved[7];
      const c10::OptionalDeviceGuard guard(v.device());
      const cpab_delta_rule r = describe(saved[0], saved[1], v, saved[3], saved[4], h0, saved[6],
                                         ctx->saved_data["scale"].toDouble());
      Tensor go = grad_of(grads[0], v.scalar_type()), gh = grad_of(grads[1], at::kFloat);
      if (go.defined()) go = go.contiguous();
      if (gh.defined()) gh = gh.contiguous();
      // h0, where it was given, is the sixth that may need a gradient
      for (int k = 0; k < (h0.defined() ? 6 : 5); ++k)
        if (ctx->needs_input_grad(k)) d[k] = at::empty(saved[k].sizes(), saved[k].options());
      const int64_t bytes = cpab_delta_rule_workspace_size(&r, 1, 1);
      at::DataPtr ws;
      if (bytes > 0) ws = scratch(bytes);
      check(cpab_delta_rule_backward(&r, in(kept), ptr(go), in(gh), ptr(d[0]), ptr(d[1]), ptr(d[2]),
                                     ptr(d[3]), ptr(d[4]), out(d[5]), ws.get(), bytes, stream_of(v)),
            "cpab_delta_rule_backward");
    }
    return once_any(std::move(d));
  }
};

variable_list delta_rule(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& decay,
                         const Tensor& beta, const Maybe& h0_, const Maybe& lengths_,
                         const std::optional<double>& scale_) {
  const Tensor h0 = of(h0_), lengths = of(lengths_);
  if (!v.is_cuda()) fail("gated_delta_rule: only GPU tensors are supported");
  if (!has_type(v)) fail("gated_delta_rule: expected float32 or bfloat16, got " + dtype_of(v));
  if (v.dim() != 4) fail("gated_delta_rule: v must be [B, T, heads, dv], got " + shape_of(v));
  const int64_t B = v.size(0), T = v.size(1), H = v.size(2);
  const auto text = [](int64_t n) { return std::to_string(n); };
  for (const auto& [t, name] : {std::make_pair(&q, "q"), std::make_pair(&k, "k")})
    if (t->device() != v.device() || t->scalar_type() != v.scalar_type() || t->dim() != 4 ||
        t->size(0) != B || t->size(1) != T || t->sizes() != q.sizes() ||
        (H > 0 && (t->size(2) == 0 || H % t->size(2) != 0)))
      fail(std::string("gated_delta_rule: ") + name + " must be [" + text(B) + ", " + text(T) +
           ", heads, dk] (the heads of v, " + text(H) + ", a multiple of q's and k's) of v's type and " +
           "device, got " + shape_of(*t) + " " + dtype_of(*t));
  const int64_t dk = q.size(3), dv = v.size(3);
  if (dk < 1 || dk > CPAB_DELTA_MOST_KEY)
    fail("gated_delta_rule: dk must be from 1 to " + text(CPAB_DELTA_MOST_KEY) + ", got " + text(dk));
  if (dv < 1) fail("gated_delta_rule: v has heads of no values");
  for (const auto& [t, name] : {std::make_pair(&decay, "decay"), std::make_pair(&beta, "beta")})
    if (t->device() != v.device() || !has_type(*t) || t->scalar_type() != decay.scalar_type() ||
        t->dim() != 3 || t->size(0) != B || t->size(1) != T || t->size(2) != H)
      fail(std::string("gated_delta_rule: ") + name + " must be float32 or bfloat16 (decay and beta of " +
           "one type) [" + text(B) + ", " + text(T) + ", " + text(H) + "] on v's device, got " +
           shape_of(*t) + " " + dtype_of(*t));
  if (h0.defined() && (h0.device() != v.device() || h0.scalar_type() != at::kFloat || h0.dim() != 4 ||
                       h0.size(0) != B || h0.size(1) != H || h0.size(2) != dk || h0.size(3) != dv))
    fail("gated_delta_rule: h0 must be float32 [" + text(B) + ", " + text(H) + ", " + text(dk) + ", " +
         text(dv) + "] on v's device, got " + shape_of(h0) + " " + dtype_of(h0));
  if (lengths.defined() &&
      (lengths.device() != v.device() || lengths.dim() != 1 || lengths.size(0) != B ||
       (lengths.scalar_type() != at::kInt && lengths.scalar_type() != at::kLong)))
    fail("gated_delta_rule: lengths must be int32 or int64 [" + text(B) + "] on v's device, got " +
         shape_of(lengths) + " " + dtype_of(lengths));
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)dk);
  const bool keep = any_grad({q, k, v, decay, beta, h0});
  py::gil_scoped_release nogil;
  const Maybe dense = lengths.defined() ? Maybe(lengths.contiguous()) : Maybe();
  return DeltaRule::apply(q, k, v, decay, beta, h0_, dense, scale, keep);
}

}  // namespace

void heads_functions(py::module& m) {
  m.def("qk_norm", &qk_norm);
  m.def("delta_rule", &delta_rule);
}
