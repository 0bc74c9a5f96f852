// The operators around the transform as torch functions over the C ABI: what
// cpab/pytorch/sequence.py calls.
#include "torch_common.hpp"

#include <array>

namespace {

using namespace cpab_torch;
// [B, T, C] with its channels contiguous, detached; no copy where they are already and its
// samples no further apart than the kernels reach.
Tensor samples_of(const Tensor& t) {
  const Tensor d = t.detach();
  const int64_t B = d.size(0), T = d.size(1), C = d.size(2);
  return (C <= 1 || d.stride(2) == 1) &&
                 (T <= 1 || d.stride(1) <= cpab_recurrence_max_stride(type_of(d), B, T, C))
             ? d : d.contiguous();
}

// ---- gated recurrence --------------------------------------------------------

std::array<int64_t, 6> strides_of(const Tensor& x, const Tensor& f, const Tensor& g) {
  return {x.stride(0), x.stride(1), f.stride(0), f.stride(1), g.defined() ? g.stride(0) : 0,
          g.defined() ? g.stride(1) : 0};
}

struct Recurrence : torch::autograd::Function<Recurrence> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Tensor& f_,
                               const Maybe& maybe_g, const Maybe& maybe_h0,
                               const Maybe& maybe_lengths, bool keep) {
    const c10::OptionalDeviceGuard guard(x_.device());
    const Tensor g_ = of(maybe_g), h0_ = of(maybe_h0), lengths = of(maybe_lengths);
    const Tensor x = samples_of(x_), f = samples_of(f_),
                 g = g_.defined() ? samples_of(g_) : Tensor();
    const Tensor h0 = h0_.defined() ? plain(h0_) : Tensor();
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
    Tensor y = at::empty({B, T, C}, x.options()), h = empty({B, C}, x), carries;
    const int type = type_of(x);
    if (keep) carries = empty({cpab_recurrence_carries(type, B, T, C)}, x);
    const int64_t bytes = cpab_recurrence_workspace_size(type, B, T, C, 0);
    at::DataPtr ws;
    if (bytes > 0) ws = scratch(bytes);
    const auto strides = strides_of(x, f, g);
    check(cpab_recurrence_forward(type, B, T, C, ptr(x), ptr(f), ptr(g), strides.data(), in(h0),
                                  ptr(lengths),
                                  lengths.defined() && lengths.scalar_type() == at::kLong, ptr(y),
                                  out(h), out(carries), ws.get(), bytes, stream_of(x)),
          "cpab_recurrence_forward");
    ctx->set_materialize_grads(false);
    if (keep) ctx->save_for_backward({x, f, g, h0, lengths, carries});
    return {y, h};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (!any_defined(grads)) return variable_list(6);
    Tensor dx, df, dg, dh0;
    {
      const at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const Tensor &x = saved[0], &f = saved[1], &g = saved[2], &h0 = saved[3], &lengths = saved[4],
                   &carries = saved[5];
      const c10::OptionalDeviceGuard guard(x.device());
      const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
      Tensor dy = grad_of(grads[0], x.scalar_type()), dh = grad_of(grads[1], at::kFloat);
      if (dy.defined()) dy = dy.contiguous();
      if (dh.defined()) dh = dh.contiguous();
      if (ctx->needs_input_grad(0)) dx = at::empty({B, T, C}, x.options());
      if (ctx->needs_input_grad(1)) df = at::empty({B, T, C}, x.options());
      // inputs that were not given have no place among those that may need a gradient
      const size_t after_g = g.defined() ? 3 : 2;
      if (g.defined() && ctx->needs_input_grad(2)) dg = at::empty({B, T, C}, x.options());
      if (h0.defined() && ctx->needs_input_grad(after_g)) dh0 = empty({B, C}, x);
      const int type = type_of(x);
      const int64_t bytes = cpab_recurrence_workspace_size(type, B, T, C, 1);
      at::DataPtr ws;
      if (bytes > 0) ws = scratch(bytes);
      const auto strides = strides_of(x, f, g);
      check(cpab_recurrence_backward(type, B, T, C, ptr(x), ptr(f), ptr(g), strides.data(), in(h0),
                                     ptr(lengths),
                                     lengths.defined() && lengths.scalar_type() == at::kLong,
                                     in(carries), ptr(dy), in(dh), ptr(dx), ptr(df), ptr(dg),
                                     out(dh0), ws.get(), bytes, stream_of(x)),
            "cpab_recurrence_backward");
    }
    return once_any({dx, df, dg, dh0, Tensor(), Tensor()});
  }
};

variable_list recurrence(const Tensor& x, const Tensor& f, const Maybe& g_, const Maybe& h0_,
                         const Maybe& lengths_) {
  const Tensor g = of(g_), h0 = of(h0_), lengths = of(lengths_);
  if (!x.is_cuda()) fail("gated_recurrence: only GPU tensors are supported");
  if (!has_type(x))
    fail("gated_recurrence: expected float32 or bfloat16, got " + dtype_of(x));
  if (x.dim() != 3) fail("gated_recurrence: x must be [B, T, C], got " + shape_of(x));
  const auto like_x = [&](const Tensor& t, const char* name) {
    if (t.device() != x.device() || t.scalar_type() != x.scalar_type() || t.sizes() != x.sizes())
      fail(std::string("gated_recurrence: ") + name + " must have x's shape " + shape_of(x) +
           ", type and device, got " + shape_of(t) + " " + dtype_of(t));
  };
  like_x(f, "f");
  if (g.defined()) like_x(g, "g");
  if (h0.defined() && (h0.device() != x.device() || h0.scalar_type() != at::kFloat ||
                       h0.dim() != 2 || h0.size(0) != x.size(0) || h0.size(1) != x.size(2)))
    fail("gated_recurrence: h0 must be float32 [" + std::to_string(x.size(0)) + ", " +
         std::to_string(x.size(2)) + "] on x's device, got " + shape_of(h0) + " " + dtype_of(h0));
  if (lengths.defined() &&
      (lengths.device() != x.device() || lengths.dim() != 1 || lengths.size(0) != x.size(0) ||
       (lengths.scalar_type() != at::kInt && lengths.scalar_type() != at::kLong)))
    fail("gated_recurrence: lengths must be int32 or int64 [" + std::to_string(x.size(0)) +
         "] on x's device, got " + shape_of(lengths) + " " + dtype_of(lengths));
  const bool keep = any_grad({x, f, g, h0});
  py::gil_scoped_release nogil;
  const Maybe dense = lengths.defined() ? Maybe(lengths.contiguous()) : Maybe();
  return Recurrence::apply(x, f, g_, h0_, dense, keep);
}

// ---- root-mean-square norm -----------------------------------------------------

// [rows, C] with one stride over the rows, without a copy where that is possible.
Tensor as_rows(const Tensor& t, int64_t C) {
  const Tensor d = t.requires_grad() ? t.detach() : t;
  const Tensor m = t.dim() == 2 ? d : d.reshape({-1, C});
  return C <= 1 || m.stride(1) == 1 ? m : m.contiguous();
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Tensor& weight_,
                               const Maybe& maybe_residual, double eps, bool keep) {
    const c10::OptionalDeviceGuard guard(x_.device());
    const Tensor residual_ = of(maybe_residual);
    const int64_t C = x_.size(-1);
    const Tensor x = as_rows(x_, C), w = plain(weight_);
    const Tensor res = residual_.defined() ? as_rows(residual_, C) : Tensor();
    const int64_t rows = x.size(0);
    Tensor y = at::empty(x_.sizes(), x.options()), sum, rstd;
    if (res.defined()) sum = at::empty(x_.sizes(), res.options());
    if (keep) rstd = empty({rows}, x);
    const int type = type_of(x);
    check(cpab_rms_norm_forward(type, res.defined() ? type_of(res) : type, type_of(w), rows, C,
                                ptr(x), x.stride(0), ptr(res), res.defined() ? res.stride(0) : 0,
                                ptr(w), (float)eps, ptr(y), ptr(sum), out(rstd), stream_of(x)),
          "cpab_rms_norm_forward");
    ctx->set_materialize_grads(false);
    // the sum; or its parts, where it was rounded to 16 bits
    const bool parts = sum.defined() && sum.scalar_type() != at::kFloat;
    if (keep && parts)
      ctx->save_for_backward({x, w, rstd, res});
    else if (keep)
      ctx->save_for_backward({sum.defined() ? sum : x, w, rstd, Tensor()});
    ctx->saved_data["dtype"] = (int64_t)x.scalar_type();
    if (sum.defined()) return {y, sum};
    return {y};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    if (!any_defined(grads)) return variable_list(5);
    Tensor dx, dres, dw;
    {
      const at::NoGradGuard no_grad;
      const auto saved = ctx->get_saved_variables();
      const Tensor &r_ = saved[0], &w = saved[1], &rstd = saved[2], &added = saved[3];
      const c10::OptionalDeviceGuard guard(r_.device());
      const bool residual = grads.size() > 1;
      const auto dtype = (at::ScalarType)ctx->saved_data["dtype"].toInt();
      const int64_t C = r_.size(-1);
      const Tensor r = as_rows(r_, C);
      const int64_t rows = r.size(0);
      const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
      const bool want_res = residual && ctx->needs_input_grad(2);
      const bool same = dtype == r.scalar_type();
      const auto shape = grads[0].defined() ? grads[0].sizes().vec() : grads[1].sizes().vec();
      const auto options = r.options().dtype(dtype);
      Tensor dy = grads[0].defined() ? as_rows(grad_of(grads[0], dtype), C) : at::zeros({rows, C}, options);
      Tensor dout;
      if (residual && grads[1].defined()) dout = as_rows(grad_of(grads[1], r.scalar_type()), C);
      // one gradient for both where they have one type
      if (want_x || (want_res && same)) dx = at::empty(shape, options);
      if (want_res) dres = same ? dx : at::empty(shape, r.options());
      if (want_w) dw = at::empty(w.sizes(), w.options());
      const int64_t bytes = want_w ? cpab_rms_norm_backward_workspace_size(rows, C) : 0;
      at::DataPtr ws;
      if (bytes > 0) ws = scratch(bytes);
      check(cpab_rms_norm_backward(dtype == at::kFloat ? CPAB_F32 : CPAB_BF16, type_of(r),
                                   type_of(w), rows, C, ptr(r), r.stride(0), ptr(added),
                                   added.defined() ? added.stride(0) : 0, in(rstd), ptr(w), ptr(dy), dy.stride(0), ptr(dout),
                                   dout.defined() ? dout.stride(0) : 0, ptr(dx),
                                   same ? nullptr : ptr(dres), ptr(dw), ws.get(), bytes,
                                   stream_of(r)),
            "cpab_rms_norm_backward");
      if (!want_x) dx = Tensor();
    }
    return once_any({dx, dw, dres, Tensor(), Tensor()});
  }
};

variable_list rms_norm(const Tensor& x, const Tensor& weight, const Maybe& residual_, double eps,
                       bool eight) {
  const Tensor residual = of(residual_);
  if (!x.is_cuda()) fail("rms_norm: only GPU tensors are supported");
  if (!has_type(x)) fail("rms_norm: expected float32 or bfloat16, got " + dtype_of(x));
  if (x.dim() < 1) fail("rms_norm: x must be [..., C], got a scalar");
  const int64_t C = x.size(-1);
  if (weight.device() != x.device() || !has_type(weight) || weight.dim() != 1 || weight.size(0) != C)
    fail("rms_norm: weight must be float32 or bfloat16 [" + std::to_string(C) +
         "] on x's device, got " + shape_of(weight) + " " + dtype_of(weight));
  if (residual.defined() &&
      (residual.device() != x.device() || residual.sizes() != x.sizes() ||
       (residual.scalar_type() != x.scalar_type() && residual.scalar_type() != at::kFloat)))
    fail("rms_norm: residual must have x's shape " + shape_of(x) +
         " and device, and x's type or float32, got " + shape_of(residual) + " " + dtype_of(residual));
  if (!(eps >= 0)) fail("rms_norm: eps must not be negative");
  const bool keep = any_grad({x, weight, residual});
  if (eight && keep)
    fail("rms_norm: the 8-bit output has no gradient; call it under torch.no_grad()");
  py::gil_scoped_release nogil;
  if (C == 0) fail("rms_norm: x has rows of no values");
  if (!eight) return RmsNorm::apply(x, weight, residual_, eps, keep);
  const c10::OptionalDeviceGuard guard(x.device());
  const Tensor xr = as_rows(x, C), w = plain(weight);
  const Tensor res = residual.defined() ? as_rows(residual, C) : Tensor();
  Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), sum;
  Tensor scale = empty(x.sizes().slice(0, x.dim() - 1), x);
  if (res.defined()) sum = at::empty(x.sizes(), res.options());
  const int type = type_of(x);
  check(cpab_rms_norm_e4m3(type, res.defined() ? type_of(res) : type, type_of(w), xr.size(0), C,
                           ptr(xr), xr.stride(0), ptr(res), res.defined() ? res.stride(0) : 0,
                           ptr(w), (float)eps, ptr(q), out(scale), ptr(sum), stream_of(xr)),
        "cpab_rms_norm_e4m3");
  if (sum.defined()) return {q, scale, sum};
  return {q, scale};
}

// ---- AdamW -----------------------------------------------------------------------

typedef std::vector<Tensor> Tensors;

void adamw(const Tensors& params, const Tensors& grads, const Tensors& exp_avgs,
           const Tensors& exp_avg_sqs, int64_t step, double lr, double beta1, double beta2,
           double eps, double weight_decay, const std::optional<Tensors>& exp_avg_scales,
           const std::optional<Tensors>& exp_avg_sq_scales, const std::optional<Tensors>& masters,
           int64_t seed) {
  const size_t n = params.size();
  if (grads.size() != n || exp_avgs.size() != n || exp_avg_sqs.size() != n ||
      (exp_avg_scales && exp_avg_scales->size() != n) ||
      (exp_avg_sq_scales && exp_avg_sq_scales->size() != n) || (masters && masters->size() != n))
    fail("adamw_step: the lists must have one entry for each of the " + std::to_string(n) +
         " parameters");
  if (exp_avg_scales.has_value() != exp_avg_sq_scales.has_value())
    fail("adamw_step: give both lists of scales (8-bit states) or neither");
  if (n == 0) return;
  const bool eight = exp_avg_scales.has_value();
  const Tensor& first = params[0];
  if (!first.is_cuda()) fail("adamw_step: only GPU tensors are supported");
  if (!has_type(first))
    fail("adamw_step: expected float32 or bfloat16 parameters, got " + dtype_of(first));
  const c10::OptionalDeviceGuard guard(first.device());
  const at::NoGradGuard no_grad;
  std::vector<cpab_adamw_tensor> tensors(n);
  Tensors copies;   // gradients in other layouts, until they are queued
  for (size_t k = 0; k < n; ++k) {
    const Tensor& p = params[k];
    const auto where = [k] { return " of parameter " + std::to_string(k); };
    if (p.device() != first.device() || p.scalar_type() != first.scalar_type())
      fail("adamw_step: the parameters must have one type and one device; parameter " +
           std::to_string(k) + " is " + dtype_of(p) + " on " + p.device().str());
    if (!p.is_non_overlapping_and_dense())
      fail("adamw_step: parameter " + std::to_string(k) + " is not dense in memory");
    // autograd counts its changes, which it refuses only after they were made
    const auto changed = [&](const Tensor& t, const char* name) {
      if (t.is_inference() && !c10::InferenceMode::is_enabled())
        fail(std::string("adamw_step: ") + name + where() +
             " is an inference tensor, which may not be changed outside inference mode");
      return t.data_ptr();
    };
    // a state in the parameter's own layout: its values lie in the same order
    const auto like_p = [&](const Tensor& t, at::ScalarType type, const char* name) {
      if (t.device() != p.device() || t.scalar_type() != type || t.sizes() != p.sizes() ||
          (t.strides() != p.strides() && !(t.is_contiguous() && p.is_contiguous())))
        fail(std::string("adamw_step: ") + name + where() + " must be " +
             c10::getDtypeNames(type).first + " in the parameter's shape " + shape_of(p) +
             ", strides and device, got " + shape_of(t) + " " + dtype_of(t));
      return changed(t, name);
    };
    const auto flat = [&](const Tensor& t, at::ScalarType type, int64_t count, const char* name) {
      if (t.device() != p.device() || t.scalar_type() != type || t.numel() != count ||
          !t.is_contiguous())
        fail(std::string("adamw_step: ") + name + where() + " must be contiguous " +
             c10::getDtypeNames(type).first + " of " + std::to_string(count) +
             " values on the parameter's device, got " + shape_of(t) + " " + dtype_of(t));
      return changed(t, name);
    };
    Tensor g = grads[k];
    if (g.device() != p.device() || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes() ||
        g.layout() != at::kStrided)
      fail("adamw_step: the gradient" + where() + " must be dense in the parameter's shape " +
           shape_of(p) + ", type and device, got " + shape_of(g) + " " + dtype_of(g));
    if (g.strides() != p.strides() && !(g.is_contiguous() && p.is_contiguous())) {
      Tensor same = at::empty_strided(p.sizes(), p.strides(), p.options());
      same.copy_(g);
      copies.push_back(same);
      g = same;
    }
    const int64_t count = p.numel();
    cpab_adamw_tensor& t = tensors[k];
    t.param = changed(p, "the value");
    t.grad = g.data_ptr();
    t.n = count;
    t.master = masters ? static_cast<float*>(like_p((*masters)[k], at::kFloat, "the master")) : nullptr;
    if (eight) {
      const int64_t groups = (count + 31) / 32;
      t.exp_avg = flat(exp_avgs[k], at::kFloat8_e4m3fn, count, "exp_avg");
      t.exp_avg_sq = flat(exp_avg_sqs[k], at::kFloat8_e4m3fn, count, "exp_avg_sq");
      t.exp_avg_scale = flat((*exp_avg_scales)[k], at::kFloat8_e8m0fnu, groups, "the exp_avg scale");
      t.exp_avg_sq_scale =
          flat((*exp_avg_sq_scales)[k], at::kFloat8_e8m0fnu, groups, "the exp_avg_sq scale");
    } else {
      t.exp_avg = like_p(exp_avgs[k], at::kFloat, "exp_avg");
      t.exp_avg_sq = like_p(exp_avg_sqs[k], at::kFloat, "exp_avg_sq");
    }
  }
  check(cpab_adamw_step(type_of(first), eight ? 8 : 32, (int64_t)n, tensors.data(), step, lr, beta1,
                        beta2, eps, weight_decay, (uint32_t)seed, stream_of(first)),
        "cpab_adamw_step");
  // autograd sees the tensors as changed in place
  for (const Tensors* list : {&params, &exp_avgs, &exp_avg_sqs})
    for (const Tensor& t : *list) torch::autograd::impl::bump_version(t);
  for (const auto* list : {&exp_avg_scales, &exp_avg_sq_scales, &masters})
    if (list->has_value())
      for (const Tensor& t : **list) torch::autograd::impl::bump_version(t);
}

// ---- Muon ------------------------------------------------------------------------

void muon(const Tensors& params, const Tensors& grads, const Tensors& momenta, const std::vector<double>& rates,
          double lr, double weight_decay, double momentum, bool nesterov,
          const std::array<double, 3>& coefficients, double eps, int64_t ns_steps,
          const std::optional<Tensors>& masters) {
  const size_t n = params.size();
  if (grads.size() != n || momenta.size() != n || rates.size() != n || (masters && masters->size() != n))
    fail("muon_step: the lists must have one entry for each of the " + std::to_string(n) + " parameters");
  if (n == 0) return;
  const Tensor& first = params[0];
  if (!first.is_cuda()) fail("muon_step: only GPU tensors are supported");
  if (!has_type(first)) fail("muon_step: expected float32 or bfloat16 parameters, got " + dtype_of(first));
  const c10::OptionalDeviceGuard guard(first.device());
  const at::NoGradGuard no_grad;
  std::vector<cpab_muon_matrix> matrices(n);
  Tensors copies;   // gradients in other layouts, until they are queued
  for (size_t k = 0; k < n; ++k) {
    const Tensor& p = params[k];
    const auto where = [k] { return " of parameter " + std::to_string(k); };
    const auto written = [&](const Tensor& t, at::ScalarType type, const char* name) {
      if (t.device() != p.device() || t.scalar_type() != type || t.sizes() != p.sizes() || !t.is_contiguous())
        fail(std::string("muon_step: ") + name + where() + " must be contiguous " + c10::getDtypeNames(type).first +
             " in the parameter's shape " + shape_of(p) + " on its device, got " + shape_of(t) + " " + dtype_of(t));
      if (t.is_inference() && !c10::InferenceMode::is_enabled())
        fail(std::string("muon_step: ") + name + where() +
             " is an inference tensor, which may not be changed outside inference mode");
      return t.data_ptr();
    };
    if (p.device() != first.device() || p.scalar_type() != first.scalar_type())
      fail("muon_step: the parameters must have one type and one device; parameter " + std::to_string(k) +
           " is " + dtype_of(p) + " on " + p.device().str());
    if (p.dim() != 2) fail("muon_step: parameter " + std::to_string(k) + " must be a matrix, got " + shape_of(p));
    Tensor g = grads[k];
    if (g.device() != p.device() || g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes() ||
        g.layout() != at::kStrided)
      fail("muon_step: the gradient" + where() + " must be dense in the parameter's shape " + shape_of(p) +
           ", type and device, got " + shape_of(g) + " " + dtype_of(g));
    if (!g.is_contiguous()) {
      g = g.contiguous();
      copies.push_back(g);
    }
    cpab_muon_matrix& t = matrices[k];
    t.param = written(p, p.scalar_type(), "the value");
    t.grad = g.data_ptr();
    t.momentum = static_cast<float*>(written(momenta[k], at::kFloat, "the momentum"));
    t.master = masters ? static_cast<float*>(written((*masters)[k], at::kFloat, "the master")) : nullptr;
    t.rows = p.size(0), t.cols = p.size(1);
  }
  if (ns_steps < 1 || ns_steps > 100) fail("muon_step: ns_steps must be from 1 to 100");
  const int64_t bytes = cpab_muon_workspace_size((int64_t)n, matrices.data());
  at::DataPtr ws;
  if (bytes > 0) ws = scratch(bytes);
  check(cpab_muon_step(type_of(first), (int64_t)n, matrices.data(), rates.data(), lr, weight_decay, momentum,
                       nesterov, coefficients.data(), eps, (int)ns_steps, ws.get(), bytes, stream_of(first)),
        "cpab_muon_step");
  // autograd sees the tensors as changed in place
  for (const Tensors* list : {&params, &momenta})
    for (const Tensor& t : *list) torch::autograd::impl::bump_version(t);
  if (masters)
    for (const Tensor& t : *masters) torch::autograd::impl::bump_version(t);
}

}  // namespace

void sequence_functions(py::module& m) {
  m.def("muon", &muon);
  m.def("recurrence", &recurrence);
  m.def("rms_norm", &rms_norm);
  m.def("adamw", &adamw);
}
