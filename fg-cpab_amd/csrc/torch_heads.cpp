// The operators over heads as torch functions over the C ABI: what
// cpab/pytorch/heads.py calls.
#include "torch_common.hpp"

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
    if (!freqs.defined()) fail("qk_norm: positions without freqs");
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

}  // namespace

void heads_functions(py::module& m) { m.def("qk_norm", &qk_norm); }
