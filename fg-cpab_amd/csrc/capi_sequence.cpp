// The operators around the transform at the extern "C" boundary: argument checks
// before any HIP call, then the launch.
#include <hip/hip_runtime.h>

#include <cmath>
#include <memory>
#include <new>

#include "capi_common.hpp"
#include "sequence_launch.hpp"

namespace {

using cpab::check_hip;
using cpab::fail;

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

int check_dtype(const char* what, int dtype) {
  if (dtype != CPAB_F32 && dtype != CPAB_BF16)
    return fail(CPAB_ERR_INVALID, "%s must be CPAB_F32 or CPAB_BF16, got %d", what, dtype);
  return CPAB_OK;
}

int size_of(int dtype) { return dtype == CPAB_F32 ? 4 : 2; }

#define CPAB_TYPED(ptr, dtype) CPAB_ALIGNED(ptr, size_of(dtype))
#define CPAB_TRY(call) \
  do { const int rc_ = (call); if (rc_ != CPAB_OK) return rc_; } while (0)

// Values of one array below 2^37, rows and channels below 2^31.
constexpr int64_t kMaxValues = 1LL << 37, kMaxCount = (1LL << 31) - 1;

int check_recurrence(int dtype, int64_t B, int64_t T, int64_t C) {
  CPAB_TRY(check_dtype("dtype", dtype));
  if (B < 0 || T < 0 || C < 0)
    return fail(CPAB_ERR_INVALID, "negative size (B=%lld, T=%lld, C=%lld)", (long long)B,
                (long long)T, (long long)C);
  if (B > kMaxCount || T > kMaxCount || C > kMaxCount ||
      (double)B * (double)(T > 0 ? T : 1) * (double)C >= (double)kMaxValues ||
      (B > 0 && C > 0 && !cpab::recurrence_fits(dtype, B, T, C)))
    return fail(CPAB_ERR_INVALID, "recurrence of %lld x %lld x %lld values is too large",
                (long long)B, (long long)T, (long long)C);
  return CPAB_OK;
}

int fill_recurrence(int dtype, int64_t B, int64_t T, int64_t C, const void* x, const void* f,
                    const void* g, const int64_t* strides, const float* h0, const void* lengths,
                    int lengths64, cpab::Recurrence* r) {
  if (T > 0) {
    CPAB_REQUIRE(x); CPAB_REQUIRE(f); CPAB_REQUIRE(strides);
  }
  CPAB_TYPED(x, dtype); CPAB_TYPED(f, dtype); CPAB_TYPED(g, dtype);
  CPAB_ALIGNED(h0, 4);
  CPAB_ALIGNED(lengths, lengths64 ? 8 : 4);
  *r = cpab::Recurrence{};
  r->B = B; r->T = T; r->C = C;
  r->x = x; r->f = f; r->g = g;
  if (strides && T > 0) {
    int64_t most = 0;
    for (int k = 0; k < (g ? 6 : 4); ++k) {
      if (strides[k] < 0) return fail(CPAB_ERR_INVALID, "strides must not be negative");
      if (k % 2 == 1 && strides[k] > most) most = strides[k];
    }
    r->xb = strides[0]; r->fb = strides[2];
    if (g) r->gb = strides[4];
    if (T > 1) {
      if (most > cpab::recurrence_max_stride(dtype, B, T, C))
        return fail(CPAB_ERR_INVALID, "samples %lld values apart are too far for 32-bit offsets",
                    (long long)most);
      r->xt = strides[1]; r->ft = strides[3];
      if (g) r->gt = strides[5];
    }
  }
  r->h0 = h0;
  r->lengths = lengths;
  r->lengths64 = lengths64;
  return CPAB_OK;
}

int check_workspace(const void* workspace, int64_t have, int64_t need) {
  if (need <= 0) return CPAB_OK;
  CPAB_REQUIRE(workspace);
  CPAB_ALIGNED(workspace, 16);
  if (have < need)
    return fail(CPAB_ERR_INVALID, "workspace too small: %lld bytes, %lld needed", (long long)have,
                (long long)need);
  return CPAB_OK;
}

// Addresses, `most` at most, that are to come once each.
class Once {
 public:
  explicit Once(int64_t most) {
    while (mask_ + 1 < 2 * most) mask_ = 2 * mask_ + 1;
    if (mask_ >= kFew) many_.reset(new (std::nothrow) uintptr_t[mask_ + 1]());
  }
  bool room() const { return mask_ < kFew || many_; }
  bool add(const void* p) {   // false: it came before
    const uintptr_t key = reinterpret_cast<uintptr_t>(p);
    uintptr_t* table = many_ ? many_.get() : few_;
    int64_t at = (int64_t)(key * 0x9E3779B97F4A7C15u >> 32) & mask_;
    for (; table[at]; at = (at + 1) & mask_)
      if (table[at] == key) return false;
    table[at] = key;
    return true;
  }

 private:
  static constexpr int64_t kFew = 1024;
  int64_t mask_ = 63;
  uintptr_t few_[kFew] = {};
  std::unique_ptr<uintptr_t[]> many_;
};

int check_norm(int dtype, int residual_dtype, int weight_dtype, int64_t rows, int64_t C) {
  CPAB_TRY(check_dtype("dtype", dtype));
  CPAB_TRY(check_dtype("residual_dtype", residual_dtype));
  CPAB_TRY(check_dtype("weight_dtype", weight_dtype));
  if (dtype == CPAB_F32 && residual_dtype != CPAB_F32)
    return fail(CPAB_ERR_INVALID, "residual_dtype must be dtype or CPAB_F32");
  if (rows < 0 || C < 0)
    return fail(CPAB_ERR_INVALID, "negative size (rows=%lld, C=%lld)", (long long)rows, (long long)C);
  if (rows > kMaxCount || C > kMaxCount || (double)rows * (double)C >= (double)kMaxValues)
    return fail(CPAB_ERR_INVALID, "norm of %lld x %lld values is too large", (long long)rows,
                (long long)C);
  return CPAB_OK;
}

int norm_forward(const char* who, int dtype, int residual_dtype, int weight_dtype, int64_t rows,
                 int64_t C, const void* x, int64_t x_stride, const void* residual,
                 int64_t residual_stride, const void* weight, float eps, void* y, bool eight,
                 float* scale, void* residual_out, float* rstd, void* stream) {
  CPAB_TRY(check_norm(dtype, residual_dtype, weight_dtype, rows, C));
  if (!(eps >= 0.0f)) return fail(CPAB_ERR_INVALID, "eps must not be negative, got %g", (double)eps);
  if (rows == 0 || C == 0) return CPAB_OK;
  CPAB_REQUIRE(x); CPAB_REQUIRE(weight); CPAB_REQUIRE(y);
  if (eight) CPAB_REQUIRE(scale);
  if (residual) CPAB_REQUIRE(residual_out);
  if (!residual && residual_out)
    return fail(CPAB_ERR_INVALID, "residual_out without a residual");
  CPAB_TYPED(x, dtype); CPAB_TYPED(weight, weight_dtype);
  CPAB_TYPED(residual, residual_dtype); CPAB_TYPED(residual_out, residual_dtype);
  if (!eight) CPAB_TYPED(y, dtype);
  CPAB_ALIGNED(scale, 4); CPAB_ALIGNED(rstd, 4);
  const cpab::RmsNorm n{dtype, residual ? residual_dtype : dtype, weight_dtype, rows, C, x, x_stride,
                        residual, residual_stride, weight, eps};
  return check_hip(cpab::launch_rms_norm_forward(n, y, eight ? scale : nullptr, residual_out, rstd,
                                                 as_stream(stream)),
                   who);
}

}  // namespace

extern "C" {

int64_t cpab_recurrence_carries(int dtype, int64_t B, int64_t T, int64_t C) {
  if (check_recurrence(dtype, B, T, C) != CPAB_OK) return 0;
  return cpab::recurrence_carries(dtype, B, T, C);
}

int64_t cpab_recurrence_max_stride(int dtype, int64_t B, int64_t T, int64_t C) {
  if (check_recurrence(dtype, B, T, C) != CPAB_OK) return 0;
  return T > 1 ? cpab::recurrence_max_stride(dtype, B, T, C) : INT64_MAX;
}

int64_t cpab_recurrence_workspace_size(int dtype, int64_t B, int64_t T, int64_t C, int backward) {
  if (check_recurrence(dtype, B, T, C) != CPAB_OK) return 0;
  return cpab::recurrence_workspace(dtype, B, T, C, backward != 0);
}

int cpab_recurrence_forward(int dtype, int64_t B, int64_t T, int64_t C, const void* x,
                            const void* f, const void* g, const int64_t* strides,
                            const float* h0, const void* lengths, int lengths64, void* y,
                            float* h_last, float* carries, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  CPAB_TRY(check_recurrence(dtype, B, T, C));
  if (B == 0 || C == 0) return CPAB_OK;
  cpab::Recurrence r;
  CPAB_TRY(fill_recurrence(dtype, B, T, C, x, f, g, strides, h0, lengths, lengths64, &r));
  if (T > 0) CPAB_REQUIRE(y);
  CPAB_REQUIRE(h_last);
  CPAB_TYPED(y, dtype); CPAB_ALIGNED(h_last, 4); CPAB_ALIGNED(carries, 4);
  CPAB_TRY(check_workspace(workspace, workspace_bytes,
                           cpab::recurrence_workspace(dtype, B, T, C, false)));
  return check_hip(cpab::launch_recurrence_forward(dtype, r, y, h_last, carries, workspace,
                                                   as_stream(stream)),
                   "cpab_recurrence_forward");
}

int cpab_recurrence_backward(int dtype, int64_t B, int64_t T, int64_t C, const void* x,
                             const void* f, const void* g, const int64_t* strides,
                             const float* h0, const void* lengths, int lengths64,
                             const float* carries, const void* grad_y, const float* grad_h_last,
                             void* grad_x, void* grad_f, void* grad_g, float* grad_h0,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  CPAB_TRY(check_recurrence(dtype, B, T, C));
  if (B == 0 || C == 0) return CPAB_OK;
  cpab::Recurrence r;
  CPAB_TRY(fill_recurrence(dtype, B, T, C, x, f, g, strides, h0, lengths, lengths64, &r));
  if (T > 0) CPAB_REQUIRE(carries);
  if (grad_g && !g) return fail(CPAB_ERR_INVALID, "grad_g without g");
  CPAB_TYPED(grad_y, dtype); CPAB_TYPED(grad_x, dtype); CPAB_TYPED(grad_f, dtype);
  CPAB_TYPED(grad_g, dtype);
  CPAB_ALIGNED(carries, 4); CPAB_ALIGNED(grad_h_last, 4); CPAB_ALIGNED(grad_h0, 4);
  CPAB_TRY(check_workspace(workspace, workspace_bytes,
                           cpab::recurrence_workspace(dtype, B, T, C, true)));
  return check_hip(cpab::launch_recurrence_backward(dtype, r, carries, grad_y, grad_h_last, grad_x,
                                                    grad_f, grad_g, grad_h0, workspace,
                                                    as_stream(stream)),
                   "cpab_recurrence_backward");
}

int cpab_rms_norm_forward(int dtype, int residual_dtype, int weight_dtype, int64_t rows, int64_t C,
                          const void* x, int64_t x_stride, const void* residual,
                          int64_t residual_stride, const void* weight, float eps, void* y,
                          void* residual_out, float* rstd, void* stream) {
  return norm_forward("cpab_rms_norm_forward", dtype, residual_dtype, weight_dtype, rows, C, x,
                      x_stride, residual, residual_stride, weight, eps, y, false, nullptr,
                      residual_out, rstd, stream);
}

int cpab_rms_norm_e4m3(int dtype, int residual_dtype, int weight_dtype, int64_t rows, int64_t C,
                       const void* x, int64_t x_stride, const void* residual,
                       int64_t residual_stride, const void* weight, float eps, void* q,
                       float* scale, void* residual_out, void* stream) {
  return norm_forward("cpab_rms_norm_e4m3", dtype, residual_dtype, weight_dtype, rows, C, x, x_stride,
                      residual, residual_stride, weight, eps, q, true, scale, residual_out, nullptr,
                      stream);
}

int64_t cpab_rms_norm_backward_workspace_size(int64_t rows, int64_t C) {
  if (check_norm(CPAB_F32, CPAB_F32, CPAB_F32, rows, C) != CPAB_OK) return 0;
  return cpab::rms_norm_backward_workspace(rows, C);
}

int cpab_rms_norm_backward(int dtype, int residual_dtype, int weight_dtype, int64_t rows, int64_t C,
                           const void* r, int64_t r_stride, const void* added,
                           int64_t added_stride, const float* rstd, const void* weight,
                           const void* grad_y, int64_t grad_y_stride,
                           const void* grad_residual_out, int64_t grad_residual_stride,
                           void* grad_x, void* grad_residual, void* grad_weight, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  CPAB_TRY(check_norm(dtype, residual_dtype, weight_dtype, rows, C));
  if (C == 0) return CPAB_OK;
  if (rows > 0) {
    CPAB_REQUIRE(r); CPAB_REQUIRE(rstd); CPAB_REQUIRE(weight); CPAB_REQUIRE(grad_y);
  }
  CPAB_TYPED(r, residual_dtype); CPAB_TYPED(added, residual_dtype); CPAB_ALIGNED(rstd, 4); CPAB_TYPED(weight, weight_dtype);
  CPAB_TYPED(grad_y, dtype); CPAB_TYPED(grad_residual_out, residual_dtype);
  CPAB_TYPED(grad_x, dtype); CPAB_TYPED(grad_residual, residual_dtype);
  CPAB_TYPED(grad_weight, weight_dtype);
  CPAB_TRY(check_workspace(workspace, workspace_bytes,
                           grad_weight ? cpab::rms_norm_backward_workspace(rows, C) : 0));
  const cpab::RmsNormGrad n{dtype, residual_dtype, weight_dtype, rows, C, r, r_stride, added,
                            added_stride, rstd, weight, grad_y, grad_y_stride, grad_residual_out,
                            grad_residual_stride};
  return check_hip(cpab::launch_rms_norm_backward(n, grad_x, grad_residual, grad_weight, workspace,
                                                  as_stream(stream)),
                   "cpab_rms_norm_backward");
}

int cpab_adamw_step(int dtype, int state_bits, int64_t n_tensors, const cpab_adamw_tensor* tensors,
                    int64_t step, double lr, double beta1, double beta2, double eps,
                    double weight_decay, uint32_t seed, void* stream) {
  CPAB_TRY(check_dtype("dtype", dtype));
  if (state_bits != 32 && state_bits != 8)
    return fail(CPAB_ERR_INVALID, "state_bits must be 32 or 8, got %d", state_bits);
  if (n_tensors < 0) return fail(CPAB_ERR_INVALID, "negative number of tensors");
  if (n_tensors > kMaxCount) return fail(CPAB_ERR_INVALID, "%lld tensors are too many", (long long)n_tensors);
  if (step < 1) return fail(CPAB_ERR_INVALID, "step must be at least 1, got %lld", (long long)step);
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0))
    return fail(CPAB_ERR_INVALID, "beta1 and beta2 must be in [0, 1), got %g and %g", beta1, beta2);
  if (!(lr >= 0.0 && eps >= 0.0 && weight_decay >= 0.0))
    return fail(CPAB_ERR_INVALID, "lr, eps and weight_decay must not be negative, got %g, %g and %g",
                lr, eps, weight_decay);
  if (n_tensors > 0) CPAB_REQUIRE(tensors);
  bool any = false;
  Once once(6 * n_tensors);
  if (!once.room()) return fail(CPAB_ERR_INVALID, "no memory to look %lld tensors over", (long long)n_tensors);
  for (int64_t k = 0; k < n_tensors; ++k) {
    const cpab_adamw_tensor& t = tensors[k];
    if (t.n < 0 || t.n > cpab::kAdamWMost)
      return fail(CPAB_ERR_INVALID, "tensor %lld has %lld values", (long long)k, (long long)t.n);
    if (t.n == 0) continue;
    any = true;
    CPAB_REQUIRE(t.param); CPAB_REQUIRE(t.grad); CPAB_REQUIRE(t.exp_avg); CPAB_REQUIRE(t.exp_avg_sq);
    CPAB_TYPED(t.param, dtype); CPAB_TYPED(t.grad, dtype); CPAB_ALIGNED(t.master, 4);
    if (state_bits == 8) {
      CPAB_REQUIRE(t.exp_avg_scale); CPAB_REQUIRE(t.exp_avg_sq_scale);
    } else {
      CPAB_ALIGNED(t.exp_avg, 4); CPAB_ALIGNED(t.exp_avg_sq, 4);
    }
    // two workgroups would move it at once
    void* const master = t.master;
    for (void* p : {t.param, t.exp_avg, t.exp_avg_sq, master, state_bits == 8 ? t.exp_avg_scale : nullptr,
                    state_bits == 8 ? t.exp_avg_sq_scale : nullptr})
      if (p && !once.add(p))
        return fail(CPAB_ERR_INVALID, "an array of tensor %lld comes twice among those that the step writes",
                    (long long)k);
  }
  if (!any) return CPAB_OK;
  cpab::AdamW a;
  a.beta1 = (float)beta1;
  a.beta2 = (float)beta2;
  a.rest1 = (float)(1.0 - beta1);
  a.rest2 = (float)(1.0 - beta2);
  a.decay = (float)(1.0 - lr * weight_decay);
  a.rate = (float)(lr / (1.0 - std::pow(beta1, (double)step)));
  a.root = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step)));
  a.eps = (float)eps;
  a.cached = true;
  a.key = cpab::adamw_mix(seed ^ ((uint32_t)step * 0x9E3779B1u));
  return check_hip(cpab::launch_adamw(dtype, state_bits, n_tensors, tensors, a, as_stream(stream)),
                   "cpab_adamw_step");
}

}  // extern "C"
