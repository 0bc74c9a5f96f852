// The operators over heads at the extern "C" boundary: argument checks before any HIP
// call, then the launch.
#include <hip/hip_runtime.h>

#include <cmath>

#include "capi_common.hpp"
#include "heads_launch.hpp"

namespace {

using cpab::check_hip;
using cpab::fail;

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

#define CPAB_TRY(call) \
  do { const int rc_ = (call); if (rc_ != CPAB_OK) return rc_; } while (0)

constexpr int64_t kMaxValues = 1LL << 37, kMaxCount = (1LL << 31) - 1, kMaxHeads = 65535;

int size_of(int dtype) { return dtype == CPAB_F32 ? 4 : 2; }

int check_dtype(const char* what, int dtype) {
  if (dtype != CPAB_F32 && dtype != CPAB_BF16)
    return fail(CPAB_ERR_INVALID, "%s must be CPAB_F32 or CPAB_BF16, got %d", what, dtype);
  return CPAB_OK;
}

int check_strides(const char* what, const int64_t* strides, int count) {
  for (int k = 0; k < count; ++k)
    if (strides[k] < 0) return fail(CPAB_ERR_INVALID, "strides of %s must not be negative", what);
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

int check_qk_sizes(const cpab_qk_norm* norm) {
  CPAB_REQUIRE(norm);
  const cpab_qk_norm& n = *norm;
  CPAB_TRY(check_dtype("dtype", n.dtype));
  CPAB_TRY(check_dtype("weight_dtype", n.weight_dtype));
  if (n.B < 0 || n.T < 0 || n.heads < 0 || n.key_heads < 0 || n.width < 0)
    return fail(CPAB_ERR_INVALID, "negative size (B=%lld, T=%lld, heads=%lld, key_heads=%lld, width=%lld)",
                (long long)n.B, (long long)n.T, (long long)n.heads, (long long)n.key_heads,
                (long long)n.width);
  if (n.width < 1 || n.width > cpab::kQkMostWidth)
    return fail(CPAB_ERR_INVALID, "width must be from 1 to %d, got %lld", cpab::kQkMostWidth,
                (long long)n.width);
  if (n.turned < 0 || n.turned > n.width || n.turned % 2 != 0)
    return fail(CPAB_ERR_INVALID, "turned must be even and at most width, got %lld", (long long)n.turned);
  if (n.heads > kMaxHeads || n.key_heads > kMaxHeads || n.B > kMaxCount || n.T > kMaxCount ||
      (double)n.B * (double)n.T > (double)kMaxCount ||
      (double)n.B * (double)n.T * (double)(n.heads + n.key_heads) * (double)n.width >= (double)kMaxValues)
    return fail(CPAB_ERR_INVALID, "norms of %lld x %lld x (%lld + %lld) x %lld values are too large",
                (long long)n.B, (long long)n.T, (long long)n.heads, (long long)n.key_heads,
                (long long)n.width);
  return CPAB_OK;
}

int check_qk(const cpab_qk_norm* norm) {
  CPAB_TRY(check_qk_sizes(norm));
  const cpab_qk_norm& n = *norm;
  if (!(n.eps >= 0.0f)) return fail(CPAB_ERR_INVALID, "eps must not be negative, got %g", (double)n.eps);
  const bool any = n.B > 0 && n.T > 0;
  if (any && n.heads > 0) { CPAB_REQUIRE(n.q); CPAB_REQUIRE(n.q_weight); }
  if (any && n.key_heads > 0) { CPAB_REQUIRE(n.k); CPAB_REQUIRE(n.k_weight); }
  if (any && n.turned > 0) CPAB_REQUIRE(n.freqs);
  CPAB_ALIGNED(n.q, size_of(n.dtype)); CPAB_ALIGNED(n.k, size_of(n.dtype));
  CPAB_ALIGNED(n.q_weight, size_of(n.weight_dtype)); CPAB_ALIGNED(n.k_weight, size_of(n.weight_dtype));
  CPAB_ALIGNED(n.freqs, 4);
  if (n.position_type < CPAB_POSITION_I32 || n.position_type > CPAB_POSITION_F32)
    return fail(CPAB_ERR_INVALID, "position_type must be one of CPAB_POSITION_*, got %d", n.position_type);
  CPAB_ALIGNED(n.positions, n.position_type == CPAB_POSITION_I64 ? 8 : 4);
  CPAB_TRY(check_strides("q", n.q_strides, 3));
  CPAB_TRY(check_strides("k", n.k_strides, 3));
  return check_strides("positions", n.position_strides, 2);
}

int check_delta_sizes(const cpab_delta_rule* rule) {
  CPAB_REQUIRE(rule);
  const cpab_delta_rule& r = *rule;
  CPAB_TRY(check_dtype("dtype", r.dtype));
  CPAB_TRY(check_dtype("gate_dtype", r.gate_dtype));
  if (r.B < 0 || r.T < 0 || r.heads < 0 || r.key_heads < 0 || r.dk < 0 || r.dv < 0)
    return fail(CPAB_ERR_INVALID, "negative size (B=%lld, T=%lld, heads=%lld, key_heads=%lld, dk=%lld, dv=%lld)",
                (long long)r.B, (long long)r.T, (long long)r.heads, (long long)r.key_heads,
                (long long)r.dk, (long long)r.dv);
  if (r.dk < 1 || r.dk > CPAB_DELTA_MOST_KEY)
    return fail(CPAB_ERR_INVALID, "dk must be from 1 to %d, got %lld", CPAB_DELTA_MOST_KEY, (long long)r.dk);
  if (r.dv < 1) return fail(CPAB_ERR_INVALID, "dv must be at least 1, got %lld", (long long)r.dv);
  if (r.heads > 0 && (r.key_heads < 1 || r.heads % r.key_heads != 0))
    return fail(CPAB_ERR_INVALID, "heads must be a multiple of key_heads, got %lld and %lld",
                (long long)r.heads, (long long)r.key_heads);
  // a launch's workgroups: a chunk, up to 1024 lanes, or 32 columns of a head, 256; the lanes
  // are counted in 32 bits
  const double heads = (double)r.B * (double)r.heads, blocks = (double)kMaxCount / 256,
               chunks = (double)(kMaxCount / 512);
  if (r.heads * (r.dv + 8) > CPAB_DELTA_MOST_STRIDE || r.key_heads * (r.dk + 8) > CPAB_DELTA_MOST_STRIDE ||
      r.heads > kMaxHeads || r.B > kMaxCount || r.T > kMaxCount - 64 || r.dv > kMaxCount / 64 ||
      heads * ((double)r.T / 64 + 1) > chunks || heads * ((double)r.dv / 32 + 1) > blocks ||
      heads * (double)(r.T + 64) * (double)(r.dv + r.dk) >= (double)kMaxValues ||
      (double)r.B * (double)r.key_heads * (double)r.T * (double)r.dk >= (double)kMaxValues ||   // also without heads
      heads * ((double)r.T / 64 + 2) * (double)r.dk * (double)r.dv >= (double)kMaxValues)
    return fail(CPAB_ERR_INVALID, "delta rule of %lld x %lld x %lld heads of %lld x %lld is too large",
                (long long)r.B, (long long)r.T, (long long)r.heads, (long long)r.dk, (long long)r.dv);
  return CPAB_OK;
}

// Whether there is anything to do.
bool any_delta(const cpab_delta_rule& r) { return r.B > 0 && r.heads > 0; }

int check_delta(const cpab_delta_rule* rule) {
  CPAB_TRY(check_delta_sizes(rule));
  const cpab_delta_rule& r = *rule;
  if (!std::isfinite(r.scale)) return fail(CPAB_ERR_INVALID, "scale must be finite");
  if (any_delta(r) && r.T > 0) {
    CPAB_REQUIRE(r.q); CPAB_REQUIRE(r.k);
    CPAB_REQUIRE(r.v);
    CPAB_REQUIRE(r.decay); CPAB_REQUIRE(r.beta);
  }
  CPAB_ALIGNED(r.q, size_of(r.dtype)); CPAB_ALIGNED(r.k, size_of(r.dtype)); CPAB_ALIGNED(r.v, size_of(r.dtype));
  CPAB_ALIGNED(r.decay, size_of(r.gate_dtype)); CPAB_ALIGNED(r.beta, size_of(r.gate_dtype));
  CPAB_ALIGNED(r.h0, 4); CPAB_ALIGNED(r.lengths, r.lengths64 ? 8 : 4);
  CPAB_TRY(check_strides("q", r.q_strides, 3));
  CPAB_TRY(check_strides("k", r.k_strides, 3));
  CPAB_TRY(check_strides("v", r.v_strides, 3));
  // a chunk's offsets have 32 bits
  if (r.T > 1)
    for (const int64_t* strides : {r.q_strides, r.k_strides, r.v_strides})
      if (strides[1] > CPAB_DELTA_MOST_STRIDE)
        return fail(CPAB_ERR_INVALID, "samples %lld values apart are too far, at most %d", (long long)strides[1],
                    CPAB_DELTA_MOST_STRIDE);
  CPAB_TRY(check_strides("decay", r.decay_strides, 3));
  return check_strides("beta", r.beta_strides, 3);
}

}  // namespace

extern "C" {

int cpab_qk_norm_forward(const cpab_qk_norm* norm, void* q_out, void* k_out, void* stream) {
  CPAB_TRY(check_qk(norm));
  if (norm->B == 0 || norm->T == 0) return CPAB_OK;
  if (norm->heads > 0) CPAB_REQUIRE(q_out);
  if (norm->key_heads > 0) CPAB_REQUIRE(k_out);
  CPAB_ALIGNED(q_out, size_of(norm->dtype)); CPAB_ALIGNED(k_out, size_of(norm->dtype));
  return check_hip(cpab::launch_qk_norm_forward(*norm, q_out, k_out, as_stream(stream)),
                   "cpab_qk_norm_forward");
}

int64_t cpab_qk_norm_backward_workspace_size(const cpab_qk_norm* norm) {
  if (check_qk_sizes(norm) != CPAB_OK) return 0;
  return cpab::qk_norm_backward_workspace(*norm);
}

int cpab_qk_norm_backward(const cpab_qk_norm* norm, const void* const* grads,
                          const int64_t* grad_strides, void* const* outs, void* const* weight_outs,
                          void* workspace, int64_t workspace_bytes, void* stream) {
  CPAB_TRY(check_qk(norm));
  CPAB_REQUIRE(grads); CPAB_REQUIRE(grad_strides); CPAB_REQUIRE(outs); CPAB_REQUIRE(weight_outs);
  const bool any = norm->B > 0 && norm->T > 0;
  if (any && norm->heads > 0) CPAB_REQUIRE(grads[0]);
  if (any && norm->key_heads > 0) CPAB_REQUIRE(grads[1]);
  for (int k = 0; k < 2; ++k) {
    CPAB_ALIGNED(grads[k], size_of(norm->dtype)); CPAB_ALIGNED(outs[k], size_of(norm->dtype));
    CPAB_ALIGNED(weight_outs[k], size_of(norm->weight_dtype));
  }
  CPAB_TRY(check_strides("the gradients", grad_strides, 6));
  CPAB_TRY(check_workspace(workspace, workspace_bytes, cpab::qk_norm_backward_workspace(*norm)));
  return check_hip(cpab::launch_qk_norm_backward(*norm, grads, grad_strides, outs, weight_outs,
                                                 workspace, as_stream(stream)),
                   "cpab_qk_norm_backward");
}

int64_t cpab_delta_rule_kept(const cpab_delta_rule* rule) {
  if (check_delta_sizes(rule) != CPAB_OK || !any_delta(*rule)) return 0;
  return cpab::delta_rule_kept(*rule);
}

int64_t cpab_delta_rule_workspace_size(const cpab_delta_rule* rule, int keep, int backward) {
  if (check_delta_sizes(rule) != CPAB_OK || !any_delta(*rule)) return 0;
  return cpab::delta_rule_workspace(*rule, keep != 0, backward != 0);
}

int cpab_delta_rule_forward(const cpab_delta_rule* rule, void* o, float* h, float* kept,
                            void* workspace, int64_t workspace_bytes, void* stream) {
  CPAB_TRY(check_delta(rule));
  const cpab_delta_rule& r = *rule;
  if (!any_delta(r)) return CPAB_OK;
  if (r.T > 0) CPAB_REQUIRE(o);
  CPAB_REQUIRE(h);
  CPAB_ALIGNED(o, size_of(r.dtype)); CPAB_ALIGNED(h, 4); CPAB_ALIGNED(kept, 4);
  CPAB_TRY(check_workspace(workspace, workspace_bytes, cpab::delta_rule_workspace(r, kept != nullptr, false)));
  return check_hip(cpab::launch_delta_rule_forward(r, o, h, kept, workspace, as_stream(stream)),
                   "cpab_delta_rule_forward");
}

int cpab_delta_rule_backward(const cpab_delta_rule* rule, const float* kept, const void* grad_o,
                             const float* grad_h, void* grad_q, void* grad_k, void* grad_v,
                             void* grad_decay, void* grad_beta, float* grad_h0, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  CPAB_TRY(check_delta(rule));
  const cpab_delta_rule& r = *rule;
  CPAB_ALIGNED(grad_q, size_of(r.dtype)); CPAB_ALIGNED(grad_k, size_of(r.dtype));
  if (!any_delta(r))   // queries and keys may be there all the same
    return check_hip(cpab::launch_delta_rule_unread(r, grad_q, grad_k, as_stream(stream)), "cpab_delta_rule_backward");
  if (r.T > 0) CPAB_REQUIRE(kept);
  CPAB_ALIGNED(kept, 4); CPAB_ALIGNED(grad_h, 4); CPAB_ALIGNED(grad_h0, 4);
  CPAB_ALIGNED(grad_o, size_of(r.dtype)); CPAB_ALIGNED(grad_v, size_of(r.dtype));
  CPAB_ALIGNED(grad_decay, size_of(r.gate_dtype)); CPAB_ALIGNED(grad_beta, size_of(r.gate_dtype));
  CPAB_TRY(check_workspace(workspace, workspace_bytes, cpab::delta_rule_workspace(r, true, true)));
  return check_hip(cpab::launch_delta_rule_backward(r, kept, grad_o, grad_h, grad_q, grad_k, grad_v,
                                                    grad_decay, grad_beta, grad_h0, workspace,
                                                    as_stream(stream)),
                   "cpab_delta_rule_backward");
}

}  // extern "C"
