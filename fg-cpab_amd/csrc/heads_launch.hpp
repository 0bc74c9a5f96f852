// Launch interface of the operators over heads (qk_norm.hip, delta_rule.hip,
// delta_rule_backward.hip).  Arguments are validated by the caller (capi_heads.cpp); a
// launcher only enqueues work on `s`.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cpab_hip.h"

namespace cpab {

int compute_units();   // of the current device (capi.cpp)

constexpr int kQkMostWidth = 512;
hipError_t launch_qk_norm_forward(const cpab_qk_norm& n, void* q_out, void* k_out, hipStream_t s);
int64_t qk_norm_backward_workspace(const cpab_qk_norm& n);
hipError_t launch_qk_norm_backward(const cpab_qk_norm& n, const void* const grads[2],
                                   const int64_t grad_strides[6], void* const outs[2],
                                   void* const weight_outs[2], void* workspace, hipStream_t s);


// Floats that a forward keeps for its backward; bytes of workspace.
int64_t delta_rule_kept(const cpab_delta_rule& r);
int64_t delta_rule_workspace(const cpab_delta_rule& r, bool keep, bool backward);
hipError_t launch_delta_rule_forward(const cpab_delta_rule& r, void* o, float* h, float* kept,
                                     void* workspace, hipStream_t s);
hipError_t launch_delta_rule_backward(const cpab_delta_rule& r, const float* kept, const void* grad_o,
                                      const float* grad_h, void* grad_q, void* grad_k, void* grad_v,
                                      void* grad_decay, void* grad_beta, float* grad_h0,
                                      void* workspace, hipStream_t s);
// The gradients of queries and keys that no head of values reads.
hipError_t launch_delta_rule_unread(const cpab_delta_rule& r, void* grad_q, void* grad_k, hipStream_t s);

}  // namespace cpab
