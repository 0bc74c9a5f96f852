// Launch interface of the operators around the transform (recurrence.hip,
// rms_norm.hip, adamw.hip).  Arguments are validated by the caller
// (capi_sequence.cpp); a launcher only enqueues work on `s`.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cpab_hip.h"

namespace cpab {

int compute_units();   // of the current device (capi.cpp)

// Sizes and inputs of a gated recurrence; strides in elements.
struct Recurrence {
  int64_t B, T, C;
  const void *x, *f, *g;
  int64_t xb, xt, fb, ft, gb, gt;
  const float* h0;
  const void* lengths;
  int lengths64;
};
// The most values from an input's sample to the next that a tile's samples are reached over
// with offsets of 31 bits.
int64_t recurrence_max_stride(int dtype, int64_t B, int64_t T, int64_t C);
// Whether that holds for the outputs, and the launches' lanes can be counted in 32 bits, as
// a grid's are.
bool recurrence_fits(int dtype, int64_t B, int64_t T, int64_t C);
int64_t recurrence_carries(int dtype, int64_t B, int64_t T, int64_t C);
int64_t recurrence_workspace(int dtype, int64_t B, int64_t T, int64_t C, bool backward);
hipError_t launch_recurrence_forward(int dtype, const Recurrence& r, void* y, float* h_last,
                                     float* carries, void* workspace, hipStream_t s);
hipError_t launch_recurrence_backward(int dtype, const Recurrence& r, const float* carries,
                                      const void* grad_y, const float* grad_h_last, void* grad_x,
                                      void* grad_f, void* grad_g, float* grad_h0, void* workspace,
                                      hipStream_t s);

struct RmsNorm {
  int dtype, residual_dtype, weight_dtype;
  int64_t rows, C;
  const void* x;
  int64_t x_stride;
  const void* residual;
  int64_t residual_stride;
  const void* weight;
  float eps;
};
// scale: the row scales of an 8-bit y (NULL: y of n.dtype).
hipError_t launch_rms_norm_forward(const RmsNorm& n, void* y, float* scale, void* residual_out,
                                   float* rstd, hipStream_t s);
struct RmsNormGrad {
  int dtype, residual_dtype, weight_dtype;
  int64_t rows, C;
  const void* r;
  int64_t r_stride;
  const void* added;   // to r, in 32 bits; may be NULL
  int64_t added_stride;
  const float* rstd;
  const void* weight;
  const void* grad_y;
  int64_t grad_y_stride;
  const void* grad_out;   // of the residual; may be NULL
  int64_t grad_out_stride;
};
int64_t rms_norm_backward_workspace(int64_t rows, int64_t C);
hipError_t launch_rms_norm_backward(const RmsNormGrad& n, void* grad_x, void* grad_residual,
                                    void* grad_weight, void* workspace, hipStream_t s);

struct AdamW {
  float beta1, beta2, rest1, rest2;   // rest: 1 - beta
  float decay;                        // 1 - lr weight_decay
  float rate;                         // lr / (1 - beta1^step)
  float root;                         // 1 / sqrt(1 - beta2^step)
  float eps;
  uint32_t key;                       // mix(seed xor step * 0x9E3779B1)
  bool cached;                        // the parameters are stored through the caches
};
constexpr int64_t kAdamWMost = (1LL << 34) - 1024;   // values of one tensor
hipError_t launch_adamw(int dtype, int state_bits, int64_t n_tensors,
                        const cpab_adamw_tensor* tensors, const AdamW& a, hipStream_t s);
uint32_t adamw_mix(uint32_t z);

}  // namespace cpab
