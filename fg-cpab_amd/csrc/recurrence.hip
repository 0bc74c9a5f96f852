// Gated linear recurrence: a = sigmoid(f), h_t = a_t h_{t-1} + (1 - a_t) x_t,
// y = h g sigmoid(g), and its gradient.
//
// Backward: with l_t the gradient of h_t through everything after it,
//   l_t = dy_t silu(g_t) + a_{t+1} l_{t+1},   l at the row's end also + grad_h_last,
//   dx = (1 - a) l,  df = l (h_{t-1} - x) a (1 - a)  (sigmoid' = a (1 - a)),
//   dg = dy h s (1 + g (1 - s)),  s = sigmoid(g),  dh0 = a_0 l_0.
// h is computed again from the state that the forward kept before each kTile samples.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

constexpr int kTile = 16;
constexpr int kLanes = 256;

__device__ __forceinline__ int64_t row_length(const Recurrence& r, int64_t b) {
  if (!r.lengths) return r.T;
  const int64_t n = r.lengths64 ? static_cast<const int64_t*>(r.lengths)[b]
                                : (int64_t)static_cast<const int32_t*>(r.lengths)[b];
  return n < 0 ? 0 : (n > r.T ? r.T : n);
}

template <typename T>
__global__ void __launch_bounds__(kLanes)
recurrence_forward_kernel(Recurrence r, T* y, float* h_last, float* carries) {
  const int64_t i = blockIdx.x * (int64_t)kLanes + threadIdx.x;
  if (i >= r.B * r.C) return;
  const int64_t b = i / r.C, c = i - b * r.C;
  const int64_t n = row_length(r, b), tiles = (r.T + kTile - 1) / kTile;
  const T* x = static_cast<const T*>(r.x) + b * r.xb + c;
  const T* f = static_cast<const T*>(r.f) + b * r.fb + c;
  const T* g = r.g ? static_cast<const T*>(r.g) + b * r.gb + c : nullptr;
  y += b * r.T * r.C + c;
  float h = r.h0 ? r.h0[i] : 0.0f;
  for (int64_t t = 0; t < n; ++t) {
    if (carries && t % kTile == 0) carries[(b * tiles + t / kTile) * r.C + c] = h;
    const Gate a = sigmoids(to_float(f[t * r.ft]));
    h = fmaf(a.pos, h, a.neg * to_float(x[t * r.xt]));
    float out = h;
    if (g) {
      const float gv = to_float(g[t * r.gt]);
      out *= gv * sigmoids(gv).pos;
    }
    y[t * r.C] = from_float<T>(out);
  }
  for (int64_t t = n; t < r.T; ++t) y[t * r.C] = from_float<T>(0.0f);
  h_last[i] = h;
}

template <typename T>
__global__ void __launch_bounds__(kLanes)
recurrence_backward_kernel(Recurrence r, const float* carries, const T* dy, const float* dh_last,
                           T* dx, T* df, T* dg, float* dh0) {
  const int64_t i = blockIdx.x * (int64_t)kLanes + threadIdx.x;
  if (i >= r.B * r.C) return;
  const int64_t b = i / r.C, c = i - b * r.C;
  const int64_t n = row_length(r, b), tiles = (r.T + kTile - 1) / kTile;
  const T* x = static_cast<const T*>(r.x) + b * r.xb + c;
  const T* f = static_cast<const T*>(r.f) + b * r.fb + c;
  const T* g = r.g ? static_cast<const T*>(r.g) + b * r.gb + c : nullptr;
  const int64_t row = b * r.T * r.C + c;
  for (int64_t t = n; t < r.T; ++t) {
    const int64_t at = row + t * r.C;
    if (dx) dx[at] = from_float<T>(0.0f);
    if (df) df[at] = from_float<T>(0.0f);
    if (dg) dg[at] = from_float<T>(0.0f);
  }
  float l = dh_last ? dh_last[i] : 0.0f;   // a_{t+1} l_{t+1}
  for (int64_t k = (n + kTile - 1) / kTile - 1; k >= 0; --k) {
    float h[kTile + 1];
    h[0] = carries[(b * tiles + k) * r.C + c];
#pragma unroll
    for (int j = 0; j < kTile; ++j) {
      const int64_t t = k * kTile + j;
      h[j + 1] = h[j];
      if (t >= n) continue;
      const Gate a = sigmoids(to_float(f[t * r.ft]));
      h[j + 1] = fmaf(a.pos, h[j], a.neg * to_float(x[t * r.xt]));
    }
#pragma unroll
    for (int j = kTile - 1; j >= 0; --j) {
      const int64_t t = k * kTile + j;
      if (t >= n) continue;
      const int64_t at = row + t * r.C;
      float d = dy ? to_float(dy[at]) : 0.0f;
      if (g) {
        const float gv = to_float(g[t * r.gt]);
        const Gate s = sigmoids(gv);
        if (dg) dg[at] = from_float<T>(d * h[j + 1] * s.pos * fmaf(gv, s.neg, 1.0f));
        d *= gv * s.pos;
      }
      l += d;
      const Gate a = sigmoids(to_float(f[t * r.ft]));
      if (dx) dx[at] = from_float<T>(a.neg * l);
      if (df) df[at] = from_float<T>(l * (h[j] - to_float(x[t * r.xt])) * (a.pos * a.neg));
      l *= a.pos;
    }
  }
  if (dh0) dh0[i] = l;
}

unsigned blocks_for(const Recurrence& r) { return (unsigned)((r.B * r.C + kLanes - 1) / kLanes); }

}  // namespace

int64_t recurrence_carries(int, int64_t B, int64_t T, int64_t C) {
  return B * ((T + kTile - 1) / kTile) * C;
}
int64_t recurrence_workspace(int, int64_t, int64_t, int64_t, bool) { return 0; }

hipError_t launch_recurrence_forward(int dtype, const Recurrence& r, void* y, float* h_last,
                                     float* carries, void*, hipStream_t s) {
  if (dtype == CPAB_F32)
    recurrence_forward_kernel<float><<<blocks_for(r), kLanes, 0, s>>>(r, (float*)y, h_last, carries);
  else
    recurrence_forward_kernel<bf16><<<blocks_for(r), kLanes, 0, s>>>(r, (bf16*)y, h_last, carries);
  return hipGetLastError();
}

hipError_t launch_recurrence_backward(int dtype, const Recurrence& r, const float* carries,
                                      const void* dy, const float* dh_last, void* dx, void* df,
                                      void* dg, float* dh0, void*, hipStream_t s) {
  if (dtype == CPAB_F32)
    recurrence_backward_kernel<float><<<blocks_for(r), kLanes, 0, s>>>(
        r, carries, (const float*)dy, dh_last, (float*)dx, (float*)df, (float*)dg, dh0);
  else
    recurrence_backward_kernel<bf16><<<blocks_for(r), kLanes, 0, s>>>(
        r, carries, (const bf16*)dy, dh_last, (bf16*)dx, (bf16*)df, (bf16*)dg, dh0);
  return hipGetLastError();
}

}  // namespace cpab
