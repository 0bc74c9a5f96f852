// Root-mean-square norm with the residual's addition, to the input's type or to
// 8 bits with a scale per row, and its gradient.
//
// s = 1 / sqrt(mean(r^2) + eps), y = r s w.  Backward, with u = w dy:
//   dr = s (u - r s^2 mean(u r)) + dr_out,  dw = sum over rows of dy r s.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

constexpr int kLanes = 256;

struct Sum {
  __device__ float operator()(float a, float b) const { return a + b; }
};
struct Max {   // a NaN stays
  __device__ float operator()(float a, float b) const { return a != a || a > b ? a : b; }
};

// The same value in every lane of the workgroup; `room` holds a float per wave.
template <typename Op>
__device__ float over_workgroup(float v, float* room, Op op) {
  for (int d = 1; d < 64; d *= 2) v = op(v, __shfl_xor(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
  __syncthreads();
  v = room[0];
  for (int w = 1; w < (int)blockDim.x >> 6; ++w) v = op(v, room[w]);
  return v;
}

__device__ __forceinline__ uint8_t to_e4m3(float v) {   // |v| <= 448 or NaN
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

template <typename T, typename R, typename W>
__global__ void __launch_bounds__(kLanes)
rms_norm_forward_kernel(RmsNorm n, T* y, uint8_t* q, float* scale, R* residual_out, float* rstd) {
  __shared__ float room[kLanes / 64];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(n.x) + row * n.x_stride;
  const R* res = n.residual ? static_cast<const R*>(n.residual) + row * n.residual_stride : nullptr;
  const W* w = static_cast<const W*>(n.weight);
  const auto value = [&](int64_t c) { return to_float(x[c]) + (res ? to_float(res[c]) : 0.0f); };
  float sum = 0.0f;
  for (int64_t c = threadIdx.x; c < n.C; c += kLanes) {
    const float r = value(c);
    sum = fmaf(r, r, sum);
  }
  sum = over_workgroup(sum, room, Sum());
  const float s = 1.0f / sqrtf(sum / (float)n.C + n.eps);
  if (rstd && threadIdx.x == 0) rstd[row] = s;
  float inv = 0.0f;
  if (q) {
    float top = 0.0f;
    for (int64_t c = threadIdx.x; c < n.C; c += kLanes)
      top = Max()(fabsf(value(c) * s * to_float(w[c])), top);
    top = over_workgroup(top, room, Max());
    const float sc = top == 0.0f ? 1.0f : top / 448.0f;
    if (threadIdx.x == 0) scale[row] = sc;
    inv = 1.0f / sc;
  }
  for (int64_t c = threadIdx.x; c < n.C; c += kLanes) {
    const float r = value(c), v = r * s * to_float(w[c]);
    if (q) {
      const float z = v * inv;
      q[row * n.C + c] = to_e4m3(fabsf(z) > 448.0f ? copysignf(448.0f, z) : z);
    } else {
      y[row * n.C + c] = from_float<T>(v);
    }
    if (residual_out) residual_out[row * n.C + c] = from_float<R>(r);
  }
}

template <typename T, typename R, typename W>
__global__ void __launch_bounds__(kLanes)
rms_norm_backward_kernel(RmsNormGrad n, T* dx, R* dres) {
  __shared__ float room[kLanes / 64];
  const int64_t row = blockIdx.x;
  const R* r = static_cast<const R*>(n.r) + row * n.r_stride;
  const T* dy = static_cast<const T*>(n.grad_y) + row * n.grad_y_stride;
  const R* dout = n.grad_out ? static_cast<const R*>(n.grad_out) + row * n.grad_out_stride : nullptr;
  const W* w = static_cast<const W*>(n.weight);
  const float s = n.rstd[row];
  float sum = 0.0f;
  for (int64_t c = threadIdx.x; c < n.C; c += kLanes)
    sum = fmaf(to_float(dy[c]) * to_float(w[c]), to_float(r[c]) * s, sum);
  const float mean = over_workgroup(sum, room, Sum()) / (float)n.C;
  for (int64_t c = threadIdx.x; c < n.C; c += kLanes) {
    const float u = to_float(dy[c]) * to_float(w[c]);
    const float d = s * (u - to_float(r[c]) * s * mean) + (dout ? to_float(dout[c]) : 0.0f);
    if (dx) dx[row * n.C + c] = from_float<T>(d);
    if (dres) dres[row * n.C + c] = from_float<R>(d);
  }
}

// grad_weight, a lane per channel.
template <typename T, typename R, typename W>
__global__ void __launch_bounds__(kLanes) rms_norm_weight_kernel(RmsNormGrad n, W* dw) {
  const int64_t c = blockIdx.x * (int64_t)kLanes + threadIdx.x;
  if (c >= n.C) return;
  const R* r = static_cast<const R*>(n.r) + c;
  const T* dy = static_cast<const T*>(n.grad_y) + c;
  float sum = 0.0f;
  for (int64_t row = 0; row < n.rows; ++row)
    sum = fmaf(to_float(dy[row * n.grad_y_stride]), to_float(r[row * n.r_stride]) * n.rstd[row], sum);
  dw[c] = from_float<W>(sum);
}

// f(T(), R(), W()) for the arrays' types.
template <typename F>
void with_types(int dtype, int residual, int weight, F f) {
  if (dtype == CPAB_F32) return weight == CPAB_F32 ? f(0.0f, 0.0f, 0.0f) : f(0.0f, 0.0f, bf16());
  if (residual == CPAB_F32)
    return weight == CPAB_F32 ? f(bf16(), 0.0f, 0.0f) : f(bf16(), 0.0f, bf16());
  return weight == CPAB_F32 ? f(bf16(), bf16(), 0.0f) : f(bf16(), bf16(), bf16());
}

}  // namespace

hipError_t launch_rms_norm_forward(const RmsNorm& n, void* y, float* scale, void* residual_out,
                                   float* rstd, hipStream_t st) {
  with_types(n.dtype, n.residual_dtype, n.weight_dtype, [&](auto t, auto r, auto w) {
    typedef decltype(t) T;
    typedef decltype(r) R;
    typedef decltype(w) W;
    rms_norm_forward_kernel<T, R, W><<<(unsigned)n.rows, kLanes, 0, st>>>(
        n, scale ? nullptr : (T*)y, scale ? (uint8_t*)y : nullptr, scale, (R*)residual_out, rstd);
  });
  return hipGetLastError();
}

int64_t rms_norm_backward_workspace(int64_t, int64_t) { return 0; }

hipError_t launch_rms_norm_backward(const RmsNormGrad& n, void* grad_x, void* grad_residual,
                                    void* grad_weight, void*, hipStream_t st) {
  with_types(n.dtype, n.residual_dtype, n.weight_dtype, [&](auto t, auto r, auto w) {
    typedef decltype(t) T;
    typedef decltype(r) R;
    typedef decltype(w) W;
    if (grad_x || grad_residual)
      rms_norm_backward_kernel<T, R, W><<<(unsigned)n.rows, kLanes, 0, st>>>(n, (T*)grad_x,
                                                                            (R*)grad_residual);
    if (grad_weight)
      rms_norm_weight_kernel<T, R, W><<<(unsigned)((n.C + kLanes - 1) / kLanes), kLanes, 0, st>>>(
          n, (W*)grad_weight);
  });
  return hipGetLastError();
}

}  // namespace cpab
