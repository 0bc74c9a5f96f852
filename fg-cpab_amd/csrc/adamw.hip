// One AdamW step over many tensors, states in 32 bits or in 8.
//
// m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
// p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps).
//
// 8-bit states are E4M3 values (3 bits of mantissa, 2^-9 to 448) with one
// power-of-two scale to each 32, so that neither scaling rounds; the second moment
// is kept as its square root, which halves the range that its exponent has to
// cover.  A step changes v by a thousandth: to nearest it would never change, so
// both states are rounded up or down at random in proportion, from a hash of the
// step's seed and the value's place: the same call gives the same states.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

constexpr int kLanes = 256;
constexpr int kGroup = 32;   // values that share a scale

// Scrambles 32 bits: xorshifts and odd multipliers, the leading digits of the golden
// section and of the square root of two.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t z) {
  z ^= z >> 16;
  z *= 0x9E3779B1u;
  z ^= z >> 15;
  z *= 0xB504F333u;
  return z ^ (z >> 16);
}

// The least k from -127 with top <= 448 * 2^k, for finite top >= 0: 448 is 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(k, -127);
}
__device__ __forceinline__ float power_of_two(int k) {   // k in [-127, 127]
  return __uint_as_float(k > -127 ? (uint32_t)(k + 127) << 23 : 1u << 22);
}

// a in [0, 448], rounded to an E4M3 value: up with the probability of what lies
// between it and the value below, against the 16 random bits r.  Normal values keep
// the float's upper 3 mantissa bits; below the least of them, 2^-6, the spacing is
// even, as it is from 2^-6 to 2^-5, where those are moved.
__device__ __forceinline__ float round_at_random(float a, uint32_t r) {
  const bool small = a < 0.015625f;
  if (small) a += 0.015625f;
  a = __uint_as_float((__float_as_uint(a) + (r << 4)) & ~0xfffffu);
  return small ? a - 0.015625f : a;
}

__device__ __forceinline__ float from_e4m3(uint8_t v) {
  return __builtin_amdgcn_cvt_f32_fp8((int)v, 0);
}
// z an E4M3 value, or NaN.
__device__ __forceinline__ uint8_t to_e4m3(float z) {
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(z, z, 0, false) & 0xff);
}

// The weight after a step, from the new moments and the root of the second.
__device__ __forceinline__ float moved(const AdamW& a, float w, float m, float root) {
  return w * a.decay - a.rate * m / (root * a.root + a.eps);
}

// A lane per value; 32 lanes share a scale.
template <typename T, bool EIGHT>
__global__ void __launch_bounds__(kLanes)
adamw_kernel(cpab_adamw_tensor t, AdamW a, uint32_t key) {
  const int64_t i = blockIdx.x * (int64_t)kLanes + threadIdx.x;
  const bool in = i < t.n;
  T* p = static_cast<T*>(t.param);
  float g = 0.0f, m = 0.0f, v = 0.0f, w = 0.0f;
  if (in) {
    g = to_float(static_cast<const T*>(t.grad)[i]);
    w = t.master ? t.master[i] : to_float(p[i]);
    if (EIGHT) {
      m = from_e4m3(static_cast<const uint8_t*>(t.exp_avg)[i]) *
          power_of_two((int)static_cast<const uint8_t*>(t.exp_avg_scale)[i / kGroup] - 127);
      v = from_e4m3(static_cast<const uint8_t*>(t.exp_avg_sq)[i]) *
          power_of_two((int)static_cast<const uint8_t*>(t.exp_avg_sq_scale)[i / kGroup] - 127);
      v *= v;
    } else {
      m = static_cast<const float*>(t.exp_avg)[i];
      v = static_cast<const float*>(t.exp_avg_sq)[i];
    }
  }
  m = a.beta1 * m + a.rest1 * g;
  v = a.beta2 * v + a.rest2 * g * g;
  const float root = sqrtf(v);
  if (in) {
    w = moved(a, w, m, root);
    p[i] = from_float<T>(w);
    if (t.master) t.master[i] = w;
  }
  if (!EIGHT) {
    if (in) {
      static_cast<float*>(t.exp_avg)[i] = m;
      static_cast<float*>(t.exp_avg_sq)[i] = v;
    }
    return;
  }
  const bool fine_m = fabsf(m) < INFINITY, fine_v = root < INFINITY;
  float top_m = fine_m ? fabsf(m) : 0.0f, top_v = fine_v ? root : 0.0f;
  for (int d = 1; d < kGroup; d *= 2) {
    top_m = fmaxf(top_m, __shfl_xor(top_m, d));
    top_v = fmaxf(top_v, __shfl_xor(top_v, d));
  }
  if (!in) return;
  const int km = scale_exponent(top_m), kv = scale_exponent(top_v);
  const uint32_t bits = mix((uint32_t)i + key);
  const float am = round_at_random(fabsf(m) * power_of_two(-km), bits & 0xffffu);
  float av = round_at_random(root * power_of_two(-kv), bits >> 16);
  if (root > 0.0f) av = fmaxf(av, 0.001953125f);
  static_cast<uint8_t*>(t.exp_avg)[i] = to_e4m3(fine_m ? copysignf(am, m) : NAN);
  static_cast<uint8_t*>(t.exp_avg_sq)[i] = to_e4m3(fine_v ? av : NAN);
  if (i % kGroup == 0) {
    static_cast<uint8_t*>(t.exp_avg_scale)[i / kGroup] = (uint8_t)(km + 127);
    static_cast<uint8_t*>(t.exp_avg_sq_scale)[i / kGroup] = (uint8_t)(kv + 127);
  }
}

}  // namespace

uint32_t adamw_mix(uint32_t z) { return mix(z); }

hipError_t launch_adamw(int dtype, int state_bits, int64_t n_tensors,
                        const cpab_adamw_tensor* tensors, const AdamW& a, hipStream_t s) {
  for (int64_t k = 0; k < n_tensors; ++k) {
    const cpab_adamw_tensor& t = tensors[k];
    if (t.n == 0) continue;
    const unsigned blocks = (unsigned)((t.n + kLanes - 1) / kLanes);
    const uint32_t key = mix(a.key + (uint32_t)k);
    if (dtype == CPAB_F32)
      state_bits == 8 ? adamw_kernel<float, true><<<blocks, kLanes, 0, s>>>(t, a, key)
                      : adamw_kernel<float, false><<<blocks, kLanes, 0, s>>>(t, a, key);
    else
      state_bits == 8 ? adamw_kernel<bf16, true><<<blocks, kLanes, 0, s>>>(t, a, key)
                      : adamw_kernel<bf16, false><<<blocks, kLanes, 0, s>>>(t, a, key);
  }
  return hipGetLastError();
}

}  // namespace cpab
