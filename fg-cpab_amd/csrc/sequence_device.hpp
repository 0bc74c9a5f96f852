// Device-side helpers shared by the operators around the transform: values of
// 32-bit floats and bfloat16 in memory, 32-bit floats in registers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace cpab {

typedef __bf16 bf16;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(bf16 v) {
  return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16);
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  return (T)v;   // bfloat16: to nearest, ties to even
}

// sigmoid(v) and sigmoid(-v) = 1 - sigmoid(v), each to a few units in its last
// place: with e = exp(-|v|) they are 1 / (1 + e) and e / (1 + e), and nothing is
// subtracted from 1.
struct Gate {
  float pos, neg;
};
__device__ __forceinline__ Gate sigmoids(float v) {
  const float e = __expf(-fabsf(v));
  const float big = __builtin_amdgcn_rcpf(1.0f + e);
  const float small = e * big;
  return v < 0.0f ? Gate{small, big} : Gate{big, small};
}

}  // namespace cpab
