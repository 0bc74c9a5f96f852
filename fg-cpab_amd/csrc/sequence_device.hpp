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

// sigmoid(v) and sigmoid(-v) = 1 - sigmoid(v): with e = exp(-|v|) the smaller is
// e / (1 + e), to a few units in its last place (and |v| units from the scaling of exp's
// argument), and 1 less that the larger, off by half a unit and the smaller's share:
// gates near 1, whose products run over hundreds of samples, come nearer so than by the
// approximate reciprocal.
struct Gate {
  float pos, neg;
};
// Both in one register: the smaller, under v's sign, which says which of the two it is.
// The larger alone would not do: 1 less it keeps nothing of a smaller below 2^-24.
__device__ __forceinline__ float folded(float v) {
  const float e = __expf(-fabsf(v));
  return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), v);
}
__device__ __forceinline__ Gate unfolded(float half) {
  const float small = fabsf(half), big = 1.0f - small;
  return __float_as_int(half) < 0 ? Gate{small, big} : Gate{big, small};
}
__device__ __forceinline__ Gate sigmoids(float v) { return unfolded(folded(v)); }

}  // namespace cpab
