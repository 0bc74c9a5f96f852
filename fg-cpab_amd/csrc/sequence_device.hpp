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
// e / (1 + e), and 1 less that the larger, off by half a unit and the smaller's share:
// gates near 1, whose products run over hundreds of samples, come nearer so than by the
// approximate reciprocal.  v is of type T: the smaller carries a few units in its last place
// in 32 bits, and |v| units from the scaling of exp's argument beside them in 16, where no
// result shows it (8 x 4096 x 1280 trained, without them: bfloat16 215 and 224 us, 32 bits
// 358 and 360).
struct Gate {
  float pos, neg;
};
// Both in one register: the smaller, under v's sign, which says which of the two it is.
// The larger alone would not do: 1 less it keeps nothing of a smaller below 2^-24.
template <typename T>
__device__ __forceinline__ float folded(float v) {
  constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0c0p-26f, kLn2 = 0x1.62e430p-1f;
  const float t = -fabsf(v) * kLog2e;
  float e = __builtin_amdgcn_exp2f(t);
  if (sizeof(T) == 4) {
    // what t was rounded by; held to 1 where t is infinite and e is 0
    const float rest = fmaf(-fabsf(v), kLog2eRest, fmaf(-fabsf(v), kLog2e, -t));
    e = fmaf(e, __builtin_amdgcn_fmed3f(rest, -1.0f, 1.0f) * kLn2, e);
  }
  return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), v);
}
__device__ __forceinline__ Gate unfolded(float half) {
  const float small = fabsf(half), big = 1.0f - small;
  return __float_as_int(half) < 0 ? Gate{small, big} : Gate{big, small};
}
template <typename T>
__device__ __forceinline__ Gate sigmoids(float v) { return unfolded(folded<T>(v)); }

}  // namespace cpab
