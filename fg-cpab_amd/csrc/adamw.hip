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
#include <type_traits>

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
// The weight after a step, from the new moments and the root of the second.
__device__ __forceinline__ float moved(const AdamW& a, float w, float m, float root) {
  return w * a.decay - a.rate * m / (root * a.root + a.eps);
}

// N values at any alignment of theirs, N * sizeof(T) a power of two up to 16 bytes.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = N * (int)sizeof(T);
  typedef uint32_t Words __attribute__((ext_vector_type(kBytes / 4)));
  typedef Words __attribute__((aligned(sizeof(T)))) Unit;
  T v[N];
  // Past the caches: nothing of this comes again before the next step.
  __device__ __forceinline__ static Pack load(const T* p) {
    return __builtin_bit_cast(Pack, (Words)__builtin_nontemporal_load(reinterpret_cast<const Unit*>(p)));
  }
  __device__ __forceinline__ void store(T* p) const {
    __builtin_nontemporal_store((Unit)__builtin_bit_cast(Words, *this), reinterpret_cast<Unit*>(p));
  }
  __device__ __forceinline__ void store_cached(T* p) const {
    *reinterpret_cast<Unit*>(p) = __builtin_bit_cast(Words, *this);
  }
};

constexpr int kEach = 4;                       // values of a lane
constexpr int kSpan = kLanes * kEach;          // of a workgroup
constexpr int kTensors = 48;                   // of a launch: 64 bytes of arguments each

// The tensors of a launch and where each one's spans begin among the launch's.
struct Batch {
  cpab_adamw_tensor t[kTensors];
  uint32_t first[kTensors + 1];
  uint32_t ordinal;   // of the first tensor, in the step's list
};

// Four E4M3 values, or NaN.
__device__ __forceinline__ Pack<uint8_t, kEach> pack_e4m3(const float z[kEach]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], w, true);
  return __builtin_bit_cast(Pack<uint8_t, kEach>, w);
}

// One value's step: the new moments, their root, and the moved weight.
__device__ __forceinline__ void advance(const AdamW& a, float g, float& m, float& v, float& root,
                                        float& w) {
  m = a.beta1 * m + a.rest1 * g;
  v = a.beta2 * v + a.rest2 * g * g;
  root = sqrtf(v);
  w = moved(a, w, m, root);
}

// A span of a tensor to a workgroup, four neighbouring values to a lane; eight lanes hold
// the 32 that share a scale.
template <typename T, bool EIGHT, bool MASTER>
__global__ void __launch_bounds__(kLanes) adamw_kernel(Batch batch, int count, AdamW a) {
  // the tensor of this span: the last that begins at or before it
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (batch.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const cpab_adamw_tensor& t = batch.t[lo];
  const int64_t at = (int64_t)(blockIdx.x - batch.first[lo]) * kSpan + threadIdx.x * kEach;
  const int here = (int)max((int64_t)0, min((int64_t)kEach, t.n - at));   // values of this lane
  T* p = static_cast<T*>(t.param) + at;
  const T* gp = static_cast<const T*>(t.grad) + at;
  float* wp = MASTER ? t.master + at : nullptr;
  float g[kEach] = {}, w[kEach] = {}, m[kEach] = {}, v[kEach] = {}, root[kEach];
  float* mp = static_cast<float*>(t.exp_avg) + at;
  float* vp = static_cast<float*>(t.exp_avg_sq) + at;
  uint8_t* m8 = static_cast<uint8_t*>(t.exp_avg) + at;
  uint8_t* v8 = static_cast<uint8_t*>(t.exp_avg_sq) + at;
  uint8_t* ms = static_cast<uint8_t*>(t.exp_avg_scale) + at / kGroup;
  uint8_t* vs = static_cast<uint8_t*>(t.exp_avg_sq_scale) + at / kGroup;
  if (here == kEach) {
    const auto gs = Pack<T, kEach>::load(gp);
    if (MASTER) {
      const auto ws = Pack<float, kEach>::load(wp);
#pragma unroll
      for (int e = 0; e < kEach; ++e) w[e] = ws.v[e];
    } else {
      const auto ws = Pack<T, kEach>::load(p);
#pragma unroll
      for (int e = 0; e < kEach; ++e) w[e] = to_float(ws.v[e]);
    }
    if (EIGHT) {
      const auto mq = Pack<uint8_t, kEach>::load(m8), vq = Pack<uint8_t, kEach>::load(v8);
      const float mk = power_of_two((int)*ms - 127), vk = power_of_two((int)*vs - 127);
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        m[e] = from_e4m3(mq.v[e]) * mk;
        v[e] = from_e4m3(vq.v[e]) * vk;
      }
    } else {
      const auto mq = Pack<float, kEach>::load(mp), vq = Pack<float, kEach>::load(vp);
#pragma unroll
      for (int e = 0; e < kEach; ++e) m[e] = mq.v[e], v[e] = vq.v[e];
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) g[e] = to_float(gs.v[e]);
  } else if (here > 0) {   // a tensor's end
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (e >= here) continue;
      g[e] = to_float(gp[e]);
      w[e] = MASTER ? wp[e] : to_float(p[e]);
      m[e] = EIGHT ? from_e4m3(m8[e]) * power_of_two((int)*ms - 127) : mp[e];
      v[e] = EIGHT ? from_e4m3(v8[e]) * power_of_two((int)*vs - 127) : vp[e];
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (EIGHT) v[e] *= v[e];
    advance(a, g[e], m[e], v[e], root[e], w[e]);
  }
  Pack<T, kEach> po;
  Pack<float, kEach> wo, mo, vo;
  Pack<uint8_t, kEach> mq, vq;
  int km = 0, kv = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    po.v[e] = from_float<T>(w[e]), wo.v[e] = w[e], mo.v[e] = m[e], vo.v[e] = v[e];
  if (EIGHT) {
    float top_m = 0.0f, top_v = 0.0f;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      top_m = fmaxf(top_m, fabsf(m[e]) < INFINITY ? fabsf(m[e]) : 0.0f);
      top_v = fmaxf(top_v, root[e] < INFINITY ? root[e] : 0.0f);
    }
    for (int d = 1; d < kGroup / kEach; d *= 2) {
      top_m = fmaxf(top_m, __shfl_xor(top_m, d));
      top_v = fmaxf(top_v, __shfl_xor(top_v, d));
    }
    km = scale_exponent(top_m), kv = scale_exponent(top_v);
    const float im = power_of_two(-km), iv = power_of_two(-kv);
    const uint32_t key = mix(a.key + batch.ordinal + (uint32_t)lo);
    float am[kEach], av[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const uint32_t bits = mix((uint32_t)at + e + key);
      am[e] = copysignf(round_at_random(fabsf(m[e]) * im, bits & 0xffffu), m[e]);
      av[e] = round_at_random(root[e] * iv, bits >> 16);
      if (root[e] > 0.0f) av[e] = fmaxf(av[e], 0.001953125f);
      if (!(fabsf(m[e]) < INFINITY)) am[e] = NAN;
      if (!(root[e] < INFINITY)) av[e] = NAN;
    }
    mq = pack_e4m3(am);
    vq = pack_e4m3(av);
  }
  if (here == kEach) {
    if (a.cached) {
      asm volatile("");   // or the compiler makes the two one, through the caches
      po.store_cached(p);
      asm volatile("");
    } else {
      po.store(p);
    }
    if (MASTER) wo.store(wp);
    if (EIGHT) {
      mq.store(m8);
      vq.store(v8);
    } else {
      mo.store(mp);
      vo.store(vp);
    }
  } else if (here > 0) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (e >= here) continue;
      p[e] = po.v[e];
      if (MASTER) wp[e] = wo.v[e];
      if (EIGHT)
        m8[e] = mq.v[e], v8[e] = vq.v[e];
      else
        mp[e] = mo.v[e], vp[e] = vo.v[e];
    }
  }
  if (EIGHT && here > 0 && at % kGroup == 0) {
    *ms = (uint8_t)(km + 127);
    *vs = (uint8_t)(kv + 127);
  }
}

}  // namespace

uint32_t adamw_mix(uint32_t z) { return mix(z); }

hipError_t launch_adamw(int dtype, int state_bits, int64_t n_tensors,
                        const cpab_adamw_tensor* tensors, const AdamW& step, hipStream_t s) {
  constexpr int64_t kMost = kAdamWMost / kSpan;   // a launch's lanes are counted in 32 bits
  // The parameters are what the next pass reads: through the cache, where it holds them
  // (half of the 256 MB before memory; 134 million weights in 32 bits, 616 us past it
  // with everything, 650 with the parameters through it, 688 with all through it).
  int64_t bytes = 0;
  for (int64_t k = 0; k < n_tensors; ++k) bytes += tensors[k].n * (dtype == CPAB_F32 ? 4 : 2);
  AdamW a = step;
  a.cached = bytes <= (128 << 20);
  for (int64_t k = 0; k < n_tensors;) {
    Batch batch;
    batch.ordinal = (uint32_t)k;
    const bool master = tensors[k].master != nullptr;
    int count = 0;
    int64_t spans = 0;
    for (; k < n_tensors && count < kTensors && (tensors[k].master != nullptr) == master; ++k, ++count) {
      const int64_t more = (tensors[k].n + kSpan - 1) / kSpan;
      if (spans + more > kMost) break;
      batch.t[count] = tensors[k];
      batch.first[count] = (uint32_t)spans;
      spans += more;
    }
    if (count == 0) return hipErrorInvalidValue;   // capi_sequence.cpp lets none so large in
    if (spans == 0) continue;
    const auto launch = [&](auto t, auto eight, auto with) {
      adamw_kernel<decltype(t), decltype(eight)::value, decltype(with)::value>
          <<<(unsigned)spans, kLanes, 0, s>>>(batch, count, a);
    };
    const auto masters = [&](auto t, auto eight) {
      master ? launch(t, eight, std::true_type()) : launch(t, eight, std::false_type());
    };
    const auto states = [&](auto t) {
      state_bits == 8 ? masters(t, std::true_type()) : masters(t, std::false_type());
    };
    dtype == CPAB_F32 ? states(0.0f) : states(bf16());
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace cpab
