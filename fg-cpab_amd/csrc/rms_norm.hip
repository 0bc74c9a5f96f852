// Root-mean-square norm with the residual's addition, to the input's type or to
// 8 bits with a scale per row, and its gradient.
//
// s = 1 / sqrt(mean(r^2) + eps), y = r s w.  Backward, with u = w dy and n = r s:
//   dr = s (u - n mean(u n)) + dr_out,  dw = sum over rows of dy n.
//
// The forward's norm is of r before it is rounded to the residual's type, and the backward
// is its gradient: where that type has 16 bits it takes x and the residual again and not the
// rounded r, whose rounding the gradients would show beside their own (the weight's is
// 0.0017 from 64 bits so, 0.0024 from the rounded r, for a quarter more to read and write).
//
// Bound by memory: each value is read once and written once.  A row is held in the
// registers of `tpr` lanes (a part of a wave, so that a narrow row does not leave one
// idle, or several waves), in pieces of V neighbouring values (16
// bytes); the sums go over the lanes by shuffles and, beyond a wave, LDS.  Rows wider
// than the registers of the largest workgroup are read again from the cache instead.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

constexpr int kMaxLanes = 1024;   // of a workgroup
constexpr int kMinBlock = 256;

struct Sum {
  __device__ float operator()(float a, float b) const { return a + b; }
};
struct Max {   // a NaN stays
  __device__ float operator()(float a, float b) const { return a != a || a > b ? a : b; }
};

// The same value in each of a row's `tpr` lanes; `room` holds a float for each wave.
// Called by every lane of the workgroup.
template <typename Op>
__device__ __forceinline__ float over_row(float v, int tpr, float* room, Op op) {
  const int most = min(tpr, 64);
  for (int d = 1; d < most; d *= 2) v = op(v, __shfl_xor(v, d));
  if (tpr > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
    __syncthreads();
    const int waves = tpr >> 6, first = (int)(threadIdx.x >> 6) / waves * waves;
    v = room[first];
    for (int w = 1; w < waves; ++w) v = op(v, room[first + w]);
  }
  return v;
}

__device__ __forceinline__ uint32_t to_e4m3(float v) {   // |v| <= 448 or NaN
  return __builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff;
}
// A row in 8 bits.  s cancels between y and its scale: with s = m 2^k, m in [1, 2), and
// z = (r 2^k) w, of y's size and one rounding from y / m, y / scale is
// z / (max |z| / 448), two roundings from the definition, and the scale max |z| m / 448.
__device__ __forceinline__ float power_of(float s) {   // 2^k; 0 and infinity stay, NaN is infinity
  return __uint_as_float(__float_as_uint(s) & 0x7f800000u);
}
struct Eight {
  float scale, up, by, inv;
  __device__ Eight(float top, float s) {   // top = max |z|
    const float y = top * __uint_as_float((__float_as_uint(s) & 0x7fffffu) | 0x3f800000u);
    scale = y == 0.0f ? 1.0f : y / 448.0f;
    up = top < 0x1p-100f ? 0x1p100f : 1.0f;   // or 1 / by would pass the largest float
    by = y == 0.0f ? 1.0f : top * up / 448.0f;
    inv = y == 0.0f ? 0.0f : 1.0f / by;
  }
  // z / by, of z times `up`, the product's rounding taken back, so that what lies between
  // two 8-bit values falls to the nearer.
  __device__ __forceinline__ float value(float z) const {
    const float q = z * inv, v = fmaf(fmaf(-q, by, z), inv, q);
    return fabsf(v) > 448.0f ? copysignf(448.0f, v) : v;
  }
};

template <int V>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float in[V]) {
  if constexpr (V == 1) {
    *p = (uint8_t)to_e4m3(in[0]);
  } else {
    typedef Piece<V, 1> P;
    uint32_t words[V / 4];
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * k], in[4 * k + 1], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * k + 2], in[4 * k + 3], w, true);
      words[k] = (uint32_t)w;
    }
    typename P::Bits bits;
    __builtin_memcpy(&bits, words, sizeof(words));
    *reinterpret_cast<typename P::Unit*>(p) = bits;
  }
}

// Where a lane's piece `k` lies.  The last piece of a row that V does not divide is moved
// back to end with the row; `again` of its first values are another lane's too, and are
// not summed a second time (stored they are, the same).  V <= C.
struct Place {
  int64_t at;
  int again;   // V or more: no piece
  __device__ Place(int k, int tpr, int lane, int V, int64_t C) {
    const int64_t from = ((int64_t)k * tpr + lane) * V;
    at = min(from, C - V);
    again = (int)min(from - at, (int64_t)V);
  }
};

template <typename T, typename R, typename W, bool EIGHT, int V, int CH>
__global__ void __launch_bounds__(kMaxLanes)
rms_norm_forward_kernel(RmsNorm n, T* y, uint8_t* q, float* scale, R* residual_out, float* rstd,
                        int tpr) {
  __shared__ float room[kMaxLanes / 64];
  const int group = threadIdx.x / tpr, lane = threadIdx.x - group * tpr;
  const int per = blockDim.x / tpr;
  const int64_t rounds = (n.rows + per - 1) / per;
  float w[CH][V];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const Place p(k, tpr, lane, V, n.C);
    if (p.again < V) load<V>(static_cast<const W*>(n.weight) + p.at, w[k]);
  }
  for (int64_t round = blockIdx.x; round < rounds; round += gridDim.x) {
    const bool live = round * per + group < n.rows;
    const int64_t row = min(round * per + group, n.rows - 1);
    const T* x = static_cast<const T*>(n.x) + row * n.x_stride;
    const R* res = static_cast<const R*>(n.residual) + row * n.residual_stride;
    float r[CH][V];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again < V) load<V>(x + p.at, r[k]);
    }
    if (n.residual) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const Place p(k, tpr, lane, V, n.C);
        if (p.again >= V) continue;
        float more[V];
        load<V>(res + p.at, more);
#pragma unroll
        for (int e = 0; e < V; ++e) r[k][e] += more[e];
      }
    }
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again >= V) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) sum += e >= p.again ? r[k][e] * r[k][e] : 0.0f;
      if (residual_out && live) store<V>(residual_out + row * n.C + p.at, r[k]);
    }
    sum = over_row(sum, tpr, room, Sum());
    const float s = 1.0f / sqrtf(sum / (float)n.C + n.eps), by_s = EIGHT ? power_of(s) : s;
    if (rstd && live && lane == 0) rstd[row] = s;
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again >= V) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        r[k][e] = r[k][e] * by_s * w[k][e];
        if (EIGHT) top = Max()(fabsf(r[k][e]), top);
      }
      if (!EIGHT && live) store<V>(y + row * n.C + p.at, r[k]);
    }
    if (!EIGHT) continue;
    top = over_row(top, tpr, room, Max());
    const Eight by(top, s);
    if (live && lane == 0) scale[row] = by.scale;
    if (by.up != 1.0f) {   // hardly ever
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) r[k][e] *= by.up;
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again >= V) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) r[k][e] = by.value(r[k][e]);
      if (live) store_e4m3<V>(q + row * n.C + p.at, r[k]);
    }
  }
}

// Each workgroup takes every gridDim.x-th round of rows and adds up its part of dw in
// registers; the parts, [gridDim.x, C], are joined by the next kernel in their order, and
// the part of a workgroup that is alone is the whole, `direct`.
template <typename T, typename R, typename W, int V, int CH>
__global__ void __launch_bounds__(kMaxLanes)
rms_norm_backward_kernel(RmsNormGrad n, T* dx, R* dres, float* parts, W* direct, int tpr) {
  __shared__ float room[kMaxLanes / 64];
  extern __shared__ float sums[];   // [per - 1][tpr][CH][V], where rows share a workgroup
  const int group = threadIdx.x / tpr, lane = threadIdx.x - group * tpr;
  const int per = blockDim.x / tpr;
  const int64_t rounds = (n.rows + per - 1) / per;
  float w[CH][V], dw[CH][V];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < V; ++e) dw[k][e] = 0.0f;
    const Place p(k, tpr, lane, V, n.C);
    if (p.again < V) load<V>(static_cast<const W*>(n.weight) + p.at, w[k]);
  }
  for (int64_t round = blockIdx.x; round < rounds; round += gridDim.x) {
    const bool live = round * per + group < n.rows;
    const int64_t row = min(round * per + group, n.rows - 1);
    const R* r = static_cast<const R*>(n.r) + row * n.r_stride;
    const T* dy = static_cast<const T*>(n.grad_y) + row * n.grad_y_stride;
    const R* dout = static_cast<const R*>(n.grad_out) + row * n.grad_out_stride;
    const float s = n.rstd[row];
    float v[CH][V], u[CH][V];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again >= V) continue;
      load<V>(r + p.at, v[k]);
      load<V>(dy + p.at, u[k]);
    }
    if (n.added) {
      const R* more = static_cast<const R*>(n.added) + row * n.added_stride;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const Place p(k, tpr, lane, V, n.C);
        if (p.again >= V) continue;
        float a[V];
        load<V>(more + p.at, a);
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] += a[e];
      }
    }
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again >= V) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[k][e] *= s;
        if (live) dw[k][e] = fmaf(u[k][e], v[k][e], dw[k][e]);
        u[k][e] *= w[k][e];
        sum += e >= p.again ? u[k][e] * v[k][e] : 0.0f;
      }
    }
    if (!dx && !dres) continue;
    const float mean = over_row(sum, tpr, room, Sum()) / (float)n.C;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const Place p(k, tpr, lane, V, n.C);
      if (p.again >= V || !live) continue;
      float d[V] = {};
      if (n.grad_out) load<V>(dout + p.at, d);
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] += s * (u[k][e] - v[k][e] * mean);
      if (dx) store<V>(dx + row * n.C + p.at, d);
      if (dres) store<V>(dres + row * n.C + p.at, d);
    }
  }
  if (!parts && !direct) return;
  if (per > 1) {
    // the other rows' lanes of the same channels, in their order
    if (group > 0) {
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e)
          sums[((group - 1) * CH * V + k * V + e) * tpr + lane] = dw[k][e];
    }
    __syncthreads();
    if (group > 0) return;
    for (int g = 0; g < per - 1; ++g)
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) dw[k][e] += sums[(g * CH * V + k * V + e) * tpr + lane];
  }
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const Place p(k, tpr, lane, V, n.C);
    if (p.again >= V) continue;
    if (direct)
      store<V>(direct + p.at, dw[k]);
    else
      store<V>(parts + (int64_t)blockIdx.x * n.C + p.at, dw[k]);
  }
}

// dw[c] = the sum of `count` parts.  A workgroup has 16 channels and 64 runs of parts,
// joined over a wave's four and then the 16 waves.  Latency counts (4 MB of parts for
// 32768 x 1024: 4.8 us with 64 channels and 16 runs).
template <typename W>
__global__ void __launch_bounds__(1024)
rms_norm_weight_kernel(const float* parts, int count, int64_t C, W* dw) {
  __shared__ float sums[16][16];
  const int lane = threadIdx.x & 15, run = threadIdx.x >> 4;
  const int64_t c = blockIdx.x * (int64_t)16 + lane;
  float sum = 0.0f;
  if (c < C)
#pragma unroll 8
    for (int k = run; k < count; k += 64) sum += parts[k * C + c];
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if ((run & 3) == 0) sums[run >> 2][lane] = sum;
  __syncthreads();
  if (run > 0 || c >= C) return;
#pragma unroll
  for (int k = 1; k < 16; ++k) sum += sums[k][lane];
  dw[c] = from_float<W>(sum);
}

// ---- rows of any width: read once for each sum and once for the result -------------

template <typename T, typename R, typename W, bool EIGHT>
__global__ void __launch_bounds__(kMaxLanes)
rms_norm_wide_forward_kernel(RmsNorm n, T* y, uint8_t* q, float* scale, R* residual_out, float* rstd) {
  __shared__ float room[kMaxLanes / 64];
  const W* w = static_cast<const W*>(n.weight);
  for (int64_t row = blockIdx.x; row < n.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(n.x) + row * n.x_stride;
    const R* res = n.residual ? static_cast<const R*>(n.residual) + row * n.residual_stride : nullptr;
    const auto value = [&](int64_t c) { return to_float(x[c]) + (res ? to_float(res[c]) : 0.0f); };
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < n.C; c += kMaxLanes) sum += value(c) * value(c);
    sum = over_row(sum, kMaxLanes, room, Sum());
    const float s = 1.0f / sqrtf(sum / (float)n.C + n.eps), by_s = EIGHT ? power_of(s) : s;
    if (rstd && threadIdx.x == 0) rstd[row] = s;
    float top = 0.0f;
    if (EIGHT) {
      for (int64_t c = threadIdx.x; c < n.C; c += kMaxLanes)
        top = Max()(fabsf(value(c) * by_s * to_float(w[c])), top);
      top = over_row(top, kMaxLanes, room, Max());
    }
    const Eight by(top, s);
    if (EIGHT && threadIdx.x == 0) scale[row] = by.scale;
    for (int64_t c = threadIdx.x; c < n.C; c += kMaxLanes) {
      const float r = value(c);
      if (EIGHT)
        q[row * n.C + c] = (uint8_t)to_e4m3(by.value(r * by_s * to_float(w[c]) * by.up));
      else
        y[row * n.C + c] = from_float<T>(r * by_s * to_float(w[c]));
      if (residual_out) residual_out[row * n.C + c] = from_float<R>(r);
    }
  }
}

// parts [gridDim.x, C]: this workgroup's rows' part of dw, zero before.
template <typename T, typename R, typename W>
__global__ void __launch_bounds__(kMaxLanes)
rms_norm_wide_backward_kernel(RmsNormGrad n, T* dx, R* dres, float* parts) {
  __shared__ float room[kMaxLanes / 64];
  const W* w = static_cast<const W*>(n.weight);
  float* part = parts ? parts + (int64_t)blockIdx.x * n.C : nullptr;
  for (int64_t row = blockIdx.x; row < n.rows; row += gridDim.x) {
    const R* r = static_cast<const R*>(n.r) + row * n.r_stride;
    const T* dy = static_cast<const T*>(n.grad_y) + row * n.grad_y_stride;
    const R* dout = n.grad_out ? static_cast<const R*>(n.grad_out) + row * n.grad_out_stride : nullptr;
    const R* more = n.added ? static_cast<const R*>(n.added) + row * n.added_stride : nullptr;
    const auto value = [&](int64_t c) { return to_float(r[c]) + (more ? to_float(more[c]) : 0.0f); };
    const float s = n.rstd[row];
    float sum = 0.0f;
    for (int64_t c = threadIdx.x; c < n.C; c += kMaxLanes) {
      const float g = to_float(dy[c]), v = value(c) * s;
      sum += g * to_float(w[c]) * v;
      if (part) part[c] += g * v;   // the lane's own channels
    }
    if (!dx && !dres) continue;
    const float mean = over_row(sum, kMaxLanes, room, Sum()) / (float)n.C;
    for (int64_t c = threadIdx.x; c < n.C; c += kMaxLanes) {
      const float u = to_float(dy[c]) * to_float(w[c]);
      const float d = s * (u - value(c) * s * mean) + (dout ? to_float(dout[c]) : 0.0f);
      if (dx) dx[row * n.C + c] = from_float<T>(d);
      if (dres) dres[row * n.C + c] = from_float<R>(d);
    }
  }
}

// How a launch lays rows on lanes.
struct Layout {
  int V, CH, tpr, block;   // tpr: a power of two up to a wave, or whole waves
  int64_t rounds;          // of rows, one workgroup each
  bool wide;
};
// Few lanes with several pieces each leave few idle where a width is not a power of two,
// and make more workgroups to a compute unit; the registers bound what a lane holds, the
// backward's most.  2^27 values, us, by the most pieces to a lane (2, 3, 4):
//   forward to 8 bits, float32    333: 285, 201, 201    4096: 227, 226, 176
//                      bfloat16   333: 140, 118, 117    4096: 112, 112, 119
//   backward,          float32    333: 346, 304, 304    4096: 284, 285, 292
//                      bfloat16   333: 178, 227, 226    4096: 158, 157, 395
// In the forward 32 values to a lane come before 1024 lanes, of which one workgroup alone
// finds room (16384, 8 bits: 190 us in 32 bits, 245 with 16; bfloat16 129 and 173).  Where
// 1024 lanes are not enough a lane takes up to four pieces in the backward too: in bfloat16
// (16385 to 32768) they do not all fit its registers (12 to 83 words a lane in scratch), and
// still take less than reading the row again (4096 rows of 17,000 145 us and 452, 24,600 332
// and 677, 32,768 393 and 905; 64 rows of 24,600 36 to 47 and 28).
Layout layout(int dtype, int64_t rows, int64_t C, bool backward) {
  Layout l;
  const bool f32 = dtype == CPAB_F32;
  l.V = f32 ? 4 : 8;
  const int most = (f32 ? 4 : 3) - backward, cap = backward ? 4 : 32 / l.V;
  if (C < l.V) l.V = 1;
  const int64_t pieces = (C + l.V - 1) / l.V;
  const auto lanes = [&](int each) {
    int n = 8;
    while (n < kMaxLanes && (int64_t)n * each < pieces) n *= 2;
    return n;
  };
  l.tpr = lanes(most);
  if (l.tpr == kMaxLanes) l.tpr = lanes(backward ? most : cap);
  const int64_t each = (pieces + l.tpr - 1) / l.tpr;
  l.wide = each > cap;
  l.CH = (int)std::min<int64_t>(each <= 4 ? each : each <= 6 ? 6 : 8, cap);
  if (backward && !f32 && l.CH == 2 && l.tpr > 64 && 3 * pieces < 4 * (int64_t)l.tpr && pieces <= kMaxLanes) {
    // less than two thirds of the pieces that the lanes have room for: one piece a lane, as
    // many waves as that takes (4200: 160 us, 201; 5000: 160, 189; 6000, not so: 179, 172)
    l.CH = 1;
    l.tpr = (int)((pieces + 63) / 64 * 64);
  }
  const int per = std::max(1, kMinBlock / l.tpr);
  l.block = l.tpr * per;
  l.rounds = (rows + per - 1) / per;
  return l;
}

// f(T(), R(), W()) for the arrays' types.
template <typename F>
void with_types(int dtype, int residual, int weight, F f) {
  if (dtype == CPAB_F32) return weight == CPAB_F32 ? f(0.0f, 0.0f, 0.0f) : f(0.0f, 0.0f, bf16());
  if (residual == CPAB_F32)
    return weight == CPAB_F32 ? f(bf16(), 0.0f, 0.0f) : f(bf16(), 0.0f, bf16());
  return weight == CPAB_F32 ? f(bf16(), bf16(), 0.0f) : f(bf16(), bf16(), bf16());
}
// f(V, CH) as constants.
template <typename T, bool BACKWARD, typename F>
void with_layout(const Layout& l, F f) {
  constexpr int V = 16 / (int)sizeof(T);
  const auto many = [&](auto ch) { f(std::integral_constant<int, V>(), ch); };
  typedef std::integral_constant<int, 1> One;
  if (l.V == 1) return f(One(), One());   // C < V: at most 8 lanes' worth
  if (l.CH == 1) return many(One());
  if (l.CH == 2) return many(std::integral_constant<int, 2>());
  if (l.CH == 3) return many(std::integral_constant<int, 3>());
  if constexpr (V == 4 && !BACKWARD) {
    if (l.CH == 6) return many(std::integral_constant<int, 6>());
    if (l.CH == 8) return many(std::integral_constant<int, 8>());
  }
  many(std::integral_constant<int, 4>());
}

// Workgroups that take rounds of rows in turn, their weights in registers: `waves` to a
// compute unit.  Forward 64, twice what runs at once (16384 x 8192 bfloat16 to 8 bits:
// 186 us, 5.0 TB/s as a large copy; 218 with 32, 208 with a workgroup for each round);
// backward 16 (32768 x 1024 from one array: 46.6 and 4.8 us for dw's parts, 51 and 4.0 with
// 12, 49 and 8.2 with 32; from x and the residual 67.7 and 4.2).
int64_t workgroups(int64_t rounds, int block, int waves) {
  return std::max<int64_t>(1, std::min<int64_t>(rounds, (int64_t)compute_units() * waves * 64 / block));
}

}  // namespace

hipError_t launch_rms_norm_forward(const RmsNorm& n, void* y, float* scale, void* residual_out,
                                   float* rstd, hipStream_t st) {
  const Layout l = layout(n.dtype, n.rows, n.C, false);
  with_types(n.dtype, n.residual_dtype, n.weight_dtype, [&](auto t, auto r, auto w) {
    typedef decltype(t) T;
    typedef decltype(r) R;
    typedef decltype(w) W;
    const auto out = [&](auto eight) {
      constexpr bool E = decltype(eight)::value;
      if (l.wide) {
        rms_norm_wide_forward_kernel<T, R, W, E>
            <<<(unsigned)workgroups(n.rows, kMaxLanes, 32), kMaxLanes, 0, st>>>(
                n, (T*)y, (uint8_t*)y, scale, (R*)residual_out, rstd);
        return;
      }
      with_layout<T, false>(l, [&](auto v, auto ch) {
        rms_norm_forward_kernel<T, R, W, E, decltype(v)::value, decltype(ch)::value>
            <<<(unsigned)workgroups(l.rounds, l.block, 64), l.block, 0, st>>>(
                n, (T*)y, (uint8_t*)y, scale, (R*)residual_out, rstd, l.tpr);
      });
    };
    scale ? out(std::true_type()) : out(std::false_type());
  });
  return hipGetLastError();
}

// The backward's layout, with dw.  Rows that one workgroup goes through in four rounds are
// one workgroup's, which saves the second launch: 64 x 1024 bfloat16, forward and backward,
// 37 us a pass and 41 with it (32 x 4096, nearer the limit: 39.7 and 40.8).
static Layout backward_layout(int dtype, int64_t rows, int64_t C) {
  Layout l = layout(dtype, rows, C, true);
  const int most = l.tpr < 64 ? 512 : kMaxLanes;   // 64 KiB of LDS for the other rows' sums
  if (!l.wide && rows <= 4 * (most / l.tpr)) {
    while (2 * l.block <= most && l.rounds > 1) {
      l.block *= 2;
      l.rounds = (rows + l.block / l.tpr - 1) / (l.block / l.tpr);
    }
  }
  return l;
}
// Its workgroups: the fewer, the fewer parts of dw to join.
static int64_t backward_parts(const Layout& l, int64_t rows) {
  if (l.wide) return workgroups(rows, kMaxLanes, 16);
  return l.rounds <= 4 ? 1 : workgroups(l.rounds, l.block, 16);
}

int64_t rms_norm_backward_workspace(int64_t rows, int64_t C) {
  int64_t most = 0;
  for (const int dtype : {CPAB_F32, CPAB_BF16}) {
    const Layout l = backward_layout(dtype, rows, C);
    const int64_t parts = backward_parts(l, rows);
    if (l.wide || rows == 0 || parts > 1) most = std::max(most, parts);
  }
  return most * C * 4;
}

hipError_t launch_rms_norm_backward(const RmsNormGrad& n, void* grad_x, void* grad_residual,
                                    void* grad_weight, void* workspace, hipStream_t st) {
  const Layout l = grad_weight ? backward_layout(n.dtype, n.rows, n.C) : layout(n.dtype, n.rows, n.C, true);
  const int64_t count = grad_weight ? backward_parts(l, n.rows)
                                    : workgroups(l.wide ? n.rows : l.rounds, l.wide ? kMaxLanes : l.block, 64);
  const bool alone = grad_weight && !l.wide && n.rows > 0 && count == 1;
  float* parts = grad_weight && !alone ? static_cast<float*>(workspace) : nullptr;
  if (parts && (l.wide || n.rows == 0)) {
    const hipError_t e = launch_fill(parts, count * n.C, 0.0f, st);
    if (e != hipSuccess) return e;
  }
  with_types(n.dtype, n.residual_dtype, n.weight_dtype, [&](auto t, auto r, auto w) {
    typedef decltype(t) T;
    typedef decltype(r) R;
    typedef decltype(w) W;
    if (n.rows > 0 && l.wide) {
      rms_norm_wide_backward_kernel<T, R, W><<<(unsigned)count, kMaxLanes, 0, st>>>(
          n, (T*)grad_x, (R*)grad_residual, parts);
    } else if (n.rows > 0) {
      with_layout<T, true>(l, [&](auto v, auto ch) {
        constexpr int V = decltype(v)::value, CH = decltype(ch)::value;
        const size_t lds = (size_t)(l.block / l.tpr - 1) * l.tpr * CH * V * 4;
        rms_norm_backward_kernel<T, R, W, V, CH><<<(unsigned)count, l.block, lds, st>>>(
            n, (T*)grad_x, (R*)grad_residual, parts, alone ? (W*)grad_weight : nullptr, l.tpr);
      });
    }
    if (parts)
      rms_norm_weight_kernel<W><<<(unsigned)((n.C + 15) / 16), 1024, 0, st>>>(parts, (int)count, n.C,
                                                                             (W*)grad_weight);
  });
  return hipGetLastError();
}

}  // namespace cpab
