// Norms of queries and keys by head, rotated by the position in the same pass, and their
// gradients.
//
// For each head's D values x: s = 1 / sqrt(mean(x^2) + eps), n = x s w; then the first R of
// them, as R / 2 pairs (a, b), turn by the angle p = position * freqs[pair]:
//   (a cos p - b sin p, b cos p + a sin p).
// Backward: the gradient turns back, g = turned by -p; dw = sum of g x s over the rows, and
// with u = w g: dx = s (u - x s mean(u x s)).  s is computed again, which costs nothing
// beside reading x.
//
// The angle is reduced in 64 bits, to a part of a turn, before its sine and cosine in 32: a
// position of 2^20 leaves a 32-bit product 0.06 radians off.
//
// Bound by memory: each value is read once and written once.  A head's row lies in the
// registers of `tpr` lanes, V pairs (or V values of what does not turn, twice) in a unit:
// the two halves of a pair are in one lane, so that turning moves nothing between lanes.
// Sines and cosines are computed once for a token and all the heads that a group of lanes
// goes through.
//
// Measured, 8 x 4096 tokens of 16 + 4 heads of 128 in bfloat16: forward 73 us (335 MB, 4.6
// TB/s), backward 128 (503 MB, 3.9 TB/s) and the weights' sums 7; a copy of the bytes takes 164
// in all.  16 x 784 tokens of 5 + 3 heads of 50 in 32 bits, one value to a load: 21 + 21 + 7.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "heads_launch.hpp"
#include "sequence_device.hpp"

namespace cpab {
namespace {

constexpr int kBlock = 256;

// What a launch knows of one side, queries or keys.
struct Side {
  const void* x;
  int64_t xb, xt, xh;
  const void* w;
  const void* dy;
  int64_t db, dt, dh;
  void* out;        // y, or dx
  void* dw;
  int heads, each;  // heads that an item goes through
  int splits;
  int blocks;       // workgroups that take this side's items in turn
  int64_t parts;    // where its parts of dw begin (floats)
};
struct Both {
  Side side[2];
  int64_t tokens;
  uint32_t T;
  int D, R;
  int turned_units, units, tpr;
  const float* freqs;
  const void* positions;
  int position_type;
  int64_t pb, pt;
  float eps;
  float* parts;
};

// Where unit u of a row lies: V values at `a` and V at `b` (`single`: b is past the end).
struct Unit {
  int a, b;
  bool single, turned, live;
};
template <int V, bool NEIGHBOURS>
__device__ __forceinline__ Unit unit_of(const Both& n, int u) {
  Unit r;
  r.turned = u < n.turned_units;
  r.live = u < n.units;
  if (r.turned && !NEIGHBOURS) {
    r.a = u * V;
    r.b = n.R / 2 + u * V;
  } else {
    r.a = r.turned ? 2 * u * V : n.R + 2 * (u - n.turned_units) * V;
    r.b = r.a + V;
  }
  r.single = V == 1 && r.b >= n.D;
  return r;
}

// x[0..V) from a, x[V..2V) from b; zeros where there is nothing.
template <int V, bool NEIGHBOURS, typename T>
__device__ __forceinline__ void load_unit(const T* row, const Unit& u, float x[2 * V]) {
  if (u.live) {
    load<V>(row + u.a, x);
    if (!u.single) {
      load<V>(row + u.b, x + V);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x[V + e] = 0.0f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) x[e] = 0.0f;
  }
}
template <int V, typename T>
__device__ __forceinline__ void store_unit(T* row, const Unit& u, const float x[2 * V]) {
  if (!u.live) return;
  store<V>(row + u.a, x);
  if (!u.single) store<V>(row + u.b, x + V);
}

// Pair e of a turned unit: its places among the unit's 2 V values.
template <int V, bool NEIGHBOURS>
__device__ __forceinline__ constexpr int first_of(int e) { return NEIGHBOURS ? 2 * e : e; }
template <int V, bool NEIGHBOURS>
__device__ __forceinline__ constexpr int second_of(int e) { return NEIGHBOURS ? 2 * e + 1 : V + e; }

__device__ __forceinline__ double position_of(const Both& n, int64_t b, int64_t t) {
  if (!n.positions) return (double)t;
  const int64_t at = b * n.pb + t * n.pt;
  if (n.position_type == CPAB_POSITION_I32) return (double)static_cast<const int32_t*>(n.positions)[at];
  if (n.position_type == CPAB_POSITION_I64) return (double)static_cast<const int64_t*>(n.positions)[at];
  return (double)static_cast<const float*>(n.positions)[at];
}

template <int V>
__device__ __forceinline__ void angles(const Both& n, double position, const Unit& u, int index,
                                       float c[V], float s[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) c[e] = 1.0f, s[e] = 0.0f;
  if (!u.turned) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    constexpr double kTurn = 0.15915494309189533577;   // 1 / (2 pi)
    const double turns = position * (double)n.freqs[index * V + e] * kTurn;
    sincospif(2.0f * (float)(turns - rint(turns)), &s[e], &c[e]);
  }
}

__device__ __forceinline__ float over_group(float v, int tpr) {
  for (int d = 1; d < tpr; d *= 2) v += __shfl_xor(v, d);
  return v;
}

template <typename T, typename W, int V, int CH, bool NEIGHBOURS>
__global__ __launch_bounds__(kBlock) void qk_norm_forward_kernel(Both n) {
  const Side& sd = n.side[blockIdx.y];
  if ((int)blockIdx.x >= sd.blocks) return;
  const int lane = threadIdx.x & (n.tpr - 1), per = kBlock / n.tpr;
  Unit u[CH];
  float w[CH][2 * V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    u[c] = unit_of<V, NEIGHBOURS>(n, lane + c * n.tpr);
    load_unit<V, NEIGHBOURS>(static_cast<const W*>(sd.w), u[c], w[c]);
  }
  const int64_t items = n.tokens * sd.splits;
  const float each = 1.0f / (float)n.D;
  for (int64_t item = (int64_t)blockIdx.x * per + threadIdx.x / n.tpr; item < items;
       item += (int64_t)sd.blocks * per) {
    const int64_t token = sd.splits == 1 ? item : item / sd.splits;
    const int first = sd.splits == 1 ? 0 : (int)(item - token * sd.splits) * sd.each;
    const int last = min(first + sd.each, sd.heads);
    const int64_t b = (uint32_t)token / n.T, t = (uint32_t)token - (uint32_t)b * n.T;
    float cs[CH][V], sn[CH][V];
    if (n.R > 0) {
      const double position = position_of(n, b, t);
#pragma unroll
      for (int c = 0; c < CH; ++c) angles<V>(n, position, u[c], lane + c * n.tpr, cs[c], sn[c]);
    }
    const T* x = static_cast<const T*>(sd.x) + b * sd.xb + t * sd.xt;
    T* y = static_cast<T*>(sd.out) + token * sd.heads * n.D;
    for (int h = first; h < last; ++h) {
      float v[CH][2 * V], sum = 0.0f;
#pragma unroll
      for (int c = 0; c < CH; ++c) load_unit<V, NEIGHBOURS>(x + h * sd.xh, u[c], v[c]);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) sum = fmaf(v[c][e], v[c][e], sum);
      sum = over_group(sum, n.tpr);
      const float s = 1.0f / sqrtf(fmaf(sum, each, n.eps));
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) v[c][e] = v[c][e] * s * w[c][e];
        if (u[c].turned) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float &p = v[c][first_of<V, NEIGHBOURS>(e)], &q = v[c][second_of<V, NEIGHBOURS>(e)];
            const float a = p, o = q;
            p = fmaf(a, cs[c][e], -o * sn[c][e]);
            q = fmaf(o, cs[c][e], a * sn[c][e]);
          }
        }
        store_unit<V>(y + (int64_t)h * n.D, u[c], v[c]);
      }
    }
  }
}

template <typename T, typename W, int V, int CH, bool NEIGHBOURS>
__global__ __launch_bounds__(kBlock) void qk_norm_backward_kernel(Both n) {
  extern __shared__ float room[];   // a row of D for each wave
  const Side& sd = n.side[blockIdx.y];
  if ((int)blockIdx.x >= sd.blocks) return;
  const int lane = threadIdx.x & (n.tpr - 1), per = kBlock / n.tpr;
  Unit u[CH];
  float w[CH][2 * V], dw[CH][2 * V];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    u[c] = unit_of<V, NEIGHBOURS>(n, lane + c * n.tpr);
    load_unit<V, NEIGHBOURS>(static_cast<const W*>(sd.w), u[c], w[c]);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) dw[c][e] = 0.0f;
  }
  const int64_t items = n.tokens * sd.splits;
  const float each = 1.0f / (float)n.D;
  for (int64_t item = (int64_t)blockIdx.x * per + threadIdx.x / n.tpr; item < items;
       item += (int64_t)sd.blocks * per) {
    const int64_t token = sd.splits == 1 ? item : item / sd.splits;
    const int first = sd.splits == 1 ? 0 : (int)(item - token * sd.splits) * sd.each;
    const int last = min(first + sd.each, sd.heads);
    const int64_t b = (uint32_t)token / n.T, t = (uint32_t)token - (uint32_t)b * n.T;
    float cs[CH][V], sn[CH][V];
    if (n.R > 0) {
      const double position = position_of(n, b, t);
#pragma unroll
      for (int c = 0; c < CH; ++c) angles<V>(n, position, u[c], lane + c * n.tpr, cs[c], sn[c]);
    }
    const T* x = static_cast<const T*>(sd.x) + b * sd.xb + t * sd.xt;
    const T* dy = static_cast<const T*>(sd.dy) + b * sd.db + t * sd.dt;
    for (int h = first; h < last; ++h) {
      float v[CH][2 * V], g[CH][2 * V], sum = 0.0f, dot = 0.0f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        load_unit<V, NEIGHBOURS>(x + h * sd.xh, u[c], v[c]);
        load_unit<V, NEIGHBOURS>(dy + h * sd.dh, u[c], g[c]);
      }
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (u[c].turned) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            float &p = g[c][first_of<V, NEIGHBOURS>(e)], &q = g[c][second_of<V, NEIGHBOURS>(e)];
            const float a = p, o = q;
            p = fmaf(a, cs[c][e], o * sn[c][e]);
            q = fmaf(o, cs[c][e], -a * sn[c][e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) sum = fmaf(v[c][e], v[c][e], sum);
      }
      sum = over_group(sum, n.tpr);
      const float s = 1.0f / sqrtf(fmaf(sum, each, n.eps));
#pragma unroll
      for (int c = 0; c < CH; ++c) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          v[c][e] *= s;
          dw[c][e] = fmaf(g[c][e], v[c][e], dw[c][e]);
          g[c][e] *= w[c][e];
          dot = fmaf(g[c][e], v[c][e], dot);
        }
      }
      dot = over_group(dot, n.tpr) * each;
      if (sd.out) {
        T* dx = static_cast<T*>(sd.out) + (token * sd.heads + h) * n.D;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) g[c][e] = s * fmaf(-v[c][e], dot, g[c][e]);
          store_unit<V>(dx, u[c], g[c]);
        }
      }
    }
  }
  if (!sd.dw) return;
  // over the groups of a wave, then over the waves
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int e = 0; e < 2 * V; ++e)
      for (int d = n.tpr; d < 64; d *= 2) dw[c][e] += __shfl_xor(dw[c][e], d);
    if ((threadIdx.x & 63) < n.tpr) store_unit<V>(room + wave * n.D, u[c], dw[c]);
  }
  __syncthreads();
  float* part = n.parts + sd.parts + (int64_t)blockIdx.x * n.D;
  for (int i = threadIdx.x; i < n.D; i += kBlock) {
    float v = room[i];
    for (int k = 1; k < kBlock / 64; ++k) v += room[k * n.D + i];
    part[i] = v;
  }
}

// dw of a side: its parts, added 64 rows at a time in an order that depends on their count.
template <typename W>
__global__ __launch_bounds__(1024) void qk_norm_weight_kernel(Both n) {
  __shared__ float room[64][17];
  const Side& sd = n.side[blockIdx.y];
  if (!sd.dw) return;
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int at = blockIdx.x * 16 + col;
  float v = 0.0f;
  if (at < n.D)
    for (int k = row; k < sd.blocks; k += 64) v += n.parts[sd.parts + (int64_t)k * n.D + at];
  room[row][col] = v;
  __syncthreads();
  for (int half = 32; half > 0; half /= 2) {
    if (row < half) room[row][col] += room[row + half][col];
    __syncthreads();
  }
  if (row == 0 && at < n.D) static_cast<W*>(sd.dw)[at] = from_float<W>(room[0][col]);
}

// V: the most pairs to a unit, 16 bytes, that divide both what turns and what does not.
struct Layout {
  int V, CH;
};
Layout lay_out(const cpab_qk_norm& n, Both* b) {
  Layout l{n.dtype == CPAB_F32 ? 4 : 8, 1};
  const auto fits = [&](int V) {
    return (n.neighbours ? n.turned % (2 * V) == 0 : n.turned / 2 % V == 0) &&
           (n.width - n.turned) % (2 * V) == 0;
  };
  while (l.V > 1 && !fits(l.V)) l.V /= 2;
  b->turned_units = n.turned / 2 / l.V;
  b->units = b->turned_units + (n.width - n.turned + 2 * l.V - 1) / (2 * l.V);
  b->tpr = 1;
  while (b->tpr < 64 && b->tpr < b->units) b->tpr *= 2;
  while (l.CH * b->tpr < b->units) l.CH *= 2;
  return l;
}

// f(V, CH) as constants: 512 values are 64 units of 4 pairs, 128 of 2 and 256 of 1.
template <typename T, typename F>
void with_layout(const Layout& l, F f) {
  typedef std::integral_constant<int, 1> I1;
  typedef std::integral_constant<int, 2> I2;
  typedef std::integral_constant<int, 4> I4;
  typedef std::integral_constant<int, 8> I8;
  if constexpr (sizeof(T) == 2)
    if (l.V == 8) return f(I8(), I1());
  if (l.V == 4) return f(I4(), I1());
  if (l.V == 2) return l.CH == 1 ? f(I2(), I1()) : f(I2(), I2());
  l.CH == 1 ? f(I1(), I1()) : l.CH == 2 ? f(I1(), I2()) : f(I1(), I4());
}
template <typename F>
void with_types(const cpab_qk_norm& n, F f) {
  if (n.dtype == CPAB_F32)
    return n.weight_dtype == CPAB_F32 ? f(0.0f, 0.0f) : f(0.0f, bf16());
  n.weight_dtype == CPAB_F32 ? f(bf16(), 0.0f) : f(bf16(), bf16());
}

Both both_of(const cpab_qk_norm& n) {
  Both b{};
  b.tokens = n.B * n.T;
  b.T = (uint32_t)n.T;
  b.D = (int)n.width;
  b.R = (int)n.turned;
  b.freqs = n.freqs;
  b.positions = n.positions;
  b.position_type = n.position_type;
  b.pb = n.position_strides[0], b.pt = n.position_strides[1];
  b.eps = n.eps;
  Side &q = b.side[0], &k = b.side[1];
  q.x = n.q, q.xb = n.q_strides[0], q.xt = n.q_strides[1], q.xh = n.q_strides[2];
  k.x = n.k, k.xb = n.k_strides[0], k.xt = n.k_strides[1], k.xh = n.k_strides[2];
  q.w = n.q_weight, k.w = n.k_weight;
  q.heads = (int)n.heads, k.heads = (int)n.key_heads;
  return b;
}

// An item is a token with all its heads, whose angles are computed once; where there are
// fewer items than the lanes that run at once, a part of its heads.
void split(Both* b, int waves) {
  const int64_t most = (int64_t)compute_units() * waves * 64 / b->tpr;   // groups that run at once
  const int per = kBlock / b->tpr;
  for (Side& s : b->side) {
    const int64_t want = b->tokens > 0 ? (most + b->tokens - 1) / b->tokens : 1;
    const int splits = (int)std::min<int64_t>(std::max(s.heads, 1), std::max<int64_t>(want, 1));
    s.each = (s.heads + splits - 1) / splits;
    s.splits = s.each > 0 ? (s.heads + s.each - 1) / s.each : 0;
    s.blocks = (int)std::min((b->tokens * s.splits + per - 1) / per, most / per);
  }
}
constexpr int kForwardWaves = 64, kBackwardWaves = 16;

}  // namespace

hipError_t launch_qk_norm_forward(const cpab_qk_norm& n, void* q_out, void* k_out, hipStream_t st) {
  Both b = both_of(n);
  const Layout l = lay_out(n, &b);
  split(&b, kForwardWaves);
  b.side[0].out = q_out, b.side[1].out = k_out;
  const int blocks = std::max(b.side[0].blocks, b.side[1].blocks);
  if (blocks == 0) return hipSuccess;
  with_types(n, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    with_layout<T>(l, [&](auto v, auto ch) {
      constexpr int V = decltype(v)::value, CH = decltype(ch)::value;
      if (n.neighbours)
        qk_norm_forward_kernel<T, W, V, CH, true><<<dim3(blocks, 2), kBlock, 0, st>>>(b);
      else
        qk_norm_forward_kernel<T, W, V, CH, false><<<dim3(blocks, 2), kBlock, 0, st>>>(b);
    });
  });
  return hipGetLastError();
}

int64_t qk_norm_backward_workspace(const cpab_qk_norm& n) {
  Both b = both_of(n);
  lay_out(n, &b);
  split(&b, kBackwardWaves);
  return ((int64_t)b.side[0].blocks + b.side[1].blocks) * n.width * 4;
}

hipError_t launch_qk_norm_backward(const cpab_qk_norm& n, const void* const grads[2],
                                   const int64_t grad_strides[6], void* const outs[2],
                                   void* const weight_outs[2], void* workspace, hipStream_t st) {
  Both b = both_of(n);
  const Layout l = lay_out(n, &b);
  split(&b, kBackwardWaves);
  b.parts = static_cast<float*>(workspace);
  for (int k = 0; k < 2; ++k) {
    Side& s = b.side[k];
    s.dy = grads[k];
    s.db = grad_strides[3 * k], s.dt = grad_strides[3 * k + 1], s.dh = grad_strides[3 * k + 2];
    s.out = outs[k];
    s.dw = weight_outs[k];
    if (!s.out && !s.dw) s.blocks = 0;   // nothing is wanted of this side
  }
  b.side[1].parts = (int64_t)b.side[0].blocks * n.width;
  const int blocks = std::max(b.side[0].blocks, b.side[1].blocks);
  with_types(n, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    if (blocks > 0)
      with_layout<T>(l, [&](auto v, auto ch) {
        constexpr int V = decltype(v)::value, CH = decltype(ch)::value;
        const size_t lds = (size_t)kBlock / 64 * n.width * 4;
        if (n.neighbours)
          qk_norm_backward_kernel<T, W, V, CH, true><<<dim3(blocks, 2), kBlock, lds, st>>>(b);
        else
          qk_norm_backward_kernel<T, W, V, CH, false><<<dim3(blocks, 2), kBlock, lds, st>>>(b);
      });
    if (weight_outs[0] || weight_outs[1])
      qk_norm_weight_kernel<W><<<dim3((unsigned)(n.width + 15) / 16, 2), 1024, 0, st>>>(b);
  });
  return hipGetLastError();
}

}  // namespace cpab
