// Gated linear recurrence: a = sigmoid(f), h_t = a_t h_{t-1} + (1 - a_t) x_t,
// y = h g sigmoid(g), and its gradient.
//
// Backward: with l_t the gradient of h_t through everything after it,
//   l_t = dy_t silu(g_t) + a_{t+1} l_{t+1},   l at the row's end also + grad_h_last,
//   dx = (1 - a) l,  df = l (h_{t-1} - x) a (1 - a)  (sigmoid' = a (1 - a)),
//   dg = dy h s (1 + g (1 - s)),  s = sigmoid(g),  dh0 = a_0 l_0.
// h is computed again from the state that the forward kept before each tile.
//
// A run of samples maps the state before it to the state after it by h -> A h + B,
// with A the product of its a, so runs can be worked on side by side and joined.  A
// workgroup takes a tile: `lanes` lanes of V channels across, `segs` segments of L
// samples each along the time, one segment to a lane, its samples in registers from
// one load to the end.  A segment's (A, B) goes to LDS, the tile's to memory; with the
// state before the tile each lane then runs through its samples once more.
//
// The state before a tile comes from the tiles before it in the same launch: each
// publishes its (A, B) as soon as it has it, and the state after it once it knows the
// state before it.  A tile looks at its `segs` nearest predecessors until one of them
// has its state, and applies the (A, B) in between in the order of time.  Since a
// state is always fma(A, state before, B), it has the same bits wherever the look-back
// finds one, so results do not depend on timing.  Tiles are taken in the order of
// their tickets, so a tile's predecessors are held by workgroups that run already, and
// each of those publishes its (A, B) without waiting: every wait ends.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cpab_launch.hpp"
#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

constexpr int kForwardSteps = 16, kBackwardSteps = 8;   // L
constexpr int kBlock = 512;                             // lanes of a workgroup, at most

// How a launch cuts [B, T, C] into tiles.
struct Tiling {
  int lanes, segs, block;
  int64_t tiles, across, chains;   // tiles along T and C; across * B
};

__device__ __forceinline__ int64_t row_length(const Recurrence& r, int64_t b) {
  if (!r.lengths) return r.T;
  const int64_t n = r.lengths64 ? static_cast<const int64_t*>(r.lengths)[b]
                                : (int64_t)static_cast<const int32_t*>(r.lengths)[b];
  return n < 0 ? 0 : (n > r.T ? r.T : n);
}

// ---- a tile's map or state as one 64-bit word ------------------------------------
// One relaxed atomic carries it whole, so nothing else has to be ordered.  0: nothing
// yet.  A map has A, which is in [0, 1] or NaN, with its sign bit set in the upper half
// and B in the lower; a state is under the pattern of -2.
typedef unsigned long long Word;
constexpr uint32_t kState = 0xC0000000u;
__device__ __forceinline__ Word map_word(float A, float B) {
  return (Word)(__float_as_uint(A) | 0x80000000u) << 32 | __float_as_uint(B);
}
__device__ __forceinline__ Word state_word(float h) { return (Word)kState << 32 | __float_as_uint(h); }
__device__ __forceinline__ bool is_state(Word w) { return (uint32_t)(w >> 32) == kState; }
__device__ __forceinline__ float word_B(Word w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ float word_A(Word w) {
  return __uint_as_float((uint32_t)(w >> 32) & 0x7fffffffu);
}
__device__ __forceinline__ void publish(Word* at, Word w) {
  __hip_atomic_store(at, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Word await(Word* at) {
  Word w;
  while ((w = __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == 0)
    __builtin_amdgcn_s_sleep(1);
  return w;
}

// What joins a workgroup's segments and tiles; `before` counts tiles in the order in
// which the state travels (forward: time, backward: against it).
template <int V>
struct Join {
  const Tiling& s;
  float2* agg;     // LDS [segs][lanes * V]: the segments' (A, B)
  Word* window;    // LDS [segs][lanes * V]
  Word* words;     // [chains' tiles, B, C]
  int seg, lane;

  __device__ float2& at(int sg, int v) const { return agg[(sg * s.lanes + lane) * V + v]; }
  // Of the whole tile, segments taken from `first` in steps of `dir`.
  __device__ void whole(int first, int dir, float A[V], float B[V]) const {
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
    for (int k = 0, sg = first; k < s.segs; ++k, sg += dir)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = at(sg, v);
        B[v] = fmaf(m.x, B[v], m.y);
        A[v] *= m.x;
      }
  }
  // The state before this tile, from the tiles before it (`before` > 0 of them):
  // word of the k-th before is words[k * stride + channel].  Called by every lane.
  __device__ void look_back(int64_t before, Word* last, int64_t stride, float h[V]) const {
    bool all;
    do {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        Word w = state_word(0.0f);   // beyond the first tile: not looked at
        if (seg < before) w = await(last - seg * stride + v);
        window[(seg * s.lanes + lane) * V + v] = w;
      }
      __syncthreads();
      bool found = true;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        int k = 0;
        Word w = 0;
        for (; k < s.segs; ++k) {
          w = window[(k * s.lanes + lane) * V + v];
          if (is_state(w)) break;
        }
        found &= k < s.segs;
        h[v] = word_B(w);
        for (--k; k >= 0; --k) {
          w = window[(k * s.lanes + lane) * V + v];
          h[v] = fmaf(word_A(w), h[v], word_B(w));
        }
      }
      all = __syncthreads_and(found);
    } while (!all);
  }
};

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float out[V]) {
  T raw[V];
  __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = to_float(raw[v]);
}
template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float in[V]) {
  T raw[V];
#pragma unroll
  for (int v = 0; v < V; ++v) raw[v] = from_float<T>(in[v]);
  __builtin_memcpy(p, raw, sizeof(raw));
}

// This workgroup's tile: its ticket where tiles wait for others, else its index.
__device__ __forceinline__ int64_t take_tile(const Tiling& s, unsigned* ticket) {
  __shared__ unsigned mine;
  if (s.tiles == 1) return blockIdx.x;
  if (threadIdx.x == 0) mine = atomicAdd(ticket, 1u);
  __syncthreads();
  return mine;
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(kBlock)
recurrence_forward_kernel(Recurrence r, Tiling s, T* y, float* h_last, float* carries,
                          Tiling back, Word* words, unsigned* ticket) {
  constexpr int L = kForwardSteps;
  extern __shared__ char room[];
  const int seg = threadIdx.x / s.lanes, lane = threadIdx.x % s.lanes;
  const int64_t mine = take_tile(s, ticket);
  const int64_t tile = mine / s.chains, chain = mine - tile * s.chains;
  const int64_t b = chain / s.across;
  // lanes beyond the last channels repeat those
  const int64_t c = min(((chain - b * s.across) * s.lanes + lane) * V, r.C - V);
  const int64_t n = row_length(r, b), t0 = tile * s.segs * L, t1 = t0 + s.segs * L;
  const int64_t ts = t0 + seg * L;
  T* out = y + (b * r.T + ts) * r.C + c;
  const float none[V] = {};
  if (t0 >= n && tile > 0) {
    for (int j = 0; j < L && ts + j < r.T; ++j) store<T, V>(out + j * r.C, none);
    return;
  }
  const int live = (int)max((int64_t)0, min((int64_t)L, n - ts));
  float a[L][V], u[L][V], g[L][V];
  const T* x = static_cast<const T*>(r.x) + b * r.xb + ts * r.xt + c;
  const T* f = static_cast<const T*>(r.f) + b * r.fb + ts * r.ft + c;
  const T* gp = GATE ? static_cast<const T*>(r.g) + b * r.gb + ts * r.gt + c : nullptr;
#pragma unroll
  for (int j = 0; j < L; ++j) {
#pragma unroll
    for (int v = 0; v < V; ++v) a[j][v] = INFINITY, u[j][v] = 0.0f, g[j][v] = 0.0f;
    if (j < live) {
      load<T, V>(f + j * r.ft, a[j]);
      load<T, V>(x + j * r.xt, u[j]);
      if (GATE) load<T, V>(gp + j * r.gt, g[j]);
    }
  }
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
  for (int j = 0; j < L; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gate k = sigmoids(a[j][v]);
      a[j][v] = k.pos;
      u[j][v] *= k.neg;
      B[v] = fmaf(k.pos, B[v], u[j][v]);
      A[v] *= k.pos;
    }
  const Join<V> join{s, reinterpret_cast<float2*>(room),
                     reinterpret_cast<Word*>(room) + s.segs * s.lanes * V, words, seg, lane};
#pragma unroll
  for (int v = 0; v < V; ++v) join.at(seg, v) = make_float2(A[v], B[v]);
  __syncthreads();
  float h[V];
  Word* own = words + (tile * r.B + b) * r.C + c;
  if (tile == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = r.h0 ? r.h0[b * r.C + c + v] : 0.0f;
  }
  const bool follows = t1 < n;   // a live tile comes after this one
  if (seg == 0 && follows) join.whole(0, 1, A, B);
  if (tile > 0) {
    if (seg == 0 && follows)
#pragma unroll
      for (int v = 0; v < V; ++v) publish(own + v, map_word(A[v], B[v]));
    join.look_back(tile, own - r.B * r.C, r.B * r.C, h);
  }
  if (seg == 0 && follows)
#pragma unroll
    for (int v = 0; v < V; ++v) publish(own + v, state_word(fmaf(A[v], h[v], B[v])));
  for (int sg = 0; sg < seg; ++sg)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = join.at(sg, v);
      h[v] = fmaf(m.x, h[v], m.y);
    }
  if (carries) {   // where a tile of the backward begins, at the start of a segment
    const int span = back.segs * kBackwardSteps;
    if (ts % span == 0 && ts < r.T)
#pragma unroll
      for (int v = 0; v < V; ++v) carries[(b * back.tiles + ts / span) * r.C + c + v] = h[v];
  }
#pragma unroll
  for (int j = 0; j < L; ++j) {
    float o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = fmaf(a[j][v], h[v], u[j][v]);
      o[v] = GATE ? h[v] * (g[j][v] * sigmoids(g[j][v]).pos) : h[v];
    }
    if (j < live)
      store<T, V>(out + j * r.C, o);
    else if (ts + j < r.T)
      store<T, V>(out + j * r.C, none);
  }
  if (!follows && seg == s.segs - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) h_last[b * r.C + c + v] = h[v];
  }
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(kBlock)
recurrence_backward_kernel(Recurrence r, Tiling s, const float* carries, const T* dy,
                           const float* dh_last, T* dx, T* df, T* dg, float* dh0, Word* words,
                           unsigned* ticket) {
  constexpr int L = kBackwardSteps;
  extern __shared__ char room[];
  const int seg = threadIdx.x / s.lanes, lane = threadIdx.x % s.lanes;
  const int64_t mine = take_tile(s, ticket);
  const int64_t order = mine / s.chains, chain = mine - order * s.chains;
  const int64_t tile = s.tiles - 1 - order;
  const int64_t b = chain / s.across;
  const int64_t c = min(((chain - b * s.across) * s.lanes + lane) * V, r.C - V);
  const int64_t n = row_length(r, b), t0 = tile * s.segs * L, t1 = t0 + s.segs * L;
  const int64_t ts = t0 + seg * L;
  const int64_t row = (b * r.T + ts) * r.C + c;
  const float none[V] = {};
  if (t0 >= n && tile > 0) {
    for (int j = 0; j < L && ts + j < r.T; ++j) {
      if (dx) store<T, V>(dx + row + j * r.C, none);
      if (df) store<T, V>(df + row + j * r.C, none);
      if (GATE && dg) store<T, V>(dg + row + j * r.C, none);
    }
    return;
  }
  const int live = (int)max((int64_t)0, min((int64_t)L, n - ts));
  float f[L][V], x[L][V], g[L][V], d[L][V];
  const T* xp = static_cast<const T*>(r.x) + b * r.xb + ts * r.xt + c;
  const T* fp = static_cast<const T*>(r.f) + b * r.fb + ts * r.ft + c;
  const T* gp = GATE ? static_cast<const T*>(r.g) + b * r.gb + ts * r.gt + c : nullptr;
#pragma unroll
  for (int j = 0; j < L; ++j) {
#pragma unroll
    for (int v = 0; v < V; ++v) f[j][v] = INFINITY, x[j][v] = 0.0f, g[j][v] = 0.0f, d[j][v] = 0.0f;
    if (j < live) {
      load<T, V>(fp + j * r.ft, f[j]);
      load<T, V>(xp + j * r.xt, x[j]);
      if (GATE) load<T, V>(gp + j * r.gt, g[j]);
      if (dy) load<T, V>(dy + row + j * r.C, d[j]);
    }
  }
  float A[V], B[V], h[V];
  float a[L][V], k[L][V];   // the gate and its complement
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
  for (int j = 0; j < L; ++j)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const Gate q = sigmoids(f[j][v]);
      a[j][v] = q.pos;
      k[j][v] = q.neg;
      B[v] = fmaf(q.pos, B[v], q.neg * x[j][v]);
      A[v] *= q.pos;
    }
  const Join<V> join{s, reinterpret_cast<float2*>(room),
                     reinterpret_cast<Word*>(room) + s.segs * s.lanes * V, words, seg, lane};
#pragma unroll
  for (int v = 0; v < V; ++v) join.at(seg, v) = make_float2(A[v], B[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = carries[(b * s.tiles + tile) * r.C + c + v];
  __syncthreads();
  for (int sg = 0; sg < seg; ++sg)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = join.at(sg, v);
      h[v] = fmaf(m.x, h[v], m.y);
    }
  // through the samples: dg, and f becomes (h_{t-1} - x) a (1 - a), d what reaches h_t
#pragma unroll
  for (int j = 0; j < L; ++j) {
    float o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      f[j][v] = (h[v] - x[j][v]) * (a[j][v] * k[j][v]);
      h[v] = fmaf(a[j][v], h[v], k[j][v] * x[j][v]);
      if (GATE) {
        const Gate q = sigmoids(g[j][v]);
        o[v] = d[j][v] * h[v] * q.pos * fmaf(g[j][v], q.neg, 1.0f);
        d[j][v] *= g[j][v] * q.pos;
      }
    }
    if (GATE && dg) {
      if (j < live)
        store<T, V>(dg + row + j * r.C, o);
      else if (ts + j < r.T)
        store<T, V>(dg + row + j * r.C, none);
    }
  }
  // what a segment hands to the sample before it: A (what it is handed) + B
#pragma unroll
  for (int v = 0; v < V; ++v) B[v] = 0.0f;
#pragma unroll
  for (int j = L - 1; j >= 0; --j)
#pragma unroll
    for (int v = 0; v < V; ++v) B[v] = a[j][v] * (B[v] + d[j][v]);
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) join.at(seg, v) = make_float2(A[v], B[v]);
  __syncthreads();
  float l[V];
  Word* own = words + (tile * r.B + b) * r.C + c;
  const bool last = t1 >= n;   // the row's last live tile
  if (last) {
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = dh_last ? dh_last[b * r.C + c + v] : 0.0f;
  }
  if (seg == 0 && tile > 0) join.whole(s.segs - 1, -1, A, B);
  if (!last) {
    if (seg == 0 && tile > 0)
#pragma unroll
      for (int v = 0; v < V; ++v) publish(own + v, map_word(A[v], B[v]));
    // tiles after this one that are live
    const int64_t span = (int64_t)s.segs * L;
    join.look_back((n + span - 1) / span - 1 - tile, own + r.B * r.C, -(r.B * r.C), l);
  }
  if (seg == 0 && tile > 0)
#pragma unroll
    for (int v = 0; v < V; ++v) publish(own + v, state_word(fmaf(A[v], l[v], B[v])));
  for (int sg = s.segs - 1; sg > seg; --sg)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 m = join.at(sg, v);
      l[v] = fmaf(m.x, l[v], m.y);
    }
#pragma unroll
  for (int j = L - 1; j >= 0; --j) {
    float ox[V], of[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      l[v] += d[j][v];
      ox[v] = k[j][v] * l[v];
      of[v] = l[v] * f[j][v];
      l[v] *= a[j][v];
    }
    const bool in = j < live;
    if (ts + j < r.T) {
      if (dx) store<T, V>(dx + row + j * r.C, in ? ox : none);
      if (df) store<T, V>(df + row + j * r.C, in ? of : none);
    }
  }
  if (dh0 && tile == 0 && seg == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) dh0[b * r.C + c + v] = l[v];
  }
}

int pow2_at_least(int64_t n, int most) {
  int p = 1;
  while (p < n && p < most) p *= 2;
  return p;
}

// Channels of a lane.
int channels(int dtype, int64_t C) { return dtype == CPAB_BF16 && C > 64 ? 2 : 1; }

Tiling tiling(int dtype, int64_t B, int64_t T, int64_t C, int L) {
  Tiling s;
  const int V = channels(dtype, C);
  s.lanes = pow2_at_least((C + V - 1) / V, 64);
  // as many segments as the samples fill, up to the workgroup's lanes
  s.segs = pow2_at_least((T + L - 1) / L, kBlock / s.lanes);
  s.segs = std::max(s.segs, 64 / s.lanes);
  s.block = s.lanes * s.segs;
  s.tiles = std::max<int64_t>(1, (T + (int64_t)s.segs * L - 1) / ((int64_t)s.segs * L));
  s.across = (C + (int64_t)s.lanes * V - 1) / ((int64_t)s.lanes * V);
  s.chains = s.across * B;
  return s;
}

size_t lds_bytes(const Tiling& s, int V) {
  return (size_t)s.block * V * (sizeof(float2) + (s.tiles > 1 ? sizeof(Word) : 0));
}

// f(T(), V, GATE) for the call's types, as constants.
template <typename F>
void with_shape(int dtype, int V, bool gate, F f) {
  const auto types = [&](auto g) {
    if (dtype == CPAB_F32) return f(0.0f, std::integral_constant<int, 1>(), g);
    if (V == 1) return f(bf16(), std::integral_constant<int, 1>(), g);
    return f(bf16(), std::integral_constant<int, 2>(), g);
  };
  gate ? types(std::true_type()) : types(std::false_type());
}

}  // namespace

bool recurrence_fits(int dtype, int64_t B, int64_t T, int64_t C) {
  for (const int L : {kForwardSteps, kBackwardSteps}) {
    const Tiling s = tiling(dtype, B, T, C, L);
    if ((double)s.tiles * (double)s.chains * s.block >= 4294967296.0) return false;
  }
  return true;
}

int64_t recurrence_carries(int dtype, int64_t B, int64_t T, int64_t C) {
  return T == 0 ? 0 : B * tiling(dtype, B, T, C, kBackwardSteps).tiles * C;
}

// A ticket (16 bytes) and a word for each tile and channel.
int64_t recurrence_workspace(int dtype, int64_t B, int64_t T, int64_t C, bool backward) {
  const int64_t tiles = tiling(dtype, B, T, C, backward ? kBackwardSteps : kForwardSteps).tiles;
  return tiles > 1 ? 16 + tiles * B * C * (int64_t)sizeof(Word) : 0;
}

hipError_t launch_recurrence_forward(int dtype, const Recurrence& r, void* y, float* h_last,
                                     float* carries, void* workspace, hipStream_t st) {
  const Tiling s = tiling(dtype, r.B, r.T, r.C, kForwardSteps);
  const Tiling back = tiling(dtype, r.B, r.T, r.C, kBackwardSteps);
  const int64_t bytes = recurrence_workspace(dtype, r.B, r.T, r.C, false);
  if (bytes) {
    const hipError_t e = launch_fill(static_cast<float*>(workspace), bytes / 4, 0.0f, st);
    if (e != hipSuccess) return e;
  }
  const int V = channels(dtype, r.C);
  with_shape(dtype, V, r.g != nullptr, [&](auto t, auto vs, auto gate) {
    typedef decltype(t) T;
    recurrence_forward_kernel<T, decltype(vs)::value, decltype(gate)::value>
        <<<(unsigned)(s.tiles * s.chains), s.block, lds_bytes(s, V), st>>>(
            r, s, (T*)y, h_last, carries, back, bytes ? (Word*)workspace + 2 : nullptr,
            (unsigned*)workspace);
  });
  return hipGetLastError();
}

hipError_t launch_recurrence_backward(int dtype, const Recurrence& r, const float* carries,
                                      const void* dy, const float* dh_last, void* dx, void* df,
                                      void* dg, float* dh0, void* workspace, hipStream_t st) {
  if (r.T == 0) {
    if (!dh0) return hipSuccess;
    if (!dh_last) return launch_fill(dh0, r.B * r.C, 0.0f, st);
    return hipMemcpyAsync(dh0, dh_last, r.B * r.C * 4, hipMemcpyDeviceToDevice, st);
  }
  const Tiling s = tiling(dtype, r.B, r.T, r.C, kBackwardSteps);
  const int64_t bytes = recurrence_workspace(dtype, r.B, r.T, r.C, true);
  if (bytes) {
    const hipError_t e = launch_fill(static_cast<float*>(workspace), bytes / 4, 0.0f, st);
    if (e != hipSuccess) return e;
  }
  const int V = channels(dtype, r.C);
  with_shape(dtype, V, r.g != nullptr, [&](auto t, auto vs, auto gate) {
    typedef decltype(t) T;
    recurrence_backward_kernel<T, decltype(vs)::value, decltype(gate)::value>
        <<<(unsigned)(s.tiles * s.chains), s.block, lds_bytes(s, V), st>>>(
            r, s, carries, (const T*)dy, dh_last, (T*)dx, (T*)df, (T*)dg, dh0,
            bytes ? (Word*)workspace + 2 : nullptr, (unsigned*)workspace);
  });
  return hipGetLastError();
}

}  // namespace cpab
