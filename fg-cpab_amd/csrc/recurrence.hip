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
// state before it.  A tile looks at its kWindow predecessors until one of them has its
// state, and applies the (A, B) in between in the order of time.  Since the state after a
// tile is always fma(A, state before, B), it has the same bits wherever the look-back
// finds one, so results do not depend on timing.  Tiles are taken by tickets, so those
// before a tile are held by workgroups that run already, and each publishes its (A, B)
// without waiting: every wait ends.
//
// One wave of a workgroup polls, and only a flag to each tile; the words of the channels
// are read once, when the flags say that they are there (all lanes polling the words took
// the memory's bandwidth from the samples).
//
// Bound by memory: 8 x 4096 x 1280 bfloat16 forward 74 us and backward 143, 4.5 and 4.1
// TB/s of what has to be read and written (a profile's 77 and 147; 69 and 132 without the
// look-back).  With few chains the look-back counts: one row of 131,072 x 512, forward, 127
// us, 99 without; 16 ragged rows of 10,000 x 64 in 32 bits 32 and 45, 28 and 42 without.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

constexpr int kBlock = 512;   // lanes of a workgroup, at most
constexpr int kWindow = 64;   // tiles that a look-back sees: a lane of a wave to each

// Samples of a lane: what registers hold at four waves to a SIMD; forward one, where the
// samples are few and their latency counts (64 x 1 x 512 bfloat16: 6.0 us with 16).
constexpr int kForwardSteps = 16, kFewSamples = 16;
int forward_steps(int64_t T) { return T <= kFewSamples ? 1 : kForwardSteps; }
constexpr int backward_steps(int V) { return 16 / V; }

// How a launch cuts [B, T, C] into tiles.
struct Tiling {
  int lanes, segs, block;          // lanes and block powers of two
  unsigned tiles, across, chains;   // tiles along T and C; across * B
};

// Samples of row b (T below 2^31), the same in every lane for the compiler too.
__device__ __forceinline__ int row_length(const Recurrence& r, int64_t b) {
  int64_t n = r.T;
  if (r.lengths)
    n = r.lengths64 ? static_cast<const int64_t*>(r.lengths)[b]
                    : (int64_t)static_cast<const int32_t*>(r.lengths)[b];
  return __builtin_amdgcn_readfirstlane((int)(n < 0 ? 0 : (n > r.T ? r.T : n)));
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
// A barrier for what lanes hand each other in LDS: unlike __syncthreads it does not wait
// for a wave's stores to memory.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr unsigned kHasMap = 1, kHasState = 2;   // a tile's flag
template <typename W>
__device__ __forceinline__ void publish(W* at, W w) {
  __hip_atomic_store(at, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename W>
__device__ __forceinline__ W peek(W* at) {
  return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What joins a workgroup's segments and the tiles.  Tiles are numbered from 0 in the
// order in which a row's state travels (forward: time, backward: against it).  A tile's
// channels are its `slots`, at most a wave of them: the first wave has a lane to each.
template <int V>
struct Join {
  const Tiling& s;
  int slots, seg, lane;
  float2* agg;     // LDS [segs][slots]: the segments' (A, B)
  Word* window;    // LDS [kWindow][slots]: the tiles before, newest first
  float* entry;    // LDS [slots]: the state before the tile
  int* nearest;    // LDS: how many tiles back the nearest state is

  __device__ Join(const Tiling& t, char* room, int* one, int sg, int ln)
      : s(t), slots(t.lanes * V), seg(sg), lane(ln), agg(reinterpret_cast<float2*>(room)),
        window(reinterpret_cast<Word*>(agg + t.segs * slots)),
        entry(reinterpret_cast<float*>(window + min(kWindow, (int)t.tiles) * slots)), nearest(one) {}
  __device__ float2& at(int sg, int v) const { return agg[sg * slots + lane * V + v]; }
  // h: from the state before the tile to that before a segment, over `count` segments
  // from `first` in steps of `dir`.
  __device__ void to_segment(int first, int count, int dir, float h[V]) const {
#pragma unroll 2
    for (int k = 0, sg = first; k < count; ++k, sg += dir)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 m = at(sg, v);
        h[v] = fmaf(m.x, h[v], m.y);
      }
  }
  // (A, B) of the whole tile in a slot, segments taken from `first` in steps of `dir`,
  // read four ahead: a step waits for a multiplication then, and not for LDS.
  __device__ float2 whole(int slot, int first, int dir) const {
    float2 all = make_float2(1.0f, 0.0f);
    for (int k = 0; k < s.segs; k += 4) {
      float2 m[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) m[q] = agg[(first + min(k + q, s.segs - 1) * dir) * slots + slot];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (k + q >= s.segs) continue;
        all.y = fmaf(m[q].x, all.y, m[q].y);
        all.x *= m[q].x;
      }
    }
    return all;
  }
  // h: the state before tile `number`, given as the state before tile 0; the segments'
  // (A, B) are in LDS, taken as in whole().  `follows`: tiles come after it.  The chain's
  // words, [tiles][slots], and flags, tile by tile.  Called by every lane.
  __device__ void state_before(int number, bool follows, int segment, int dir, Word* words,
                               unsigned* flags, float h[V]) const {
    const int slot = threadIdx.x;
    const bool carries = slot < slots;
    Word* own = words + (int64_t)number * slots + slot;
    if (number == 0) {
      if (!follows) return;
      if (seg == 0)
#pragma unroll
        for (int v = 0; v < V; ++v) entry[lane * V + v] = h[v];
      lds_barrier();
      if (carries) {
        const float2 all = whole(slot, segment, dir);
        publish(own, state_word(fmaf(all.x, entry[slot], all.y)));
        if (slot == 0) publish(flags, kHasState);
      }
      return;
    }
    // other tiles wait for this wave
    if (slot < 64) __builtin_amdgcn_s_setprio(3);
    float2 all;
    if (carries && follows) {
      all = whole(slot, segment, dir);
      publish(own, map_word(all.x, all.y));
      if (slot == 0) publish(flags + number, kHasMap);
    }
    if (threadIdx.x >= blockDim.x - 64) {   // the last wave, beside the first
      // lane k: the tile k + 1 before; what lies before tile 0 is not asked
      const int mine = number - 1 - (int)(threadIdx.x & 63);
      for (;;) {
        const unsigned f = mine >= 0 ? peek(flags + mine) : kHasMap;
        const uint64_t state = __ballot(f == kHasState), any = __ballot(f != 0);
        const int k = __builtin_ctzll(state | 1ull << 63);
        if ((state >> k & 1) && !(~any & ((1ull << k) - 1))) {
          if ((threadIdx.x & 63) == 0) *nearest = k;
          break;
        }
        __builtin_amdgcn_s_sleep(2);
      }
    }
    lds_barrier();
    // Words of the tiles up to the nearest state, two of each lane on their way at once.
    // The flags are no more than a hint: a word says itself what it is.
    const int k = *nearest, count = (k + 1) * slots, lanes = blockDim.x;
    const Word* newest = words + (int64_t)(number - 1) * slots;
    const auto ready = [&](Word w, int i) { return w != 0 && (i < k * slots || is_state(w)); };
    const auto from = [&](int i) {   // tile i / slots back, slot i % slots
      return const_cast<Word*>(newest) - (i & -slots) + (i & (slots - 1));
    };
    for (int i = threadIdx.x; i < count; i += 2 * lanes) {
      const bool two = i + lanes < count;
      Word w = peek(from(i)), x = two ? peek(from(i + lanes)) : 0;
      while (!ready(w, i)) w = peek(from(i));
      window[i] = w;
      if (!two) continue;
      while (!ready(x, i + lanes)) x = peek(from(i + lanes));
      window[i + lanes] = x;
    }
    lds_barrier();
    if (carries) {
      float state = 0.0f;
      for (int q = k; q >= 0; q -= 4) {   // read four ahead, as in whole()
        Word w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = window[max(q - e, 0) * slots + slot];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e > q) continue;
          // a tile may have come to its state since: that is then the one to take
          state = is_state(w[e]) ? word_B(w[e]) : fmaf(word_A(w[e]), state, word_B(w[e]));
        }
      }
      entry[slot] = state;
      if (follows) {
        publish(own, state_word(fmaf(all.x, state, all.y)));
        if (slot == 0) publish(flags + number, kHasState);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    lds_barrier();
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = entry[lane * V + v];
  }
};

// V neighbouring channels as they lie in memory, in registers of 32 bits.
template <typename T, int V>
struct Raw {
  static constexpr int kBytes = V * (int)sizeof(T), kWords = (kBytes + 3) / 4;
  static_assert(kBytes == 2 || kBytes == 4 || kBytes == 8, "one load");
  typedef typename std::conditional<
      kBytes == 8, uint64_t, typename std::conditional<kBytes == 4, uint32_t, uint16_t>::type>::type Bits;
  typedef Bits __attribute__((aligned(sizeof(T)))) Unit;   // in memory
  uint32_t w[kWords];
  __device__ __forceinline__ float operator[](int v) const {
    if (sizeof(T) == 4) return __uint_as_float(w[v]);
    return __uint_as_float(v & 1 ? w[v / 2] & 0xffff0000u : w[v / 2] << 16);
  }
  // Keeps the compiler from unpacking before this point (twice the registers).
  __device__ __forceinline__ void hold() {
#pragma unroll
    for (int k = 0; k < kWords; ++k) asm volatile("" : "+v"(w[k]));
  }
  static __device__ __forceinline__ Raw all(float value) {
    Raw raw;
    const uint32_t bits = __float_as_uint(value);
#pragma unroll
    for (int k = 0; k < kWords; ++k) raw.w[k] = sizeof(T) == 4 ? bits : bits >> 16 | (bits & 0xffff0000u);
    return raw;
  }
};
// A pointer that is the same for the workgroup's lanes and walks from sample to sample;
// a lane adds its 32-bit offset.
template <typename T>
struct Walk {
  __attribute__((address_space(1))) char* p;
  int64_t step;
  __device__ __forceinline__ Walk(const T* from, int64_t stride)
      : p((__attribute__((address_space(1))) char*)from), step(stride * (int64_t)sizeof(T)) {}
  __device__ __forceinline__ void next() { p += step; }
};
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load(const Walk<T>& w, uint32_t off) {
  typedef typename Raw<T, V>::Unit Unit;
  const typename Raw<T, V>::Bits bits = *(const __attribute__((address_space(1))) Unit*)(w.p + off);
  Raw<T, V> raw;
#pragma unroll
  for (int k = 0; k < Raw<T, V>::kWords; ++k) raw.w[k] = (uint32_t)((uint64_t)bits >> (32 * k));
  return raw;
}
template <typename T, int V>
__device__ __forceinline__ void store(const Walk<T>& w, uint32_t off, const float in[V]) {
  typedef typename Raw<T, V>::Unit Unit;
  T raw[V];
#pragma unroll
  for (int v = 0; v < V; ++v) raw[v] = from_float<T>(in[v]);
  // past the second-level cache, which the inputs need (16 x 10,000 x 64 in 32 bits, forward
  // and backward, through it and past it: 39 and 58 us, 33 and 49)
  __builtin_nontemporal_store((Unit)__builtin_bit_cast(Unit, raw),
                              (__attribute__((address_space(1))) Unit*)(w.p + off));
}

// Bytes from a tile's first sample to channel c of its sample t; below 2^31 for the samples
// that there are (recurrence_max_stride), and not used for others.
template <typename T>
__device__ __forceinline__ uint32_t offset(int t, int64_t stride, int64_t c) {
  return (uint32_t)((uint32_t)t * (uint32_t)stride + (uint32_t)c) * (uint32_t)sizeof(T);
}

// This workgroup's tile: by a ticket where tiles wait for others, else its index.
__device__ __forceinline__ unsigned take_tile(unsigned* counter, unsigned* room) {
  unsigned mine = blockIdx.x;
  if (counter) {
    if (threadIdx.x == 0) *room = atomicAdd(counter, 1u);
    lds_barrier();
    mine = *room;
  }
  return (unsigned)__builtin_amdgcn_readfirstlane((int)mine);
}

template <typename T, int V, bool GATE, int L>
__global__ void __launch_bounds__(kBlock, 4)
recurrence_forward_kernel(Recurrence r, Tiling s, T* y, float* h_last, float* carries,
                          Tiling back, Word* words, unsigned* flags, unsigned* counter) {
  extern __shared__ char room[];
  __shared__ unsigned mine_of;
  __shared__ int nearest;
  const int lane = threadIdx.x & (s.lanes - 1), seg = threadIdx.x >> (31 - __clz(s.lanes));
  const Join<V> join(s, room, &nearest, seg, lane);
  const float none[V] = {};
  const unsigned mine = take_tile(counter, &mine_of);
  const unsigned tile = mine / s.chains, chain = mine - tile * s.chains;
  const unsigned block = chain / s.across;
  const int64_t b = block;
  // lanes beyond the last channels repeat those
  const int64_t c = min((int64_t)((chain - block * s.across) * s.lanes + lane) * V, r.C - V);
  const int64_t n = row_length(r, b), t0 = (int64_t)tile * (s.segs * L), t1 = t0 + s.segs * L;
  const int64_t ts = t0 + seg * L;
  const int rest = (int)min((int64_t)L, r.T - ts);   // of the lane's samples those in T,
  const int live = (int)min((int64_t)L, n - ts);     // and those in the row (none: <= 0)
  Walk<T> out(y + (b * r.T + t0) * r.C, r.C);
  const uint32_t at = offset<T>(seg * L, r.C, c);
  // a tile that is whole, the usual one, needs no question at each sample
  const auto work = [&](auto whole) {
    constexpr bool full = decltype(whole)::value;
    float a[L][V], u[L][V];
    Raw<T, V> rf[L], rx[L], g[L];   // no sample: a gate that keeps the state
    Walk<T> x(static_cast<const T*>(r.x) + b * r.xb + t0 * r.xt, r.xt);
    Walk<T> f(static_cast<const T*>(r.f) + b * r.fb + t0 * r.ft, r.ft);
    Walk<T> gp(GATE ? static_cast<const T*>(r.g) + b * r.gb + t0 * r.gt : nullptr, r.gt);
    const uint32_t atx = offset<T>(seg * L, r.xt, c), atf = offset<T>(seg * L, r.ft, c);
    const uint32_t atg = offset<T>(seg * L, r.gt, c);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      rf[j] = Raw<T, V>::all(INFINITY);
      rx[j] = g[j] = Raw<T, V>::all(0.0f);
      if (full || j < live) {
        rf[j] = load<T, V>(f, atf);
        rx[j] = load<T, V>(x, atx);
        if (GATE) g[j] = load<T, V>(gp, atg);
      }
      f.next(), x.next();
      if (GATE) gp.next();
    }
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
    for (int j = 0; j < L; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate k = sigmoids<T>(rf[j][v]);
        a[j][v] = k.pos;
        u[j][v] = k.neg * rx[j][v];
        B[v] = fmaf(k.pos, B[v], u[j][v]);
        A[v] *= k.pos;
      }
#pragma unroll
    for (int v = 0; v < V; ++v) join.at(seg, v) = make_float2(A[v], B[v]);
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = r.h0 ? r.h0[b * r.C + c + v] : 0.0f;
    lds_barrier();
    const bool follows = t1 < n;   // a live tile comes after this one
    if (s.tiles > 1)
      join.state_before((int)tile, follows, 0, 1, words + (int64_t)chain * s.tiles * join.slots,
                        flags + chain * s.tiles, h);
    join.to_segment(0, seg, 1, h);
    if (carries) {   // where a tile of the backward begins, at the start of a segment
      const int span = back.segs * backward_steps(V);
      if (ts % span == 0 && ts < r.T)
#pragma unroll
        for (int v = 0; v < V; ++v)
          carries[(b * (int64_t)back.tiles + ts / span) * r.C + c + v] = h[v];
    }
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float o[V];
      if (GATE) g[j].hold();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = fmaf(a[j][v], h[v], u[j][v]);
        o[v] = GATE ? h[v] * (g[j][v] * sigmoids<T>(g[j][v]).pos) : h[v];
      }
      if (full || j < live)
        store<T, V>(out, at, o);
      else if (j < rest)
        store<T, V>(out, at, none);
      out.next();
    }
    if (!follows && seg == s.segs - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) h_last[b * r.C + c + v] = h[v];
    }
  };
  if (t0 >= n && tile > 0) {   // behind the row's end
    for (int j = 0; j < L; ++j, out.next())
      if (j < rest) store<T, V>(out, at, none);
  } else if (t1 <= n) {
    work(std::true_type());
  } else {
    work(std::false_type());
  }
}

template <typename T, int V, bool GATE>
__global__ void __launch_bounds__(kBlock, 4)
recurrence_backward_kernel(Recurrence r, Tiling s, const float* carries, const T* dy,
                           const float* dh_last, T* dx, T* df, T* dg, float* dh0,
                           Word* words, unsigned* flags, unsigned* counter) {
  constexpr int L = backward_steps(V);
  extern __shared__ char room[];
  __shared__ unsigned mine_of;
  __shared__ int nearest;
  const int lane = threadIdx.x & (s.lanes - 1), seg = threadIdx.x >> (31 - __clz(s.lanes));
  const Join<V> join(s, room, &nearest, seg, lane);
  const float none[V] = {};
  const unsigned mine = take_tile(counter, &mine_of);
  const unsigned order = mine / s.chains, chain = mine - order * s.chains;
  const unsigned tile = s.tiles - 1 - order, block = chain / s.across;
  const int64_t b = block;
  const int64_t c = min((int64_t)((chain - block * s.across) * s.lanes + lane) * V, r.C - V);
  const int64_t n = row_length(r, b), t0 = (int64_t)tile * (s.segs * L), t1 = t0 + s.segs * L;
  const int64_t ts = t0 + seg * L;
  const int rest = (int)min((int64_t)L, r.T - ts), live = (int)min((int64_t)L, n - ts);
  const int64_t row = (b * r.T + t0) * r.C;
  const uint32_t at = offset<T>(seg * L, r.C, c);
  const auto work = [&](auto whole) {
    constexpr bool full = decltype(whole)::value;
    Raw<T, V> rf[L], x[L], g[L], rd[L];
    Walk<T> xp(static_cast<const T*>(r.x) + b * r.xb + t0 * r.xt, r.xt);
    Walk<T> fp(static_cast<const T*>(r.f) + b * r.fb + t0 * r.ft, r.ft);
    Walk<T> gp(GATE ? static_cast<const T*>(r.g) + b * r.gb + t0 * r.gt : nullptr, r.gt);
    Walk<T> dyp(dy + row, r.C), dgp(dg + row, r.C);
    const uint32_t atx = offset<T>(seg * L, r.xt, c), atf = offset<T>(seg * L, r.ft, c);
    const uint32_t atg = offset<T>(seg * L, r.gt, c);
#pragma unroll
    for (int j = 0; j < L; ++j) {
      rf[j] = Raw<T, V>::all(INFINITY);
      x[j] = g[j] = rd[j] = Raw<T, V>::all(0.0f);
      if (full || j < live) {
        rf[j] = load<T, V>(fp, atf);
        x[j] = load<T, V>(xp, atx);
        if (GATE) g[j] = load<T, V>(gp, atg);
        if (dy) rd[j] = load<T, V>(dyp, at);
      }
      fp.next(), xp.next(), dyp.next();
      if (GATE) gp.next();
    }
    float A[V], B[V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.0f, B[v] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = carries[(b * (int64_t)s.tiles + tile) * r.C + c + v];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      rf[j].hold(), x[j].hold();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate q = sigmoids<T>(rf[j][v]);
        B[v] = fmaf(q.pos, B[v], q.neg * x[j][v]);
        A[v] *= q.pos;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) join.at(seg, v) = make_float2(A[v], B[v]);
    lds_barrier();
    join.to_segment(0, seg, 1, h);
    // Through the samples: dg; k the gate, folded, f (h_{t-1} - x) a (1 - a), d what
    // reaches h_t.  The gates are computed again (two registers a value less across the
    // join) and kept folded: l may come to a sample through closed gates alone, so a has to
    // be held to its own last places, as 1 - a has.
    float k[L][V], f[L][V], d[L][V];
#pragma unroll
    for (int j = 0; j < L; ++j) {
      float o[V];
      rf[j].hold(), x[j].hold(), rd[j].hold();
      if (GATE) g[j].hold();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        k[j][v] = folded<T>(rf[j][v]);
        const Gate q = unfolded(k[j][v]);
        f[j][v] = (h[v] - x[j][v]) * (q.pos * q.neg);
        h[v] = fmaf(q.pos, h[v], q.neg * x[j][v]);
        if (GATE) {
          const Gate z = sigmoids<T>(g[j][v]);
          o[v] = rd[j][v] * h[v] * z.pos * fmaf(g[j][v], z.neg, 1.0f);
          d[j][v] = rd[j][v] * (g[j][v] * z.pos);
        } else {
          d[j][v] = rd[j][v];
        }
        // here and not where it is used: the parts would take more registers
        asm volatile("" : "+v"(f[j][v]), "+v"(d[j][v]));
      }
      if (GATE && dg) {
        if (full || j < live)
          store<T, V>(dgp, at, o);
        else if (j < rest)
          store<T, V>(dgp, at, none);
      }
      if (GATE) dgp.next();
    }
    // what a segment hands to the sample before it: A (what it is handed) + B
#pragma unroll
    for (int v = 0; v < V; ++v) B[v] = 0.0f;
#pragma unroll
    for (int j = L - 1; j >= 0; --j)
#pragma unroll
      for (int v = 0; v < V; ++v) B[v] = unfolded(k[j][v]).pos * (B[v] + d[j][v]);
    lds_barrier();
#pragma unroll
    for (int v = 0; v < V; ++v) join.at(seg, v) = make_float2(A[v], B[v]);
    float l[V];
#pragma unroll
    for (int v = 0; v < V; ++v) l[v] = dh_last ? dh_last[b * r.C + c + v] : 0.0f;
    lds_barrier();
    if (s.tiles > 1) {
      const int span = s.segs * L;
      const int after = n > 0 ? (int)((n - 1) / span) - (int)tile : 0;   // live tiles after it
      join.state_before(after, tile > 0, s.segs - 1, -1,
                        words + (int64_t)chain * s.tiles * join.slots, flags + chain * s.tiles, l);
    }
    join.to_segment(s.segs - 1, s.segs - 1 - seg, -1, l);
    Walk<T> dxp(dx + row + (L - 1) * r.C, -r.C), dfp(df + row + (L - 1) * r.C, -r.C);
#pragma unroll
    for (int j = L - 1; j >= 0; --j) {
      float ox[V], of[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const Gate q = unfolded(k[j][v]);
        l[v] += d[j][v];
        ox[v] = q.neg * l[v];
        of[v] = l[v] * f[j][v];
        l[v] *= q.pos;
      }
      const bool in = full || j < live;
      if (full || j < rest) {
        if (dx) store<T, V>(dxp, at, in ? ox : none);
        if (df) store<T, V>(dfp, at, in ? of : none);
      }
      dxp.next(), dfp.next();
    }
    if (dh0 && tile == 0 && seg == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) dh0[b * r.C + c + v] = l[v];
    }
  };
  if (t0 >= n && tile > 0) {
    Walk<T> dxp(dx + row, r.C), dfp(df + row, r.C), dgp(dg + row, r.C);
    for (int j = 0; j < L; ++j, dxp.next(), dfp.next(), dgp.next()) {
      if (j >= rest) continue;
      if (dx) store<T, V>(dxp, at, none);
      if (df) store<T, V>(dfp, at, none);
      if (GATE && dg) store<T, V>(dgp, at, none);
    }
  } else if (t1 <= n) {
    work(std::true_type());
  } else {
    work(std::false_type());
  }
}

int pow2_at_least(int64_t n, int most) {
  int p = 1;
  while (p < n && p < most) p *= 2;
  return p;
}

int channels(int dtype, int64_t C) { return dtype == CPAB_BF16 && C > 1 ? 2 : 1; }

Tiling tiling(int dtype, int64_t B, int64_t T, int64_t C, bool backward) {
  Tiling s;
  const int V = channels(dtype, C), L = backward ? backward_steps(V) : forward_steps(T);
  // 32 lanes of 4 bytes are a cache line across, and the more segments the fewer tiles
  // for a state to pass (8 x 4096 x 1280 bfloat16, forward and backward: 74 and 143 us, with
  // 16 lanes 93 and 192, in half as many segments 87 and 143; one row of 131,072 x 512,
  // forward, 124, 141 and 188; 16 x 10,000 x 64 in 32 bits 33 and 47, 39 and 64, 46 and 51).
  // At least 8, so that a few channels do not make thousands of segments.  Rows of 32-bit
  // values that are not whole lines have the line at a tile's edge read twice and written
  // in two parts: 64 lanes, where there is work enough, beside each step too, that half as
  // many segments do not tell.  Forward and backward, us, 32 and 64 lanes:
  //   by the rows beside each step   1 x 60,000 x 150 152 and 153   1 x 40,000 x 200 124 and 128
  //     1 x 40,000 x 232 133 and 129   1 x 40,000 x 300 181 and 162   2 x 40,000 x 116 149 and 132
  //   by the values                  64 x 200 x 300 77 and 85       64 x 300 x 300 98 and 86
  //     128 x 100 x 500 94 and 79      16 x 1700 x 300 126 and 104    4 x 8000 x 1111 588 and 442
  //   whole lines                    4 x 26,204 x 160 131 and 144
  // A wave cannot have a lane to each of twice as many channels of 16 bits.
  const bool edges = dtype == CPAB_F32 && C % 32 != 0 && T > kFewSamples && B * C > 216 &&
                     B * T * C > (1 << 22);
  s.lanes = std::max(8, pow2_at_least((C + V - 1) / V, edges ? 64 : 32));
  // as many segments as the samples fill, up to the workgroup's lanes
  s.segs = pow2_at_least((T + L - 1) / L, kBlock / s.lanes);
  s.segs = std::max(s.segs, 64 / s.lanes);
  s.block = s.lanes * s.segs;
  s.tiles = (unsigned)std::max<int64_t>(1, (T + (int64_t)s.segs * L - 1) / ((int64_t)s.segs * L));
  s.across = (unsigned)((C + (int64_t)s.lanes * V - 1) / ((int64_t)s.lanes * V));
  s.chains = (unsigned)(s.across * B);
  return s;
}

size_t lds_bytes(const Tiling& s, int V) {
  const size_t row = (size_t)s.lanes * V * sizeof(float2);
  return s.segs * row + (s.tiles > 1 ? std::min<size_t>(kWindow, s.tiles) * row + row / 2 : 0);
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

// The workspace: a ticket counter (16 bytes), a word for each channel of each tile, and
// a flag for each tile.
struct Room {
  unsigned *counter = nullptr, *flags = nullptr;
  Word* words = nullptr;
  hipError_t clear(const Tiling& s, int V, void* workspace, hipStream_t st) {
    if (s.tiles == 1) return hipSuccess;
    counter = static_cast<unsigned*>(workspace);
    words = static_cast<Word*>(workspace) + 2;
    flags = reinterpret_cast<unsigned*>(words + (int64_t)s.tiles * s.chains * s.lanes * V);
    return launch_fill(static_cast<float*>(workspace), bytes(s, V) / 4, 0.0f, st);
  }
  static int64_t bytes(const Tiling& s, int V) {
    if (s.tiles == 1) return 0;
    return 16 + (int64_t)s.tiles * s.chains * (s.lanes * V * (int64_t)sizeof(Word) + 4);
  }
};

}  // namespace

int64_t recurrence_max_stride(int dtype, int64_t B, int64_t T, int64_t C) {
  int64_t span = 2;   // samples of a tile, those that there are
  for (const bool backward : {false, true}) {
    const int L = backward ? backward_steps(channels(dtype, C)) : forward_steps(T);
    span = std::max(span, std::min<int64_t>(tiling(dtype, B, T, C, backward).segs * L, T));
  }
  return ((1LL << 31) / (dtype == CPAB_F32 ? 4 : 2) - 1 - C) / (span - 1);
}

bool recurrence_fits(int dtype, int64_t B, int64_t T, int64_t C) {
  for (const bool backward : {false, true}) {
    const Tiling s = tiling(dtype, B, T, C, backward);
    if ((double)s.tiles * (double)s.across * (double)B * s.block >= 4294967296.0) return false;
  }
  return T <= 1 || recurrence_max_stride(dtype, B, T, C) >= C;   // y's samples
}

int64_t recurrence_carries(int dtype, int64_t B, int64_t T, int64_t C) {
  return T == 0 ? 0 : B * (int64_t)tiling(dtype, B, T, C, true).tiles * C;
}

int64_t recurrence_workspace(int dtype, int64_t B, int64_t T, int64_t C, bool backward) {
  return Room::bytes(tiling(dtype, B, T, C, backward), channels(dtype, C));
}

hipError_t launch_recurrence_forward(int dtype, const Recurrence& r, void* y, float* h_last,
                                     float* carries, void* workspace, hipStream_t st) {
  const Tiling s = tiling(dtype, r.B, r.T, r.C, false), back = tiling(dtype, r.B, r.T, r.C, true);
  const int V = channels(dtype, r.C);
  Room room;
  const hipError_t e = room.clear(s, V, workspace, st);
  if (e != hipSuccess) return e;
  with_shape(dtype, V, r.g != nullptr, [&](auto t, auto vs, auto gate) {
    typedef decltype(t) T;
    constexpr int W = decltype(vs)::value;
    constexpr bool G = decltype(gate)::value;
    const auto k = forward_steps(r.T) == 1 ? recurrence_forward_kernel<T, W, G, 1>
                                           : recurrence_forward_kernel<T, W, G, kForwardSteps>;
    k<<<s.tiles * s.chains, s.block, lds_bytes(s, V), st>>>(r, s, (T*)y, h_last, carries, back,
                                                            room.words, room.flags, room.counter);
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
  const Tiling s = tiling(dtype, r.B, r.T, r.C, true);
  const int V = channels(dtype, r.C);
  Room room;
  const hipError_t e = room.clear(s, V, workspace, st);
  if (e != hipSuccess) return e;
  with_shape(dtype, V, r.g != nullptr, [&](auto t, auto vs, auto gate) {
    typedef decltype(t) T;
    recurrence_backward_kernel<T, decltype(vs)::value, decltype(gate)::value>
        <<<s.tiles * s.chains, s.block, lds_bytes(s, V), st>>>(
            r, s, carries, (const T*)dy, dh_last, (T*)dx, (T*)df, (T*)dg, dh0, room.words,
            room.flags, room.counter);
  });
  return hipGetLastError();
}

}  // namespace cpab
