// Gated delta rule, backward: the states' gradients through the chain of chunks, then
// everything else by chunks.  The formulas stand in delta_device.hpp.
#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "delta_device.hpp"

namespace cpab {
namespace {

// ---- the chain of chunks, backwards --------------------------------------------

// As the forward's chain: 32 columns of the state's gradient in registers, back through a
// segment's chunks.  Keeps the gradient after each chunk and E, and writes grad_v and
// grad_h0.  M and P lie transposed.  ENDS: only what the segment adds to the gradient before
// it.
template <typename T, int DP, bool ENDS>
__global__ __launch_bounds__(kDeltaBlock, 2) void delta_back_chain_kernel(
    Delta d, const Squares<T>* squares, const Keys<T, DP>* keys, Cut cut, const T* grad_o,
    const float* grad_h, const float* starts, T* grad_v, float* grad_h0, float* dstates, float* es,
    float* adds) {
  typedef Shares<DP> Sh;
  constexpr int E = kWide, kPitch = DP + 8, NV = Parts<T>::kValue, NI = Parts<T>::kInput, kSteps = DP / 32;
  constexpr int kState = E * kPitch, kSamples = E * kRow;   // planes
  extern __shared__ __align__(16) bf16 lds[];
  bf16* St = lds;                       // the gradient, [32][DP]
  bf16* Bt = St + NV * kState;          // beta dU, [32][64]
  bf16* Zt = Bt + NV * kSamples;        // - exp(G) Z
  bf16* Ot = Zt + NV * kSamples;        // dO, as the input that it is
  bf16* Gt = Ot + NI * kSamples;        // scale exp(G) dO
  const int dk = (int)d.r.dk, dv = (int)d.r.dv, wide = (dv + 7) / 8 * 8;
  const int64_t heads = d.r.B * d.r.heads;
  const Where at = where(heads, cut.segs, (dv + E - 1) / E);
  if (!at.in) return;
  const int64_t bh = at.bh, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group, e0 = at.block * E, hs = (int)d.r.heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int64_t length = live_of(d, b);
  const int d0 = wave % Sh::WD * Sh::MT * 16, s0 = wave / Sh::WD * Sh::NT * 16;
  const int w0 = 16 * wave;
  const int chunks = (int)((length + kChunk - 1) / kChunk);
  const int first = at.seg * cut.each, last = min(first + cut.each, chunks);
  // what comes from behind: the state's own gradient, or that of the segment behind
  const bool end = last == chunks;
  const float* start = ENDS ? nullptr : end ? (grad_h ? grad_h + bh * dk * dv : nullptr)
                                            : starts + (bh * cut.segs + at.seg) * dk * dv;
  f32x4 S[Sh::MT][Sh::NT];
#pragma unroll
  for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
    for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
        S[m][n][e] = start && row < dk && col < dv ? start[(int64_t)row * dv + col] : 0.0f;
      }
  const auto put_state = [&](float* to) {
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
          if (row < dk && col < dv) to[row * dv + col] = S[m][n][e];
        }
  };
  const Frag<1> eye[2] = {unit_frag(0), unit_frag(1)};
  // Fetched as in the forward's chain.  Without grad_o as many bytes of E's place, as zeros.
  const T* go = grad_o ? grad_o : reinterpret_cast<const T*>(es);
  Raw<T> kf[kSteps], ktf[Sh::MT][2], qtf[Sh::MT][2], of;
  Frag<NV> mf[2], pf[2];
  f32x4 since, until, beta;
  float total;
  const Squares<T>* sqs = squares + bh * d.chunks;
  const Keys<T, DP>* kys = keys + (b * d.r.key_heads + kh) * d.chunks;
  const auto orows = [&](int c) {
    const int64_t t0 = (int64_t)c * kChunk;
    return Rows<T>{go + ((b * d.r.T + t0) * d.r.heads + h) * wide, hs * wide, (int)min(length - t0, (int64_t)kChunk), wide};
  };
  const auto fetch_o = [&](int c) { of.fetch(orows(c).template place<8>(w0 + i, e0 + 8 * g)); };
  const auto fetch_k = [&](int c) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) kf[s].fetch(kys[c].k[wave][s][lane]);
#pragma unroll
    for (int s = 0; s < 2; ++s) pf[s] = plane_frag<NV>(sqs[c].p[0][wave][s][lane], kSquare);
    until = *reinterpret_cast<const f32x4*>(sqs[c].gates.until + w0 + 4 * g);
  };
  const auto fetch_m = [&](int c) {
#pragma unroll
    for (int s = 0; s < 2; ++s) mf[s] = plane_frag<NV>(sqs[c].m[0][wave][s][lane], kSquare);
    since = *reinterpret_cast<const f32x4*>(sqs[c].gates.since + w0 + 4 * g);
    beta = *reinterpret_cast<const f32x4*>(sqs[c].gates.beta + w0 + 4 * g);
  };
  const auto fetch_turned = [&](int c) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < Sh::MT; ++m) {
        ktf[m][s].fetch(kys[c].kt[d0 / 16 + m][s][lane]);
        qtf[m][s].fetch(kys[c].qt[d0 / 16 + m][s][lane]);
      }
    total = sqs[c].gates.since[kChunk - 1];
  };
  loaded();
  if (first < last) {
    fetch_o(last - 1);
    fetch_k(last - 1);
    fetch_m(last - 1);
    fetch_turned(last - 1);
  }
  for (int c = last - 1; c >= first; --c) {
    const int64_t t0 = (int64_t)c * kChunk, row0 = (b * d.r.T + t0) * d.r.heads + h;
    const int live = (int)min(length - t0, (int64_t)kChunk), next = max(c - 1, first);
    renew(lane);
    i = lane & 15, g = lane >> 4;
    if (!ENDS) {
      float* to = dstates + (bh * d.chunks + c) * dk * wide;
#pragma unroll
      for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
        for (int n = 0; n < Sh::NT; ++n) {
          const int row = d0 + 16 * m + 4 * g + (i & 3), col = e0 + s0 + 16 * n + (i & 12);
          const f32x4 x = across(S[m][n]);
          if (row < dk && col < wide) store4(to + row * wide + col, x);
        }
    }
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
        put4<NV>(St + (s0 + 16 * n + i) * kPitch + d0 + 16 * m + 4 * g, kState, S[m][n]);
    if (live < kChunk || e0 + E > wide || !grad_o) of.keep(grad_o && orows(c).in(w0 + i, e0 + 8 * g));
    f32x4 O[1][2];   // dO as the sums lie
    clear(O);
    {
      const Frag<NI> ov = of.frag();
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        mma(O[0][n], ov, eye[n]);
        put4<NI>(Ot + (16 * n + i) * kRow + w0 + 4 * g, kSamples, O[0][n]);
      }
    }
    fetch_o(next);
    __syncthreads();
    f32x4 U[1][2], V[1][2];
    clear(U);
    clear(V);
    {
      Frag<NV> st[2][2];
      const auto read = [&](int s) {
#pragma unroll
        for (int n = 0; n < 2; ++n) st[s & 1][n] = plane_frag<NV>(St + (16 * n + i) * kPitch + 32 * s + 8 * g, kState);
      };
      read(0);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s + 1 < kSteps) read(s + 1);
        const Frag<NI> kv[1] = {kf[s].frag()};
        mma(U, kv, st[s & 1]);
      }
    }
    {
      Frag<NI> ot[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) ot[s][n] = plane_frag<NI>(Ot + (16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
#pragma unroll
      for (int n = 0; n < 2; ++n) U[0][n] *= until;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Frag<NV> pv[1] = {pf[s]};
        mma(U, pv, ot[s]);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) put4<NV>(Bt + (16 * n + i) * kRow + w0 + 4 * g, kSamples, beta * U[0][n]);
    fetch_k(next);
    __syncthreads();
    {
      Frag<NV> bt[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) bt[s][n] = plane_frag<NV>(Bt + (16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Frag<NV> mv[1] = {mf[s]};
        mma(V, mv, bt[s]);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const f32x4 ev = U[0][n] - V[0][n], z = beta * ev;
      const int to = (16 * n + i) * kRow + w0 + 4 * g;
      put4<NV>(Zt + to, kSamples, -since * z);
      put4<NV>(Gt + to, kSamples, d.r.scale * since * O[0][n]);
      if (ENDS) continue;
      const int t = w0 + 4 * g + (i & 3), col = e0 + 16 * n + (i & 12);
      const f32x4 er = across(ev), zr = across(z);
      if (t < live && col < wide) {
        store4(es + row0 * wide + t * hs * wide + col, er);
        if (grad_v && col < dv) store_some(grad_v + row0 * dv + t * hs * dv + col, zr, dv - col);
      }
    }
    fetch_m(next);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) S[m][n] *= total;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      Frag<NV> gt[Sh::NT], zt[Sh::NT];
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) {
        const int from = (s0 + 16 * n + i) * kRow + 32 * s + 8 * g;
        gt[n] = plane_frag<NV>(Gt + from, kSamples);
        zt[n] = plane_frag<NV>(Zt + from, kSamples);
      }
      Frag<NI> qv[Sh::MT], kv[Sh::MT];
#pragma unroll
      for (int m = 0; m < Sh::MT; ++m) qv[m] = qtf[m][s].frag(), kv[m] = ktf[m][s].frag();
      mma(S, qv, gt);
      mma(S, kv, zt);
    }
    fetch_turned(next);
  }
  if (ENDS) {
    put_state(adds + (bh * cut.segs + at.seg) * dk * dv);
    return;
  }
  if (grad_h0 && at.seg == 0) put_state(grad_h0 + bh * dk * dv);
  if (grad_v) {
    const int64_t rest = max(length, (int64_t)first * kChunk), stop = min((int64_t)(first + cut.each) * kChunk, d.r.T);
    for (int64_t n = rest * E + threadIdx.x; n < stop * E; n += kDeltaBlock) {
      const int64_t t = n / E;
      const int col = e0 + (int)(n % E);
      if (col < dv) grad_v[((b * d.r.T + t) * d.r.heads + h) * dv + col] = from_float<T>(0.0f);
    }
  }
}

// ---- everything else, by chunks ------------------------------------------------

__device__ __forceinline__ void put_gate(const Delta& d, void* p, int64_t at, float v) {
  if (d.r.gate_dtype == CPAB_F32)
    static_cast<float*>(p)[at] = v;
  else
    static_cast<bf16*>(p)[at] = from_float<bf16>(v);
}

__device__ __forceinline__ f32x4 masked(f32x4 v, bool in) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = in ? v[e] : 0.0f;
  return v;
}

constexpr int kWidePitch = kWide + 8;

// NP: the parts that a value goes as: two where every output has 16 bits.
template <typename T, int DP, int NP>
struct PartsRoom {
  // groups of waves over the columns: with 32-bit inputs four would leave too few registers
  static constexpr int kGroups = DP == 32 || sizeof(T) == 4 ? 2 : 4, kBlock = 256 * kGroups;
  static constexpr int kState = DP * kWidePitch, kSamples = kChunk * kWidePitch, kFlat = kChunk * kRow;
  // S, its gradient, U and Z, then in their place W, its transpose and the other square
  static constexpr int kLoop = NP * (2 * kState + 2 * kSamples), kAfter = 3 * NP * kFlat;
  static constexpr int kParts = kLoop > kAfter ? kLoop : kAfter;   // 16-bit values
  static constexpr int kSquares = 2 * kParts + 4 * kChunk * (kChunk + 1);
  // keys and queries too where there is room, which leaves 12 KB to the rest
  static constexpr bool kStaged = kSquares + sizeof(Keys<T, DP>) <= 148 * 1024;
  static constexpr int kBytes = kSquares + (kStaged ? sizeof(Keys<T, DP>) : 0);
};

// A chunk of a key's head: the gradients of its queries and keys, added up over the heads
// that share them, and of those heads' gates.  Four waves share the samples, and groups of
// four the columns.
// 8 x 4096 samples of 16 heads of 128 in bfloat16 take 667 us: the 1.65 GB of states, their
// gradients, X, E, dO and results would take 325, and the products after them, where memory
// only brings the next head's first columns, the rest; the waves wait for half of their cycles.
// Sixteen waves are one workgroup to a compute unit, and the registers' limit; eight took
// longer.  Keys and queries in LDS take 0.89 of the time from the cache, the next head fetched
// ahead 0.89 of that.
template <typename T, int DP, int NP>
__global__ __launch_bounds__((PartsRoom<T, DP, NP>::kBlock)) void delta_parts_kernel(
    Delta d, const Squares<T>* squares, const Keys<T, DP>* keys, const float* states, const float* xs,
    const float* dstates, const float* es, const T* grad_o, T* grad_q, T* grad_k, void* grad_decay,
    void* grad_beta) {
  typedef PartsRoom<T, DP, NP> Room;
  constexpr int kGroups = Room::kGroups, kBlock = Room::kBlock, kWaves = kBlock / 64;
  constexpr int NI = Parts<T>::kInput, kSteps = DP / 32;
  constexpr int NT = DP / 16 / kGroups, NJ = 4 / kGroups;   // tiles of DP and of the 64 to a wave
  extern __shared__ __align__(16) bf16 lds[];
  __shared__ double G[kChunk];
  __shared__ float betas[kChunk], since[kChunk], until[kChunk], dbeta[kChunk], before[kGroups][kChunk], after[kGroups][kChunk], whole[kWaves],
      sums[kWaves][kChunk];
  bf16* S = lds;                              // [DP][32]
  bf16* L = S + NP * Room::kState;            // the gradient, [DP][32]
  bf16* U = L + NP * Room::kState;            // [64][32]
  bf16* Z = U + NP * Room::kSamples;
  bf16* W = lds;                              // scale D dP, [64][64]
  bf16* Wt = W + NP * Room::kFlat;
  bf16* Y = Wt + NP * Room::kFlat;            // D dA + (D dA)^T
  float* H = reinterpret_cast<float*>(lds + Room::kParts);   // dP P + dA A, [64][65]
  const int c = blockIdx.x % d.chunks;
  const int64_t rest = blockIdx.x / d.chunks, b = rest / d.r.key_heads;
  const int kh = (int)(rest - b * d.r.key_heads);
  const int dk = (int)d.r.dk, dv = (int)d.r.dv, wide = (dv + 7) / 8 * 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int i = lane & 15, g = lane >> 4;
  const int tile = wave & 3, w0 = 16 * tile, group = wave >> 2;   // samples; columns of DP and of 64
  const int d0 = group * NT, j0 = group * NJ;                     // tiles
  const int64_t t0 = (int64_t)c * kChunk;
  const int live = (int)min(max(live_of(d, b) - t0, (int64_t)0), (int64_t)kChunk);
  const int rows = (int)min(d.r.T - t0, (int64_t)kChunk);   // that there are
  const Keys<T, DP>& theirs = keys[(b * d.r.key_heads + kh) * d.chunks + c];
  Keys<T, DP>& here = *reinterpret_cast<Keys<T, DP>*>(reinterpret_cast<char*>(lds) + Room::kSquares);
  const Keys<T, DP>& own = Room::kStaged ? here : theirs;
  if (Room::kStaged && live > 0) {
    typedef typename Raw<T>::U4 U4;
    const U4* from = reinterpret_cast<const U4*>(&theirs);
    U4* to = reinterpret_cast<U4*>(&here);
    constexpr int kAll = sizeof(Keys<T, DP>) / 16 / kBlock;
    U4 v[kAll];
#pragma unroll
    for (int n = 0; n < kAll; ++n) v[n] = from[n * kBlock + threadIdx.x];
#pragma unroll
    for (int n = 0; n < kAll; ++n) to[n * kBlock + threadIdx.x] = v[n];
  }
  const auto own_frag = [&](const auto& of, int row, int step) {
    Raw<T> r;
    r.take(of[row][step][threadIdx.x & 63]);
    return r.frag();
  };
  if (live == 0) {
    for (int n = threadIdx.x; n < rows * d.group; n += kBlock) {
      const int64_t at = (b * d.r.T + t0 + n / d.group) * d.r.heads + kh * d.group + n % d.group;
      if (grad_decay) put_gate(d, grad_decay, at, 0.0f);
      if (grad_beta) put_gate(d, grad_beta, at, 0.0f);
    }
    for (int n = threadIdx.x; n < rows * dk; n += kBlock) {
      const int64_t at = ((b * d.r.T + t0 + n / dk) * d.r.key_heads + kh) * dk + n % dk;
      if (grad_q) grad_q[at] = from_float<T>(0.0f);
      if (grad_k) grad_k[at] = from_float<T>(0.0f);
    }
    return;
  }
  const int64_t token = (b * d.r.T + t0) * d.r.heads + kh * d.group;
  const int64_t state = ((b * d.r.heads + kh * d.group) * d.chunks + c) * dk * wide;
  const int next_row = (int)d.r.heads * wide;
  Rows<T> orows{(grad_o ? grad_o : reinterpret_cast<const T*>(es)) + token * wide, next_row, live, wide};
  // the library's own: rows of whole eights, zeros beyond dv
  Rows<float> srows{states + state, wide, dk, wide}, lrows{dstates + state, wide, dk, wide};
  Rows<float> xrows{xs + token * wide, next_row, live, wide}, erows{es + token * wide, next_row, live, wide};
  // A block of columns is fetched while the matrix unit has the one before, the next head's
  // first during the rest of this one's.
  constexpr int kAll = DP * (kWide / 4), kQuads = (kAll + kBlock - 1) / kBlock, kValues = kChunk * (kWide / 4);
  static_assert(kValues <= kBlock, "a quad of X to a lane");
  int tid = threadIdx.x;
  f32x4 sq4[kQuads], lq4[kQuads], xq, eq;
  Raw<T> oraw;
  const auto load4 = [](const Rows<float>& r, int row, int col) {
    float w[4];
    load<4>(r.template place<4>(row, col), w);
    return f32x4{w[0], w[1], w[2], w[3]};
  };
  const auto fetch = [&](int e0) {
#pragma unroll
    for (int n = 0; n < kQuads; ++n) {
      const int at = tid + n * kBlock, row = at / (kWide / 4), col = at % (kWide / 4) * 4;
      sq4[n] = load4(srows, row, e0 + col);
      lq4[n] = load4(lrows, row, e0 + col);
    }
    const int t = tid / (kWide / 4), col = tid % (kWide / 4) * 4;
    xq = load4(xrows, t, e0 + col);
    eq = load4(erows, t, e0 + col);
    oraw.fetch(orows.template place<8>(w0 + i, e0 + 8 * g));   // this wave's own samples of dO
  };
  const auto next_head = [&] {
    orows.p += wide, xrows.p += wide, erows.p += wide;
    srows.p += (int64_t)d.chunks * dk * wide, lrows.p += (int64_t)d.chunks * dk * wide;
  };
  fetch(0);
  f32x4 dQ[1][NT], dK[1][NT];
  clear(dQ);
  clear(dK);
  for (int hh = 0; hh < d.group; ++hh) {
    const int h = kh * d.group + hh;
    const int64_t bh = b * d.r.heads + h;
    const Squares<T>& sq = squares[bh * d.chunks + c];
    if (threadIdx.x < kChunk) {
      const int t = threadIdx.x;
      G[t] = sq.gates.log[t];
      betas[t] = sq.gates.beta[t];
      since[t] = sq.gates.since[t];
      until[t] = sq.gates.until[t];
      dbeta[t] = 0.0f;
    }
    f32x4 qs[1][NT], k1[1][NT], k2[1][NT], P[1][NJ], ZU[1][NJ];
    clear(qs);
    clear(k1);
    clear(k2);
    clear(P);
    clear(ZU);
    float dot = 0.0f;
    __syncthreads();
#pragma unroll 1
    for (int e0 = 0; e0 < dv; e0 += kWide) {
      renew(tid);
      i = tid & 15, g = tid >> 4 & 3;
#pragma unroll
      for (int n = 0; n < kQuads; ++n) {
        const int at = tid + n * kBlock, row = at / (kWide / 4), col = at % (kWide / 4) * 4;
        if (kAll % kBlock == 0 || at < kAll) {
          const bool in = row < dk && e0 + col < wide;
          const f32x4 s = masked(sq4[n], in), l = masked(lq4[n], in);
          put4<NP>(S + row * kWidePitch + col, Room::kState, s);
          put4<NP>(L + row * kWidePitch + col, Room::kState, l);
#pragma unroll
          for (int e = 0; e < 4; ++e) dot = fmaf(s[e], l[e], dot);
        }
      }
      if (kValues == kBlock || tid < kValues) {
        const int t = tid / (kWide / 4), col = tid % (kWide / 4) * 4;
        const bool in = t < live && e0 + col < wide;
        const f32x4 x = masked(xq, in), ev = masked(eq, in);
        put4<NP>(U + t * kWidePitch + col, Room::kSamples, betas[t] * x);
        put4<NP>(Z + t * kWidePitch + col, Room::kSamples, betas[t] * ev);
        float part = x[0] * ev[0];
#pragma unroll
        for (int e = 1; e < 4; ++e) part = fmaf(x[e], ev[e], part);
        part = over8(part);
        if (col == 0) dbeta[t] += part;
      }
      oraw.keep(grad_o && orows.in(w0 + i, e0 + 8 * g));
      const Frag<NI> of[1] = {oraw.frag()};
      int next = e0 + kWide;
      if (next >= dv) {   // the last head's is not used
        next = 0;
        if (hh + 1 < d.group) next_head();
      }
      fetch(next);
      __syncthreads();
      const int mine = (w0 + i) * kWidePitch + 8 * g;
      const Frag<NP> uf[1] = {plane_frag<NP>(U + mine, Room::kSamples)}, zf[1] = {plane_frag<NP>(Z + mine, Room::kSamples)};
      Frag<NP> sf[NT], lf[NT], tf[NJ];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int at = (16 * (d0 + n) + i) * kWidePitch + 8 * g;
        sf[n] = plane_frag<NP>(S + at, Room::kState), lf[n] = plane_frag<NP>(L + at, Room::kState);
      }
#pragma unroll
      for (int n = 0; n < NJ; ++n) tf[n] = plane_frag<NP>(U + (16 * (j0 + n) + i) * kWidePitch + 8 * g, Room::kSamples);
      mma(qs, of, sf);
      mma(k2, zf, sf);
      mma(k1, uf, lf);
      mma(P, of, tf);
      mma(ZU, zf, tf);
      __syncthreads();
    }
    // keys and queries as the sums lie
    f32x4 qv[1][NT], kv[1][NT];
    clear(qv);
    clear(kv);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const Frag<1> one = unit_frag((d0 + n) & 1);   // tiles of both halves of a step
      mma(qv[0][n], own_frag(own.q, tile, (d0 + n) / 2), one);
      mma(kv[0][n], own_frag(own.k, tile, (d0 + n) / 2), one);
    }
    // what passes a sample's decay from the state before the chunk, and to the one after
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = w0 + 4 * g + e;
      const float early = since[row], late = until[row], ss = d.r.scale * early;
      float from = 0.0f, to = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float a = ss * qs[0][n][e], z = early * k2[0][n][e], u = late * k1[0][n][e];
        from = fmaf(qv[0][n][e], a, from);
        from = fmaf(-kv[0][n][e], z, from);
        to = fmaf(kv[0][n][e], u, to);
        dQ[0][n][e] += a;
        dK[0][n][e] += u - z;
      }
      from = over16(from);
      to = over16(to);
      if (i == 0) before[group][row] = from, after[group][row] = to;
    }
    // the products that M and P were made of
    f32x4 kk[1][NJ], qk[1][NJ];
    clear(kk);
    clear(qk);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const Frag<NI> ak[1] = {own_frag(own.k, tile, s)}, aq[1] = {own_frag(own.q, tile, s)};
      Frag<NI> bk[NJ];
#pragma unroll
      for (int n = 0; n < NJ; ++n) bk[n] = own_frag(own.k, j0 + n, s);
      mma(kk, ak, bk);
      mma(qk, aq, bk);
    }
    dot = over_rows(over16(dot));
    if (lane == 0) whole[wave] = dot;
#pragma unroll
    for (int n = 0; n < NJ; ++n) {
      const int other = j0 + n, col = 16 * other + i, flat = Room::kFlat;
      f32x4 w, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = w0 + 4 * g + e;
        const float decay = col <= row ? expf((float)(G[row] - G[col])) : 0.0f;
        w[e] = d.r.scale * decay * P[0][n][e];
        y[e] = col < row ? -decay * ZU[0][n][e] : 0.0f;
        H[row * (kChunk + 1) + col] = w[e] * qk[0][n][e] + y[e] * kk[0][n][e];
      }
      const int row4 = (w0 + 4 * g + (i & 3)) * kRow + 16 * other + (i & 12);
      put4<NP>(Wt + col * kRow + w0 + 4 * g, flat, w);
      put4<NP>(W + row4, flat, across(w));
      // Y: a tile below the diagonal, and its mirror image above it
      if (other < tile) {
        put4<NP>(Y + col * kRow + w0 + 4 * g, flat, y);
        put4<NP>(Y + row4, flat, across(y));
      } else if (other == tile) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = w0 + 4 * g + e;
          bf16x2 p[NP];
          split<NP>(y[e], y[e], p);
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            if (col <= row) Y[k * flat + row * kRow + col] = p[k][0];
            if (col < row) Y[k * flat + col * kRow + row] = p[k][0];
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int from = (w0 + i) * kRow + 32 * s + 8 * g;
      const Frag<NP> wf[1] = {plane_frag<NP>(W + from, Room::kFlat)}, wt[1] = {plane_frag<NP>(Wt + from, Room::kFlat)},
                     yf[1] = {plane_frag<NP>(Y + from, Room::kFlat)};
      Frag<NI> kf[NT], qf[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) kf[n] = own_frag(own.kt, d0 + n, s), qf[n] = own_frag(own.qt, d0 + n, s);
      mma(dQ, wf, kf);
      mma(dK, wt, qf);
      mma(dK, yf, kf);
    }
    // the decays: the waves share the rows, a lane has a sample; what crosses it from the
    // columns before, for each row from it on
    {
      float sum = 0.0f;
      for (int n = 0; n < kChunk / kWaves; ++n) {
        const int row = kChunk / kWaves * wave + n;
        const float v = lanes_before(H[row * (kChunk + 1) + lane]);
        float from = 0.0f, to = 0.0f;
#pragma unroll
        for (int m = 0; m < kGroups; ++m) from += before[m][row], to += after[m][row];
        sum += row >= lane ? v + from : to;
      }
      sums[wave][lane] = sum;
    }
    __syncthreads();
    if (threadIdx.x < kChunk) {
      const int t = threadIdx.x;
      float dots = 0.0f, sum = 0.0f;
#pragma unroll
      for (int n = 0; n < kWaves; ++n) dots += whole[n], sum += sums[n][t];
      sum = fmaf(since[kChunk - 1], dots, sum);
      if (t < rows) {
        const int64_t at = (b * d.r.T + t0 + t) * d.r.heads + h;
        if (grad_decay) put_gate(d, grad_decay, at, t < live ? sum : 0.0f);
        if (grad_beta) put_gate(d, grad_beta, at, t < live ? dbeta[t] : 0.0f);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = w0 + 4 * g + e, col = 16 * (d0 + n) + i;
      if (t >= rows || col >= dk) continue;
      const int64_t at = ((b * d.r.T + t0 + t) * d.r.key_heads + kh) * dk + col;
      if (grad_q) grad_q[at] = from_float<T>(dQ[0][n][e]);
      if (grad_k) grad_k[at] = from_float<T>(dK[0][n][e]);
    }
}

template <typename T>
__global__ __launch_bounds__(kDeltaBlock) void delta_zero_kernel(T* a, T* b, int64_t n) {
  for (int64_t at = (int64_t)blockIdx.x * kDeltaBlock + threadIdx.x; at < n; at += (int64_t)gridDim.x * kDeltaBlock) {
    if (a) a[at] = (T)0.0f;
    if (b) b[at] = (T)0.0f;
  }
}

// The backward's workspace (bytes).
struct Space {
  int64_t squares, keys, dstates, es, adds, starts, padded, grads, all;
};
Space space_of(const Delta& d, const Cut& cut) {
  const int64_t heads = d.r.B * d.r.heads;
  const auto next = [](int64_t n) { return (n + 255) / 256 * 256; };
  Space w;
  w.squares = 0;
  w.keys = next(heads * d.chunks * squares_bytes(d.r.dtype));
  w.dstates = w.keys + next(d.r.B * d.r.key_heads * d.chunks * keys_bytes(d.r));
  w.es = w.dstates + next(heads * d.chunks * d.r.dk * wide_of(d.r) * 4);
  w.adds = w.es + next(heads * d.r.T * wide_of(d.r) * 4);
  const int64_t segments = cut.segs > 1 ? next(heads * cut.segs * d.r.dk * d.r.dv * 4) : 0;
  w.starts = w.adds + segments;
  w.padded = w.starts + segments;
  w.grads = w.padded + next(padded_keys(d.r));
  w.all = w.grads + padded_values(d.r);
  return w;
}

}  // namespace

hipError_t launch_delta_rule_unread(const cpab_delta_rule& r, void* grad_q, void* grad_k, hipStream_t st) {
  const int64_t n = r.B * r.T * r.key_heads * r.dk;
  if (n == 0 || !(grad_q || grad_k)) return hipSuccess;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + kDeltaBlock - 1) / kDeltaBlock, 1 << 16);
  if (r.dtype == CPAB_F32)
    delta_zero_kernel<float><<<blocks, kDeltaBlock, 0, st>>>((float*)grad_q, (float*)grad_k, n);
  else
    delta_zero_kernel<bf16><<<blocks, kDeltaBlock, 0, st>>>((bf16*)grad_q, (bf16*)grad_k, n);
  return hipGetLastError();
}

int64_t delta_backward_workspace(const Delta& d) { return space_of(d, cut_of(d)).all; }

hipError_t launch_delta_rule_backward(const cpab_delta_rule& r, const float* kept, const void* grad_o,
                                      const float* grad_h, void* grad_q, void* grad_k, void* grad_v,
                                      void* grad_decay, void* grad_beta, float* grad_h0,
                                      void* workspace, hipStream_t st) {
  Delta d = delta_of(r);
  const Cut cut = cut_of(d);
  const Space w = space_of(d, cut);
  const Kept k = kept_of(d, cut);
  const int64_t heads = r.B * r.heads;
  char* room = static_cast<char*>(workspace);
  float* dstates = reinterpret_cast<float*>(room + w.dstates);
  float* es = reinterpret_cast<float*>(room + w.es);
  float* adds = reinterpret_cast<float*>(room + w.adds);
  float* starts = reinterpret_cast<float*>(room + w.starts);
  hipError_t e = hipSuccess;
  if (r.dv % 8 != 0 && grad_o) {
    const int64_t strides[3] = {r.T * r.heads * r.dv, r.heads * r.dv, r.dv};
    e = launch_delta_pad(r.dtype, grad_o, strides, r.B, r.T, r.heads, r.dv, room + w.grads, st);
    grad_o = room + w.grads;
  }
  if (e == hipSuccess && d.chunks > 0) e = pad_keys(&d, room + w.padded, st);
  if (e == hipSuccess && d.chunks > 0) e = launch_delta_squares(d, room + w.squares, room + w.keys, true, st);
  if (e != hipSuccess) return e;
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value, NV = Parts<T>::kValue, NI = Parts<T>::kInput;
    const Squares<T>* squares = reinterpret_cast<const Squares<T>*>(room + w.squares);
    const Keys<T, DP>* keys = reinterpret_cast<const Keys<T, DP>*>(room + w.keys);
    const auto run = [&](auto only_ends) {
      constexpr bool ENDS = decltype(only_ends)::value;
      constexpr int kRoom = 2 * kWide * (NV * (DP + 8) + (3 * NV + NI) * kRow);
      static LdsAllowed allowed;
      e = allow_lds(reinterpret_cast<const void*>(delta_back_chain_kernel<T, DP, ENDS>), kRoom, allowed);
      if (e != hipSuccess) return;
      delta_back_chain_kernel<T, DP, ENDS>
          <<<(unsigned)((heads * cut.segs + 7) / 8 * 8 * ((r.dv + kWide - 1) / kWide)), kDeltaBlock, kRoom, st>>>(
              d, squares, keys, cut, (const T*)grad_o, grad_h, starts, (T*)grad_v, grad_h0, dstates, es, adds);
      e = hipGetLastError();
    };
    if (cut.segs > 1) {
      run(std::true_type());
      if (e == hipSuccess) e = launch_delta_join(d, cut, false, kept + k.maps, adds, grad_h, starts, st);
      if (e != hipSuccess) return;
    }
    run(std::false_type());
    if (e != hipSuccess || d.chunks == 0 || !(grad_q || grad_k || grad_decay || grad_beta)) return;
    const auto parts = [&](auto np) {
      constexpr int NP = decltype(np)::value;
      typedef PartsRoom<T, DP, NP> Room;
      static LdsAllowed allowed;
      e = allow_lds(reinterpret_cast<const void*>(delta_parts_kernel<T, DP, NP>), Room::kBytes, allowed);
      if (e != hipSuccess) return;
      delta_parts_kernel<T, DP, NP><<<(unsigned)(r.B * r.key_heads * d.chunks), Room::kBlock, Room::kBytes, st>>>(
          d, squares, keys, kept + k.states, kept + k.xs, dstates, es, (const T*)grad_o, (T*)grad_q,
          (T*)grad_k, grad_decay, grad_beta);
      e = hipGetLastError();
    };
    if constexpr (sizeof(T) == 2)
      if (r.gate_dtype == CPAB_BF16) return parts(std::integral_constant<int, 2>());
    parts(std::integral_constant<int, 3>());
  });
  return e;
}

}  // namespace cpab
