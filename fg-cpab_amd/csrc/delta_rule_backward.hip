// Gated delta rule, backward: the states' gradients through the chain of chunks, then
// everything else by chunks.  The formulas stand in delta_device.hpp.
#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "delta_device.hpp"

namespace cpab {
namespace {

// ---- the chain of chunks, backwards --------------------------------------------

// As the forward's chain: E columns of the state's gradient in registers, back through a
// segment's chunks.  Keeps the gradient after each chunk and E, and writes grad_v and
// grad_h0.  M and P lie transposed.  ENDS: only what the segment adds to the gradient before
// it.
template <typename T, int DP, int E, bool ENDS>
__global__ __launch_bounds__(8 * E) void delta_back_chain_kernel(
    Delta d, const Squares<T>* squares, const T* kt, const T* qt, Cut cut, const T* grad_o,
    const float* grad_h, const float* starts, T* grad_v, float* grad_h0, float* dstates, float* es,
    float* adds) {
  typedef Shares<DP, E> Sh;
  constexpr int kPitch = DP + 8, NV = Parts<T>::kValue, NI = Parts<T>::kInput, kSteps = DP / 32;
  constexpr int kState = E * kPitch, kSamples = E * kRow;   // planes
  extern __shared__ __align__(16) bf16 lds[];
  bf16* St = lds;                       // the gradient, [E][DP]
  bf16* Bt = St + NV * kState;          // beta dU, [E][64]
  bf16* Zt = Bt + NV * kSamples;        // - exp(G) Z
  bf16* Ot = Zt + NV * kSamples;        // dO, as the input that it is
  bf16* Gt = Ot + NI * kSamples;        // scale exp(G) dO
  const int dk = (int)d.r.dk, dv = (int)d.r.dv, wide = (dv + 7) / 8 * 8;
  const int64_t heads = d.r.B * d.r.heads;
  const Where at = where(heads, cut.segs, (dv + E - 1) / E);
  if (!at.in) return;
  const int64_t bh = at.bh, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group, e0 = at.block * E;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int i = lane & 15, g = lane >> 4;
  const int64_t length = live_of(d, b);
  const T* k = static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + kh * d.r.k_strides[2];
  const int ks = (int)d.r.k_strides[1];
  const int d0 = wave % Sh::WD * Sh::MT * 16, s0 = wave / Sh::WD * Sh::NT * 16;
  const int w0 = 16 * (wave & 3), c0 = wave / 4 * 32;
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
  const auto put_state = [&](float* to, int pitch) {
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
          if (row < dk && col < dv) to[row * pitch + col] = S[m][n][e];
        }
  };
  // Fetched as in the forward's chain.  Without grad_o as many bytes of E's place, as zeros.
  const T* go = grad_o ? grad_o : reinterpret_cast<const T*>(es);
  Raw<T> kf[kSteps], ktf[Sh::MT][2], qtf[Sh::MT][2];
  Frag<NV> mf[2], pf[2];
  RawOne<T> of[2][4];
  f32x4 since, until, beta;
  float total;
  const auto krows_of = [&](int c) {
    const int64_t t0 = (int64_t)c * kChunk;
    return Rows<T>{k + t0 * ks, ks, (int)min(length - t0, (int64_t)kChunk), d.read};
  };
  const auto orows_of = [&](int c) {
    const int64_t t0 = (int64_t)c * kChunk;
    return Rows<T>{go + ((b * d.r.T + t0) * d.r.heads + h) * wide, (int)d.r.heads * wide,
                   (int)min(length - t0, (int64_t)kChunk), dv};
  };
  const auto fetch_k = [&](int c) {
    const Rows<T> krows = krows_of(c);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) kf[s].fetch(krows.template place<8>(w0 + i, 32 * s + 8 * g));
  };
  const auto fetch_o = [&](int c) {
    const Rows<T> orows = orows_of(c);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) of[n][e].fetch(orows.template place<1>(w0 + 4 * g + e, e0 + c0 + 16 * n + i));
  };
  const auto mask_rows = [&](int c) {   // zeros where there was nothing to fetch
    const Rows<T> krows = krows_of(c), orows = orows_of(c);
    if (krows.live == kChunk && d.read == DP && e0 + E <= dv && grad_o) return;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) kf[s].keep(krows.in(w0 + i, 32 * s + 8 * g));
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        of[n][e].keep(grad_o && orows.in(w0 + 4 * g + e, e0 + c0 + 16 * n + i));
  };
  const auto fetch_p = [&](const Squares<T>& sq) {
#pragma unroll
    for (int s = 0; s < 2; ++s) pf[s] = plane_frag<NV>(&sq.p[0][w0 + i][32 * s + 8 * g], kSquare);
    until = *reinterpret_cast<const f32x4*>(sq.gates.until + w0 + 4 * g);
  };
  const auto fetch_m = [&](const Squares<T>& sq) {
#pragma unroll
    for (int s = 0; s < 2; ++s) mf[s] = plane_frag<NV>(&sq.m[0][w0 + i][32 * s + 8 * g], kSquare);
    since = *reinterpret_cast<const f32x4*>(sq.gates.since + w0 + 4 * g);
    beta = *reinterpret_cast<const f32x4*>(sq.gates.beta + w0 + 4 * g);
  };
  const auto fetch_turned = [&](const Squares<T>& sq, int c) {
    const int64_t turned = ((b * d.r.key_heads + kh) * d.chunks + c) * DP * kChunk;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < Sh::MT; ++m) {
        const int from = (d0 + 16 * m + i) * kChunk + 32 * s + 8 * g;
        ktf[m][s].fetch(kt + turned + from);
        qtf[m][s].fetch(qt + turned + from);
      }
    total = sq.gates.since[kChunk - 1];
  };
  const Squares<T>* sqs = squares + bh * d.chunks;
  loaded();
  if (first < last) {
    fetch_o(last - 1);
    fetch_k(last - 1);
    fetch_p(sqs[last - 1]);
    fetch_m(sqs[last - 1]);
    fetch_turned(sqs[last - 1], last - 1);
  }
  for (int c = last - 1; c >= first; --c) {
    const int64_t t0 = (int64_t)c * kChunk;
    const int live = (int)min(length - t0, (int64_t)kChunk), next = max(c - 1, first);
    float* ec = es + ((b * d.r.T + t0) * d.r.heads + h) * wide;
    T* vc = grad_v ? grad_v + ((b * d.r.T + t0) * d.r.heads + h) * dv : nullptr;
    renew(i, g);
    if (!ENDS) put_state(dstates + (bh * d.chunks + c) * dk * wide, wide);
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
        put4<NV>(St + (s0 + 16 * n + i) * kPitch + d0 + 16 * m + 4 * g, kState, S[m][n]);
    mask_rows(c);
    f32x4 ov[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) ov[n][e] = of[n][e].value();
      put4<NI>(Ot + (c0 + 16 * n + i) * kRow + w0 + 4 * g, kSamples, ov[n]);
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
        for (int n = 0; n < 2; ++n)
          st[s & 1][n] = plane_frag<NV>(St + (c0 + 16 * n + i) * kPitch + 32 * s + 8 * g, kState);
      };
      read(0);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s + 1 < kSteps) read(s + 1);
        const Frag<NI> kv = kf[s].frag();
#pragma unroll
        for (int n = 0; n < 2; ++n) mma(U[0][n], kv, st[s & 1][n]);
      }
    }
    {
      Frag<NI> ot[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          ot[s][n] = plane_frag<NI>(Ot + (c0 + 16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
#pragma unroll
      for (int n = 0; n < 2; ++n) U[0][n] *= until;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) mma(U[0][n], pf[s], ot[s][n]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
      put4<NV>(Bt + (c0 + 16 * n + i) * kRow + w0 + 4 * g, kSamples, beta * U[0][n]);
    fetch_k(next);
    fetch_p(sqs[next]);
    __syncthreads();
    {
      Frag<NV> bt[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          bt[s][n] = plane_frag<NV>(Bt + (c0 + 16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) mma(V[0][n], mf[s], bt[s][n]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const f32x4 ev = U[0][n] - V[0][n], z = beta * ev;
      const int at = (c0 + 16 * n + i) * kRow + w0 + 4 * g;
      put4<NV>(Zt + at, kSamples, -since * z);
      put4<NV>(Gt + at, kSamples, d.r.scale * since * ov[n]);
      if (ENDS) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = w0 + 4 * g + e, col = e0 + c0 + 16 * n + i;
        if (t < live && col < dv) {
          const int to = t * (int)d.r.heads;
          ec[to * wide + col] = ev[e];
          if (vc) vc[to * dv + col] = from_float<T>(z[e]);
        }
      }
    }
    fetch_m(sqs[next]);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) S[m][n] *= total;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) {
        const int from = (s0 + 16 * n + i) * kRow + 32 * s + 8 * g;
        const Frag<NV> go = plane_frag<NV>(Gt + from, kSamples), z = plane_frag<NV>(Zt + from, kSamples);
#pragma unroll
        for (int m = 0; m < Sh::MT; ++m) {
          mma(S[m][n], qtf[m][s].frag(), go);
          mma(S[m][n], ktf[m][s].frag(), z);
        }
      }
    fetch_turned(sqs[next], next);
  }
  if (ENDS) {
    put_state(adds + (bh * cut.segs + at.seg) * dk * dv, dv);
    return;
  }
  if (grad_h0 && at.seg == 0) put_state(grad_h0 + bh * dk * dv, dv);
  if (grad_v) {
    const int64_t rest = max(length, (int64_t)first * kChunk), stop = min((int64_t)(first + cut.each) * kChunk, d.r.T);
    for (int64_t n = rest * E + threadIdx.x; n < stop * E; n += 8 * E) {
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

// The first `left` of four values, zeros behind them.
__device__ __forceinline__ f32x4 edge(f32x4 v, int left) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e < left ? v[e] : 0.0f;
  return v;
}

constexpr int kPartsBlock = 512;
constexpr int kWide = 32, kWidePitch = kWide + 8;   // columns of values at once

template <typename T, int DP>
struct PartsRoom {
  static constexpr int NV = Parts<T>::kValue;
  static constexpr int kState = DP * kWidePitch, kSamples = kChunk * kWidePitch, kFlat = kChunk * kRow;
  // S, its gradient and U, then in their place W, its transpose and the other square
  static constexpr int kLoop = NV * (2 * kState + kSamples), kAfter = 3 * NV * kFlat;
  static constexpr int kParts = kLoop > kAfter ? kLoop : kAfter;   // 16-bit values
  static constexpr int kBytes = 2 * kParts + 4 * kChunk * (kChunk + 1);
};

// A chunk of a key's head: the gradients of its queries and keys, added up over the heads
// that share them, and of those heads' gates.  Of the eight waves four share the samples and
// two the columns.
template <typename T, int DP>
__global__ __launch_bounds__(kPartsBlock) void delta_parts_kernel(
    Delta d, const Squares<T>* squares, const T* kt, const T* qt, const float* states, const float* xs,
    const float* dstates, const float* es, const T* grad_o, T* grad_q, T* grad_k, void* grad_decay,
    void* grad_beta) {
  typedef PartsRoom<T, DP> Room;
  constexpr int NV = Parts<T>::kValue, NI = Parts<T>::kInput, kSteps = DP / 32, NT = DP / 32;
  extern __shared__ __align__(16) bf16 lds[];
  __shared__ double G[kChunk];
  __shared__ float betas[kChunk], dbeta[kChunk], before[2][kChunk], after[2][kChunk], whole[8], sums[8][kChunk];
  bf16* S = lds;                              // [DP][32]
  bf16* L = S + NV * Room::kState;            // the gradient, [DP][32]
  bf16* U = L + NV * Room::kState;            // [64][32]
  bf16* W = lds;                              // scale D dP, [64][64]
  bf16* Wt = W + NV * Room::kFlat;
  bf16* Y = Wt + NV * Room::kFlat;            // D dA + (D dA)^T
  float* H = reinterpret_cast<float*>(lds + Room::kParts);   // dP P + dA A, [64][65]
  const int c = blockIdx.x % d.chunks;
  const int64_t rest = blockIdx.x / d.chunks, b = rest / d.r.key_heads;
  const int kh = (int)(rest - b * d.r.key_heads);
  const int dk = (int)d.r.dk, dv = (int)d.r.dv, wide = (dv + 7) / 8 * 8;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int i = lane & 15, g = lane >> 4;
  const int w0 = 16 * (wave & 3), half = wave >> 2;   // samples; columns of DP and of 64
  const int d0 = half * (DP / 2), j0 = half * 32;
  const int64_t t0 = (int64_t)c * kChunk;
  const int live = (int)min(max(live_of(d, b) - t0, (int64_t)0), (int64_t)kChunk);
  const int rows = (int)min(d.r.T - t0, (int64_t)kChunk);   // that there are
  const T* k = static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + t0 * d.r.k_strides[1] + kh * d.r.k_strides[2];
  const T* q = static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + t0 * d.r.q_strides[1] + kh * d.r.q_strides[2];
  const Rows<T> krows{k, (int)d.r.k_strides[1], live, d.read}, qrows{q, (int)d.r.q_strides[1], live, d.read};
  const int64_t turned = ((b * d.r.key_heads + kh) * d.chunks + c) * DP * kChunk;
  f32x4 dQ[1][NT], dK[1][NT];
  clear(dQ);
  clear(dK);
  for (int hh = 0; hh < d.group; ++hh) {
    const int h = kh * d.group + hh;
    const int64_t bh = b * d.r.heads + h;
    if (live == 0) {
      if ((int)threadIdx.x < rows) {
        const int64_t at = (b * d.r.T + t0 + threadIdx.x) * d.r.heads + h;
        if (grad_decay) put_gate(d, grad_decay, at, 0.0f);
        if (grad_beta) put_gate(d, grad_beta, at, 0.0f);
      }
      continue;
    }
    const Squares<T>& sq = squares[bh * d.chunks + c];
    if (threadIdx.x < kChunk) {
      const int t = threadIdx.x;
      double sum = 0.0;
      if (t < live)
        sum = (double)clamped(gate_at(d, d.r.decay, b * d.r.decay_strides[0] + (t0 + t) * d.r.decay_strides[1] +
                                                        h * d.r.decay_strides[2]));
      for (int n = 1; n < 64; n *= 2) {
        const double prior = __shfl_up(sum, n);
        if (t >= n) sum += prior;
      }
      G[t] = sum;
      betas[t] = sq.gates.beta[t];
      dbeta[t] = 0.0f;
    }
    const float* state = states + (bh * d.chunks + c) * dk * wide;
    const float* dstate = dstates + (bh * d.chunks + c) * dk * wide;
    f32x4 qs[1][NT], k1[1][NT], k2[1][NT], P[1][2], ZU[1][2];
    clear(qs);
    clear(k1);
    clear(k2);
    clear(P);
    clear(ZU);
    float dot = 0.0f;
    const int64_t token = (b * d.r.T + t0) * d.r.heads + h;
    const int across = (int)d.r.heads * wide;
    const Rows<T> orows{(grad_o ? grad_o : reinterpret_cast<const T*>(es)) + token * wide, across, live, wide};
    // rows of whole eights, in which the library itself wrote nothing beyond dv
    const Rows<float> srows{state, wide, dk, wide}, lrows{dstate, wide, dk, wide};
    const Rows<float> xrows{xs + token * wide, across, live, wide}, erows{es + token * wide, across, live, wide};
    // A block of columns is fetched while the matrix unit has the one before.
    constexpr int kQuads = (DP * (kWide / 4) + kPartsBlock - 1) / kPartsBlock;
    static_assert(kChunk * (kWide / 4) == kPartsBlock, "a quad of X to a lane");
    int tid = threadIdx.x, unused = 0;
    f32x4 sq4[kQuads], lq4[kQuads], xq, eq, zq[2];
    Raw<T> oraw;
    const auto load4 = [](const Rows<float>& r, int row, int col) {
      float w[4];
      load<4>(r.template place<4>(row, col), w);
      return f32x4{w[0], w[1], w[2], w[3]};
    };
    const auto fetch = [&](int e0) {
#pragma unroll
      for (int n = 0; n < kQuads; ++n) {
        const int at = tid + n * kPartsBlock, row = at / (kWide / 4), col = at % (kWide / 4) * 4;
        sq4[n] = load4(srows, row, e0 + col);
        lq4[n] = load4(lrows, row, e0 + col);
      }
      const int t = tid / (kWide / 4), col = tid % (kWide / 4) * 4;
      xq = load4(xrows, t, e0 + col);
      eq = load4(erows, t, e0 + col);
      // this wave's own samples of dO and Z
      oraw.fetch(orows.template place<8>(w0 + i, e0 + 8 * g));
      zq[0] = load4(erows, w0 + i, e0 + 8 * g);
      zq[1] = load4(erows, w0 + i, e0 + 8 * g + 4);
    };
    __syncthreads();
    fetch(0);
#pragma unroll 1
    for (int e0 = 0; e0 < dv; e0 += kWide) {
      renew(i, g);
      renew(tid, unused);
#pragma unroll
      for (int n = 0; n < kQuads; ++n) {
        const int at = tid + n * kPartsBlock, row = at / (kWide / 4), col = at % (kWide / 4) * 4;
        const int left = row < dk ? dv - e0 - col : 0;
        const f32x4 s = edge(sq4[n], left), l = edge(lq4[n], left);
        if (DP * (kWide / 4) % kPartsBlock == 0 || at < DP * (kWide / 4)) {
          put4<NV>(S + row * kWidePitch + col, Room::kState, s);
          put4<NV>(L + row * kWidePitch + col, Room::kState, l);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) dot = fmaf(s[e], l[e], dot);
      }
      {
        const int t = tid / (kWide / 4), col = tid % (kWide / 4) * 4, left = t < live ? dv - e0 - col : 0;
        const f32x4 x = edge(xq, left), ev = edge(eq, left);
        put4<NV>(U + t * kWidePitch + col, Room::kSamples, betas[t] * x);
        float part = x[0] * ev[0];
#pragma unroll
        for (int e = 1; e < 4; ++e) part = fmaf(x[e], ev[e], part);
        part += __shfl_xor(part, 1);
        part += __shfl_xor(part, 2);
        part += __shfl_xor(part, 4);
        if (col == 0) dbeta[t] += part;
      }
      const int row = w0 + i, col = 8 * g, left = row < live ? dv - e0 - col : 0;
      oraw.keep(grad_o && left > 0);
      const Frag<NI> of = oraw.frag();
      float z[8];
      const f32x4 z0 = edge(zq[0], left), z1 = edge(zq[1], left - 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = betas[row] * z0[e], z[4 + e] = betas[row] * z1[e];
      const Frag<NV> zf = frag_of<NV>(z);
      fetch(min(e0 + kWide, (dv - 1) / kWide * kWide));
      __syncthreads();
      const Frag<NV> uf = plane_frag<NV>(U + row * kWidePitch + col, Room::kSamples);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int at = (d0 + 16 * n + i) * kWidePitch + col;
        const Frag<NV> s = plane_frag<NV>(S + at, Room::kState), l = plane_frag<NV>(L + at, Room::kState);
        mma(qs[0][n], of, s);
        mma(k2[0][n], zf, s);
        mma(k1[0][n], uf, l);
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const Frag<NV> u = plane_frag<NV>(U + (j0 + 16 * n + i) * kWidePitch + col, Room::kSamples);
        mma(P[0][n], of, u);
        mma(ZU[0][n], zf, u);
      }
      __syncthreads();
    }
    renew(i, g);
    // the products that M and P were made of
    f32x4 kk[1][2], qk[1][2];
    clear(kk);
    clear(qk);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int col = 32 * s + 8 * g;
      const Frag<NI> ak = krows.at(w0 + i, col), aq = qrows.at(w0 + i, col);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const Frag<NI> bk = krows.at(j0 + 16 * n + i, col);
        mma(kk[0][n], ak, bk);
        mma(qk[0][n], aq, bk);
      }
    }
    renew(i, g);
    // what passes a sample's decay from the state before the chunk, and to the one after
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = w0 + 4 * g + e;
      const float since = sq.gates.since[row], until = sq.gates.until[row], ss = d.r.scale * since;
      float from = 0.0f, to = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int col = d0 + 16 * n + i;
        const float qv = qrows.one(row, col), kv = krows.one(row, col);
        const float a = ss * qs[0][n][e], z = since * k2[0][n][e], u = until * k1[0][n][e];
        from = fmaf(qv, a, from);
        from = fmaf(-kv, z, from);
        to = fmaf(kv, u, to);
        dQ[0][n][e] += a;
        dK[0][n][e] += u - z;
      }
#pragma unroll
      for (int n = 1; n < 16; n *= 2) {
        from += __shfl_xor(from, n);
        to += __shfl_xor(to, n);
      }
      if (i == 0) before[half][row] = from, after[half][row] = to;
    }
#pragma unroll
    for (int n = 1; n < 64; n *= 2) dot += __shfl_xor(dot, n);
    if (lane == 0) whole[wave] = dot;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int col = j0 + 16 * n + i;
      f32x4 w, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = w0 + 4 * g + e;
        const float decay = col <= row ? expf((float)(G[row] - G[col])) : 0.0f;
        w[e] = d.r.scale * decay * P[0][n][e];
        y[e] = col < row ? -decay * ZU[0][n][e] : 0.0f;
        H[row * (kChunk + 1) + col] = w[e] * qk[0][n][e] + y[e] * kk[0][n][e];
      }
      put4<NV>(Wt + col * kRow + w0 + 4 * g, Room::kFlat, w);
      // both halves of Y: above the diagonal its mirror image
      const int top = w0 + 4 * g;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = top + e;
        bf16 p[NV], r[NV];
        split<NV>(w[e], p);
        split<NV>(y[e], r);
#pragma unroll
        for (int n2 = 0; n2 < NV; ++n2) {
          W[n2 * Room::kFlat + row * kRow + col] = p[n2];
          if (col <= row) Y[n2 * Room::kFlat + row * kRow + col] = r[n2];
          if (col < row) Y[n2 * Room::kFlat + col * kRow + row] = r[n2];
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int from = (w0 + i) * kRow + 32 * s + 8 * g;
      const Frag<NV> wf = plane_frag<NV>(W + from, Room::kFlat), wt = plane_frag<NV>(Wt + from, Room::kFlat),
                     yf = plane_frag<NV>(Y + from, Room::kFlat);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int64_t at = turned + (d0 + 16 * n + i) * kChunk + 32 * s + 8 * g;
        const Frag<NI> kf = eight(kt + at), qf = eight(qt + at);
        mma(dQ[0][n], wf, kf);
        mma(dK[0][n], wt, qf);
        mma(dK[0][n], yf, kf);
      }
    }
    // the decays: a wave has 8 of the rows, a lane a sample; what crosses it from the columns
    // before, for each row from it on
    {
      float sum = 0.0f;
      for (int n = 0; n < 8; ++n) {
        const int row = 8 * wave + n;
        float v = H[row * (kChunk + 1) + lane];
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
          const float prior = __shfl_up(v, m);
          if (lane >= m) v += prior;
        }
        v = __shfl_up(v, 1);   // of the columns before
        if (lane == 0) v = 0.0f;
        if (row >= lane) sum += v + (before[0][row] + before[1][row]);
        else sum += after[0][row] + after[1][row];
      }
      sums[wave][lane] = sum;
    }
    __syncthreads();
    if (threadIdx.x < kChunk) {
      const int t = threadIdx.x;
      float dots = 0.0f, sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 8; ++n) dots += whole[n], sum += sums[n][t];
      sum = fmaf(sq.gates.since[kChunk - 1], dots, sum);
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
      const int t = w0 + 4 * g + e, col = d0 + 16 * n + i;
      if (t >= rows || col >= dk) continue;
      const int64_t at = ((b * d.r.T + t0 + t) * d.r.key_heads + kh) * dk + col;
      if (grad_q) grad_q[at] = from_float<T>(dQ[0][n][e]);
      if (grad_k) grad_k[at] = from_float<T>(dK[0][n][e]);
    }
}

// The backward's workspace (bytes).
struct Space {
  int64_t squares, kt, qt, dstates, es, adds, starts, keys, grads, all;
};
Space space_of(const Delta& d, const Cut& cut) {
  const int64_t heads = d.r.B * d.r.heads, turned = d.r.B * d.r.key_heads * d.chunks * turned_bytes(d.r);
  const auto next = [](int64_t n) { return (n + 255) / 256 * 256; };
  Space w;
  w.squares = 0;
  w.kt = next(heads * d.chunks * squares_bytes(d.r.dtype));
  w.qt = w.kt + next(turned);
  w.dstates = w.qt + next(turned);
  w.es = w.dstates + next(heads * d.chunks * d.r.dk * wide_of(d.r) * 4);
  w.adds = w.es + next(heads * d.r.T * wide_of(d.r) * 4);
  const int64_t segments = cut.segs > 1 ? next(heads * cut.segs * d.r.dk * d.r.dv * 4) : 0;
  w.starts = w.adds + segments;
  w.keys = w.starts + segments;
  w.grads = w.keys + next(padded_keys(d.r));
  w.all = w.grads + (d.r.dv % 8 ? heads * d.r.T * wide_of(d.r) * (d.r.dtype == CPAB_F32 ? 4 : 2) : 0);
  return w;
}

}  // namespace

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
  if (e == hipSuccess && d.chunks > 0) e = pad_keys(&d, room + w.keys, st);
  if (e == hipSuccess && d.chunks > 0) e = launch_delta_squares(d, room + w.squares, room + w.kt, room + w.qt, st);
  if (e != hipSuccess) return e;
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value, NV = Parts<T>::kValue, NI = Parts<T>::kInput;
    const Squares<T>* squares = reinterpret_cast<const Squares<T>*>(room + w.squares);
    const T *kt = reinterpret_cast<const T*>(room + w.kt), *qt = reinterpret_cast<const T*>(room + w.qt);
    const auto run = [&](auto width, auto only_ends) {
      constexpr int E = decltype(width)::value;
      constexpr bool ENDS = decltype(only_ends)::value;
      constexpr int kRoom = 2 * E * (NV * (DP + 8) + (3 * NV + NI) * kRow);
      static LdsAllowed allowed;
      e = allow_lds(reinterpret_cast<const void*>(delta_back_chain_kernel<T, DP, E, ENDS>), kRoom, allowed);
      if (e != hipSuccess) return;
      delta_back_chain_kernel<T, DP, E, ENDS>
          <<<(unsigned)((heads * cut.segs + 7) / 8 * 8 * ((r.dv + E - 1) / E)), 8 * E, kRoom, st>>>(
              d, squares, kt, qt, cut, (const T*)grad_o, grad_h, starts, (T*)grad_v, grad_h0, dstates, es, adds);
      e = hipGetLastError();
    };
    const auto both = [&](auto only_ends) {
      if constexpr (sizeof(T) == 2)
        if (r.dv > 32) return run(std::integral_constant<int, 64>(), only_ends);
      run(std::integral_constant<int, 32>(), only_ends);
    };
    if (cut.segs > 1) {
      both(std::true_type());
      if (e == hipSuccess) e = launch_delta_join(d, cut, false, kept + k.ends, adds, grad_h, starts, st);
      if (e != hipSuccess) return;
    }
    both(std::false_type());
    if (e != hipSuccess || d.chunks == 0 || !(grad_q || grad_k || grad_decay || grad_beta)) return;
    constexpr int kRoom = PartsRoom<T, DP>::kBytes;
    static LdsAllowed allowed;
    e = allow_lds(reinterpret_cast<const void*>(delta_parts_kernel<T, DP>), kRoom, allowed);
    if (e != hipSuccess) return;
    delta_parts_kernel<T, DP><<<(unsigned)(r.B * r.key_heads * d.chunks), kPartsBlock, kRoom, st>>>(
        d, squares, kt, qt, kept + k.states, kept + k.xs, dstates, es, (const T*)grad_o, (T*)grad_q,
        (T*)grad_k, grad_decay, grad_beta);
    e = hipGetLastError();
  });
  return e;
}

}  // namespace cpab
