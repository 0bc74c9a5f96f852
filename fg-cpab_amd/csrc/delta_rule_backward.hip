// Gated delta rule, backward: the states' gradients through the chain of chunks, then
// everything else by chunks.  The formulas stand in delta_device.hpp.
#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "delta_device.hpp"

namespace cpab {
namespace {

constexpr int kRow = kChunk + 4;
constexpr int kWide = 32, kWidePitch = kWide + 4;   // columns of values at once

// One workgroup goes back through a head's chunks with 32 columns of the state's gradient
// in registers.  Keeps the gradient after each chunk and E, and writes grad_v and grad_h0.
template <typename T, int DP>
__global__ __launch_bounds__(kDeltaBlock) void delta_back_chain_kernel(
    Delta d, const float* squares, const T* grad_o, const float* grad_h, T* grad_v, float* grad_h0,
    float* dstates, float* es) {
  typedef Shares<DP, kWide> Sh;
  constexpr int kPitch = DP + 4, NT = kWide / 16;
  extern __shared__ float room[];
  __shared__ Gates gates;
  __shared__ float scaled[kChunk];   // scale exp(G_i)
  float* K = room;
  float* Q = K + kChunk * kPitch;
  float* St = Q + kChunk * kPitch;   // the gradient [32][DP]
  float* Ot = St + kWide * kPitch;   // dO [32][64]
  float* Zt = Ot + kWide * kRow;
  float* M = Zt + kWide * kRow;
  float* P = M + kChunk * kRow;
  const int64_t heads = d.r.B * d.r.heads, bh = blockIdx.x % heads, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group, e0 = (int)(blockIdx.x / heads) * kWide;
  const int dk = (int)d.r.dk, dv = (int)d.r.dv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int64_t length = live_of(d, b);
  const T* q = static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + kh * d.r.q_strides[2];
  const T* k = static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + kh * d.r.k_strides[2];
  const int d0 = wave % Sh::WD * Sh::MT * 16, s0 = wave / Sh::WD * Sh::NT * 16;
  f32x4 S[Sh::MT][Sh::NT];
#pragma unroll
  for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
    for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
        S[m][n][e] = grad_h && row < dk && col < dv ? grad_h[(bh * dk + row) * dv + col] : 0.0f;
      }
  const auto put_state = [&](float* to) {
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
          if (row < dk && col < dv) to[(int64_t)row * dv + col] = S[m][n][e];
        }
  };
  const int chunks = (int)((length + kChunk - 1) / kChunk);
  for (int c = chunks - 1; c >= 0; --c) {
    const int64_t t0 = (int64_t)c * kChunk;
    const int live = (int)min(length - t0, (int64_t)kChunk);
    put_state(dstates + (bh * d.chunks + c) * dk * dv);
    load_gates(gates, d, b, h, t0, live);
    load_rows<DP>(K, kPitch, k + t0 * d.r.k_strides[1], d.r.k_strides[1], live, dk);
    load_rows<DP>(Q, kPitch, q + t0 * d.r.q_strides[1], d.r.q_strides[1], live, dk);
    const float* sq = squares + (bh * d.chunks + c) * kSquares;
    load_rows<kChunk>(M, kRow, sq, (int64_t)kChunk, kChunk, kChunk);
    load_rows<kChunk>(P, kRow, sq + kSquare, (int64_t)kChunk, kChunk, kChunk);
    for (int at = threadIdx.x; at < kChunk * kWide; at += kDeltaBlock) {
      const int t = at / kWide, col = at % kWide;
      Ot[col * kRow + t] = grad_o && t < live && e0 + col < dv
                               ? to_float(grad_o[((b * d.r.T + t0 + t) * d.r.heads + h) * dv + e0 + col]) : 0.0f;
    }
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
        *reinterpret_cast<f32x4*>(St + (s0 + 16 * n + i) * kPitch + d0 + 16 * m + 4 * g) = S[m][n];
    __syncthreads();
    if (threadIdx.x < kChunk) scaled[threadIdx.x] = d.r.scale * gates.since[threadIdx.x];
    const int w0 = 16 * wave + 4 * g;
    f32x4 U[1][NT], V[1][NT];
    clear(U);
    clear(V);
    multiply<false, false>(U, K + 16 * wave * kPitch, kPitch, St, kPitch, DP);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) U[0][n][e] *= gates.until[w0 + e];
    multiply<true, false>(U, P + 16 * wave, kRow, Ot, kRow, kChunk);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 bu;
#pragma unroll
      for (int e = 0; e < 4; ++e) bu[e] = gates.beta[w0 + e] * U[0][n][e];
      *reinterpret_cast<f32x4*>(Zt + (16 * n + i) * kRow + w0) = bu;
    }
    __syncthreads();
    multiply<true, false>(V, M + 16 * wave, kRow, Zt, kRow, kChunk);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 gz;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = w0 + e, col = e0 + 16 * n + i;
        const float ev = U[0][n][e] - V[0][n][e], z = gates.beta[t] * ev;
        gz[e] = -gates.since[t] * z;
        if (t < live && col < dv) {
          const int64_t at = ((b * d.r.T + t0 + t) * d.r.heads + h) * dv + col;
          es[at] = ev;
          if (grad_v) grad_v[at] = from_float<T>(z);
        }
      }
      *reinterpret_cast<f32x4*>(Zt + (16 * n + i) * kRow + w0) = gz;
    }
    __syncthreads();
    const float total = gates.since[kChunk - 1];
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) S[m][n] *= total;
    multiply<true, false>(S, Q + d0, kPitch, Ot + s0 * kRow, kRow, kChunk, scaled);
    multiply<true, false>(S, K + d0, kPitch, Zt + s0 * kRow, kRow, kChunk);
    __syncthreads();
  }
  if (grad_h0) put_state(grad_h0 + bh * dk * dv);
  if (grad_v)
    for (int64_t at = length * kWide + threadIdx.x; at < d.r.T * kWide; at += kDeltaBlock) {
      const int64_t t = at / kWide;
      const int col = e0 + (int)(at % kWide);
      if (col < dv) grad_v[((b * d.r.T + t) * d.r.heads + h) * dv + col] = from_float<T>(0.0f);
    }
}

__device__ __forceinline__ void put_gate(const Delta& d, void* p, int64_t at, float v) {
  if (d.r.gate_dtype == CPAB_F32)
    static_cast<float*>(p)[at] = v;
  else
    static_cast<bf16*>(p)[at] = from_float<bf16>(v);
}

// [rows, 32] columns of a 32-bit array in LDS, zeros beyond `live` rows and `cols` columns.
__device__ __forceinline__ f32x4 quad(const float* row, bool in, int left) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (!in) return v;
  if (left >= 4) {
    float w[4];
    load<4>(row, w);
    return f32x4{w[0], w[1], w[2], w[3]};
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) v[e] = row[e];
  return v;
}

// A chunk of a key's head: the gradients of its queries and keys, added up over the heads
// that share them, and of those heads' gates.
template <typename T, int DP>
__global__ __launch_bounds__(kDeltaBlock) void delta_parts_kernel(
    Delta d, const float* squares, const float* states, const float* xs, const float* dstates,
    const float* es, const T* grad_o, T* grad_q, T* grad_k, void* grad_decay, void* grad_beta) {
  constexpr int kPitch = DP + 4, NT = DP / 16;
  extern __shared__ float room[];
  __shared__ Gates gates;
  __shared__ float dbeta[kChunk], before[kChunk], after[kChunk], whole[4];
  float* K = room;
  float* Q = K + kChunk * kPitch;
  float* S = Q + kChunk * kPitch;      // [DP][32]
  float* L = S + DP * kWidePitch;      // the gradient's, [DP][32]
  float* O = L + DP * kWidePitch;      // dO [64][32]
  float* U = O + kChunk * kWidePitch;
  float* Z = U + kChunk * kWidePitch;
  float* W1 = S;                       // the chunk's squares, in the same place afterwards
  float* W2 = W1 + kChunk * kRow;
  float* H = W2 + kChunk * kRow;       // [64][65]
  const int c = blockIdx.x % d.chunks;
  const int64_t rest = blockIdx.x / d.chunks, b = rest / d.r.key_heads;
  const int kh = (int)(rest - b * d.r.key_heads);
  const int dk = (int)d.r.dk, dv = (int)d.r.dv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int64_t t0 = (int64_t)c * kChunk;
  const int live = (int)min(max(live_of(d, b) - t0, (int64_t)0), (int64_t)kChunk);
  const int rows = (int)min(d.r.T - t0, (int64_t)kChunk);   // that there are
  if (live > 0) {
    load_rows<DP>(K, kPitch, static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + t0 * d.r.k_strides[1] + kh * d.r.k_strides[2],
                  d.r.k_strides[1], live, dk);
    load_rows<DP>(Q, kPitch, static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + t0 * d.r.q_strides[1] + kh * d.r.q_strides[2],
                  d.r.q_strides[1], live, dk);
  }
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
    load_gates(gates, d, b, h, t0, live);
    if (threadIdx.x < kChunk) dbeta[threadIdx.x] = 0.0f;
    const float* state = states + (bh * d.chunks + c) * dk * dv;
    const float* dstate = dstates + (bh * d.chunks + c) * dk * dv;
    f32x4 qs[1][NT], k1[1][NT], k2[1][NT], P[1][4], ZU[1][4];
    clear(qs);
    clear(k1);
    clear(k2);
    clear(P);
    clear(ZU);
    float dot = 0.0f;
    __syncthreads();
    for (int e0 = 0; e0 < dv; e0 += kWide) {
      for (int at = threadIdx.x; at < DP * (kWide / 4); at += kDeltaBlock) {
        const int row = at / (kWide / 4), col = at % (kWide / 4) * 4;
        const int64_t from = (int64_t)row * dv + e0 + col;
        const f32x4 s = quad(state + from, row < dk, dv - e0 - col), l = quad(dstate + from, row < dk, dv - e0 - col);
        *reinterpret_cast<f32x4*>(S + row * kWidePitch + col) = s;
        *reinterpret_cast<f32x4*>(L + row * kWidePitch + col) = l;
#pragma unroll
        for (int e = 0; e < 4; ++e) dot = fmaf(s[e], l[e], dot);
      }
      for (int at = threadIdx.x; at < kChunk * (kWide / 4); at += kDeltaBlock) {
        const int t = at / (kWide / 4), col = at % (kWide / 4) * 4;
        const int64_t from = ((b * d.r.T + t0 + t) * d.r.heads + h) * dv + e0 + col;
        const f32x4 x = quad(xs + from, t < live, dv - e0 - col), ev = quad(es + from, t < live, dv - e0 - col);
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        if (grad_o && t < live)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (e0 + col + e < dv) o[e] = to_float(grad_o[from + e]);
        const float beta = gates.beta[t];
        *reinterpret_cast<f32x4*>(O + t * kWidePitch + col) = o;
        *reinterpret_cast<f32x4*>(U + t * kWidePitch + col) = beta * x;
        *reinterpret_cast<f32x4*>(Z + t * kWidePitch + col) = beta * ev;
        float part = x[0] * ev[0];
#pragma unroll
        for (int e = 1; e < 4; ++e) part = fmaf(x[e], ev[e], part);
        part += __shfl_xor(part, 1);
        part += __shfl_xor(part, 2);
        part += __shfl_xor(part, 4);
        if (col == 0) dbeta[t] += part;
      }
      __syncthreads();
      const int w = 16 * wave * kWidePitch;
      multiply<false, false>(qs, O + w, kWidePitch, S, kWidePitch, kWide);
      multiply<false, false>(k1, U + w, kWidePitch, L, kWidePitch, kWide);
      multiply<false, false>(k2, Z + w, kWidePitch, S, kWidePitch, kWide);
      multiply<false, false>(P, O + w, kWidePitch, U, kWidePitch, kWide);
      multiply<false, false>(ZU, Z + w, kWidePitch, U, kWidePitch, kWide);
      __syncthreads();
    }
    // what passes a sample's decay from the state before the chunk, and to the one after
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * wave + 4 * g + e;
      const float since = gates.since[row], until = gates.until[row], ss = d.r.scale * since;
      float from = 0.0f, to = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float qv = Q[row * kPitch + 16 * n + i], kv = K[row * kPitch + 16 * n + i];
        const float a = ss * qs[0][n][e], z = since * k2[0][n][e], u = until * k1[0][n][e];
        from = fmaf(qv, a, from);
        from = fmaf(-kv, z, from);
        to = fmaf(kv, u, to);
        dQ[0][n][e] += a;
        dK[0][n][e] += u - z;
      }
#pragma unroll
      for (int k = 1; k < 16; k *= 2) {
        from += __shfl_xor(from, k);
        to += __shfl_xor(to, k);
      }
      if (i == 0) before[row] = from, after[row] = to;
    }
#pragma unroll
    for (int k = 1; k < 64; k *= 2) dot += __shfl_xor(dot, k);
    if (lane == 0) whole[wave] = dot;
    const float* sq = squares + (bh * d.chunks + c) * kSquares;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * wave + 4 * g + e, col = 16 * n + i;
        const float decay = col <= row ? expf((float)(gates.G[row] - gates.G[col])) : 0.0f;
        W1[row * kRow + col] = d.r.scale * decay * P[0][n][e];
        W2[row * kRow + col] = col < row ? -decay * ZU[0][n][e] : 0.0f;
        H[row * (kChunk + 1) + col] = P[0][n][e] * sq[kSquare + row * kChunk + col] -
                                      ZU[0][n][e] * sq[2 * kSquare + row * kChunk + col];
      }
    __syncthreads();
    multiply<false, true>(dQ, W1 + 16 * wave * kRow, kRow, K, kPitch, kChunk);
    multiply<true, true>(dK, W1 + 16 * wave, kRow, Q, kPitch, kChunk);
    multiply<false, true>(dK, W2 + 16 * wave * kRow, kRow, K, kPitch, kChunk);
    multiply<true, true>(dK, W2 + 16 * wave, kRow, K, kPitch, kChunk);
    if (threadIdx.x < kChunk) {   // H: each row's sum of the columns before
      float sum = 0.0f;
      for (int k = 0; k < kChunk; ++k) {
        float& v = H[threadIdx.x * (kChunk + 1) + k];
        const float now = v;
        v = sum;
        sum += now;
      }
    }
    __syncthreads();
    if (threadIdx.x < kChunk) {
      const int t = threadIdx.x;
      float sum = gates.since[kChunk - 1] * ((whole[0] + whole[1]) + (whole[2] + whole[3]));
      for (int k = 0; k < t; ++k) sum += after[k];
      for (int k = t; k < kChunk; ++k) sum += before[k] + H[k * (kChunk + 1) + t];
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
      const int t = 16 * wave + 4 * g + e, col = 16 * n + i;
      if (t >= rows || col >= dk) continue;
      const int64_t at = ((b * d.r.T + t0 + t) * d.r.key_heads + kh) * dk + col;
      if (grad_q) grad_q[at] = from_float<T>(dQ[0][n][e]);
      if (grad_k) grad_k[at] = from_float<T>(dK[0][n][e]);
    }
}

}  // namespace

hipError_t launch_delta_rule_backward(const cpab_delta_rule& r, const float* kept, const void* grad_o,
                                      const float* grad_h, void* grad_q, void* grad_k, void* grad_v,
                                      void* grad_decay, void* grad_beta, float* grad_h0,
                                      void* workspace, hipStream_t st) {
  const Delta d = delta_of(r);
  const int64_t heads = r.B * r.heads, states = heads * d.chunks * r.dk * r.dv;
  float* squares = static_cast<float*>(workspace);
  float* dstates = squares + heads * d.chunks * kSquares;
  float* es = dstates + states;
  hipError_t e = hipSuccess;
  if (d.chunks > 0) e = launch_delta_squares(d, squares, st);
  if (e != hipSuccess) return e;
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value;
    constexpr int kChain = 4 * ((2 * kChunk + kWide) * (DP + 4) + (2 * kWide + 2 * kChunk) * kRow);
    static LdsAllowed chain, parts;
    if (r.dv > 0) {
      e = allow_lds(reinterpret_cast<const void*>(delta_back_chain_kernel<T, DP>), kChain, chain);
      if (e != hipSuccess) return;
      delta_back_chain_kernel<T, DP><<<(unsigned)(heads * ((r.dv + kWide - 1) / kWide)), kDeltaBlock, kChain, st>>>(
          d, squares, (const T*)grad_o, grad_h, (T*)grad_v, grad_h0, dstates, es);
      e = hipGetLastError();
    }
    if (e != hipSuccess || d.chunks == 0 || !(grad_q || grad_k || grad_decay || grad_beta)) return;
    constexpr int kAfter = 3 * kChunk * kRow, kLoop = (2 * DP + 3 * kChunk) * kWidePitch;
    constexpr int kParts = 4 * (2 * kChunk * (DP + 4) + std::max(kAfter, kLoop));
    e = allow_lds(reinterpret_cast<const void*>(delta_parts_kernel<T, DP>), kParts, parts);
    if (e != hipSuccess) return;
    delta_parts_kernel<T, DP><<<(unsigned)(r.B * r.key_heads * d.chunks), kDeltaBlock, kParts, st>>>(
        d, squares, kept, kept + states, dstates, es, (const T*)grad_o, (T*)grad_q, (T*)grad_k,
        grad_decay, grad_beta);
    e = hipGetLastError();
  });
  return e;
}

}  // namespace cpab
