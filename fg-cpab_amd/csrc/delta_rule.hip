// Gated delta rule, forward: by chunks of 64 samples, and sample by sample for a few.
// The formulas stand in delta_device.hpp.
#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "delta_device.hpp"

namespace cpab {
namespace {

// ---- a chunk's matrices ------------------------------------------------------

// M, P and A of each chunk of each head.  M by rows: M_i = A_i - sum over j < i of
// A_ij beta_j M_j; a column is four lanes', each with a quarter of the rows.
template <typename T, int DP>
__global__ __launch_bounds__(kDeltaBlock) void delta_squares_kernel(Delta d, float* squares) {
  constexpr int kPitch = DP + 4, kRow = kChunk + 4;
  extern __shared__ float room[];
  __shared__ Gates gates;
  float* K = room;
  float* Q = K + kChunk * kPitch;
  const int c = blockIdx.x % d.chunks;
  const int64_t bh = blockIdx.x / d.chunks, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group;
  const int64_t t0 = (int64_t)c * kChunk;
  const int live = (int)min(max(live_of(d, b) - t0, (int64_t)0), (int64_t)kChunk);
  if (live == 0) return;
  load_gates(gates, d, b, h, t0, live);
  load_rows<DP>(K, kPitch, static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + t0 * d.r.k_strides[1] + kh * d.r.k_strides[2],
                d.r.k_strides[1], live, (int)d.r.dk);
  load_rows<DP>(Q, kPitch, static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + t0 * d.r.q_strides[1] + kh * d.r.q_strides[2],
                d.r.q_strides[1], live, (int)d.r.dk);
  __syncthreads();
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  f32x4 kk[1][4], qk[1][4];
  clear(kk);
  clear(qk);
  multiply<false, false>(kk, K + 16 * wave * kPitch, kPitch, K, kPitch, DP);
  multiply<false, false>(qk, Q + 16 * wave * kPitch, kPitch, K, kPitch, DP);
  __syncthreads();
  float* Ab = room;                  // A beta, in K's place; its columns 4 q + p at 16 p + q
  float* A = room + kChunk * kRow;
  float* out = squares + (bh * d.chunks + c) * kSquares;
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * wave + 4 * g + e, col = 16 * n + i;
      const float decay = col <= row ? expf((float)(gates.G[row] - gates.G[col])) : 0.0f;
      const float a = col < row ? decay * kk[0][n][e] : 0.0f;
      out[kSquare + row * kChunk + col] = d.r.scale * decay * qk[0][n][e];
      out[2 * kSquare + row * kChunk + col] = a;
      Ab[row * kRow + (col & 3) * 16 + (col >> 2)] = a * gates.beta[col];
      A[row * kRow + col] = a;
    }
  __syncthreads();
  const int col = threadIdx.x >> 2, p = threadIdx.x & 3;
  float m[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) m[q] = 0.0f;
#pragma unroll
  for (int q = 0; q < 16; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 4 * q + e;
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k <= q; ++k) sum = fmaf(Ab[row * kRow + 16 * p + k], m[k], sum);
      sum += __shfl_xor(sum, 1);
      sum += __shfl_xor(sum, 2);
      const float v = A[row * kRow + col] - sum;
      if (p == e) m[q] = v;
    }
#pragma unroll
  for (int q = 0; q < 16; ++q) out[(4 * q + p) * kChunk + col] = m[q];
}

// ---- the chain of chunks -----------------------------------------------------

// One workgroup goes through a head's chunks with E columns of its state in registers, the
// sums of the matrix unit; a copy in LDS feeds the next chunk's products.
template <typename T, int DP, int E>
__global__ __launch_bounds__(kDeltaBlock) void delta_chain_kernel(Delta d, const float* squares, T* o,
                                                                float* h_out, float* states, float* xs) {
  typedef Shares<DP, E> Sh;
  constexpr int kPitch = DP + 4, kRow = kChunk + 4, NT = E / 16;
  extern __shared__ float room[];
  __shared__ Gates gates;
  float* K = room;
  float* Q = K + kChunk * kPitch;
  float* St = Q + kChunk * kPitch;   // [E][DP]
  float* Rt = St + E * kPitch;       // [E][64]
  float* M = Rt + E * kRow;
  float* P = M + kChunk * kRow;
  const int64_t heads = d.r.B * d.r.heads, bh = blockIdx.x % heads, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group, e0 = (int)(blockIdx.x / heads) * E;
  const int dk = (int)d.r.dk, dv = (int)d.r.dv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int64_t length = live_of(d, b);
  const T* q = static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + kh * d.r.q_strides[2];
  const T* k = static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + kh * d.r.k_strides[2];
  const T* v = static_cast<const T*>(d.r.v) + b * d.r.v_strides[0] + h * d.r.v_strides[2];
  const int d0 = wave % Sh::WD * Sh::MT * 16, s0 = wave / Sh::WD * Sh::NT * 16;   // this wave's part of the state
  f32x4 S[Sh::MT][Sh::NT];
  const float* h0 = d.r.h0 ? d.r.h0 + bh * dk * dv : nullptr;
#pragma unroll
  for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
    for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
        S[m][n][e] = h0 && row < dk && col < dv ? h0[(int64_t)row * dv + col] : 0.0f;
      }
  const auto put_state = [&](float* to) {   // [dk, dv]
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
  for (int c = 0; c < chunks; ++c) {
    const int64_t t0 = (int64_t)c * kChunk;
    const int live = (int)min(length - t0, (int64_t)kChunk);
    if (states) put_state(states + (bh * d.chunks + c) * dk * dv);
    load_gates(gates, d, b, h, t0, live);
    load_rows<DP>(K, kPitch, k + t0 * d.r.k_strides[1], d.r.k_strides[1], live, dk);
    load_rows<DP>(Q, kPitch, q + t0 * d.r.q_strides[1], d.r.q_strides[1], live, dk);
    const float* sq = squares + (bh * d.chunks + c) * kSquares;
    load_rows<kChunk>(M, kRow, sq, (int64_t)kChunk, kChunk, kChunk);
    load_rows<kChunk>(P, kRow, sq + kSquare, (int64_t)kChunk, kChunk, kChunk);
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n)
        *reinterpret_cast<f32x4*>(St + (s0 + 16 * n + i) * kPitch + d0 + 16 * m + 4 * g) = S[m][n];
    __syncthreads();
    // this wave's 16 samples from here on
    const int w0 = 16 * wave + 4 * g;
    f32x4 R[1][NT], O[1][NT], X[1][NT];
    clear(R);
    clear(O);
    multiply<false, false>(R, K + 16 * wave * kPitch, kPitch, St, kPitch, DP);
    multiply<false, false>(O, Q + 16 * wave * kPitch, kPitch, St, kPitch, DP);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 br;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = w0 + e, col = e0 + 16 * n + i;
        const float val = t < live && col < dv ? to_float(v[(t0 + t) * d.r.v_strides[1] + col]) : 0.0f;
        R[0][n][e] = fmaf(-gates.since[t], R[0][n][e], val);
        O[0][n][e] *= d.r.scale * gates.since[t];
        br[e] = gates.beta[t] * R[0][n][e];
      }
      *reinterpret_cast<f32x4*>(Rt + (16 * n + i) * kRow + w0) = br;
    }
    __syncthreads();
    clear(X);
    multiply<false, false>(X, M + 16 * wave * kRow, kRow, Rt, kRow, kChunk);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4 u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = w0 + e, col = e0 + 16 * n + i;
        const float x = R[0][n][e] - X[0][n][e];
        u[e] = gates.beta[t] * x;
        if (xs && t < live && col < dv) xs[((b * d.r.T + t0 + t) * d.r.heads + h) * dv + col] = x;
      }
      *reinterpret_cast<f32x4*>(Rt + (16 * n + i) * kRow + w0) = u;
    }
    __syncthreads();
    multiply<false, false>(O, P + 16 * wave * kRow, kRow, Rt, kRow, kChunk);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = w0 + e, col = e0 + 16 * n + i;
        if (t < live && col < dv) o[((b * d.r.T + t0 + t) * d.r.heads + h) * dv + col] = from_float<T>(O[0][n][e]);
      }
    const float total = gates.since[kChunk - 1];
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) S[m][n] *= total;
    multiply<true, false>(S, K + d0, kPitch, Rt + s0 * kRow, kRow, kChunk, gates.until);
    __syncthreads();
  }
  put_state(h_out + bh * dk * dv);
  for (int64_t at = length * E + threadIdx.x; at < d.r.T * E; at += kDeltaBlock) {
    const int64_t t = at / E;
    const int col = e0 + (int)(at % E);
    if (col < dv) o[((b * d.r.T + t) * d.r.heads + h) * dv + col] = from_float<T>(0.0f);
  }
}

// ---- a few samples -----------------------------------------------------------

// The definition: 64 columns of a head's state in a workgroup's registers, four to a lane
// and dk / 16 of the rows.  o = scale (S'^T q + (q.k) u) takes both products with the state
// in one pass.
template <typename T>
__global__ __launch_bounds__(kDeltaBlock) void delta_steps_kernel(Delta d, T* o, float* h_out) {
  constexpr int kRows = CPAB_DELTA_MOST_KEY / 16;
  __shared__ float ks[CPAB_DELTA_MOST_KEY], qs[CPAB_DELTA_MOST_KEY];
  __shared__ f32x4 sums[2][4][16];
  const int64_t heads = d.r.B * d.r.heads, bh = blockIdx.x % heads, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group;
  const int dk = (int)d.r.dk, dv = (int)d.r.dv;
  const int col = (int)(blockIdx.x / heads) * 64 + 4 * (threadIdx.x & 15), r = threadIdx.x >> 4;
  const int here = min(4, dv - col);   // columns of this lane; may be less than 1
  const int64_t length = live_of(d, b);
  float S[kRows][4];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int row = r + 16 * k;
#pragma unroll
    for (int e = 0; e < 4; ++e) S[k][e] = 0.0f;
    if (d.r.h0 && row < dk && here > 0) {
      const float* p = d.r.h0 + (bh * dk + row) * dv + col;
      if (here == 4) {
        load<4>(p, S[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < here) S[k][e] = p[e];
      }
    }
  }
  const T* q = static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + kh * d.r.q_strides[2];
  const T* k = static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + kh * d.r.k_strides[2];
  const T* v = static_cast<const T*>(d.r.v) + b * d.r.v_strides[0] + h * d.r.v_strides[2];
  for (int64_t t = 0; t < length; ++t) {
    __syncthreads();
    if (threadIdx.x < CPAB_DELTA_MOST_KEY) {
      const bool in = (int)threadIdx.x < dk;
      ks[threadIdx.x] = in ? to_float(k[t * d.r.k_strides[1] + threadIdx.x]) : 0.0f;
      qs[threadIdx.x] = in ? to_float(q[t * d.r.q_strides[1] + threadIdx.x]) : 0.0f;
    }
    const float a = expf(clamped(gate_at(d, d.r.decay, b * d.r.decay_strides[0] + t * d.r.decay_strides[1] + h * d.r.decay_strides[2])));
    const float beta = gate_at(d, d.r.beta, b * d.r.beta_strides[0] + t * d.r.beta_strides[1] + h * d.r.beta_strides[2]);
    float val[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < here) val[e] = to_float(v[t * d.r.v_strides[1] + col + e]);
    __syncthreads();
    float sk[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0}, kq = 0.0f, kv[kRows];
#pragma unroll
    for (int n = 0; n < kRows; ++n) {
      kv[n] = ks[r + 16 * n];
      const float qv = qs[r + 16 * n];
      kq = fmaf(kv[n], qv, kq);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        S[n][e] *= a;
        sk[e] = fmaf(kv[n], S[n][e], sk[e]);
        sq[e] = fmaf(qv, S[n][e], sq[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sk[e] += __shfl_xor(sk[e], 16);
      sk[e] += __shfl_xor(sk[e], 32);
      sq[e] += __shfl_xor(sq[e], 16);
      sq[e] += __shfl_xor(sq[e], 32);
    }
    kq += __shfl_xor(kq, 16);
    kq += __shfl_xor(kq, 32);
    __shared__ float kqs[4];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < 16) {
      sums[0][wave][threadIdx.x & 15] = f32x4{sk[0], sk[1], sk[2], sk[3]};
      sums[1][wave][threadIdx.x & 15] = f32x4{sq[0], sq[1], sq[2], sq[3]};
      kqs[wave] = kq;
    }
    __syncthreads();
    const int lane = threadIdx.x & 15;
    const f32x4 k_all = (sums[0][0][lane] + sums[0][1][lane]) + (sums[0][2][lane] + sums[0][3][lane]);
    const f32x4 q_all = (sums[1][0][lane] + sums[1][1][lane]) + (sums[1][2][lane] + sums[1][3][lane]);
    const float dot = (kqs[0] + kqs[1]) + (kqs[2] + kqs[3]);
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = beta * (val[e] - k_all[e]);
#pragma unroll
    for (int n = 0; n < kRows; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[n][e] = fmaf(kv[n], u[e], S[n][e]);
    if (r == 0) {
      T* to = o + ((b * d.r.T + t) * d.r.heads + h) * dv + col;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < here) to[e] = from_float<T>(d.r.scale * fmaf(dot, u[e], q_all[e]));
    }
  }
#pragma unroll
  for (int n = 0; n < kRows; ++n) {
    const int row = r + 16 * n;
    if (row < dk && here > 0) {
      float* p = h_out + (bh * dk + row) * dv + col;
      if (here == 4) {
        store<4>(p, S[n]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < here) p[e] = S[n][e];
      }
    }
  }
  if (r == 0)
    for (int64_t t = length; t < d.r.T; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < here) o[((b * d.r.T + t) * d.r.heads + h) * dv + col + e] = from_float<T>(0.0f);
}

// Sample by sample where there are so few of them.
bool steps(const cpab_delta_rule& r, bool keep) { return r.T <= (keep ? 0 : 16); }

}  // namespace

hipError_t launch_delta_squares(const Delta& d, float* squares, hipStream_t st) {
  hipError_t e = hipSuccess;
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value;
    constexpr int kRoom = 4 * 2 * std::max(kChunk * (DP + 4), kChunk * (kChunk + 4));
    static LdsAllowed allowed;
    e = allow_lds(reinterpret_cast<const void*>(delta_squares_kernel<T, DP>), kRoom, allowed);
    if (e != hipSuccess) return;
    delta_squares_kernel<T, DP><<<(unsigned)(d.r.B * d.r.heads * d.chunks), kDeltaBlock, kRoom, st>>>(d, squares);
    e = hipGetLastError();
  });
  return e;
}

int64_t delta_rule_kept(const cpab_delta_rule& r) {
  const Delta d = delta_of(r);
  return r.B * r.heads * (d.chunks * r.dk + r.T) * r.dv;
}

int64_t delta_rule_workspace(const cpab_delta_rule& r, bool keep, bool backward) {
  const Delta d = delta_of(r);
  if (!backward && steps(r, keep)) return 0;
  int64_t n = r.B * r.heads * d.chunks * kSquares;
  if (backward) n += r.B * r.heads * (d.chunks * r.dk + r.T) * r.dv;
  return 4 * n;
}

hipError_t launch_delta_rule_forward(const cpab_delta_rule& r, void* o, float* h, float* kept,
                                     void* workspace, hipStream_t st) {
  const Delta d = delta_of(r);
  const int64_t heads = r.B * r.heads;
  if (steps(r, kept != nullptr)) {
    const unsigned blocks = (unsigned)(heads * ((r.dv + 63) / 64));
    if (r.dtype == CPAB_F32)
      delta_steps_kernel<float><<<blocks, kDeltaBlock, 0, st>>>(d, (float*)o, h);
    else
      delta_steps_kernel<bf16><<<blocks, kDeltaBlock, 0, st>>>(d, (bf16*)o, h);
    return hipGetLastError();
  }
  float* squares = static_cast<float*>(workspace);
  hipError_t e = launch_delta_squares(d, squares, st);
  if (e != hipSuccess) return e;
  float* xs = kept ? kept + heads * d.chunks * r.dk * r.dv : nullptr;
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value;
    const auto run = [&](auto width) {
      constexpr int E = decltype(width)::value;
      constexpr int kRoom = 4 * ((2 * kChunk + E) * (DP + 4) + (E + 2 * kChunk) * (kChunk + 4));
      static LdsAllowed allowed;
      e = allow_lds(reinterpret_cast<const void*>(delta_chain_kernel<T, DP, E>), kRoom, allowed);
      if (e != hipSuccess) return;
      delta_chain_kernel<T, DP, E><<<(unsigned)(heads * ((r.dv + E - 1) / E)), kDeltaBlock, kRoom, st>>>(
          d, squares, (T*)o, h, kept, xs);
      e = hipGetLastError();
    };
    r.dv <= 32 ? run(std::integral_constant<int, 32>()) : run(std::integral_constant<int, 64>());
  });
  return e;
}

}  // namespace cpab
