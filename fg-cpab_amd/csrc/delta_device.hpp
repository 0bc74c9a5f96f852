// What the kernels of the gated delta rule share.
//
// A chunk of 64 samples at once.  With the decays' logarithms added up from the chunk's
// start, G_i, and S the state before it:
//   A_ij = exp(G_i - G_j) k_i.k_j  (j < i),      P_ij = scale exp(G_i - G_j) q_i.k_j  (j <= i),
//   X = (I + A beta)^-1 R,  R_i = v_i - exp(G_i) S^T k_i,  U = beta X,
//   o_i = scale exp(G_i) S^T q_i + (P U)_i,
//   S after = exp(G_63) S + sum of exp(G_63 - G_j) k_j u_j^T.
// With M = A (I + beta A)^-1 the inverse is I - M beta, and its transpose's counterpart in
// the backward I - M^T beta: nothing is divided by beta.  Backward, from the gradients dO and
// dS of the state after:
//   dU = P^T dO + exp(G_63 - G_j) dS^T k_j,  E = dU - M^T (beta dU),  Z = beta E = dV,
//   dbeta_j = X_j.E_j,
//   dS before = exp(G_63) dS + sum of scale exp(G_i) q_i do_i^T - exp(G_i) k_i z_i^T,
//   dP = dO U^T,  dA_ij = -beta_j Z_i.X_j,
//   dQ_i = scale exp(G_i) S do_i + (scale D dP) K,
//   dK = (scale D dP)^T Q + exp(G_63 - G_j) dS u_j - exp(G_i) S z_i + (D dA) K + (D dA)^T K,
// and the gradient of a sample's decay is what passes from before it to it and after:
//   sum over i >= t > j of dP P + dA A, over i >= t of scale exp(G_i) q_i.S do_i -
//   exp(G_i) k_i.S z_i, over j < t of exp(G_63 - G_j) k_j.dS u_j, and exp(G_63) <S, dS>:
// every term carries the decay itself, so that none of them cancel where it is small.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "heads_launch.hpp"
#include "sequence_device.hpp"

namespace cpab {

constexpr int kChunk = 64;    // samples
constexpr int kDeltaBlock = 256;
constexpr int kSquare = kChunk * kChunk;
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A call as the kernels take it.
struct Delta {
  cpab_delta_rule r;
  int chunks, group;
};

__device__ __forceinline__ int64_t live_of(const Delta& d, int64_t b) {
  if (!d.r.lengths) return d.r.T;
  const int64_t n = d.r.lengths64 ? static_cast<const int64_t*>(d.r.lengths)[b]
                                  : (int64_t)static_cast<const int32_t*>(d.r.lengths)[b];
  return n < 0 ? 0 : n > d.r.T ? d.r.T : n;
}

__device__ __forceinline__ float gate_at(const Delta& d, const void* p, int64_t at) {
  return d.r.gate_dtype == CPAB_F32 ? static_cast<const float*>(p)[at]
                                    : to_float(static_cast<const bf16*>(p)[at]);
}
__device__ __forceinline__ float clamped(float decay) { return decay < -128.0f ? -128.0f : decay; }

// The gates of a chunk.  The logarithms are added in 64 bits: their differences are what
// counts, and a sample that clears the state (-128) would leave 32 bits 2^-17 of it.
struct Gates {
  double G[kChunk];
  float since[kChunk];   // exp(G_i)
  float until[kChunk];   // exp(G_63 - G_i)
  float beta[kChunk];
};
// By the first wave; the caller synchronises.
__device__ __forceinline__ void load_gates(Gates& s, const Delta& d, int64_t b, int h, int64_t t0, int live) {
  if (threadIdx.x >= 64) return;
  const int t = threadIdx.x;
  double g = 0.0;
  float beta = 0.0f;
  if (t < live) {
    g = (double)clamped(gate_at(d, d.r.decay, b * d.r.decay_strides[0] + (t0 + t) * d.r.decay_strides[1] +
                                                  h * d.r.decay_strides[2]));
    beta = gate_at(d, d.r.beta, b * d.r.beta_strides[0] + (t0 + t) * d.r.beta_strides[1] +
                                    h * d.r.beta_strides[2]);
  }
  for (int k = 1; k < 64; k *= 2) {
    const double before = __shfl_up(g, k);
    if (t >= k) g += before;
  }
  s.G[t] = g;
  s.beta[t] = beta;
  s.since[t] = expf((float)g);
  s.until[t] = expf((float)(__shfl(g, 63) - g));
}

// [64, D] of a chunk as 32-bit floats in LDS, zeros beyond `live` and D (up to DP).
template <int DP, typename T>
__device__ __forceinline__ void load_rows(float* to, int pitch, const T* from, int64_t stride, int live, int D) {
  constexpr int kQuads = DP / 4;
#pragma unroll 4
  for (int k = threadIdx.x; k < kChunk * kQuads; k += kDeltaBlock) {
    const int row = k / kQuads, col = k % kQuads * 4;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row < live) {
      const T* p = from + row * stride + col;
      if (col + 4 <= D) {
        load<4>(p, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < D) v[e] = to_float(p[e]);
      }
    }
    *reinterpret_cast<f32x4*>(to + row * pitch + col) = f32x4{v[0], v[1], v[2], v[3]};
  }
}

// acc += A B^T of 16 x 16 tiles by the matrix unit: A [16 MT, n], B [16 NT, n] in LDS, the
// summed index contiguous, or with AT / BT the other one; `scale`: of the summed index (or
// NULL).  A lane takes four neighbours of the summed index at once, the same of A and B, so
// that one wide read feeds four products.
template <bool ACROSS>
__device__ __forceinline__ f32x4 operand(const float* p, int pitch, int row, int k) {
  if (!ACROSS) return *reinterpret_cast<const f32x4*>(p + row * pitch + k);
  return f32x4{p[k * pitch + row], p[(k + 1) * pitch + row], p[(k + 2) * pitch + row], p[(k + 3) * pitch + row]};
}
template <bool AT, bool BT, int MT, int NT>
__device__ __forceinline__ void multiply(f32x4 (&acc)[MT][NT], const float* A, int lda, const float* B,
                                         int ldb, int n, const float* scale = nullptr) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll 2
  for (int k0 = 0; k0 < n; k0 += 16) {
    const int k = k0 + 4 * g;
    f32x4 a[MT], b[NT];
#pragma unroll
    for (int m = 0; m < MT; ++m) a[m] = operand<AT>(A, lda, 16 * m + i, k);
#pragma unroll
    for (int c = 0; c < NT; ++c) b[c] = operand<BT>(B, ldb, 16 * c + i, k);
    if (scale) {
      const f32x4 s = *reinterpret_cast<const f32x4*>(scale + k);
#pragma unroll
      for (int m = 0; m < MT; ++m) a[m] *= s;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int c = 0; c < NT; ++c)
          acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m][e], b[c][e], acc[m][c], 0, 0, 0);
  }
}
template <int MT, int NT>
__device__ __forceinline__ void clear(f32x4 (&acc)[MT][NT]) {
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[m][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// How four waves share a state's block of [DP, E]: WD of them over DP.
template <int DP, int E>
struct Shares {
  static constexpr int WD = DP / 16 < 4 ? DP / 16 : 4, WE = 4 / WD;
  static constexpr int MT = DP / 16 / WD, NT = E / 16 / WE;
};

// f(T(), DP) as types and constants.
template <typename F>
void with_key(const Delta& d, F f) {
  const auto typed = [&](auto t) {
    if (d.r.dk <= 32) return f(t, std::integral_constant<int, 32>());
    if (d.r.dk <= 64) return f(t, std::integral_constant<int, 64>());
    f(t, std::integral_constant<int, 128>());
  };
  d.r.dtype == CPAB_F32 ? typed(0.0f) : typed(bf16());
}

inline Delta delta_of(const cpab_delta_rule& r) {
  return Delta{r, (int)((r.T + kChunk - 1) / kChunk), (int)(r.heads / r.key_heads)};
}

// Workspace of a chunk of a head: M, P, A.
constexpr int64_t kSquares = 3 * kSquare;

hipError_t launch_delta_squares(const Delta& d, float* squares, hipStream_t s);

}  // namespace cpab
