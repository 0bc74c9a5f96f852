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
constexpr int kRow = kChunk + 8;   // pitch of 64 16-bit values in LDS: rows begin 4 banks apart
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A call as the kernels take it.  q and k are read in eights: rows of `read`, a multiple of
// 8, are dk wide or a copy that is padded with zeros.
struct Delta {
  cpab_delta_rule r;
  int chunks, group, read;
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

// ---- products ------------------------------------------------------------------

// The matrix unit's 32-bit products run at a sixteenth of the bfloat16 ones' rate, so that
// values of 32 bits go as sums of three bfloat16 parts, each the nearest to what the ones
// before leave: 24 bits.  A 16-bit input is its own first part, a 32-bit one has three.  Of
// the products of parts those are taken that are not below the last part's rounding: three
// with an input of 16 bits, six of two values.  Outputs of 16 bits are made of two parts, 17
// bits (two throughout left the 32-bit states behind 16-bit inputs 3e-6 to 1e-5 off).
template <typename T>
struct Parts {
  static constexpr int kInput = 1, kValue = 3, kOut = 2;
};
template <>
struct Parts<float> {
  static constexpr int kInput = 3, kValue = 3, kOut = 3;
};
template <int N>
struct Frag {   // 8 neighbours of the summed index
  bf16x8 p[N];
};
// Two values at once, as the conversion takes them.
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int N>
__device__ __forceinline__ void split(float v0, float v1, bf16x2 (&p)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    p[k] = __builtin_convertvector(f32x2{v0, v1}, bf16x2);
    if (k + 1 == N) break;
    const uint32_t both = __builtin_bit_cast(uint32_t, p[k]);
    v0 -= __uint_as_float(both << 16);
    v1 -= __uint_as_float(both & 0xffff0000u);
  }
}
template <int N>
__device__ __forceinline__ Frag<N> frag_of(const float v[8]) {
  Frag<N> f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    bf16x2 p[N];
    split<N>(v[e], v[e + 1], p);
#pragma unroll
    for (int k = 0; k < N; ++k) f.p[k][e] = p[k][0], f.p[k][e + 1] = p[k][1];
  }
  return f;
}
// acc[m][n] += A[m] B[n]^T: 16 x 16 each, over 32 of the summed index.  The tiles in turn for
// each pair of parts: a product waits for the one before it in its own sums.
template <int MT, int NT, int NA, int NB>
__device__ __forceinline__ void mma(f32x4 (&acc)[MT][NT], const Frag<NA> (&a)[MT], const Frag<NB> (&b)[NT]) {
  constexpr int kLast = (NA > NB ? NA : NB) - 1;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j <= kLast)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m].p[i], b[n].p[j], acc[m][n], 0, 0, 0);
}
template <int NA, int NB>
__device__ __forceinline__ void mma(f32x4& acc, const Frag<NA>& a, const Frag<NB>& b) {
  constexpr int kLast = (NA > NB ? NA : NB) - 1;
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j <= kLast) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
}

// The first parts of an operand.
template <int N, int M>
__device__ __forceinline__ Frag<N> first_of(const Frag<M>& f) {
  Frag<N> r;
#pragma unroll
  for (int k = 0; k < N; ++k) r.p[k] = f.p[k];
  return r;
}

// 8 neighbours of a row as they come from memory, and what they are as an operand.  What is
// fetched ahead stays as it came: anything done with it would wait for it.
template <typename T>
struct Raw {
  typedef uint32_t U4 __attribute__((ext_vector_type(4)));
  static constexpr int kWords = sizeof(T) / 2;   // of 16 bytes
  U4 v[kWords];
  __device__ __forceinline__ void fetch(const T* p) {
    typedef U4 __attribute__((aligned(2))) Unit;
#pragma unroll
    for (int k = 0; k < kWords; ++k) v[k] = reinterpret_cast<const Unit*>(p)[k];
  }
  __device__ __forceinline__ void take(const T* p) {   // 16-byte aligned
#pragma unroll
    for (int k = 0; k < kWords; ++k) v[k] = reinterpret_cast<const U4*>(p)[k];
  }
  __device__ __forceinline__ void put(T* p) const {   // 16-byte aligned
#pragma unroll
    for (int k = 0; k < kWords; ++k) reinterpret_cast<U4*>(p)[k] = v[k];
  }
  __device__ __forceinline__ void keep(bool in) {
#pragma unroll
    for (int k = 0; k < kWords; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = in ? v[k][e] : 0u;
  }
  __device__ __forceinline__ Frag<Parts<T>::kInput> frag() const {
    if constexpr (sizeof(T) == 2) {
      return Frag<1>{{__builtin_bit_cast(bf16x8, v[0])}};
    } else {
      float f[8];
      __builtin_memcpy(f, v, 32);
      return frag_of<3>(f);
    }
  }
};

// Rows of an input: `live` of them, `width` values each, zeros beyond.  The last row or
// column is read again where there is nothing to read: without a branch between the lanes
// loads are not waited for one by one.  Offsets within a chunk have 32 bits
// (CPAB_DELTA_MOST_STRIDE), beside a base that is the whole wave's.
template <typename T>
struct Rows {
  const T* p;
  int stride, live, width;
  template <int N>
  __device__ __forceinline__ const T* place(int row, int col) const {   // of N neighbours; the width a multiple of N
    const uint32_t at = (uint32_t)(min(row, live - 1) * stride + min(col, width - N)) * (uint32_t)sizeof(T);
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + at);
  }
  __device__ __forceinline__ bool in(int row, int col) const { return row < live && col < width; }
  __device__ __forceinline__ void fetch(Raw<T>& r, int row, int col) const {
    r.fetch(place<8>(row, col));
    r.keep(in(row, col));
  }
  __device__ __forceinline__ Frag<Parts<T>::kInput> at(int row, int col) const {
    Raw<T> r;
    fetch(r, row, col);
    return r.frag();
  }
  __device__ __forceinline__ f32x4 four(int row, int col) const {
    float w[4];
    load<4>(place<4>(row, col), w);
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = in(row, col) ? w[e] : 0.0f;
    return v;
  }
};
// Makes a lane's number new to the compiler, which else computes every address that a loop
// takes from it once, before the loop, and has no registers for them.
__device__ __forceinline__ void renew(int& a) { asm volatile("" : "+v"(a)); }

// A value of another lane, by the vector unit's own exchanges; 0 where there is none.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float lane_at(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
// The sum over 8 or 16 neighbouring lanes.
__device__ __forceinline__ float over8(float v) {
  v += lane_at<0xb1>(v);    // the pair's other
  v += lane_at<0x4e>(v);    // of two pairs
  return v + lane_at<0x141>(v);   // mirrored in eights
}
__device__ __forceinline__ float over16(float v) {
  v = over8(v);
  return v + lane_at<0x140>(v);   // mirrored in sixteens
}
// The sum over the lanes 16, 32 and 48 on.
__device__ __forceinline__ float over_rows(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// The sum over the lanes before.
__device__ __forceinline__ float lanes_before(float v) {
  v += lane_at<0x111>(v);   // from 1, 2, 4 and 8 lanes below in the sixteen
  v += lane_at<0x112>(v);
  v += lane_at<0x114>(v);
  v += lane_at<0x118>(v);
  v += lane_at<0x142, 0xa>(v);   // the last of the sixteen before, to the second and the fourth
  v += lane_at<0x143, 0xc>(v);   // and of the half before
  return lane_at<0x138>(v);
}

// Waits for what has been loaded.  Before a loop whose registers begin with loads: the
// compiler, which does not tell its first round from the others, would wait in each of them,
// for everything that is fetched ahead.
__device__ __forceinline__ void loaded() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0) alone

// Operands in planes of 16-bit parts, in LDS or the workspace: 8 neighbours to a lane.
template <int N>
__device__ __forceinline__ Frag<N> plane_frag(const bf16* at, int plane) {
  Frag<N> f;
#pragma unroll
  for (int k = 0; k < N; ++k) f.p[k] = *reinterpret_cast<const bf16x8*>(at + k * plane);
  return f;
}
// Four neighbours of the summed index, as the sums of a product lie in a lane.
template <int N>
__device__ __forceinline__ void put4(bf16* at, int plane, const f32x4& v) {
  bf16x2 lo[N], hi[N];
  split<N>(v[0], v[1], lo);
  split<N>(v[2], v[3], hi);
#pragma unroll
  for (int k = 0; k < N; ++k)
    *reinterpret_cast<bf16x4*>(at + k * plane) = bf16x4{lo[k][0], lo[k][1], hi[k][0], hi[k][1]};
}

template <int MT, int NT>
__device__ __forceinline__ void clear(f32x4 (&acc)[MT][NT]) {
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[m][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// A chain's workgroup has 32 columns of a state; its four waves share its [DP, 32], WD of
// them over DP.
constexpr int kWide = 32;
template <int DP>
struct Shares {
  static constexpr int WD = DP / 16 < 4 ? DP / 16 : 4, WE = 4 / WD;
  static constexpr int MT = DP / 16 / WD, NT = kWide / 16 / WE;
};

// The unit matrix, 16 of its columns from 16 n on: A times it is A, as a product's sums lie.
// One wide load of a row and a product so bring an input to the sums' layout.
__device__ __forceinline__ Frag<1> unit_frag(int n) {
  const int at = 16 * n + (threadIdx.x & 15) - 8 * ((threadIdx.x >> 4) & 3);
  Frag<1> f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f.p[0][e] = (bf16)(e == at ? 1.0f : 0.0f);
  return f;
}

// A product's sums, four rows of a column to a lane, as four columns of a row: lane i of 16
// then has row i mod 4 and columns from i - i mod 4 on.  One wide store in place of four.
__device__ __forceinline__ float exchanged(float v, bool two) {
  const int i = __float_as_int(v);
  return __int_as_float(two ? __builtin_amdgcn_update_dpp(i, i, 0x4e, 0xf, 0xf, true)
                            : __builtin_amdgcn_update_dpp(i, i, 0xb1, 0xf, 0xf, true));
}
__device__ __forceinline__ f32x4 across(f32x4 v) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const float got = exchanged(odd ? v[k] : v[k + 1], false);
    v[k] = odd ? got : v[k];
    v[k + 1] = odd ? v[k + 1] : got;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float got = exchanged(high ? v[k] : v[k + 2], true);
    v[k] = high ? got : v[k];
    v[k + 2] = high ? v[k + 2] : got;
  }
  return v;
}
__device__ __forceinline__ void store4(float* p, const f32x4& v) {
  const float w[4] = {v[0], v[1], v[2], v[3]};
  store<4>(p, w);
}
// Four neighbours of a row of an output; `left` of them are there.
template <typename T>
__device__ __forceinline__ void store_some(T* p, const f32x4& v, int left) {
  if (left >= 4) {
    const float w[4] = {v[0], v[1], v[2], v[3]};
    store<4>(p, w);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = from_float<T>(v[e]);
  }
}

// ---- workspace -----------------------------------------------------------------

// What the first kernel leaves lies as the matrix unit's operands do, 8 values to a lane:
// [tile of 16 rows][32 of the summed index][64 lanes][8], so that a wave reads whole lines
// (rows of 64 bytes, 16 of them, took the vector memory unit three times as long).  Of a
// chunk of a head: exp(G_i), exp(G_63 - G_i) and beta; M and P (their transposes for the
// backward) in planes.
struct Gates {
  double log[kChunk];   // the decays' logarithms, added up
  float since[kChunk], until[kChunk], beta[kChunk];
};
template <typename T>
struct Squares {
  Gates gates;
  bf16 m[Parts<T>::kValue][4][2][64][8];
  bf16 p[Parts<T>::kValue][4][2][64][8];
};
inline int64_t squares_bytes(int dtype) {
  return dtype == CPAB_F32 ? (int64_t)sizeof(Squares<float>) : (int64_t)sizeof(Squares<bf16>);
}
// And of a chunk of a key's head, zeros beyond its rows and columns: k and q [64, DP], and
// their transposes [DP, 64].
inline int key_rows(const cpab_delta_rule& r) { return r.dk <= 32 ? 32 : r.dk <= 64 ? 64 : 128; }
template <typename T, int DP>
struct Keys {
  typedef T Own[4][DP / 32][64][8];
  typedef T Turned[DP / 16][2][64][8];
  Own k, q;
  Turned kt, qt;   // qt for the backward
};
inline int64_t keys_bytes(const cpab_delta_rule& r) {
  return 4 * (int64_t)key_rows(r) * kChunk * (r.dtype == CPAB_F32 ? 4 : 2);
}

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
  return Delta{r, (int)((r.T + kChunk - 1) / kChunk), (int)(r.heads / r.key_heads), (int)(r.dk + 7) / 8 * 8};
}
// Widths that the library's own arrays of values have: rows of whole eights.
inline int64_t wide_of(const cpab_delta_rule& r) { return (r.dv + 7) / 8 * 8; }

// Rows of `width` values (three strides before them) to contiguous rows of whole eights,
// padded with zeros.
hipError_t launch_delta_pad(int dtype, const void* from, const int64_t strides[3], int64_t B, int64_t T,
                            int64_t heads, int64_t width, void* to, hipStream_t s);
// Padded copies of q and k where their width is not whole eights: bytes of both, and the
// call on them; of v likewise.
inline int64_t padded_keys(const cpab_delta_rule& r) {
  return r.dk % 8 == 0 ? 0 : 2 * r.B * r.T * r.key_heads * ((r.dk + 7) / 8 * 8) * (r.dtype == CPAB_F32 ? 4 : 2);
}
hipError_t pad_keys(Delta* d, void* room, hipStream_t s);
inline int64_t padded_values(const cpab_delta_rule& r) {
  return r.dv % 8 == 0 ? 0 : r.B * r.T * r.heads * wide_of(r) * (r.dtype == CPAB_F32 ? 4 : 2);
}

// How a call is cut: a head's chunks in `segs` segments of `each`.
struct Cut {
  int segs, each;
};
Cut cut_of(const Delta& d);

// Which part of a head a workgroup has.  The column blocks of one segment lie on one XCD,
// whose cache they share: workgroup n runs on XCD n mod 8.
struct Where {
  int64_t bh;
  int seg, block;
  bool in;
};
__device__ __forceinline__ Where where(int64_t heads, int segs, int blocks) {
  const int64_t slot = blockIdx.x / 8, group = slot / blocks * 8 + blockIdx.x % 8;
  return Where{group % heads, (int)(group / heads), (int)(slot % blocks), group < heads * segs};
}

// What a forward keeps, in floats: the states before each chunk, X, and the segments' maps,
// transposed.
struct Kept {
  int64_t states, xs, maps, all;
};
Kept kept_of(const Delta& d, const Cut& cut);

// squares: of each chunk of each head; keys: of each of each key's head.
hipError_t launch_delta_squares(const Delta& d, void* squares, void* keys, bool backward, hipStream_t s);
hipError_t launch_delta_join(const Delta& d, const Cut& cut, bool forward, const float* maps, const float* adds,
                             const float* given, float* to, hipStream_t s);
int64_t delta_backward_workspace(const Delta& d);   // bytes

}  // namespace cpab
