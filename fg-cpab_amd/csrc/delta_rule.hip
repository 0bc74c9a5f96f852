// Gated delta rule, forward: by chunks of 64 samples, and sample by sample for a few.
// The formulas stand in delta_device.hpp.
#include <algorithm>
#include <type_traits>

#include "cpab_launch.hpp"
#include "delta_device.hpp"

namespace cpab {
namespace {

// ---- a chunk's matrices ------------------------------------------------------

// 64 x 64 values from LDS to planes of operands in the workspace, or their transpose.
template <int N, bool TURNED, int M>
__device__ __forceinline__ void put_square(const float* from, int pitch, bf16 (&to)[M][4][2][64][8]) {
  for (int n = threadIdx.x; n < 512; n += kDeltaBlock) {
    const int lane = n & 63, step = n >> 6 & 1, tile = n >> 7;
    const int row = 16 * tile + (lane & 15), col = 32 * step + 8 * (lane >> 4);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = TURNED ? from[(col + e) * pitch + row] : from[row * pitch + col + e];
    const Frag<N> f = frag_of<N>(v);
#pragma unroll
    for (int k = 0; k < N; ++k) *reinterpret_cast<bf16x8*>(to[k][tile][step][lane]) = f.p[k];
  }
}

// A chunk of an input, transposed, to the workspace: zeros beyond its rows and columns.
// Four samples of four columns to a lane.  Called by the whole workgroup; `room` holds DP
// rows of kRow values.
template <int DP, typename T>
__device__ __forceinline__ void put_turned(T* room, const Rows<T>& from, T (&to)[DP / 16][2][64][8]) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  for (int k = threadIdx.x; k < 16 * (DP / 4); k += kDeltaBlock) {
    const int row = k % 16 * 4, col = k / 16 * 4;
    f32x4 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = from.four(row + e, col);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<T4*>(room + (col + e) * kRow + row) = T4{(T)v[0][e], (T)v[1][e], (T)v[2][e], (T)v[3][e]};
  }
  __syncthreads();
  for (int n = threadIdx.x; n < DP * 8; n += kDeltaBlock) {
    const int lane = n & 63, step = n >> 6 & 1, tile = n >> 7;
    Raw<T> r;
    r.fetch(room + (16 * tile + (lane & 15)) * kRow + 32 * step + 8 * (lane >> 4));
    r.put(to[tile][step][lane]);
  }
  __syncthreads();
}

// [16 x 16] += A B with 32-bit products, B as a product's sums lie in a lane: column i, rows
// 4 g to 4 g + 3, which are the summed index, in the order in which A is read.
__device__ __forceinline__ void multiply16(f32x4& acc, const float* A, int pitch, const f32x4& B) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const f32x4 a = *reinterpret_cast<const f32x4*>(A + i * pitch + 4 * g);
#pragma unroll
  for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], B[e], acc, 0, 0, 0);
}

// The gates, M and P of each chunk of each head, and the transposes of its keys and queries.
// The decays' logarithms are added in 64 bits: their differences are what counts, and a
// sample that clears the state (-128) would leave 32 bits 2^-17 of it.
// M by blocks of 16 rows, all in 32 bits: with T_b = (I + A_bb beta_b)^-1 of the blocks on the
// diagonal, by rows, a wave each, M_b = T_b (A_b - sum over c < b of A_bc beta_c M_c); a wave
// has 16 columns.
// 8 x 4096 samples of 16 heads of 128 in bfloat16, two to a key, take 198 us for 0.66 GB (0.55
// of them written: M and P in their parts, the keys and queries as the products take them),
// 3.4 TB/s; the backward, which makes all of it again rather than keep it, 239 for 0.85.
// Memory alone would take 130 and 166: the waves wait for two thirds of their cycles.
template <typename T, int DP, bool BACKWARD>
__global__ __launch_bounds__(kDeltaBlock) void delta_squares_kernel(Delta d, Squares<T>* squares, Keys<T, DP>* keys) {
  constexpr int kPitch = kChunk + 4, NV = Parts<T>::kValue, NI = Parts<T>::kInput;
  extern __shared__ float room[];
  __shared__ double G[kChunk];
  __shared__ float betas[kChunk];
  const int c = blockIdx.x % d.chunks;
  const int64_t bh = blockIdx.x / d.chunks, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group;
  const int64_t t0 = (int64_t)c * kChunk;
  const int live = (int)min(max(live_of(d, b) - t0, (int64_t)0), (int64_t)kChunk);
  if (live == 0) return;
  Squares<T>& out = squares[bh * d.chunks + c];
  if (threadIdx.x < kChunk) {
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
    G[t] = g;
    betas[t] = beta;
    out.gates.log[t] = g;
    out.gates.since[t] = expf((float)g);
    out.gates.until[t] = expf((float)(__shfl(g, 63) - g));
    out.gates.beta[t] = beta;
  }
  const Rows<T> krows{static_cast<const T*>(d.r.k) + b * d.r.k_strides[0] + t0 * d.r.k_strides[1] + kh * d.r.k_strides[2],
                      (int)d.r.k_strides[1], live, d.read};
  const Rows<T> qrows{static_cast<const T*>(d.r.q) + b * d.r.q_strides[0] + t0 * d.r.q_strides[1] + kh * d.r.q_strides[2],
                      (int)d.r.q_strides[1], live, d.read};
  const bool first = h % d.group == 0;   // of those that share a key
  Keys<T, DP>& own = keys[(b * d.r.key_heads + kh) * d.chunks + c];
  if (first) {
    put_turned<DP>(reinterpret_cast<T*>(room), krows, own.kt);
    if (BACKWARD) put_turned<DP>(reinterpret_cast<T*>(room), qrows, own.qt);
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  f32x4 kk[1][4], qk[1][4];
  clear(kk);
  clear(qk);
#pragma unroll
  for (int s = 0; s < DP / 32; ++s) {
    const int col = 32 * s + 8 * g;
    Raw<T> rk, rq;
    krows.fetch(rk, 16 * wave + i, col);
    qrows.fetch(rq, 16 * wave + i, col);
    if (first) {
      rk.put(own.k[wave][s][lane]);
      rq.put(own.q[wave][s][lane]);
    }
    const Frag<NI> ak[1] = {rk.frag()}, aq[1] = {rq.frag()};
    Frag<NI> bk[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) bk[n] = krows.at(16 * n + i, col);
    mma(kk, ak, bk);
    mma(qk, aq, bk);
  }
  __syncthreads();
  float* Ab = room;                   // A beta
  float* A = Ab + kChunk * kPitch;
  float* Ti = A + kChunk * kPitch;    // the four T
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * wave + 4 * g + e, col = 16 * n + i;
      const float decay = col <= row ? expf((float)(G[row] - G[col])) : 0.0f;
      const float a = col < row ? decay * kk[0][n][e] : 0.0f;
      qk[0][n][e] *= d.r.scale * decay;
      Ab[row * kPitch + col] = a * betas[col];
      A[row * kPitch + col] = a;
    }
  __syncthreads();
  {
    // column i of T, rows 4 g to 4 g + 3 of it: T_r = e_r - sum over j < r of (A beta)_rj T_j
    const float* block = Ab + 16 * wave * kPitch + 16 * wave;
    f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(block + r * kPitch + 4 * g);
      float sum = a[0] * t[0];   // rows that are not there yet are 0
#pragma unroll
      for (int e = 1; e < 4; ++e) sum = fmaf(a[e], t[e], sum);
      sum = over_rows(sum);
      const float v = (i == r ? 1.0f : 0.0f) - sum;
      t[r & 3] = g == r >> 2 ? v : t[r & 3];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) Ti[(16 * wave + 4 * g + e) * 20 + i] = t[e];
  }
  __syncthreads();
  f32x4 m[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {   // the block row; what lies above this wave's diagonal block is 0
    m[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (n < wave) continue;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f}, y;
#pragma unroll
    for (int c2 = 0; c2 < n; ++c2)
      if (c2 >= wave) multiply16(sum, Ab + 16 * n * kPitch + 16 * c2, kPitch, m[c2]);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = A[(16 * n + 4 * g + e) * kPitch + 16 * wave + i] - sum[e];
    multiply16(m[n], Ti + 16 * n * 20, 20, y);
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      A[(16 * n + 4 * g + e) * kPitch + 16 * wave + i] = m[n][e];
      Ab[(16 * wave + 4 * g + e) * kPitch + 16 * n + i] = qk[0][n][e];
    }
  __syncthreads();
  put_square<NV, BACKWARD>(A, kPitch, out.m);
  put_square<BACKWARD ? NV : Parts<T>::kOut, BACKWARD>(Ab, kPitch, out.p);
}

// ---- the chain of chunks -----------------------------------------------------

// One workgroup goes through the chunks of a segment with 32 columns of a head's state in
// registers, the sums of the matrix unit; LDS holds its parts for the next chunk's products.
// Keys, queries, M and P go from memory to the lanes as the matrix unit takes them.
// ENDS: no outputs but the state after the segment, from zeros, and, in columns of their
// own, from the unit matrix without values: what the segment adds and what it makes of the
// state before it.
// Bound by a chunk's chain of five products, each behind the other's LDS: 8 x 4096 samples of
// 16 heads of 128 in bfloat16 take 526 us, 8.2 a chunk with two workgroups to a compute unit in
// turn, of which the matrix unit has a sixth; the 1.45 GB that they read and write would take
// 285.  Half of the LDS' cycles are counted as conflicts of banks.
// 32 columns: 64, with the same matrices read half as often but one workgroup to a unit, took
// longer.  Operands in the order in which lanes take them: from rows of 256 bytes a third more.
template <typename T, int DP, bool ENDS>
__global__ __launch_bounds__(kDeltaBlock, 2) void delta_chain_kernel(
    Delta d, const Squares<T>* squares, const Keys<T, DP>* keys, const float* starts, Cut cut, T* o,
    float* h_out, float* states, float* xs, float* adds, float* maps, float* turned, int segs) {
  typedef Shares<DP> Sh;
  constexpr int E = kWide, kPitch = DP + 8, kSteps = DP / 32;
  constexpr int NV = Parts<T>::kValue, NI = Parts<T>::kInput, NO = Parts<T>::kOut;
  constexpr int kState = E * kPitch, kSamples = E * kRow;   // planes
  extern __shared__ __align__(16) bf16 lds[];
  bf16* St = lds;                  // [32][DP]
  bf16* Rt = St + NV * kState;     // beta R, [32][64]
  bf16* Ut = Rt + NV * kSamples;
  bf16* Ht = Ut + NO * kSamples;   // U until the chunk's end
  const int dk = (int)d.r.dk, dv = (int)d.r.dv, blocks_v = (dv + E - 1) / E, wide = (dv + 7) / 8 * 8;
  const int64_t heads = d.r.B * d.r.heads;
  const Where at = where(heads, segs, blocks_v + (ENDS ? DP / E : 0));
  if (!at.in) return;
  const int64_t bh = at.bh, b = bh / d.r.heads;
  const int h = (int)(bh - b * d.r.heads), kh = h / d.group;
  const bool unit = ENDS && at.block >= blocks_v;
  const int e0 = (unit ? at.block - blocks_v : at.block) * E;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int64_t length = live_of(d, b);
  const T* v = static_cast<const T*>(d.r.v) + b * d.r.v_strides[0] + h * d.r.v_strides[2];
  const int vs = (int)d.r.v_strides[1], hs = (int)d.r.heads;
  const int d0 = wave % Sh::WD * Sh::MT * 16, s0 = wave / Sh::WD * Sh::NT * 16;   // this wave's part of the state
  const int w0 = 16 * wave;                                                       // and of a chunk's samples
  f32x4 S[Sh::MT][Sh::NT];
  const float* start = ENDS ? nullptr : at.seg > 0 ? starts + (bh * cut.segs + at.seg) * dk * dv
                                      : d.r.h0     ? d.r.h0 + bh * dk * dv : nullptr;
#pragma unroll
  for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
    for (int n = 0; n < Sh::NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = d0 + 16 * m + 4 * g + e, col = e0 + s0 + 16 * n + i;
        S[m][n][e] = unit ? (row == col ? 1.0f : 0.0f)
                          : start && row < dk && col < dv ? start[(int64_t)row * dv + col] : 0.0f;
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
  const int chunks = (int)((length + kChunk - 1) / kChunk);
  const int first = at.seg * cut.each, last = min(first + cut.each, chunks);
  const Frag<1> eye[2] = {unit_frag(0), unit_frag(1)};
  // What a chunk's products take is fetched as soon as the chunk before is done with the
  // registers: memory has most of a chunk's time to answer.
  Raw<T> kf[kSteps], qf[kSteps], ktf[Sh::MT][2], vf;
  Frag<NV> mf[2];
  Frag<NO> pf[2];
  f32x4 since, until, beta;
  float mine, total;   // exp(G) of this lane's sample, and of the chunk's last
  const Squares<T>* sqs = squares + bh * d.chunks;
  const Keys<T, DP>* kys = keys + (b * d.r.key_heads + kh) * d.chunks;
  const auto vrows = [&](int c) {
    const int64_t t0 = (int64_t)c * kChunk;
    return Rows<T>{v + t0 * vs, vs, (int)min(length - t0, (int64_t)kChunk), wide};
  };
  const auto fetch_rows = [&](int c) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      kf[s].fetch(kys[c].k[wave][s][lane]);
      if (!ENDS) qf[s].fetch(kys[c].q[wave][s][lane]);
    }
    if (!unit) vf.fetch(vrows(c).template place<8>(w0 + i, e0 + 8 * g));
  };
  const auto fetch_m = [&](int c) {
#pragma unroll
    for (int s = 0; s < 2; ++s) mf[s] = plane_frag<NV>(sqs[c].m[0][wave][s][lane], kSquare);
    since = *reinterpret_cast<const f32x4*>(sqs[c].gates.since + w0 + 4 * g);
    until = *reinterpret_cast<const f32x4*>(sqs[c].gates.until + w0 + 4 * g);
    beta = *reinterpret_cast<const f32x4*>(sqs[c].gates.beta + w0 + 4 * g);
    if (!ENDS) mine = sqs[c].gates.since[w0 + i];
  };
  const auto fetch_rest = [&](int c) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (!ENDS) pf[s] = plane_frag<NO>(sqs[c].p[0][wave][s][lane], kSquare);
#pragma unroll
      for (int m = 0; m < Sh::MT; ++m) ktf[m][s].fetch(kys[c].kt[d0 / 16 + m][s][lane]);
    }
    total = sqs[c].gates.since[kChunk - 1];
  };
  loaded();
  if (first < last) {
    fetch_rows(first);
    fetch_m(first);
    fetch_rest(first);
  }
  for (int c = first; c < last; ++c) {
    const int64_t t0 = (int64_t)c * kChunk, row0 = (b * d.r.T + t0) * d.r.heads + h;
    const int live = (int)min(length - t0, (int64_t)kChunk), next = min(c + 1, last - 1);
    renew(lane);
    i = lane & 15, g = lane >> 4;
    if (!ENDS && states) {
      float* to = states + (bh * d.chunks + c) * dk * wide;
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
    if (!unit) {
      const Rows<T> rows = vrows(c);
      if (live < kChunk || e0 + E > wide) vf.keep(rows.in(w0 + i, e0 + 8 * g));
    }
    __syncthreads();
    f32x4 R[1][2], O[2][1], X[1][2];   // O: rows are columns of values, columns are samples
    clear(R);
    clear(O);
    {
      Frag<NV> st[2][2];   // this step's and the next's: LDS answers while the matrix unit works
      const auto read = [&](int s) {
#pragma unroll
        for (int n = 0; n < 2; ++n) st[s & 1][n] = plane_frag<NV>(St + (16 * n + i) * kPitch + 32 * s + 8 * g, kState);
      };
      read(0);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (s + 1 < kSteps) read(s + 1);
        const Frag<NI> kv[1] = {kf[s].frag()};
        mma(R, kv, st[s & 1]);
        if (!ENDS) {
          const Frag<NI> qv[1] = {qf[s].frag()};
          const Frag<NO> so[2] = {first_of<NO>(st[s & 1][0]), first_of<NO>(st[s & 1][1])};
          mma(O, so, qv);
        }
      }
    }
    const Frag<NI> vv = vf.frag();
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      R[0][n] *= -since;
      if (!unit) mma(R[0][n], vv, eye[n]);
      if (!ENDS) O[n][0] *= d.r.scale * mine;
      put4<NV>(Rt + (16 * n + i) * kRow + w0 + 4 * g, kSamples, beta * R[0][n]);
    }
    fetch_rows(next);
    __syncthreads();
    clear(X);
    {
      Frag<NV> rt[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < 2; ++n) rt[s][n] = plane_frag<NV>(Rt + (16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const Frag<NV> mv[1] = {mf[s]};
        mma(X, mv, rt[s]);
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const f32x4 x = R[0][n] - X[0][n], u = beta * x;
      const int to = (16 * n + i) * kRow + w0 + 4 * g;
      if (!ENDS) put4<NO>(Ut + to, kSamples, u);
      put4<NV>(Ht + to, kSamples, until * u);
      if (!ENDS && xs) {
        const int t = w0 + 4 * g + (i & 3), col = e0 + 16 * n + (i & 12);
        const f32x4 row = across(x);
        if (t < live && col < wide) store4(xs + row0 * wide + t * hs * wide + col, row);
      }
    }
    fetch_m(next);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) S[m][n] *= total;
    {
      Frag<NV> ht[2][Sh::NT];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int n = 0; n < Sh::NT; ++n)
          ht[s][n] = plane_frag<NV>(Ht + (s0 + 16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Frag<NI> kv[Sh::MT];
#pragma unroll
        for (int m = 0; m < Sh::MT; ++m) kv[m] = ktf[m][s].frag();
        mma(S, kv, ht[s]);
      }
    }
    if (!ENDS) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Frag<NO> ut[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) ut[n] = plane_frag<NO>(Ut + (16 * n + i) * kRow + 32 * s + 8 * g, kSamples);
        const Frag<NO> pv[1] = {pf[s]};
        mma(O, ut, pv);
      }
    }
    fetch_rest(next);
    if (ENDS) continue;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int t = w0 + i, col = e0 + 16 * n + 4 * g;
      if (t < live && col < dv) store_some(o + row0 * dv + t * hs * dv + col, O[n][0], dv - col);
    }
  }
  if (ENDS) {
    const int64_t segment = bh * cut.segs + at.seg;
    if (!unit) {
      put_state(adds + segment * dk * dv, dv);
      return;
    }
    // the map [DP, DP], as the join takes its rows, and transposed for the backward's
#pragma unroll
    for (int m = 0; m < Sh::MT; ++m)
#pragma unroll
      for (int n = 0; n < Sh::NT; ++n) {
        const int row = d0 + 16 * m + 4 * g, col = e0 + s0 + 16 * n;
        store4(maps + (segment * DP + row + (i & 3)) * DP + col + (i & 12), across(S[m][n]));
        if (turned) store4(turned + (segment * DP + col + i) * DP + row, S[m][n]);
      }
    return;
  }
  if (at.seg == (chunks > 0 ? (chunks - 1) / cut.each : 0)) put_state(h_out + bh * dk * dv, dv);
  const int64_t rest = max(length, (int64_t)first * kChunk), stop = min((int64_t)(first + cut.each) * kChunk, d.r.T);
  for (int64_t n = rest * E + threadIdx.x; n < stop * E; n += kDeltaBlock) {
    const int64_t t = n / E;
    const int col = e0 + (int)(n % E);
    if (col < dv) o[((b * d.r.T + t) * d.r.heads + h) * dv + col] = from_float<T>(0.0f);
  }
}

// The states that the segments begin with, one after another: 16 columns to a workgroup.
// FORWARD: to[s + 1] = what segment s makes of to[s] and what it adds.  Else the gradients
// that they end with: to[s - 1] = the transposed map of s on to[s], and what s adds.  The map
// and what is added are fetched a segment ahead.
template <int DP, bool FORWARD>
__global__ __launch_bounds__(kDeltaBlock) void delta_join_kernel(Delta d, Cut cut, const float* maps,
                                                               const float* adds, const float* given, float* to) {
  constexpr int kPitch = DP + 8, kPlane = 16 * kPitch, kSteps = DP / 32, kTiles = (DP / 16 + 3) / 4;
  __shared__ __align__(16) bf16 St[3 * kPlane];
  const int dk = (int)d.r.dk, dv = (int)d.r.dv;
  const int64_t heads = d.r.B * d.r.heads, bh = blockIdx.x % heads, b = bh / d.r.heads;
  const int col = (int)(blockIdx.x / heads) * 16 + (threadIdx.x & 15);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const int chunks = (int)((live_of(d, b) + kChunk - 1) / kChunk);
  const int live = min((chunks + cut.each - 1) / cut.each, cut.segs);   // segments with samples
  const auto at = [&](int m) { return min(16 * (wave + 4 * m), DP - 16); };   // a wave's tile; waves beyond repeat the last
  f32x4 S[kTiles], added[kTiles];
  Raw<float> map[kTiles][kSteps];
  const auto fetch = [&](int n) {
    const int64_t s = bh * cut.segs + (FORWARD ? n : live - 1 - n);
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k) map[m][k].fetch(maps + (s * DP + at(m) + i) * DP + 32 * k + 8 * g);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        added[m][e] = adds[(s * dk + min(at(m) + 4 * g + e, dk - 1)) * dv + min(col, dv - 1)];
    }
  };
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = at(m) + 4 * g + e;
      S[m][e] = given && row < dk && col < dv ? given[(bh * dk + row) * dv + col] : 0.0f;
    }
  loaded();
  if (live > 1) fetch(0);
  for (int n = 0; n + 1 < live; ++n) {
    const int s = FORWARD ? n : live - 1 - n;
#pragma unroll
    for (int m = 0; m < kTiles; ++m) put4<3>(St + i * kPitch + at(m) + 4 * g, kPlane, S[m]);
    Frag<3> a[kTiles][kSteps];
#pragma unroll
    for (int m = 0; m < kTiles; ++m) {
      S[m] = added[m];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) a[m][k] = map[m][k].frag();
    }
    fetch(min(n + 1, live - 2));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const Frag<3> st = plane_frag<3>(St + i * kPitch + 32 * k + 8 * g, kPlane);
#pragma unroll
      for (int m = 0; m < kTiles; ++m) mma(S[m], a[m][k], st);
    }
    __syncthreads();
    float* out = to + (bh * cut.segs + (FORWARD ? s + 1 : s - 1)) * dk * dv;
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = at(m) + 4 * g + e;
        if (row < dk && col < dv) out[(int64_t)row * dv + col] = S[m][e];
        else S[m][e] = 0.0f;
      }
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
      sk[e] = over_rows(sk[e]);
      sq[e] = over_rows(sq[e]);
    }
    kq = over_rows(kq);
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

template <typename T>
__global__ __launch_bounds__(kDeltaBlock) void delta_pad_kernel(const T* from, int64_t s0, int64_t s1, int64_t s2,
                                                              int64_t T_, int64_t heads, int width, int wide,
                                                              int64_t n, T* to) {
  for (int64_t at = (int64_t)blockIdx.x * kDeltaBlock + threadIdx.x; at < n; at += (int64_t)gridDim.x * kDeltaBlock) {
    const int64_t row = at / wide, token = row / heads, b = token / T_;
    const int col = (int)(at - row * wide);
    to[at] = col < width ? from[b * s0 + (token - b * T_) * s1 + (row - token * heads) * s2 + col] : (T)0.0f;
  }
}

// Sample by sample where there are so few of them (64 rows of 4 heads of 64 in bfloat16: 4
// samples take 11 us and 21 in a chunk, 8 17 and 21, 16 28 and 21; 16 heads of 128: 8 50 and 82,
// 16 85 and 85), but never where something is kept: the backward goes by chunks.
bool steps(const cpab_delta_rule& r, bool keep) { return r.T <= (keep ? 0 : 8); }

}  // namespace

hipError_t launch_delta_pad(int dtype, const void* from, const int64_t strides[3], int64_t B, int64_t T,
                            int64_t heads, int64_t width, void* to, hipStream_t st) {
  const int wide = (int)((width + 7) / 8 * 8);
  const int64_t n = B * T * heads * wide;
  if (n == 0) return hipSuccess;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + kDeltaBlock - 1) / kDeltaBlock, 1 << 16);
  const auto run = [&](auto t) {
    typedef decltype(t) V;
    delta_pad_kernel<V><<<blocks, kDeltaBlock, 0, st>>>((const V*)from, strides[0], strides[1], strides[2], T, heads,
                                                        (int)width, wide, n, (V*)to);
  };
  dtype == CPAB_F32 ? run(0.0f) : run(bf16());
  return hipGetLastError();
}

hipError_t pad_keys(Delta* d, void* room, hipStream_t st) {
  cpab_delta_rule& r = d->r;
  if (r.dk % 8 == 0) return hipSuccess;
  char* second = static_cast<char*>(room) + padded_keys(r) / 2;
  hipError_t e = launch_delta_pad(r.dtype, r.q, r.q_strides, r.B, r.T, r.key_heads, r.dk, room, st);
  if (e == hipSuccess) e = launch_delta_pad(r.dtype, r.k, r.k_strides, r.B, r.T, r.key_heads, r.dk, second, st);
  r.q = room, r.k = second;
  for (int64_t* s : {r.q_strides, r.k_strides}) {
    s[2] = d->read;
    s[1] = r.key_heads * d->read;
    s[0] = r.T * s[1];
  }
  return e;
}

hipError_t launch_delta_squares(const Delta& d, void* squares, void* keys, bool backward, hipStream_t st) {
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value;
    constexpr int kRoom = std::max<int>(4 * kChunk * (2 * (kChunk + 4) + 20), DP * kRow * (int)sizeof(T));
    const unsigned blocks = (unsigned)(d.r.B * d.r.heads * d.chunks);
    if (backward)
      delta_squares_kernel<T, DP, true><<<blocks, kDeltaBlock, kRoom, st>>>(d, (Squares<T>*)squares, (Keys<T, DP>*)keys);
    else
      delta_squares_kernel<T, DP, false><<<blocks, kDeltaBlock, kRoom, st>>>(d, (Squares<T>*)squares, (Keys<T, DP>*)keys);
  });
  return hipGetLastError();
}

hipError_t launch_delta_join(const Delta& d, const Cut& cut, bool forward, const float* maps, const float* adds,
                             const float* given, float* to, hipStream_t st) {
  with_key(d, [&](auto, auto dp) {
    constexpr int DP = decltype(dp)::value;
    const unsigned blocks = (unsigned)(d.r.B * d.r.heads * ((d.r.dv + 15) / 16));
    if (forward)
      delta_join_kernel<DP, true><<<blocks, kDeltaBlock, 0, st>>>(d, cut, maps, adds, given, to);
    else
      delta_join_kernel<DP, false><<<blocks, kDeltaBlock, 0, st>>>(d, cut, maps, adds, given, to);
  });
  return hipGetLastError();
}

// Two workgroups to a compute unit between them, in segments of at least 8 chunks, or 4 where
// a head is short: the segments' ends and their joining are then paid for.  One head of 128 of
// four in bfloat16, forward and with the backward, us: 8192 samples 364 and 978 in one piece,
// 117 and 332 in 16 segments, 153 and 406 in 32; 1024 64 and 182 in one, 54 and 154 in 4; 131072
// 5626 and 16203, 1020 and 3460 in 32 (16: 1023 and 3584).  Fewer than 4 segments cost more than they give: 64
// rows of 4096 samples, 2 heads of 64, 320 and 1206 in one, 403 and 1508 in 2.
Cut cut_of(const Delta& d) {
  const int64_t columns = d.r.B * d.r.heads * ((d.r.dv + 31) / 32);
  const int64_t want = columns > 0 ? 2 * compute_units() / columns : 1;
  const int segs = (int)std::min<int64_t>(want, std::max(d.chunks / 8, std::min(d.chunks / 4, 8)));
  if (segs < 4) return Cut{1, std::max(d.chunks, 1)};
  const int each = (d.chunks + segs - 1) / segs;
  return Cut{(d.chunks + each - 1) / each, each};
}

Kept kept_of(const Delta& d, const Cut& cut) {
  const int64_t heads = d.r.B * d.r.heads;
  Kept k;
  k.states = 0;
  k.xs = heads * d.chunks * d.r.dk * wide_of(d.r);
  k.maps = k.xs + heads * d.r.T * wide_of(d.r);
  k.all = k.maps + (cut.segs > 1 ? heads * cut.segs * key_rows(d.r) * key_rows(d.r) : 0);
  return k;
}
int64_t delta_rule_kept(const cpab_delta_rule& r) {
  const Delta d = delta_of(r);
  return kept_of(d, cut_of(d)).all;
}

namespace {

// The forward's workspace (bytes).
struct Room {
  int64_t squares, keys, starts, adds, maps, padded, values, all;
};
Room room_of(const Delta& d, const Cut& cut) {
  const int64_t heads = d.r.B * d.r.heads;
  const auto next = [](int64_t n) { return (n + 255) / 256 * 256; };
  Room w;
  w.squares = 0;
  w.keys = next(heads * d.chunks * squares_bytes(d.r.dtype));
  w.starts = w.keys + next(d.r.B * d.r.key_heads * d.chunks * keys_bytes(d.r));
  const int64_t segments = cut.segs > 1 ? heads * cut.segs : 0;
  w.adds = w.starts + next(segments * d.r.dk * d.r.dv * 4);
  w.maps = w.adds + next(segments * d.r.dk * d.r.dv * 4);
  w.padded = w.maps + next(segments * key_rows(d.r) * key_rows(d.r) * 4);
  w.values = w.padded + next(padded_keys(d.r));
  w.all = w.values + padded_values(d.r);
  return w;
}

}  // namespace

int64_t delta_rule_workspace(const cpab_delta_rule& r, bool keep, bool backward) {
  const Delta d = delta_of(r);
  if (backward) return delta_backward_workspace(d);
  return steps(r, keep) ? 0 : room_of(d, cut_of(d)).all;
}

hipError_t launch_delta_rule_forward(const cpab_delta_rule& r, void* o, float* h, float* kept,
                                     void* workspace, hipStream_t st) {
  Delta d = delta_of(r);
  const int64_t heads = r.B * r.heads;
  if (steps(r, kept != nullptr)) {
    const unsigned blocks = (unsigned)(heads * ((r.dv + 63) / 64));
    if (r.dtype == CPAB_F32)
      delta_steps_kernel<float><<<blocks, kDeltaBlock, 0, st>>>(d, (float*)o, h);
    else
      delta_steps_kernel<bf16><<<blocks, kDeltaBlock, 0, st>>>(d, (bf16*)o, h);
    return hipGetLastError();
  }
  const Cut cut = cut_of(d);
  const Room w = room_of(d, cut);
  const Kept k = kept_of(d, cut);
  char* room = static_cast<char*>(workspace);
  float* starts = reinterpret_cast<float*>(room + w.starts);
  float* adds = reinterpret_cast<float*>(room + w.adds);
  float* maps = reinterpret_cast<float*>(room + w.maps);
  hipError_t e = pad_keys(&d, room + w.padded, st);
  if (e == hipSuccess && r.dv % 8 != 0) {
    e = launch_delta_pad(r.dtype, r.v, r.v_strides, r.B, r.T, r.heads, r.dv, room + w.values, st);
    d.r.v = room + w.values;
    d.r.v_strides[2] = wide_of(r);
    d.r.v_strides[1] = r.heads * wide_of(r);
    d.r.v_strides[0] = r.T * r.heads * wide_of(r);
  }
  if (e == hipSuccess) e = launch_delta_squares(d, room + w.squares, room + w.keys, false, st);
  if (e != hipSuccess) return e;
  with_key(d, [&](auto t, auto dp) {
    typedef decltype(t) T;
    constexpr int DP = decltype(dp)::value, NV = Parts<T>::kValue, NO = Parts<T>::kOut;
    const Squares<T>* squares = reinterpret_cast<const Squares<T>*>(room + w.squares);
    const Keys<T, DP>* keys = reinterpret_cast<const Keys<T, DP>*>(room + w.keys);
    const auto run = [&](auto only_ends, int segs) {
      constexpr bool ENDS = decltype(only_ends)::value;
      constexpr int kRoom = 2 * kWide * (NV * (DP + 8) + (2 * NV + NO) * kRow);
      static LdsAllowed allowed;
      e = allow_lds(reinterpret_cast<const void*>(delta_chain_kernel<T, DP, ENDS>), kRoom, allowed);
      if (e != hipSuccess) return;
      const int64_t blocks = (r.dv + kWide - 1) / kWide + (ENDS ? DP / kWide : 0);
      delta_chain_kernel<T, DP, ENDS><<<(unsigned)((heads * segs + 7) / 8 * 8 * blocks), kDeltaBlock, kRoom, st>>>(
          d, squares, keys, starts, cut, (T*)o, h, kept, kept ? kept + k.xs : nullptr, adds, maps,
          kept ? kept + k.maps : nullptr, segs);
      e = hipGetLastError();
    };
    if (cut.segs > 1) {
      // the backward takes what the last segment makes of the state too
      run(std::true_type(), kept ? cut.segs : cut.segs - 1);
      if (e == hipSuccess) e = launch_delta_join(d, cut, true, maps, adds, r.h0, starts, st);
      if (e != hipSuccess) return;
    }
    run(std::false_type(), cut.segs);
  });
  return e;
}

}  // namespace cpab
