// A Muon step over many matrices: the momentum, the orthogonalisation of its update by
// Newton-Schulz products, and the parameters' move.
//
// m = mu m + (1 - mu) g, u = mu m + (1 - mu) g (Nesterov) or m, X = u / max(|u|, eps),
// then some times  A = X X^T,  B = c1 A + c2 A A,  X = c0 X + B X,  at last
// p = p (1 - lr wd) - rate X.  X is taken with its shorter side first.
//
// Bound by the matrix unit.  Its 32-bit products run at a seventh of the 16-bit ones' rate in a
// large library product here (154 and 1113 TFLOP/s), so X, A and B are held as two 16-bit
// floats, the nearest to 2^10 times the value and to what is left, and a product is three, hi
// hi, hi lo and lo hi, in one sum of 32 bits; lo lo, 2^-22 of the whole, is left out.  2^10:
// the second float's last place is 2^-34 of 1, which gives 22 bits to what is above 2^-12 and
// 2^-35 to what is below; what is above 63 has none, but X's values stay near 1 and the
// polynomial's near 5.  (The second float times 2^11, with a sum of its own, would hold
// 22 bits to 2^-24, for twice the sums' registers: tiles of 128 had one workgroup less, and the
// error against 64 bits was the same, 5e-8 of the whole and 6e-8.)
// All products are of rows with rows, the summed index contiguous, since A and B are their
// own transposes and X is kept both ways; of A and B the half above the diagonal is computed
// and written twice.  Each step is one launch for all matrices together.
//
// Measured: four layers of 6144 x 2048 and 2048 x 2048 and a matrix of 49 x 2048 in 32 bits 9.3 ms
// a step, of which the products' 2.4 TFLOP, threefold, would take 6.5 at the library's rate:
// X's step runs at 930 TFLOP/s (3 x 275 GFLOP in 883 us), X X^T at 800, the polynomial at 710;
// the last step, which moves the parameters, takes 1088 us, the momentum 132 (6.1 TB/s) and X's
// making 248 (4.4 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cpab_launch.hpp"
#include "sequence_device.hpp"
#include "sequence_launch.hpp"

namespace cpab {
namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kLanes = 256;
constexpr int kWholeSide = 64, kWholeLong = 256;   // of the matrices that one workgroup keeps
constexpr int kWholeLanes = 1024;
constexpr int kMatrices = 40;      // of a launch
constexpr int kSpan = kLanes * 16; // values of a workgroup of the momentum's kernel
constexpr float kUp = 1024.0f, kDown = 1.0f / 1024.0f;

// A matrix and where its parts lie in the workspace (bytes).  X is [m, n], m <= n, of
// padded sizes; planes of 16-bit floats: hi, then lo.
struct Matrix {
  void* param;
  const void* grad;
  float* momentum;
  float* master;
  int64_t at;
  int rows, cols;
  float rate;
};
struct Batch {
  Matrix m[kMatrices];
  uint32_t first[kMatrices + 1];   // workgroups before each matrix's
};

// How a matrix' products go: in one workgroup that keeps it in LDS where it fits (0: 16
// matrices of 64 x 64 take 21 us a step and 93 in tiles, of 256 x 64 38 and 113), else in
// tiles of up to 64, 128 or 256, to which the matrix is padded: the longer its shorter side,
// the less that costs.
__host__ __device__ __forceinline__ int tile_of(int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
  return m <= kWholeSide && n <= kWholeLong ? 0 : m > 1024 ? 256 : m > 256 ? 128 : 64;
}
__host__ __device__ constexpr int lanes_of(int tile) { return tile > 128 ? 512 : 256; }
__host__ __device__ __forceinline__ int64_t padded(int64_t n, int tile) { return (n + tile - 1) / tile * tile; }
struct Places {
  int64_t m, n;   // padded
  int64_t sums, x0, x1, xt0, xt1, a, b, end;   // x: [m, n]; xt: [n, m]
  __host__ __device__ int64_t x(int k) const { return k ? x1 : x0; }
  __host__ __device__ int64_t xt(int k) const { return k ? xt1 : xt0; }
};
__host__ __device__ __forceinline__ Places places(int64_t rows, int64_t cols) {
  Places p;
  const int tile = tile_of(rows, cols);
  p.m = padded(rows < cols ? rows : cols, tile);
  p.n = padded(rows < cols ? cols : rows, tile);
  const int64_t spans = (rows * cols + kSpan - 1) / kSpan;
  p.sums = 0;
  p.x0 = (spans * 8 + 255) / 256 * 256;
  const int64_t whole = 4 * p.m * p.n, square = 4 * p.m * p.m;
  p.x1 = p.x0 + whole;
  p.xt0 = p.x1 + whole;
  p.xt1 = p.xt0 + whole;
  p.a = p.xt1 + whole;
  p.b = p.a + square;
  p.end = p.b + square;
  return p;
}

__device__ __forceinline__ int find(const Batch& batch, int count) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (batch.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

struct Momentum {
  float mu, rest, eps;
  bool nesterov;
};
__device__ __forceinline__ float update(const Momentum& s, float m, float g) {
  return s.nesterov ? fmaf(s.mu, m, s.rest * g) : m;
}

// The momentum, and each span's sum of the update's squares (in 64 bits: squares of small
// gradients leave the 32-bit range).
template <typename T>
__global__ __launch_bounds__(kLanes) void muon_momentum_kernel(Batch batch, int count, Momentum s, char* room) {
  __shared__ double parts[kLanes / 64];
  const int which = find(batch, count);
  const Matrix& t = batch.m[which];
  const int64_t n = (int64_t)t.rows * t.cols, span = blockIdx.x - batch.first[which];
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t at = span * kSpan + 4 * (k * kLanes + (int64_t)threadIdx.x);
    const int here = (int)min(n - at, (int64_t)4);
    if (here <= 0) continue;
    float m[4] = {}, g[4] = {};
    const T* gp = static_cast<const T*>(t.grad) + at;
    float* mp = t.momentum + at;
    if (here == 4) {
      load<4>(gp, g);
      load<4>(mp, m);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < here) g[e] = to_float(gp[e]), m[e] = mp[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = fmaf(s.mu, m[e], s.rest * g[e]);
      const double u = e < here ? (double)update(s, m[e], g[e]) : 0.0;
      sum = fma(u, u, sum);
    }
    if (here == 4) {
      store<4>(mp, m);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < here) mp[e] = m[e];
    }
  }
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0)
    reinterpret_cast<double*>(room + t.at)[span] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
}

// Where a matrix of so many (padded) rows has a value: 32 columns of all rows after another,
// so that a tile's 32 of the summed index are one piece of memory.
__host__ __device__ __forceinline__ int64_t place(int64_t row, int64_t col, int64_t rows) {
  return (col / 32 * rows + row) * 32 + col % 32;
}

// 2^10 times a value in two 16-bit floats.
struct Two {
  f16 hi, lo;
};
__device__ __forceinline__ Two two_of(float x) {
  const float v = x * kUp;
  const f16 hi = (f16)v;
  return Two{hi, (f16)(v - (float)hi)};
}

// X and its transpose from the update, 64 x 64 values to a workgroup; zeros in the padding.
template <typename T>
__global__ __launch_bounds__(kLanes) void muon_start_kernel(Batch batch, int count, Momentum s, char* room) {
  __shared__ f16 turn[2][64][66];
  __shared__ double parts[kLanes / 64];
  const int which = find(batch, count);
  const Matrix& t = batch.m[which];
  const Places p = places(t.rows, t.cols);
  const double* sums = reinterpret_cast<const double*>(room + t.at);
  const int64_t spans = ((int64_t)t.rows * t.cols + kSpan - 1) / kSpan;
  double sum = 0.0;
  for (int64_t k = threadIdx.x; k < spans; k += kLanes) sum += sums[k];
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double norm = sqrt((parts[0] + parts[1]) + (parts[2] + parts[3]));
  const float by = (float)(1.0 / (norm < (double)s.eps ? (double)s.eps : norm));
  // the parameter's own layout, [rows, cols], is X's or its transpose's
  const bool wide = t.rows <= t.cols;
  const int64_t prows = wide ? p.m : p.n, pcols = wide ? p.n : p.m;
  f16* own = reinterpret_cast<f16*>(room + t.at + (wide ? p.x0 : p.xt0));
  f16* other = reinterpret_cast<f16*>(room + t.at + (wide ? p.xt0 : p.x0));
  const int64_t plane = p.m * p.n;
  const int64_t tile = blockIdx.x - batch.first[which], across = pcols / 64;
  const int64_t r0 = tile / across * 64, c0 = tile % across * 64;
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int r = k * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63;
    const int64_t row = r0 + r, col = c0 + c;
    float x = 0.0f;
    if (row < t.rows && col < t.cols) {
      const int64_t at = row * t.cols + col;
      x = update(s, t.momentum[at], to_float(static_cast<const T*>(t.grad)[at])) * by;
    }
    const Two v = two_of(x);
    const int64_t to = place(row, col, prows);
    own[to] = v.hi;
    own[plane + to] = v.lo;
    turn[0][c][r] = v.hi;
    turn[1][c][r] = v.lo;
  }
  __syncthreads();
#pragma unroll 4
  for (int k = 0; k < 16; ++k) {
    const int c = k * 4 + (threadIdx.x >> 6), r = threadIdx.x & 63;
    const int64_t to = place(c0 + c, r0 + r, pcols);
    other[to] = turn[0][c][r];
    other[plane + to] = turn[1][c][r];
  }
}

struct Coefficients {
  float c0, c1, c2, decay;
  int from;   // which of the two X
};

template <typename T>
__device__ __forceinline__ void put(const Matrix& t, int64_t at, float w) {
  static_cast<T*>(t.param)[at] = from_float<T>(w);
  if (t.master) t.master[at] = w;
}
// The parameter's move, from the master weight where there is one.
template <typename T>
__device__ __forceinline__ void move(const Matrix& t, int64_t at, float decay, float v) {
  put<T>(t, at, (t.master ? t.master[at] : to_float(static_cast<const T*>(t.param)[at])) * decay - t.rate * v);
}

// As a sum of three products of two 16-bit floats each.
__device__ __forceinline__ f32x4 mma(const f16x8 (&l)[2], const f16x8 (&r)[2], f32x4 acc) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0], r[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0], r[1], acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(l[1], r[0], acc, 0, 0, 0);
}

// The whole step of a matrix of up to 64 x 256: X, its transpose and A, later B, lie in LDS;
// a wave has 16 of X's columns in its registers, in 32 bits, and one 16 x 16 tile of A and B.
// One launch instead of two and three to an iteration, which is what small matrices wait for:
// 17 matrices of 192 x 64, 64 x 64 and 49 x 64 take 31 us, in tiles 103.  What is left is 10 us
// around the iterations and 4.2 for each of them at 192 x 64, 2.5 at 64 x 64: a compute unit alone
// writes X twice to LDS and reads it for A, and four barriers stand between.
template <typename T>
__global__ __launch_bounds__(kWholeLanes) void muon_whole_kernel(Batch batch, Momentum s, Coefficients c, int steps) {
  constexpr int kP = kWholeSide + 8;   // pitch of A and of X's transpose
  extern __shared__ __align__(16) f16 lds[];
  __shared__ double parts[kWholeLanes / 64];
  const Matrix& t = batch.m[blockIdx.x];
  const bool wide = t.rows <= t.cols;
  const int m = wide ? t.rows : t.cols, n = wide ? t.cols : t.rows, across = (n + 31) / 32 * 32, pitch = across + 8;
  f16* const x = lds;                                   // [2][64][pitch]
  f16* const xt = x + 2 * kWholeSide * pitch;           // [2][across][kP]
  f16* const a = xt + 2 * across * kP;                  // [2][64][kP]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4, col = 16 * wave + i;
  const bool busy = 16 * wave < across;
  // Memory's values in its own order, through LDS in X's: of a matrix whose longer side comes
  // first a lane's values else lie 16 rows apart (45 us for 33).
  constexpr int kEach = kWholeSide * kWholeLong / kWholeLanes, kTurn = kWholeSide + 1;
  float* const stage = reinterpret_cast<float*>(lds);   // [n][kTurn]
  const int all = m * n, short_side = wide ? n : m;     // a row of the parameter
  struct Turned {   // of this lane's values, one after another
    int r, c, down, right, across;
    bool wide;
    __device__ int next() {
      const int at = wide ? c * kTurn + r : r * kTurn + c;
      r += down, c += right;
      if (c >= across) c -= across, ++r;
      return at;
    }
  };
  const auto turned = [&](int tid) {
    const int r = tid / short_side;
    return Turned{r, tid - r * short_side, kWholeLanes / short_side, kWholeLanes % short_side, short_side, wide};
  };
  double sum = 0.0;
  {
    float grad[kEach], mom[kEach];
    Turned to = turned(threadIdx.x);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = min(k * kWholeLanes + (int)threadIdx.x, all - 1);
      grad[k] = to_float(static_cast<const T*>(t.grad)[at]);
      mom[k] = t.momentum[at];
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = k * kWholeLanes + (int)threadIdx.x;
      if (at < all) {
        mom[k] = fmaf(s.mu, mom[k], s.rest * grad[k]);
        t.momentum[at] = mom[k];
        const float u = update(s, mom[k], grad[k]);
        sum = fma((double)u, (double)u, sum);
        stage[to.next()] = u;
      }
    }
  }
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) parts[wave] = sum;
  __syncthreads();
  sum = 0.0;
  for (int k = 0; k < kWholeLanes / 64; ++k) sum += parts[k];
  const double norm = sqrt(sum);
  const float by = (float)(1.0 / (norm < (double)s.eps ? (double)s.eps : norm));
  f32x4 own[4];   // rows 16 k + 4 g .. of column col
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * k + 4 * g + e;
      own[k][e] = row < m && col < n ? stage[col * kTurn + row] * by : 0.0f;
    }
  __syncthreads();
  const auto frag = [&](f16x8 (&to)[2], const f16* from, int plane) {
    to[0] = *reinterpret_cast<const f16x8*>(from);
    to[1] = *reinterpret_cast<const f16x8*>(from + plane);
  };
  const int tr = 16 * (wave >> 2), tc = 16 * (wave & 3);   // this wave's tile of A
  const auto keep = [&](const f32x4& v) {                  // A is its own transpose
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Two w = two_of(v[e]);
      hi[e] = w.hi, lo[e] = w.lo;
    }
    f16* const to = a + (tc + i) * kP + tr + 4 * g;
    *reinterpret_cast<f16x4*>(to) = hi;
    *reinterpret_cast<f16x4*>(to + kWholeSide * kP) = lo;
  };
  for (int step = 0;; ++step) {
    if (busy) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Two w = two_of(own[k][e]);
          hi[e] = w.hi, lo[e] = w.lo;
          x[(16 * k + 4 * g + e) * pitch + col] = w.hi;
          x[(kWholeSide + 16 * k + 4 * g + e) * pitch + col] = w.lo;
        }
        *reinterpret_cast<f16x4*>(xt + col * kP + 16 * k + 4 * g) = hi;
        *reinterpret_cast<f16x4*>(xt + (across + col) * kP + 16 * k + 4 * g) = lo;
      }
    }
    __syncthreads();
    f16x8 l[2], r[2];
    f32x4 gram = {};
#pragma unroll 1
    for (int k = 0; k < across; k += 32) {
      frag(l, x + (tr + i) * pitch + k + 8 * g, kWholeSide * pitch);
      frag(r, x + (tc + i) * pitch + k + 8 * g, kWholeSide * pitch);
      gram = mma(l, r, gram);
    }
    gram *= kDown * kDown;
    keep(gram);
    __syncthreads();
    f32x4 poly = {};
#pragma unroll
    for (int k = 0; k < kWholeSide; k += 32) {
      frag(l, a + (tr + i) * kP + k + 8 * g, kWholeSide * kP);
      frag(r, a + (tc + i) * kP + k + 8 * g, kWholeSide * kP);
      poly = mma(l, r, poly);
    }
    __syncthreads();
    keep(gram * c.c1 + poly * (c.c2 * kDown * kDown));
    __syncthreads();
    if (busy) {
#pragma unroll
      for (int k = 0; k < 4; ++k) own[k] *= c.c0 * (kUp * kUp);
#pragma unroll
      for (int k = 0; k < kWholeSide; k += 32) {
        frag(r, xt + col * kP + k + 8 * g, across * kP);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          frag(l, a + (16 * u + i) * kP + k + 8 * g, kWholeSide * kP);
          own[u] = mma(l, r, own[u]);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) own[k] *= kDown * kDown;
    }
    if (step + 1 == steps) break;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = 16 * k + 4 * g + e;
      if (row < m && col < n) stage[col * kTurn + row] = own[k][e];
    }
  __syncthreads();
  int tid = threadIdx.x;   // the places again, which else keep their registers all along
  asm volatile("" : "+v"(tid));
  float w[kEach];
  Turned from = turned(tid);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = min(k * kWholeLanes + tid, all - 1);
    w[k] = (t.master ? t.master[at] : to_float(static_cast<const T*>(t.param)[at]));
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = k * kWholeLanes + tid;
    if (at < all) put<T>(t, at, w[k] * c.decay - t.rate * stage[from.next()]);
  }
}

enum Product { kGram, kPolynomial, kStep, kLast };

// One tile of a product: a wave has a quarter of it, of a tile of 256 an eighth.  32 of the
// summed index lie in LDS twice, as the matrix unit has the one and memory brings the other;
// rows of 64 bytes begin 20 banks apart, so that a wave's wide reads meet no bank twice.  LDS
// brings a wave of 128 x 64 what it multiplies in half the matrix unit's time, one of 64 x 64
// in two thirds.  (Rows of K values apart instead of pieces of 32: X's step 1068 us for 886.)
template <Product WHAT, typename T, int TILE>
__global__ __launch_bounds__((lanes_of(TILE)), 2) void muon_product_kernel(Batch batch, int count, Coefficients c, char* room) {
  constexpr int kStepK = 32, kPitch = kStepK + 8, kThreads = lanes_of(TILE), kRows = kThreads / 4;
  constexpr int kEach = TILE / kRows, kAcross = kThreads / 128, MT = TILE / 64, NT = TILE / 32 / kAcross;
  extern __shared__ __align__(16) f16 lds[];   // [2][4][TILE][kPitch]: rows' hi and lo, columns' hi and lo
  const int which = find(batch, count);
  const Matrix& t = batch.m[which];
  const Places p = places(t.rows, t.cols);
  char* const base = room + t.at;
  // workgroups go to the eight dies in turn, each with a cache of its own: a die's tiles of a
  // matrix follow one another
  const uint32_t turn = blockIdx.x - batch.first[which], all = batch.first[which + 1] - batch.first[which];
  const int64_t tile = turn % 8 * (all / 8) + min(turn % 8, all % 8) + turn / 8;
  int64_t ti, tj;
  if (WHAT == kGram || WHAT == kPolynomial) {   // tj >= ti
    tj = (int64_t)((sqrt(8.0 * (double)tile + 1.0) - 1.0) * 0.5);
    while (tj * (tj + 1) / 2 > tile) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= tile) ++tj;
    ti = tile - tj * (tj + 1) / 2;
  } else {
    const int64_t down = p.m / TILE;
    ti = tile % down;
    tj = tile / down;
  }
  const f16* x = reinterpret_cast<const f16*>(base + p.x(c.from));
  const f16* xt = reinterpret_cast<const f16*>(base + p.xt(c.from));
  f16* a = reinterpret_cast<f16*>(base + p.a);
  f16* b = reinterpret_cast<f16*>(base + p.b);
  const int64_t whole = p.m * p.n, square = p.m * p.m;
  const int64_t K = WHAT == kGram ? p.n : p.m;
  const f16* left = WHAT == kGram ? x : WHAT == kPolynomial ? a : b;
  const f16* right = WHAT == kGram ? x : WHAT == kPolynomial ? a : xt;
  const int64_t left_plane = WHAT == kGram ? whole : square;
  const int64_t right_plane = WHAT == kPolynomial ? square : whole;
  const int64_t left_step = p.m * 32, right_step = WHAT == kStep || WHAT == kLast ? p.n * 32 : p.m * 32;
  left += ti * TILE * 32 + threadIdx.x * 8;
  right += tj * TILE * 32 + threadIdx.x * 8;
  // a lane brings 16 bytes of some rows of each of the four arrays
  const int row = threadIdx.x >> 2, part = (threadIdx.x & 3) * 8;
  u32x4 next[4][kEach];
  const auto fetch = [&] {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      next[0][e] = *reinterpret_cast<const u32x4*>(left + kRows * e * 32);
      next[1][e] = *reinterpret_cast<const u32x4*>(left + left_plane + kRows * e * 32);
      next[2][e] = *reinterpret_cast<const u32x4*>(right + kRows * e * 32);
      next[3][e] = *reinterpret_cast<const u32x4*>(right + right_plane + kRows * e * 32);
    }
    left += left_step;
    right += right_step;
  };
  fetch();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 31, g = lane >> 5;
  const int wr = wave / kAcross * (TILE / 2), wc = wave % kAcross * (32 * NT);
  f32x16 acc[MT][NT] = {};
  int buffer = 0;
  for (int64_t k0 = 0; k0 < K; k0 += kStepK, buffer ^= 1) {
    f16* const now = lds + buffer * 4 * TILE * kPitch;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        *reinterpret_cast<u32x4*>(now + (k * TILE + row + kRows * e) * kPitch + part) = next[k][e];
    __syncthreads();
    if (k0 + kStepK < K) fetch();
#pragma unroll
    for (int k = 0; k < kStepK; k += 16) {
      f16x8 l[2][MT], r[2][NT];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
          l[h][m] = *reinterpret_cast<const f16x8*>(now + (h * TILE + wr + 32 * m + i) * kPitch + k + 8 * g);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          r[h][n] = *reinterpret_cast<const f16x8*>(now + ((2 + h) * TILE + wc + 32 * n + i) * kPitch + k + 8 * g);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0][m], r[0][n], acc[m][n], 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0][m], r[1][n], acc[m][n], 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[1][m], r[0][n], acc[m][n], 0, 0, 0);
    }
  }
  // a lane's column, and 16 rows of each 32: four at a time, 8 apart
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t col = tj * TILE + wc + 32 * n + i, r0 = ti * TILE + wr + 32 * m + 8 * q + 4 * g;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = acc[m][n][4 * q + e] * (kDown * kDown);
        if (WHAT == kPolynomial) {   // A is its own transpose
          const f16x4 hi = *reinterpret_cast<const f16x4*>(a + place(col, r0, p.m));
          const f16x4 lo = *reinterpret_cast<const f16x4*>(a + square + place(col, r0, p.m));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = fmaf(c.c2, v[e], c.c1 * (((float)hi[e] + (float)lo[e]) * kDown));
        }
        if (WHAT == kStep || WHAT == kLast) {
          const f16x4 hi = *reinterpret_cast<const f16x4*>(xt + place(col, r0, p.n));
          const f16x4 lo = *reinterpret_cast<const f16x4*>(xt + whole + place(col, r0, p.n));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(c.c0, ((float)hi[e] + (float)lo[e]) * kDown, v[e]);
        }
        if (WHAT == kLast) {
          const bool wide = t.rows <= t.cols;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int64_t pr = wide ? r0 + e : col, pc = wide ? col : r0 + e;
            if (pr < t.rows && pc < t.cols) move<T>(t, pr * t.cols + pc, c.decay, v[e]);
          }
          continue;
        }
        f16* out = WHAT == kGram ? a : WHAT == kPolynomial ? b : reinterpret_cast<f16*>(base + p.x(c.from ^ 1));
        f16* turned = WHAT == kStep ? reinterpret_cast<f16*>(base + p.xt(c.from ^ 1)) : out;
        const int64_t plane = WHAT == kStep ? whole : square, across = WHAT == kStep ? p.n : p.m;
        const int64_t to = place(r0, col, p.m), over = place(col, r0, across);
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Two w = two_of(v[e]);
          hi[e] = w.hi, lo[e] = w.lo;
          out[to + 32 * e] = w.hi;
          out[plane + to + 32 * e] = w.lo;
        }
        if (WHAT == kStep || ti != tj) {
          *reinterpret_cast<f16x4*>(turned + over) = hi;
          *reinterpret_cast<f16x4*>(turned + plane + over) = lo;
        }
      }
}

// The matrices from k on, of those with this tile, that one launch takes, and their workspace.
int64_t gather(int64_t n, const cpab_muon_matrix* matrices, const double* rates, int tile, int64_t* k,
               Batch* batch, int* count) {
  int64_t bytes = 0;
  *count = 0;
  for (; *k < n && *count < kMatrices; ++*k) {
    const cpab_muon_matrix& t = matrices[*k];
    if (t.rows == 0 || t.cols == 0 || tile_of(t.rows, t.cols) != tile) continue;
    const int64_t need = tile == 0 ? 0 : (places(t.rows, t.cols).end + 255) / 256 * 256;
    if (*count > 0 && bytes + need > (1LL << 32)) break;   // a few GB of workspace are enough
    if (batch)
      batch->m[*count] = Matrix{t.param, t.grad, t.momentum, t.master, bytes, (int)t.rows, (int)t.cols,
                                (float)rates[*k]};
    ++*count;
    bytes += need;
  }
  // the longest products first, so that none begins when the others end
  if (batch)
    std::sort(batch->m, batch->m + *count, [](const Matrix& a, const Matrix& b) {
      return std::make_pair(std::max(a.rows, a.cols), a.at) > std::make_pair(std::max(b.rows, b.cols), b.at);
    });
  return bytes;
}

}  // namespace

int64_t muon_workspace(int64_t n, const cpab_muon_matrix* matrices) {
  int64_t most = 0;
  for (const int tile : {0, 64, 128, 256})
    for (int64_t k = 0; k < n;) {
      int count = 0;
      most = std::max(most, gather(n, matrices, nullptr, tile, &k, nullptr, &count));
    }
  return most;
}

namespace {

// The time of a product in so many tiles of a side, in units of what a tile of 128 takes with a
// compute unit's other one beside it.  A unit has four of 64, two of 128 or one of 256 at a
// time; one alone waits for memory at each step (128: 1.4), and the larger tile reads less for
// what it computes.  Measured, us a step all in 64, 128 or 256, and as chosen: 16 of 257 x 257
// 250, 340, -, 249; 8 of 512 x 512 269, 385, -, 267; 40 of them 926, 898, -, 896; 8 of 768 x 768
// 542, 578, -, 543; 8 of 1024 x 1024 1036, 1001, -, 1000; 8 of 1025 x 1025 1689, 1478, 1855, 1414;
// 8 of 3840 x 1280 4614, 3712, 4340, 3726; 2 of 6144 x 2048 4596, 3710, 5126, 3706; 8 of them
// 17463, 13785, 13979, 12832.
// Four layers of 6144 x 2048 and 2048 x 2048, X's step alone: 967 in 128 and 887 in 256, the
// polynomial 302 and 372, where 256 leaves most units without a tile in the second round.
double cost_of(int side, double tiles) {
  const int64_t each = (int64_t)std::ceil(tiles / compute_units());   // of a unit
  const double some[4] = {0.0, 0.7, 0.9, 1.15};
  return side == 64    ? (double)(each / 4) * 1.33 + some[each % 4]
         : side == 128 ? (double)(each / 2) * 2.0 + (double)(each % 2) * 1.4
                       : (double)each * 3.3;
}

// The step of one batch, of matrices padded to tiles of TILE.
template <typename T, int TILE>
hipError_t step(Batch& batch, int count, const Muon& s, char* room, hipStream_t st) {
  const auto tiles = [&](auto each) {   // of all matrices
    uint32_t total = 0;
    for (int i = 0; i < count; ++i) {
      batch.first[i] = total;
      total += (uint32_t)each(batch.m[i], places(batch.m[i].rows, batch.m[i].cols));
    }
    batch.first[count] = total;
    return total;
  };
  const auto product = [&](auto what, auto side, uint32_t blocks, const Coefficients& c) {
    constexpr Product WHAT = decltype(what)::value;
    constexpr int SIDE = decltype(side)::value, kRoom = 2 * 4 * SIDE * 40 * 2;
    static LdsAllowed allowed;
    const hipError_t e = allow_lds(reinterpret_cast<const void*>(muon_product_kernel<WHAT, T, SIDE>), kRoom, allowed);
    if (e != hipSuccess) return e;
    muon_product_kernel<WHAT, T, SIDE><<<blocks, lanes_of(SIDE), kRoom, st>>>(batch, count, c, room);
    return hipGetLastError();
  };
  // A product in the tiles that should take the least time for all matrices together.
  const auto best = [&](auto what, const Coefficients& c) {
    constexpr Product WHAT = decltype(what)::value;
    const auto each = [](int side, const Places& p) {
      const int64_t down = p.m / side;   // of a symmetric one the tiles on and above the diagonal
      return WHAT == kGram || WHAT == kPolynomial ? down * (down + 1) / 2 : down * (p.n / side);
    };
    const auto cost = [&](int side) {
      if (side > TILE) return HUGE_VAL;
      double sum = 0.0, longest = 1.0;   // tiles of the longest summed index
      for (int i = 0; i < count; ++i) {
        const Places p = places(batch.m[i].rows, batch.m[i].cols);
        const double k = (double)(WHAT == kGram ? p.n : p.m);
        sum += k * (double)each(side, p);
        longest = std::max(longest, k);
      }
      return cost_of(side, sum / longest);
    };
    const double by64 = cost(64), by128 = cost(128), by256 = cost(256);
    const auto go = [&](auto side) {
      constexpr int SIDE = decltype(side)::value;
      return product(what, side, tiles([&](const Matrix&, const Places& p) { return each(SIDE, p); }), c);
    };
    if constexpr (TILE >= 256)
      if (by256 <= by128 && by256 <= by64) return go(std::integral_constant<int, 256>());
    if constexpr (TILE >= 128)
      if (by128 <= by64) return go(std::integral_constant<int, 128>());
    return go(std::integral_constant<int, 64>());
  };
  const Momentum m{s.momentum, s.rest, s.eps, s.nesterov};
  uint32_t blocks = tiles([](const Matrix& a, const Places&) { return ((int64_t)a.rows * a.cols + kSpan - 1) / kSpan; });
  muon_momentum_kernel<T><<<blocks, kLanes, 0, st>>>(batch, count, m, room);
  blocks = tiles([](const Matrix&, const Places& p) { return p.m / 64 * (p.n / 64); });
  muon_start_kernel<T><<<blocks, kLanes, 0, st>>>(batch, count, m, room);
  hipError_t e = hipGetLastError();
  for (int i = 0; i < s.steps && e == hipSuccess; ++i) {
    const Coefficients c{s.c0, s.c1, s.c2, s.decay, i & 1};
    e = best(std::integral_constant<Product, kGram>(), c);
    if (e == hipSuccess) e = best(std::integral_constant<Product, kPolynomial>(), c);
    if (e != hipSuccess) break;
    e = i + 1 < s.steps ? best(std::integral_constant<Product, kStep>(), c)
                        : best(std::integral_constant<Product, kLast>(), c);
  }
  return e;
}

// The step of the matrices of one batch that are kept whole.
template <typename T>
hipError_t step_whole(const Batch& batch, int count, const Muon& s, hipStream_t st) {
  int room = 0;
  for (int i = 0; i < count; ++i) {
    const int across = (std::max(batch.m[i].rows, batch.m[i].cols) + 31) / 32 * 32;
    room = std::max(room, 2 * 2 * (kWholeSide * (across + 8) + (across + kWholeSide) * (kWholeSide + 8)));
  }
  static LdsAllowed allowed;
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(muon_whole_kernel<T>), room, allowed);
  if (e != hipSuccess) return e;
  const Momentum m{s.momentum, s.rest, s.eps, s.nesterov};
  muon_whole_kernel<T><<<count, kWholeLanes, room, st>>>(batch, m, Coefficients{s.c0, s.c1, s.c2, s.decay, 0}, s.steps);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_muon(int dtype, int64_t n, const cpab_muon_matrix* matrices, const double* rates,
                       const Muon& s, void* workspace, hipStream_t st) {
  char* room = static_cast<char*>(workspace);
  for (const int tile : {0, 64, 128, 256})
    for (int64_t k = 0; k < n;) {
      Batch batch;
      int count = 0;
      gather(n, matrices, rates, tile, &k, &batch, &count);
      if (count == 0) break;
      const auto typed = [&](auto t) {
        typedef decltype(t) T;
        return tile == 0    ? step_whole<T>(batch, count, s, st)
               : tile == 64 ? step<T, 64>(batch, count, s, room, st)
               : tile == 128 ? step<T, 128>(batch, count, s, room, st)
                             : step<T, 256>(batch, count, s, room, st);
      };
      const hipError_t e = dtype == CPAB_F32 ? typed(0.0f) : typed(bf16());
      if (e != hipSuccess) return e;
    }
  return hipSuccess;
}

}  // namespace cpab
