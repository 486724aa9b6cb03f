// The Muon step over many matrices (include/cp4/muon.h): its C ABI, matrices with a short side of up to 64, and what
// stands before the products of larger ones (muon_tiles.hip).
//
// A short side of m <= 64 (adapters, CP factors): every X of the iteration is a polynomial in the m x m matrix
// G = u u^T times u, so u itself is read twice and nothing else of its size moves.
//
//   gram      updates the momentum, adds up G over the long side - fp64 on the matrix cores: G squares u's singular
//             values, and a small one would drown in fp32's roundings of the largest -, split over workgroups;
//   iterate   one workgroup a matrix: adds up the splits, |u|^2 is G's trace, then A <- A p(A)^2 and Q <- Q p(A) in
//             fp64 in the LDS (up to 16: in registers), all of them symmetric, blocks on and below the diagonal alone;
//   apply     X = Q u and the parameters' step, in fp32 up to 5 steps, in fp64 beyond (wide()).
//
// So the step is bound by memory where matrices are long (12 bytes a value in gram, 16 in apply) and by the
// latency of three launches where they are short: 28 adapters' factors of 7 x 1001 and 777 x 7 7 + 7 + 9 us.  The entries of a
// launch are a table in the kernel's arguments.
#include <algorithm>
#include <cmath>
#include <exception>
#include <vector>

#include "muon.h"

namespace cp4 {
namespace muon {
namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr int kSmall = 72, kLarge = 16;            // entries of a launch
static_assert(kLarge <= kProducts, "a launch of products holds a group");
constexpr unsigned kSide = 64;                     // the longest short side that goes through its Gram matrix
// Whether Q and its products with u are fp64.  Q is 3.4445 to the steps in directions that u lacks, and of as much are its roundings,
// which X sees: in fp32 3e-5 of it in 5 steps (as an iteration of X in fp32 has, 4e-5), 1e-3 in 8, 0.1 in 12, 50 in 16.  fp64
// takes 131 us for 32 matrices of 64 x 4096, fp32 112; 77 and 71 of 48 x 4096; 51 and 50 for 28 adapters' 7 x 1001 and 777 x 7.
__host__ __device__ constexpr bool wide(int steps) { return steps > 5; }

// ---- a short side of up to 64 ------------------------------------------------------------

struct SmallItem {
  const void* grad;
  float* momentum;
  void *param, *copy;
  unsigned short last_row, last_col;
  unsigned char splits, param_dtype, grad_dtype, copy_dtype;       // splits: of a matrix, workgroups of gram
  __device__ unsigned rows() const { return last_row + 1u; }
  __device__ unsigned cols() const { return last_col + 1u; }
};
struct SmallArgs {
  SmallItem item[kSmall];
  unsigned gram[kSmall], iterate[kSmall], apply[kSmall];           // an entry's first workgroup of each launch; ~0: no entry
  int nesterov, steps;
  float mu, decay;
  double eps, lr;
  double* part;                                    // [gram's workgroups][blocks][16][16]
  void* q;                                         // [iterate's workgroups][M][M], fp64 where `steps` is wide(), or fp32
};
static_assert(sizeof(SmallArgs) <= 4096, "kernel arguments");

// MB: the short side in blocks of 16.  A tile is JT of the long side's places, in the LDS as u[short][long].
template <int MB>
struct Tile {
  static constexpr int M = 16 * MB, JT = MB == 1 ? 256 : MB == 2 ? 128 : 64, S = JT + 4;
  static constexpr int kBlocks = MB * (MB + 1) / 2;                // 16 x 16, on and below the diagonal
};
// Four consecutive values of u, and where they update the momentum its new values.
template <bool Update>
__device__ __forceinline__ void direction(const void* grad, int dtype, float* momentum, size_t at, int count, float mu,
                                          bool nesterov, float (&u)[4]) {
  load_values<4>(grad, dtype, at, count, u);
  if (!momentum) return;
  float m[4];
  load_values<4>(momentum, CP4_DTYPE_F32, at, count, m);
  if constexpr (Update) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = m[j] * mu + u[j];
    store_values<4>(momentum, CP4_DTYPE_F32, at, count, m);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = nesterov ? u[j] + mu * m[j] : m[j];
}
// fn(at, count, i, j) for the tile's values, four consecutive ones of memory a turn, at from the matrix's first value
// on: flat (rows <= cols) the values (i, j .. j + 3), tall the four from (i, j) on along i, then j.
template <int MB, class Fn>
__device__ __forceinline__ void for_tile(const SmallItem& it, int j0, Fn fn) {
  constexpr int JT = Tile<MB>::JT;
  const int m = min(it.rows(), it.cols()), n = max(it.rows(), it.cols());
  if (it.rows() <= it.cols()) {
    for (int e = threadIdx.x * 4; e < m * JT; e += 1024) {
      const int i = e / JT, j = e % JT;
      if (j0 + j < n) fn((size_t)i * n + j0 + j, n - j0 - j, i, j);
    }
  } else {
    const int total = min(JT, n - j0) * m;
    for (int e = threadIdx.x * 4; e < total; e += 1024) fn((size_t)j0 * m + e, total - e, e % m, e / m);
  }
}
template <int MB, bool Update>
__device__ __forceinline__ void load_tile(const SmallArgs& a, const SmallItem& it, size_t base, int j0, float* u) {
  constexpr int JT = Tile<MB>::JT, S = Tile<MB>::S;
  const int m = min(it.rows(), it.cols()), n = max(it.rows(), it.cols());
  const bool flat = it.rows() <= it.cols();
  if (j0 + JT > n)                                                 // (the last tile: what it lacks is zero)
    for (int e = threadIdx.x; e < m * JT; e += 256)
      if (j0 + e % JT >= n) u[e / JT * S + e % JT] = 0.0f;
  for_tile<MB>(it, j0, [&](size_t at, int count, int i, int j) __attribute__((always_inline)) {
    float x[4];
    direction<Update>(it.grad, it.grad_dtype, it.momentum, base + at, count, a.mu, a.nesterov, x);
    if (flat) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (q < count) u[i * S + j + q] = x[q];
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (q < count) u[i * S + j] = x[q];
        if (++i == m) {
          i = 0;
          ++j;
        }
      }
    }
  });
}

template <int MB>
__global__ __launch_bounds__(256) void gram_kernel(const SmallArgs a) {
  typedef Tile<MB> T;
  __shared__ __attribute__((aligned(16))) float u[T::M * T::S];
  __shared__ double sum[T::kBlocks * 256];
  const int entry = entry_of(a.gram, blockIdx.x);
  const SmallItem& it = a.item[entry];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const unsigned splits = it.splits, matrix = (blockIdx.x - a.gram[entry]) / splits, split = (blockIdx.x - a.gram[entry]) % splits;
  const int m = min(it.rows(), it.cols()), tiles = (max(it.rows(), it.cols()) + T::JT - 1) / T::JT;
  const size_t base = (size_t)matrix * it.rows() * it.cols();
  for (int e = m * T::S + threadIdx.x; e < T::M * T::S; e += 256) u[e] = 0.0f;
  const int first = tiles * split / splits, last = tiles * (split + 1) / splits;
  f64x4 acc[T::kBlocks] = {};
  for (int t = first; t < last; ++t) {
    __syncthreads();
    load_tile<MB, true>(a, it, base, t * T::JT, u);
    __syncthreads();
#pragma unroll 2
    for (int s = 0; s < T::JT / 16; ++s) {                         // (four places of the long side a step, each wave its quarter)
      const float* const p = u + l * T::S + wave * (T::JT / 4) + 4 * s + g;
      double x[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) x[b] = p[16 * b * T::S];
#pragma unroll
      for (int i = 0, k = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j, ++k) acc[k] = __builtin_amdgcn_mfma_f64_16x16x4f64(x[i], x[j], acc[k], 0, 0, 0);
    }
  }
  for (int w = 0; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int k = 0; k < T::kBlocks; ++k)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          double* const p = sum + k * 256 + (g + 4 * v) * 16 + l;  // (fp64: row lane / 16 + 4 v, column lane % 16)
          *p = w ? *p + acc[k][v] : acc[k][v];
        }
    }
    __syncthreads();
  }
  double* const out = a.part + (size_t)blockIdx.x * (T::kBlocks * 256);
  for (int e = threadIdx.x; e < T::kBlocks * 256; e += 256) out[e] = sum[e];
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// What is added to G's diagonal, of its trace.  A step multiplies a small eigenvalue by 11.9.  Where u has fewer directions than rows,
// G's others are roundings: some 2^-53 times the root of a wave's 16 to n / 4 sums in a row, of either sign, and negative ones
// would leave the polynomial's range in 15 steps (|X| reaches 94 for one direction in 16 rows at 16 steps).  Lifted they stay
// in it.  Singular values of 1e-6 of the norm come out 4e-3 off where that counts (from ten steps on); a fp32 iteration's own roundings
// are 6e-2 of them.
__device__ __forceinline__ double lift(const SmallItem& it, int steps) {
  return wide(steps) ? 0x1p-48 * fmax(1.0, max(it.rows(), it.cols()) / 8192.0) : 0.0;
}
__device__ __forceinline__ void put_q(const SmallArgs& a, size_t at, double q) {
  if (wide(a.steps)) static_cast<double*>(a.q)[at] = q;
  else static_cast<float*>(a.q)[at] = (float)q;
}

// A matrix of the iteration in the LDS: [MB][MB] blocks of 16 x 16, their rows 17 apart (a column is in all banks).  An fp64 product's
// result holds, at a lane's place v, row lane / 16 + 4 v and column lane % 16, which is also what its operands want there, the
// first one turned.  So X^T Y, which is X Y for a symmetric X, reads whole blocks in order.
constexpr int kRowOf = 17, kBlockOf = 16 * kRowOf;
template <int MB>
__device__ __forceinline__ void block_at(int k, int& i, int& j) {  // the k-th on or below the diagonal
  int first = 0;
  i = 0;
  while (first + i + 1 <= k) first += ++i;
  j = k - first;
}
// Such a block of X Y.
template <int MB>
__device__ __forceinline__ f64x4 block_product(const double* X, const double* Y, int k) {
  const int lane = threadIdx.x & 63;
  int i, j;
  block_at<MB>(k, i, j);
  const int at = (lane >> 4) * kRowOf + (lane & 15);
  f64x4 acc = {};
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const double *const x = X + (b * MB + i) * kBlockOf + at, *const y = Y + (b * MB + j) * kBlockOf + at;
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(x[4 * kRowOf * s], y[4 * kRowOf * s], acc, 0, 0, 0);
  }
  return acc;
}
// f(element of the matrix, sum, whether on the diagonal) of such a block into out.  What is above the diagonal is what is below it to the
// last bit: what differs would grow nine-fold with each step.
template <int MB, class Fn>
__device__ __forceinline__ void put_block(const f64x4& x, double* out, int k, Fn f) {
  const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  int i, j;
  block_at<MB>(k, i, j);
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int r = g + 4 * v, at = (i * MB + j) * kBlockOf + r * kRowOf + l;
    if (i == j && r < l) continue;
    const double y = f(at, x[v], i == j && r == l);
    out[at] = y;
    out[(j * MB + i) * kBlockOf + l * kRowOf + r] = y;
  }
}

// Three products one after the other a step: P, then A P and Q P beside each other, then (A P) P; each stays in its wave's registers
// until all have read what it takes the place of.  A wave a block: a side of 64 41 us, of 48 24, of 32 15 (four waves, whole
// matrices and A P behind Q P: 76, 39 and 16).  Of a side of 64 21 us are the matrix core's with most to do, 65 cycles a product.
constexpr int iterate_waves(int MB) { return MB == 2 ? 8 : 16; }
template <int MB>
__global__ __launch_bounds__(64 * iterate_waves(MB)) void iterate_kernel(const SmallArgs a) {
  typedef Tile<MB> T;
  constexpr int M = T::M, W = iterate_waves(MB), kThreads = 64 * W, B = T::kBlocks, kUnits = (2 * B + W - 1) / W, kAll = MB * MB * kBlockOf;
  static_assert(B <= W, "a wave a block");
  __shared__ double A[kAll], P[kAll], Q[kAll];
  const int entry = entry_of(a.iterate, blockIdx.x), wave = threadIdx.x >> 6;
  const unsigned splits = a.item[entry].splits;
  const double* const part = a.part + (a.gram[entry] + (size_t)(blockIdx.x - a.iterate[entry]) * splits) * (B * 256);
  for (int e = threadIdx.x; e < B * 256; e += kThreads) {
    double x = 0.0;
    unsigned s = 0;
    for (; s + 8 <= splits; s += 8) {
      double y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = part[(size_t)(s + k) * (B * 256) + e];
#pragma unroll
      for (int k = 0; k < 8; ++k) x += y[k];
    }
    for (; s < splits; ++s) x += part[(size_t)s * (B * 256) + e];
    int i, j;
    block_at<MB>(e / 256, i, j);
    const int r = e % 256 / 16, c = e % 16;
    if (i == j && r < c) continue;
    A[(i * MB + j) * kBlockOf + r * kRowOf + c] = x;
    A[(j * MB + i) * kBlockOf + c * kRowOf + r] = x;
  }
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const double square = wave_sum(lane < M ? A[lane / 16 * (MB + 1) * kBlockOf + lane % 16 * (kRowOf + 1)] : 0.0);
  const double over = square < INFINITY ? 1.0 / (sqrt(square) + a.eps) : (double)NAN, more = lift(a.item[entry], a.steps) * square;
  __syncthreads();
  for (int e = threadIdx.x; e < kAll; e += kThreads) {
    const int r = e % kBlockOf / kRowOf, c = e % kRowOf, i = e / kBlockOf / MB, j = e / kBlockOf % MB;
    if (c < 16) A[e] = (A[e] + (i == j && r == c ? more : 0.0)) * over * over;
  }
  __syncthreads();
  const auto plain = [](int, double x, bool) { return x; };
  for (int s = 0; s < a.steps; ++s) {
    if (wave < B)
      put_block<MB>(block_product<MB>(A, A, wave), P, wave, [&](int at, double x, bool diagonal) { return kC * x + kB * A[at] + (diagonal ? kA : 0.0); });
    __syncthreads();
    // (the first step's Q is P itself; the last step needs no A)
    const bool last = s + 1 == a.steps;
    const int from = s ? 0 : B, to = last ? B : 2 * B;
    f64x4 x[kUnits];
#pragma unroll
    for (int e = 0; e < kUnits; ++e) {
      const int k = from + wave + e * W;
      if (k < to) x[e] = block_product<MB>(k < B ? Q : A, P, k < B ? k : k - B);
    }
    __syncthreads();
    if (s == 0)
      for (int e = threadIdx.x; e < kAll; e += kThreads)
        if (e % kRowOf < 16) Q[e] = P[e];
#pragma unroll
    for (int e = 0; e < kUnits; ++e) {
      const int k = from + wave + e * W;
      if (k < to) put_block<MB>(x[e], k < B ? Q : A, k < B ? k : k - B, plain);
    }
    __syncthreads();
    if (last) break;
    if (wave < B) x[0] = block_product<MB>(A, P, wave);
    __syncthreads();
    if (wave < B) put_block<MB>(x[0], A, wave, plain);
    __syncthreads();
  }
  for (int e = threadIdx.x; e < M * M; e += kThreads) {
    const int r = e / M, c = e % M;
    put_q(a, (size_t)blockIdx.x * (M * M) + e, Q[(r / 16 * MB + c / 16) * kBlockOf + r % 16 * kRowOf + c % 16] * over);
  }
}

// A short side of up to 16: one wave does it in its registers.  An fp64 product's result holds, at a lane's place v, row
// lane / 16 + 4 v and column lane % 16, which is also what its operands want there, the first one turned: so products
// are X^T Y without a move, and X Y as long as X is symmetric but for roundings, which X^T Y does not let grow (X Y^T
// would, nine-fold with each step).
__device__ __forceinline__ f64x4 turned_product(const f64x4& x, const f64x4& y) {
  f64x4 acc = {};
#pragma unroll
  for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(x[s], y[s], acc, 0, 0, 0);
  return acc;
}
// The mean of such a matrix and its transposed.
__device__ __forceinline__ f64x4 balanced(const f64x4& x) {
  const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  f64x4 out;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int from = g + 4 * v + 16 * (l & 3);                     // (row l, column g + 4 v: there at the place l / 4)
    double y = 0.0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const double z = __shfl(x[w], from);
      y = l >> 2 == w ? z : y;
    }
    out[v] = 0.5 * (x[v] + y);
  }
  return out;
}
__global__ __launch_bounds__(256) void iterate_16_kernel(const SmallArgs a) {
  __shared__ double sums[3][256];
  const int entry = entry_of(a.iterate, blockIdx.x), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const unsigned splits = a.item[entry].splits;
  const double* const part = a.part + (a.gram[entry] + (size_t)(blockIdx.x - a.iterate[entry]) * splits) * 256;
  f64x4 A = {};
#pragma unroll 4
  for (unsigned s = wave; s < splits; s += 4)
#pragma unroll
    for (int v = 0; v < 4; ++v) A[v] += part[(size_t)s * 256 + (g + 4 * v) * 16 + l];
  if (wave)
#pragma unroll
    for (int v = 0; v < 4; ++v) sums[wave - 1][64 * v + lane] = A[v];
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int v = 0; v < 4; ++v) A[v] += sums[w][64 * v + lane];
  double trace = 0.0;
#pragma unroll
  for (int v = 0; v < 4; ++v) trace += g + 4 * v == l ? A[v] : 0.0;
  trace = wave_sum(trace);
  const double over = trace < INFINITY ? 1.0 / (sqrt(trace) + a.eps) : (double)NAN, more = lift(a.item[entry], a.steps) * trace;
#pragma unroll
  for (int v = 0; v < 4; ++v) A[v] = (A[v] + (g + 4 * v == l ? more : 0.0)) * over * over;
  f64x4 Q = {};
  for (int s = 0; s < a.steps; ++s) {
    f64x4 P = turned_product(A, A);                                // a + b A + c A A
#pragma unroll
    for (int v = 0; v < 4; ++v) P[v] = kC * P[v] + kB * A[v] + (g + 4 * v == l ? kA : 0.0);
    Q = s ? turned_product(Q, P) : P;
    if (s + 1 < a.steps) A = turned_product(turned_product(A, P), P);
    // (what A and its transposed differ by grows in directions that u lacks as their values do: 1e-8 of X in 8 steps, 1e-6 in 10,
    // 1e-2 in 14)
    if (wide(a.steps)) A = balanced(A);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) put_q(a, (size_t)blockIdx.x * 256 + (g + 4 * v) * 16 + l, Q[v] * over);
}

// F: float or double.
template <int MB, class F>
__global__ __launch_bounds__(256) void apply_kernel(const SmallArgs a) {
  typedef Tile<MB> T;
  typedef F Four __attribute__((ext_vector_type(4)));
  constexpr bool kWide = sizeof(F) == 8;
  constexpr int M = T::M, SQ = M + (kWide ? 2 : 4);
  __shared__ __attribute__((aligned(16))) float u[M * T::S];
  __shared__ F q[M * SQ];
  const int entry = entry_of(a.apply, blockIdx.x);
  const SmallItem& it = a.item[entry];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const unsigned tiles = (max(it.rows(), it.cols()) + T::JT - 1) / T::JT;
  const unsigned matrix = (blockIdx.x - a.apply[entry]) / tiles, tile = (blockIdx.x - a.apply[entry]) % tiles;
  const int m = min(it.rows(), it.cols()), j0 = tile * T::JT;
  const size_t base = (size_t)matrix * it.rows() * it.cols();
  for (int e = m * T::S + threadIdx.x; e < M * T::S; e += 256) u[e] = 0.0f;
  const F* const from = static_cast<const F*>(a.q) + (size_t)(a.iterate[entry] + matrix) * (M * M);
  for (int e = threadIdx.x; e < M * M; e += 256) q[e / M * SQ + e % M] = from[e];
  load_tile<MB, false>(a, it, base, j0, u);
  __syncthreads();
#pragma unroll 1
  for (int b = wave; b < T::JT / 16; b += 4) {                     // 16 places of the long side: this wave's alone
    Four acc[MB] = {};
#pragma unroll 4
    for (int s = 0; s < M / 4; ++s) {
      const F y = u[(4 * s + g) * T::S + 16 * b + l];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const F x = q[(16 * i + l) * SQ + 4 * s + g];
        if constexpr (kWide) acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(x, y, acc[i], 0, 0, 0);
        else acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, acc[i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) u[(16 * i + (kWide ? g + 4 * v : 4 * g + v)) * T::S + 16 * b + l] = (float)acc[i][v];
  }
  __syncthreads();
  const auto shift = [&](void* p, int dtype) { return p ? (char*)p + base * (dtype == CP4_DTYPE_F32 ? 4 : 2) : nullptr; };
  const Outputs o{shift(it.param, it.param_dtype), shift(it.copy, it.copy_dtype), it.param_dtype, it.copy_dtype};
  const bool flat = it.rows() <= it.cols();
  const Rates rates{a.decay, (float)(a.lr * sqrt(fmax(1.0, (double)it.rows() / it.cols())))};
  for_tile<MB>(it, j0, [&](size_t at, int count, int i, int j) __attribute__((always_inline)) {
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = k < count ? u[i * T::S + j] : 0.0f;
      if (flat) {
        if (k + 1 < count) ++j;
      } else if (++i == m) {
        i = 0;
        ++j;
      }
    }
    put_out<4>(o, rates, at, count, x);
  });
}

template <int MB>
hipError_t small_launch(const SmallArgs& a, unsigned gram, unsigned iterate, unsigned apply, hipStream_t st) {
  gram_kernel<MB><<<gram, 256, 0, st>>>(a);
  if constexpr (MB == 1) iterate_16_kernel<<<iterate, 256, 0, st>>>(a);
  else iterate_kernel<MB><<<iterate, 64 * iterate_waves(MB), 0, st>>>(a);
  if (wide(a.steps)) apply_kernel<MB, double><<<apply, 256, 0, st>>>(a);
  else apply_kernel<MB, float><<<apply, 256, 0, st>>>(a);
  return hipGetLastError();
}

// ---- longer sides: the momentum, the norm and X in two parts ---------------------------------

struct LargeItem {
  const void* grad;
  float* momentum;
  char *rows_out, *cols_out;                       // X as [rows][cols] and as [cols][rows], one matrix behind the other
  int grad_dtype;
  unsigned rows, cols;
  unsigned chunks, tiles;                          // of a matrix: workgroups of the norm's launch and of the split's
  float* t0;                                       // of each matrix
};
struct LargeArgs {
  LargeItem item[kLarge];
  unsigned norm[kLarge], split[kLarge];            // an entry's first workgroup of each launch; ~0: no entry
  int nesterov;
  unsigned chunk;                                  // values of a workgroup of the norm's launch
  float mu;
  double eps;
  double* part;                                    // [the norm's workgroups]
};
static_assert(sizeof(LargeArgs) <= 4096, "kernel arguments");

__global__ __launch_bounds__(256) void norm_kernel(const LargeArgs a) {
  const int entry = entry_of(a.norm, blockIdx.x);
  const LargeItem& it = a.item[entry];
  const unsigned matrix = (blockIdx.x - a.norm[entry]) / it.chunks, chunk = (blockIdx.x - a.norm[entry]) % it.chunks;
  const size_t size = (size_t)it.rows * it.cols, base = matrix * size;
  const size_t first = (size_t)chunk * a.chunk, last = min(size, first + a.chunk);
  double s = 0.0;
#pragma unroll 4
  for (size_t at = first + threadIdx.x * 4; at < last; at += 1024) {
    float u[4];
    direction<true>(it.grad, it.grad_dtype, it.momentum, base + at, (int)min((size_t)4, last - at), a.mu, a.nesterov, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) s += (double)u[j] * u[j];
  }
  __shared__ double sums[4];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) a.part[blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

// 64 x 64 values: each thread 16 of a row, and turned in the LDS 16 of a column.
__global__ __launch_bounds__(256) void split_kernel(const LargeArgs a) {
  __shared__ float lds[64][65];
  __shared__ double sums[4];
  const int entry = entry_of(a.split, blockIdx.x);
  const LargeItem& it = a.item[entry];
  const unsigned matrix = (blockIdx.x - a.split[entry]) / it.tiles, tile = (blockIdx.x - a.split[entry]) % it.tiles;
  const unsigned wide = (it.cols + 63) / 64, r0 = tile / wide * 64, c0 = tile % wide * 64;
  const size_t size = (size_t)it.rows * it.cols;
  const double* const part = a.part + a.norm[entry] + (size_t)matrix * it.chunks;
  double s = 0.0;
  for (unsigned i = threadIdx.x; i < it.chunks; i += 256) s += part[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  s = sums[0] + sums[1] + sums[2] + sums[3];
  double over = s < INFINITY ? 1.0 / (sqrt(s) + a.eps) : (double)NAN;
  int power;
  frexp(s < INFINITY ? sqrt(s) * over : 1.0, &power);              // (|X|: in (0.5, 1), times 2^power, or 0)
  power = max(-126, min(0, power));
  if (tile == 0 && threadIdx.x == 0) it.t0[matrix] = ldexpf(1.0f, power);
  over = ldexp(over * kScale, -power);
  const int line = threadIdx.x / 4, at = threadIdx.x % 4 * 16;
  const unsigned r = r0 + line, c = c0 + at;
  float x[16] = {};
  if (r < it.rows) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float u[4];
      direction<false>(it.grad, it.grad_dtype, it.momentum, matrix * size + (size_t)r * it.cols + c + 4 * k,
                       (int)it.cols - (int)c - 4 * k, a.mu, a.nesterov, u);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * k + j] = (int)c + 4 * k + j < (int)it.cols ? (float)(u[j] * over) : 0.0f;
    }
    if (c < padded(it.cols)) store_parts<16>(it.rows_out + matrix * part_bytes(it.rows, it.cols) + r * padded(it.cols) * 4, c, x);
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) lds[line][at + j] = x[j];
  __syncthreads();
  const unsigned tc = c0 + line, tr = r0 + at;                     // (a row of the turned matrix)
  if (tc >= it.cols || tr >= padded(it.rows)) return;
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = lds[at + j][line];
  store_parts<16>(it.cols_out + matrix * part_bytes(it.cols, it.rows) + tc * padded(it.rows) * 4, tr, x);
}

// ---- the step -------------------------------------------------------------------------

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// `count` matrices of an entry, from its matrix `first` on.
struct Piece { size_t entry, first, count; };
struct Group {
  bool small = false;
  int blocks = 0;                                  // (small) of 16: the short side
  std::vector<Piece> pieces;
  size_t bytes = 0;
};
// Scratch memory of a larger matrix: X twice and its transposed twice, A and B.
size_t large_bytes(const cp4_muon_matrix& x) {
  const size_t m = std::min(x.rows, x.cols);
  return 2 * (part_bytes(x.rows, x.cols) + part_bytes(x.cols, x.rows)) + 2 * part_bytes(m, m);
}
constexpr size_t kGroupBytes = (size_t)1 << 30;
constexpr size_t kNormParts = 1 << 16, kMatrices = 4096;             // at most, of a group

bool nothing(const cp4_muon_matrix& x) { return !x.count || !x.rows || !x.cols; }
// (without them the momentum alone is updated)
bool has_outputs(const cp4_muon_matrix& x) { return x.param || x.copy; }

// Sizes of gram's launch: an entry's splits.  Enough workgroups for four on a compute unit, but no more than one workgroup
// of iterate adds up in the time of a launch (10 blocks of 2 KB a split at a side of 64).
unsigned gram_splits(unsigned tiles, size_t matrices, int blocks) {
  const unsigned most = blocks == 1 ? 128 : blocks == 2 ? 64 : 32;
  const size_t wanted = std::max<size_t>(1, 4 * (size_t)num_compute_units() / std::max<size_t>(1, matrices));
  return (unsigned)std::min<size_t>({(size_t)tiles, (size_t)most, wanted});
}
unsigned tile_length(int blocks) { return blocks == 1 ? 256 : blocks == 2 ? 128 : 64; }
unsigned tiles_of(const cp4_muon_matrix& x, int blocks) {
  return (std::max(x.rows, x.cols) + tile_length(blocks) - 1) / tile_length(blocks);
}
size_t small_bytes(const cp4_muon_matrix* x, Group& g) {
  size_t matrices = 0, wgs = 0;
  for (const Piece& p : g.pieces) matrices += p.count;
  for (const Piece& p : g.pieces) wgs += p.count * gram_splits(tiles_of(x[p.entry], g.blocks), matrices, g.blocks);
  const size_t blocks = (size_t)g.blocks * (g.blocks + 1) / 2;
  return align256(wgs * blocks * 256 * 8) + align256(matrices * g.blocks * g.blocks * 256 * 8);
}

Product gram_product(const cp4_muon_matrix& x, unsigned count) {
  Product p{};
  p.R = p.N = std::min(x.rows, x.cols);
  p.K = std::max(x.rows, x.cols);
  p.count = count;
  p.symmetric = true;
  p.four_to_step = p.beta = 1.0f;
  return p;
}
// The splits of a group's first product and what they take.
int large_splits(const cp4_muon_matrix* x, const Group& g, size_t* bytes) {
  std::vector<Product> a;
  for (const Piece& p : g.pieces)
    if (has_outputs(x[p.entry])) a.push_back(gram_product(x[p.entry], (unsigned)p.count));
  const int splits = a.empty() ? 1 : product_splits(a.data(), (int)a.size());
  *bytes = 0;
  if (splits > 1)
    for (const Product& p : a) *bytes += align256((size_t)p.count * splits * p.R * p.N * 4);
  return splits;
}

std::vector<Group> groups_of(const cp4_muon_matrix* x, size_t n) {
  std::vector<Group> out;
  constexpr size_t kMostWgs = 1 << 16;             // of a launch: the chip many times over, and up to 36 KB of scratch memory each
  for (int blocks = 1; blocks <= (int)kSide / 16; ++blocks) {
    size_t tiles = 0;
    Group g;
    const auto done = [&]() {
      if (g.pieces.empty()) return;
      g.small = true;
      g.blocks = blocks;
      g.bytes = small_bytes(x, g);
      out.push_back(std::move(g));
      g = Group();
      tiles = 0;
    };
    for (size_t i = 0; i < n; ++i) {
      if (nothing(x[i]) || (int)((std::min(x[i].rows, x[i].cols) + 15) / 16) != blocks) continue;
      const size_t each = tiles_of(x[i], blocks);
      for (size_t first = 0; first < x[i].count;) {
        if (g.pieces.size() == kSmall || tiles + each > kMostWgs) done();
        const size_t count = std::min(x[i].count - first, (kMostWgs - tiles) / each);
        g.pieces.push_back(Piece{i, first, count});
        tiles += count * each;
        first += count;
      }
    }
    done();
  }
  Group g;
  const auto done = [&]() {
    if (g.pieces.empty()) return;
    size_t part;
    large_splits(x, g, &part);
    g.bytes = align256(kNormParts * 8) + align256(kMatrices * 4) + part;
    for (const Piece& p : g.pieces) g.bytes += p.count * large_bytes(x[p.entry]) + 6 * 256;
    out.push_back(std::move(g));
    g = Group();
  };
  size_t bytes = 0, matrices = 0;
  for (size_t i = 0; i < n; ++i) {
    if (nothing(x[i]) || std::min(x[i].rows, x[i].cols) <= kSide) continue;
    const size_t each = large_bytes(x[i]);
    for (size_t first = 0; first < x[i].count;) {
      if (!g.pieces.empty() && (g.pieces.size() == kLarge || bytes + each > kGroupBytes || matrices >= kMatrices)) {
        done();
        bytes = matrices = 0;
      }
      const size_t room = g.pieces.empty() ? std::max<size_t>(1, kGroupBytes / each) : (kGroupBytes - bytes) / each;
      const size_t count = std::min({x[i].count - first, room, kMatrices - matrices});
      g.pieces.push_back(Piece{i, first, count});
      bytes += count * each;
      matrices += count;
      first += count;
    }
  }
  done();
  return out;
}

struct Settings {
  double lr, weight_decay, eps;
  float mu;
  int nesterov, steps;
};
size_t bytes_of(int dtype) { return dtype == CP4_DTYPE_F32 ? 4 : 2; }
void* ahead(void* p, size_t values, int dtype) { return p ? static_cast<char*>(p) + values * bytes_of(dtype) : nullptr; }
Outputs outputs_of(const cp4_muon_matrix& x, size_t first) {
  const size_t at = first * x.rows * x.cols;
  return Outputs{ahead(x.param, at, x.param_dtype), ahead(x.copy, at, x.copy_dtype), x.param_dtype, x.copy_dtype};
}
Rates rates_of(const cp4_muon_matrix& x, const Settings& s) {
  return Rates{(float)(1.0 - s.lr * s.weight_decay), (float)(s.lr * std::sqrt(std::max(1.0, (double)x.rows / x.cols)))};
}

hipError_t run_small(const cp4_muon_matrix* x, const Group& g, const Settings& s, char* ws, hipStream_t st) {
  SmallArgs a{};
  size_t matrices = 0;
  for (const Piece& p : g.pieces) matrices += p.count;
  unsigned gram = 0, iterate = 0, apply = 0;
  for (int i = 0; i < kSmall; ++i) {
    a.gram[i] = a.iterate[i] = a.apply[i] = ~0u;
    if (i >= (int)g.pieces.size()) continue;
    const Piece& p = g.pieces[i];
    const cp4_muon_matrix& e = x[p.entry];
    SmallItem& it = a.item[i];
    const size_t at = p.first * e.rows * e.cols;
    const Outputs o = outputs_of(e, p.first);
    const unsigned tiles = tiles_of(e, g.blocks);
    it.grad = ahead(const_cast<void*>(e.grad), at, e.grad_dtype);
    it.momentum = e.momentum ? e.momentum + at : nullptr;
    it.param = o.param;
    it.copy = o.copy;
    it.param_dtype = (unsigned char)e.param_dtype;
    it.grad_dtype = (unsigned char)e.grad_dtype;
    it.copy_dtype = (unsigned char)e.copy_dtype;
    it.last_row = (unsigned short)(e.rows - 1);
    it.last_col = (unsigned short)(e.cols - 1);
    it.splits = (unsigned char)gram_splits(tiles, matrices, g.blocks);
    a.gram[i] = gram;
    a.iterate[i] = iterate;
    a.apply[i] = apply;
    gram += (unsigned)p.count * it.splits;
    iterate += (unsigned)p.count;
    apply += (unsigned)p.count * tiles;
  }
  a.decay = (float)(1.0 - s.lr * s.weight_decay);
  a.lr = s.lr;
  a.nesterov = s.nesterov;
  a.steps = s.steps;
  a.mu = s.mu;
  a.eps = s.eps;
  a.part = reinterpret_cast<double*>(ws);
  a.q = ws + align256((size_t)gram * (g.blocks * (g.blocks + 1) / 2) * 256 * 8);
  switch (g.blocks) {
    case 1: return small_launch<1>(a, gram, iterate, apply, st);
    case 2: return small_launch<2>(a, gram, iterate, apply, st);
    case 3: return small_launch<3>(a, gram, iterate, apply, st);
    default: return small_launch<4>(a, gram, iterate, apply, st);
  }
}

hipError_t run_large(const cp4_muon_matrix* x, const Group& g, const Settings& s, char* ws, hipStream_t st) {
  LargeArgs a{};
  a.nesterov = s.nesterov;
  a.mu = s.mu;
  a.eps = s.eps;
  a.part = reinterpret_cast<double*>(ws);
  ws += align256(kNormParts * 8);
  float* const t0 = reinterpret_cast<float*>(ws);
  ws += align256(kMatrices * 4);
  size_t values = 0, part_total;
  for (const Piece& p : g.pieces) values += p.count * x[p.entry].rows * x[p.entry].cols;
  // (4096 values and more; at most half of the partial sums' room beside one for each matrix's rest)
  size_t chunk = 4096;
  while (chunk < ((size_t)1 << 22) && values / chunk > 4 * (size_t)num_compute_units()) chunk *= 2;
  while (values / chunk > kNormParts / 2) chunk *= 2;
  a.chunk = (unsigned)chunk;
  const int splits = large_splits(x, g, &part_total);
  std::vector<Product> first, second, third, last;
  char* part = ws;
  ws += part_total;
  const auto take = [&](size_t bytes) {
    char* const p = ws;
    ws += align256(bytes);
    return p;
  };
  unsigned norm = 0, split = 0, matrices = 0;
  struct Buffers { char *x[2], *t[2], *a, *b; };    // X [m][n], transposed [n][m], A and B
  std::vector<Buffers> buffers;
  for (unsigned& k : a.norm) k = ~0u;
  for (unsigned& k : a.split) k = ~0u;
  for (size_t i = 0; i < g.pieces.size(); ++i) {
    const Piece& p = g.pieces[i];
    const cp4_muon_matrix& e = x[p.entry];
    LargeItem& it = a.item[i];
    const size_t at = p.first * e.rows * e.cols, m = std::min(e.rows, e.cols), n = std::max(e.rows, e.cols);
    const bool flat = e.rows <= e.cols;
    Buffers b{};
    for (int k = 0; k < 2; ++k) {
      b.x[k] = take(p.count * part_bytes(m, n));
      b.t[k] = take(p.count * part_bytes(n, m));
    }
    b.a = take(p.count * part_bytes(m, m));
    b.b = take(p.count * part_bytes(m, m));
    buffers.push_back(b);
    it.grad = ahead(const_cast<void*>(e.grad), at, e.grad_dtype);
    it.momentum = e.momentum ? e.momentum + at : nullptr;
    it.rows_out = flat ? b.x[0] : b.t[0];
    it.cols_out = flat ? b.t[0] : b.x[0];
    it.grad_dtype = e.grad_dtype;
    it.rows = e.rows;
    it.cols = e.cols;
    it.chunks = (unsigned)(((size_t)e.rows * e.cols + chunk - 1) / chunk);
    a.norm[i] = norm;
    it.tiles = has_outputs(e) ? ((e.rows + 63) / 64) * ((e.cols + 63) / 64) : 0;
    a.split[i] = split;
    norm += it.chunks * (unsigned)p.count;
    split += it.tiles * (unsigned)p.count;
    it.t0 = t0 + matrices;
    matrices += (unsigned)p.count;
  }
  norm_kernel<<<norm, 256, 0, st>>>(a);
  if (split) split_kernel<<<split, 256, 0, st>>>(a);
  if (const hipError_t e = hipGetLastError()) return e;
  if (!split) return hipSuccess;
  for (int k = 0; k < s.steps; ++k) {
    std::vector<Product> pa, pb, px;
    char* to = part;
    for (size_t i = 0; i < g.pieces.size(); ++i) {
      const cp4_muon_matrix& e = x[g.pieces[i].entry];
      if (!has_outputs(e)) continue;
      const Buffers& b = buffers[i];
      const char *const X = b.x[k % 2], *const Xt = b.t[k % 2];
      Product p = gram_product(e, (unsigned)g.pieces[i].count);
      p.P = p.Q = X;
      p.C = b.a;
      if (splits > 1) {
        p.part = reinterpret_cast<float*>(to);
        to += align256((size_t)p.count * splits * p.R * p.N * 4);
      }
      pa.push_back(p);
      p.part = nullptr;
      p.t0 = a.item[i].t0;
      p.four_to_step = std::ldexp(1.0f, 2 * k);
      p.P = p.Q = p.E = b.a;
      p.C = b.b;
      p.K = p.N;
      p.alpha = (float)kB;
      p.beta = (float)kC;
      p.diagonal = (float)kA;
      pb.push_back(p);
      p.symmetric = false;
      p.alpha = p.diagonal = 0.0f;
      p.beta = p.four_to_step = 1.0f;
      p.t0 = nullptr;
      p.E = nullptr;
      if (k + 1 < s.steps || e.rows <= e.cols) {
        p.N = std::max(e.rows, e.cols);
        p.P = b.b;
        p.Q = Xt;
      } else {                                     // (the parameters lie the other way round)
        p.R = std::max(e.rows, e.cols);
        p.P = Xt;
        p.Q = b.b;
      }
      if (k + 1 < s.steps) {
        p.C = b.x[(k + 1) % 2];
        p.Ct = b.t[(k + 1) % 2];
      } else {
        p.C = nullptr;
        p.final = true;
        p.t0 = a.item[i].t0;
        p.four_to_step = std::ldexp(1.0f, 2 * k);
        p.o = outputs_of(e, g.pieces[i].first);
        p.rates = rates_of(e, s);
      }
      px.push_back(p);
    }
    if (const hipError_t e = product_launch(pa.data(), (int)pa.size(), splits, st)) return e;
    if (const hipError_t e = product_launch(pb.data(), (int)pb.size(), 1, st)) return e;
    if (const hipError_t e = product_launch(px.data(), (int)px.size(), 1, st)) return e;
  }
  return hipSuccess;
}

bool dtype_ok(int d) { return d == CP4_DTYPE_F32 || d == CP4_DTYPE_BF16 || d == CP4_DTYPE_F16; }
cp4_status check_matrices(const cp4_muon_matrix* x, size_t n) {
  if (!x && n) return fail_with(CP4_ERR_NULL_POINTER, "matrices is NULL");
  for (size_t i = 0; i < n; ++i) {
    const cp4_muon_matrix& e = x[i];
    if (nothing(e)) continue;
    if (e.rows > 65536 || e.cols > 65536) return fail_with(CP4_ERR_SHAPE, "a matrix with a side above 65536");
    if (e.count > (size_t)1 << 24) return fail_with(CP4_ERR_SHAPE, "more than 2^24 matrices in an entry");
    if (!e.grad) return fail_with(CP4_ERR_NULL_POINTER, "a matrix's gradient is NULL");
    if (!dtype_ok(e.grad_dtype) || (e.param && !dtype_ok(e.param_dtype)) || (e.copy && !dtype_ok(e.copy_dtype)))
      return fail_with(CP4_ERR_SHAPE, "unknown dtype of a matrix");
    if ((size_t)e.grad % bytes_of(e.grad_dtype) || (size_t)e.momentum % 4 || (e.param && (size_t)e.param % bytes_of(e.param_dtype)) ||
        (e.copy && (size_t)e.copy % bytes_of(e.copy_dtype)))
      return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  }
  return CP4_OK;
}

}  // namespace
}  // namespace muon
}  // namespace cp4

using namespace cp4::muon;
using cp4::fail_hip;
using cp4::fail_with;

extern "C" size_t cp4_muon_workspace_bytes(const cp4_muon_matrix* x, size_t n) try {
  if (check_matrices(x, n) != CP4_OK) return 0;
  size_t most = 0;
  for (const Group& g : groups_of(x, n)) most = std::max(most, g.bytes);
  return most;
} catch (const std::exception& e) {
  fail_with(CP4_ERR_HIP, e.what());
  return 0;
}

extern "C" cp4_status cp4_muon_step(const cp4_muon_matrix* x, size_t n, double lr, double momentum, int nesterov,
                                    double weight_decay, double eps, unsigned steps, void* workspace,
                                    size_t workspace_bytes, cp4_stream stream) try {
  if (const cp4_status rc = check_matrices(x, n)) return rc;
  if (!(lr >= 0) || !std::isfinite(lr) || !(momentum >= 0 && momentum < 1) || !(weight_decay >= 0) || !std::isfinite(weight_decay))
    return fail_with(CP4_ERR_SHAPE, "lr and weight_decay must be 0 or more, momentum in [0, 1)");
  // (what divides by it is held in fp32)
  if (!(eps >= 1e-30) || !std::isfinite(eps)) return fail_with(CP4_ERR_SHAPE, "eps must be 1e-30 or more");
  if (steps < 1 || steps > 16) return fail_with(CP4_ERR_SHAPE, "1 to 16 steps");
  const std::vector<Group> groups = groups_of(x, n);
  size_t need = 0;
  for (const Group& g : groups) need = std::max(need, g.bytes);
  if (need && (!workspace || workspace_bytes < need || ((size_t)workspace & 255)))
    return fail_with(CP4_ERR_WORKSPACE, "workspace missing, too small or not aligned to 256 bytes");
  const Settings s{lr, weight_decay, eps, (float)momentum, nesterov != 0, (int)steps};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for (const Group& g : groups) {
    char* const ws = static_cast<char*>(workspace);
    if (const hipError_t e = g.small ? run_small(x, g, s, ws, st) : run_large(x, g, s, ws, st)) return fail_hip(e, "cp4_muon_step");
  }
  return CP4_OK;
} catch (const std::exception& e) {
  return fail_with(CP4_ERR_HIP, e.what());
}
