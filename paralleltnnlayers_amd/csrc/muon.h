// Interface between the Muon step's C ABI (muon.hip) and its products in tiles (muon_tiles.hip).
#ifndef CP4_MUON_INTERNAL_H
#define CP4_MUON_INTERNAL_H

#include <hip/hip_runtime.h>

#include "cp4/muon.h"
#include "cp4_internal.h"
#include "value_types.h"

namespace cp4 {
namespace muon {

constexpr double kA = 3.4445, kB = -4.7750, kC = 2.0315;

// X of a matrix whose norm is far below eps is small throughout: a power of two t goes with it, X' = X / t in memory.  Of |X| in
// (t0 / 2, t0] it starts as t0, is four times as much with each step (X grows by up to 3.4445) and 1 in the end; where
// eps counts little it is 1 from the start.  A' = X' X'^T, then B = (t / next t) (a + b t^2 A' + c t^4 A' A'), X' of the next
// step is B X', and X in the end next t times that.
inline __host__ __device__ float scale_at(float t0, float four_to_step) { return fminf(1.0f, t0 * four_to_step); }

// A matrix [rows][cols] in two float16 parts: each 32 columns of a row are 64 bytes of first parts, then 64 of what those
// leave (one cache line), columns behind the last one up to a multiple of 32 are zero.  Values times kScale: X's, A's
// and a + b A + c A A's magnitudes are below 1.3, 1.5 and 3.45 (of singular values in 0 .. 1.21, where the polynomial keeps them),
// so that 2^14 keeps them below float16's 65504, and the second parts of an average value of a matrix of 65536 by 65536
// above its smallest steps.
constexpr float kScale = 16384.0f;
inline __host__ __device__ size_t padded(size_t cols) { return (cols + 31) / 32 * 32; }
inline __host__ __device__ size_t part_bytes(size_t rows, size_t cols) { return rows * padded(cols) * 4; }

// How a matrix's new values leave the last product: param null: X goes to `copy`.
struct Outputs {
  void *param, *copy;                       // [rows][cols] each, one matrix behind the other; may be null
  int param_dtype, copy_dtype;
};
struct Rates {
  float decay, rate;                        // p = p decay - rate X
};

// C[r][c] = alpha E[r][c] + beta sum_k P[r][k] Q[c][k] (+ diagonal where r == c), r < R, c < N, of `count` matrices one behind the other, P [R][K],
// Q [N][K], E and C [R][N] in two parts.
struct Product {
  const char *P, *Q, *E;                    // E null: alpha is 0
  char *C, *Ct;                             // Ct: C transposed as well (may be null)
  float* part;                              // splits > 1: partial sums [count][splits][R][N], and nothing else
  Outputs o;                                // (final) instead of C
  Rates rates;
  unsigned R, N, K, count;
  const float* t0;                          // of each matrix, for B and for X in the end; or null
  float four_to_step;
  float alpha, beta, diagonal;
  bool symmetric;                           // R == N and C is symmetric: tiles on and below the diagonal, mirrored into C
  bool final;                               // of all of a launch's products, or of none
};
constexpr int kProducts = 16;               // of a launch

// In how many parts the depth of a launch's products is taken (they have to be symmetric for more than one).
int product_splits(const Product* p, int n);
hipError_t product_launch(const Product* p, int n, int splits, hipStream_t st);

// ---- device side ------------------------------------------------------------------------

// The entry that workgroup `wg` works for, first: the entries' first ones, behind the last entry ~0.  (All of them are loaded
// at once: one after the other they were 4 us of a launch of 24 entries.)
template <int n>
__device__ __forceinline__ int entry_of(const unsigned (&first)[n], unsigned wg) {
  int k = 0;
#pragma unroll
  for (int i = 1; i < n; ++i) k += wg >= first[i];
  return k;
}

__device__ __forceinline__ float load_value(const void* p, int dtype, size_t at) {
  if (dtype == CP4_DTYPE_F32) return static_cast<const float*>(p)[at];
  const unsigned short v = static_cast<const unsigned short*>(p)[at];
  return dtype == CP4_DTYPE_BF16 ? BF16::widen(v) : F16::widen(v);
}
__device__ __forceinline__ void store_value(void* p, int dtype, size_t at, float v) {
  if (dtype == CP4_DTYPE_F32) static_cast<float*>(p)[at] = v;
  else static_cast<unsigned short*>(p)[at] = dtype == CP4_DTYPE_BF16 ? BF16::narrow(v) : F16::narrow(v);
}
// Up to n consecutive values from any element's address (count may be <= 0), zero behind.
template <int n>
__device__ __forceinline__ void load_values(const void* p, int dtype, size_t at, int count, float (&v)[n]) {
  if (count < n) {
#pragma unroll
    for (int j = 0; j < n; ++j) v[j] = j < count ? load_value(p, dtype, at + j) : 0.0f;
  } else if (dtype == CP4_DTYPE_F32) {
    __builtin_memcpy(v, static_cast<const float*>(p) + at, sizeof(v));
  } else {
    unsigned short r[n];
    __builtin_memcpy(r, static_cast<const unsigned short*>(p) + at, sizeof(r));
#pragma unroll
    for (int j = 0; j < n; ++j) v[j] = dtype == CP4_DTYPE_BF16 ? BF16::widen(r[j]) : F16::widen(r[j]);
  }
}
template <int n>
__device__ __forceinline__ void store_values(void* p, int dtype, size_t at, int count, const float (&v)[n]) {
  if (count < n) {
#pragma unroll
    for (int j = 0; j < n; ++j)
      if (j < count) store_value(p, dtype, at + j, v[j]);
  } else if (dtype == CP4_DTYPE_F32) {
    __builtin_memcpy(static_cast<float*>(p) + at, v, sizeof(v));
  } else {
    unsigned short r[n];
#pragma unroll
    for (int j = 0; j < n; ++j) r[j] = dtype == CP4_DTYPE_BF16 ? BF16::narrow(v[j]) : F16::narrow(v[j]);
    __builtin_memcpy(static_cast<unsigned short*>(p) + at, r, sizeof(r));
  }
}
// The step of up to n consecutive parameters along x, and what else wants the outcome.
template <int n>
__device__ __forceinline__ void put_out(const Outputs& o, const Rates& r, size_t at, int count, const float (&x)[n]) {
  float p[n];
#pragma unroll
  for (int j = 0; j < n; ++j) p[j] = x[j];
  if (o.param) {
    load_values<n>(o.param, o.param_dtype, at, count, p);
#pragma unroll
    for (int j = 0; j < n; ++j) p[j] = p[j] * r.decay - r.rate * x[j];
    store_values<n>(o.param, o.param_dtype, at, count, p);
  }
  if (o.copy) store_values<n>(o.copy, o.copy_dtype, at, count, p);
}
// A scaled value as two float16 parts.
__device__ __forceinline__ void two_halves(float x, unsigned short& hi, unsigned short& lo) {
  hi = F16::narrow(x);
  lo = F16::narrow(x - F16::widen(hi));
}
// n (up to 32, a power of two) consecutive columns from column c (a multiple of n) of a row in two parts.
template <int n>
__device__ __forceinline__ void store_parts(char* row, size_t c, const float (&x)[n]) {
  unsigned short hi[n], lo[n];
#pragma unroll
  for (int j = 0; j < n; ++j) two_halves(x[j], hi[j], lo[j]);
  char* const to = row + c / 32 * 128 + c % 32 * 2;
  __builtin_memcpy(__builtin_assume_aligned(to, 2 * n < 16 ? 2 * n : 16), hi, sizeof(hi));
  __builtin_memcpy(__builtin_assume_aligned(to + 64, 2 * n < 16 ? 2 * n : 16), lo, sizeof(lo));
}
template <int n>
__device__ __forceinline__ void load_parts(const char* row, size_t c, float (&x)[n]) {
  unsigned short hi[n], lo[n];
  const char* const from = row + c / 32 * 128 + c % 32 * 2;
  __builtin_memcpy(hi, __builtin_assume_aligned(from, 2 * n < 16 ? 2 * n : 16), sizeof(hi));
  __builtin_memcpy(lo, __builtin_assume_aligned(from + 64, 2 * n < 16 ? 2 * n : 16), sizeof(lo));
#pragma unroll
  for (int j = 0; j < n; ++j) x[j] = F16::widen(hi[j]) + F16::widen(lo[j]);
}

}  // namespace muon
}  // namespace cp4
#endif
