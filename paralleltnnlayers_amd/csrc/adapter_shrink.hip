// h = scale A_a x, token by token (include/cp4/adapter.h): a product with as few columns as the adapters
// have ranks, bound by reading x and the adapters in use once.
//
// A workgroup takes 16 tokens and one part of the inputs, straight from memory to the matrix cores:
// nothing is read twice within it, so the LDS would only be a detour (48 tokens of 32 adapters, 4096 inputs: 139 us
// through the LDS, 6.6 so).  Its eight waves share the adapters that these tokens have - one of a prompt, sixteen of
// single tokens - and, where there are fewer, the inputs.  All rows are multiplied with each adapter and the rows
// that are not its own keep what they had; the waves' sums meet in the LDS once, at the end.  (32 tokens a workgroup:
// no gain.)  With few tokens the inputs are split over workgroups as well: each part leaves a plane of h of its own,
// which the projection of few tokens adds up as it reads them and a small launch does before any other.
//
// A lane's ranks are RB * (lane & 15) + j, not 16 j + (lane & 15), so that factors that lie rank by rank
// (B, in the backward pass) come with loads of RB values.
//
// Measured (bf16): 8192 tokens of 4096 inputs, rank 16: 26 us, 2.6 TB/s (a copy reaches 5.1), bound by loads in flight, since
// every turn waits for memory once; 48 tokens of 32 adapters 6.6 us, which is the latency of a few such waits and a launch.
#include <algorithm>

#include "adapter.h"
#include "adapter_load.h"

namespace cp4 {
namespace adapter {
namespace {

constexpr int kWaves = 8;
template <class T>
constexpr int kUnit = 128 / sizeof(typename T::raw);                 // inputs of a loop's turn: a cache line a row

// One operand's row of a turn: 16 bytes of each half (64 bytes on); zero from `left` on.
template <class Raw>
__device__ __forceinline__ void load_row(const Raw* p, int left, bool full, u32x4 (&v)[2]) {
  constexpr int n = 16 / sizeof(Raw);
  if (full) {
    v[0] = load_16(p);
    v[1] = load_16(p + 4 * n);
  } else {
    v[0] = load_16(p, left);
    v[1] = load_16(p + 4 * n, left - 4 * n);
  }
}

template <class T, bool TR, int RB>
__global__ __launch_bounds__(64 * kWaves) void shrink_kernel(const ShrinkArgs a) {
  typedef typename T::raw Raw;
  constexpr int n = 16 / sizeof(Raw), U = kUnit<T>, kRows = 16;
  __shared__ float sum[kWaves][16][16 * RB + 4];
  __shared__ int own[kRows];
  __shared__ float factor[kRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const size_t t0 = (size_t)blockIdx.x * kRows;
  const int rows = (int)min((size_t)kRows, a.T - t0);
  int id = lane < rows ? a.ids[t0 + lane] : -1;
  if (id < 0 || id >= a.G) id = -1;
  if (threadIdx.x < kRows) {
    own[lane] = id;
    factor[lane] = a.scale && id >= 0 ? a.scale[id] : 1.0f;
  }
  int different = 0;
  {
    Adapters each(id);
    int ad;
    unsigned long long whose;
    while (different < kWaves && each.take(ad, whose)) ++different;
  }
  if (!different) return;
  // ways: how many waves go through the adapters in turn; the others share the inputs
  const int ways = different >= 8 ? 8 : different >= 4 ? 4 : different >= 2 ? 2 : 1;
  const int mine = wave & (ways - 1), slice = wave / ways, slices = kWaves / ways;
  const int units = (a.K + U - 1) / U, per = (units + a.planes - 1) / a.planes;
  const int u0 = min(units, (int)blockIdx.y * per), u1 = min(units, u0 + per);
  const int each = (u1 - u0 + slices - 1) / slices;
  const int first = min(u1, u0 + slice * each), last = min(u1, first + each);
  const int whole = min(last, a.K / U);                              // (from there on a turn has fewer inputs)

  const Raw* const z = static_cast<const Raw*>(a.z) + (t0 + min(l, rows - 1)) * a.ldz + n * g;

  for (int r0 = 0; r0 < a.Rp; r0 += 16 * RB) {
    f32x4 acc[RB] = {};
    Adapters todo(id);
    int ad, turn = 0;
    unsigned long long whose;
    while (todo.take(ad, whose)) {
      if ((turn++ & (ways - 1)) != mine) continue;
      const Raw* const f = static_cast<const Raw*>(a.f) + (size_t)ad * a.R * a.K;
      f32x4 d[RB] = {};
      auto load = [&](int u, bool full, u32x4 (&zv)[2], u32x4 (&fv)[RB][2]) __attribute__((always_inline)) {
        const int k = u * U + n * g, left = full ? U : a.K - k;
        load_row(z + (size_t)u * U, left, full, zv);
        if constexpr (!TR) {
#pragma unroll
          for (int j = 0; j < RB; ++j) {
            const int r = r0 + RB * l + j;
            load_row(f + (size_t)min(r, a.R - 1) * a.K + k, left, full, fv[j]);
            if (r >= a.R) fv[j][0] = fv[j][1] = u32x4{};
          }
        } else {
          const int r = r0 + RB * l;
          Raw x[2 * n][RB];
#pragma unroll
          for (int q = 0; q < 2 * n; ++q) {
            const int kq = q < n ? q : q + 3 * n;                     // (the second half lies 4 n inputs on)
            const Raw* const p = f + (size_t)(k + kq) * a.R + r;
            load_some(p, kq < left ? a.R - r : 0, x[q]);
          }
#pragma unroll
          for (int j = 0; j < RB; ++j) {
            Raw y[2][n];
#pragma unroll
            for (int q = 0; q < 2 * n; ++q) y[q / n][q % n] = x[q][j];
            __builtin_memcpy(&fv[j][0], y[0], 16);
            __builtin_memcpy(&fv[j][1], y[1], 16);
          }
        }
      };
      auto multiply = [&](const u32x4 (&zv)[2], const u32x4 (&fv)[RB][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < RB; ++j) {
            if constexpr (__is_same(T, F32)) {
#pragma unroll
              for (int q = 0; q < 4; ++q) d[j] = mfma_f32(__uint_as_float(zv[h][q]), __uint_as_float(fv[j][h][q]), d[j]);
            } else {
              d[j] = mfma_16<T>(__builtin_bit_cast(u16x8, zv[h]), __builtin_bit_cast(u16x8, fv[j][h]), d[j]);
            }
          }
      };
      constexpr int kAhead = RB <= 2 ? 4 : 2;                   // turns whose loads come before their products
      int u = first;
      for (; u + kAhead <= whole; u += kAhead) {
        u32x4 zv[kAhead][2], fv[kAhead][RB][2];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) load(u + e, true, zv[e], fv[e]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < kAhead; ++e) multiply(zv[e], fv[e]);
      }
      for (; u < last; ++u) {
        u32x4 zv[2], fv[RB][2];
        load(u, u < whole, zv, fv);
        multiply(zv, fv);
      }
#pragma unroll
      for (int j = 0; j < RB; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (whose >> (4 * g + v) & 1) acc[j][v] = d[j][v];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < RB; ++j)
#pragma unroll
      for (int v = 0; v < 4; ++v) sum[wave][4 * g + v][RB * l + j] = acc[j][v];
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * RB; at += 64 * kWaves) {
      const int row = at / (16 * RB), r = at % (16 * RB);
      if (own[row] < 0 || r0 + r >= a.Rp) continue;
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) x += sum[w][row][r];
      a.h[((size_t)blockIdx.y * a.T + t0 + row) * a.Rp + r0 + r] = x * factor[row];
    }
  }
}

template <class T, bool TR>
void launch_ranks(const ShrinkArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.T + 15) / 16), a.planes);
  if (a.Rp <= 16) shrink_kernel<T, TR, 1><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (a.Rp <= 32) shrink_kernel<T, TR, 2><<<grid, 64 * kWaves, 0, st>>>(a);
  else shrink_kernel<T, TR, 4><<<grid, 64 * kWaves, 0, st>>>(a);
}
template <class T>
void launch(const ShrinkArgs& a, hipStream_t st) {
  a.fk != 1 ? launch_ranks<T, true>(a, st) : launch_ranks<T, false>(a, st);
}

__global__ __launch_bounds__(64) void planes_kernel(float* h, const float* from, size_t n, int planes) {
  const size_t i = ((size_t)blockIdx.x * 64 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 x = {};
  int s = 0;
  for (; s + 8 <= planes; s += 8) {
    f32x4 y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = *reinterpret_cast<const f32x4*>(from + (s + e) * n + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) x += y[e];
  }
  for (; s < planes; ++s) x += *reinterpret_cast<const f32x4*>(from + s * n + i);
  *reinterpret_cast<f32x4*>(h + i) = x;
}

}  // namespace

hipError_t planes_join(float* h, const float* from, size_t n, int planes, hipStream_t st) {
  planes_kernel<<<(unsigned)((n + 255) / 256), 64, 0, st>>>(h, from, n, planes);
  return hipGetLastError();
}

// Parts of the inputs: a workgroup for each compute unit, two turns or more a part.  (Forward pass, bf16, 4096 inputs and
// outputs, 48 adapters: 48 tokens 138 us in one part, 43 in 8, 36 in 16; 2077 tokens 119 in one, 114 in 2; 8192 tokens 239 in one,
// 242 in 2, 243 in 4; 333 tokens of 1001 inputs 23.9 us in one, 21.7 in 4, 20.7 in 8.)
int shrink_planes(size_t T, int K, int dtype) {
  const int unit = dtype == CP4_DTYPE_F32 ? kUnit<F32> : kUnit<BF16>;
  const size_t tiles = std::max<size_t>(1, (T + 15) / 16);
  const size_t most = std::max(1, (K + unit - 1) / unit / 2);
  return (int)std::max<size_t>(1, std::min({((size_t)num_compute_units() + tiles - 1) / tiles, most, (size_t)64}));
}

hipError_t shrink_launch(const ShrinkArgs& a, int dtype, hipStream_t st) {
  if (dtype == CP4_DTYPE_F32) launch<F32>(a, st);
  else if (dtype == CP4_DTYPE_BF16) launch<BF16>(a, st);
  else launch<F16>(a, st);
  return hipGetLastError();
}

}  // namespace adapter
}  // namespace cp4
