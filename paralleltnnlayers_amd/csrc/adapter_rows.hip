// The shared projection of up to 64 tokens (include/cp4/adapter.h): bound by reading W once, so nothing
// stands between memory and the matrix cores.
//
// A workgroup takes 16 columns (rows of W) of all tokens; its eight waves share the inputs, a cache
// line of every row a turn and four turns' loads ahead of their products, which keeps 64 KB of W under way
// on every compute unit.  x comes from the L2 again for every workgroup.  Where there are few columns the inputs
// are split over workgroups too.  The adapters' parts are shared out over the waves; all sums meet in the LDS.
#include <algorithm>

#include "adapter.h"
#include "adapter_load.h"

namespace cp4 {
namespace adapter {
namespace {

constexpr int kWaves = 8;

struct RowsArgs {
  ProjectArgs p;
  float* part;            // [splits][T][N], or null: y
  int splits;
};

template <class T, int MB>
__global__ __launch_bounds__(64 * kWaves, 2) void rows_kernel(const RowsArgs ra) {
  typedef typename T::raw Raw;
  constexpr int n = 16 / sizeof(Raw), U = 128 / sizeof(Raw), NB = 1, kRow = 16 * NB + 4, kAhead = 4;
  constexpr int kSum = kWaves * 16 * MB * kRow, kH = 16 * MB * 256;
  __shared__ __attribute__((aligned(16))) float lds[kSum > kH ? kSum : kH];
  float* const hl = lds;                                             // [T][Rp], and then ...
  float* const sum = lds;                                            // ... [kWaves][16 MB][kRow]
  const ProjectArgs& a = ra.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const int rows = (int)a.T, n0 = blockIdx.x * 16 * NB, split = blockIdx.y;
  int id = lane < rows ? a.ids[lane] : -1;
  if (id >= a.G) id = -1;
  const bool adapters = split == 0 && __ballot(id >= 0);
  if (adapters)
    for (int i = threadIdx.x * 4; i < rows * a.Rp; i += 64 * kWaves * 4) {
      float x[4] = {};
      sum_planes(a, 0, i, x);
      *reinterpret_cast<f32x4*>(hl + i) = f32x4{x[0], x[1], x[2], x[3]};
    }
  const Raw *z[MB], *w[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) z[i] = static_cast<const Raw*>(a.z) + min(16 * i + l, rows - 1) * a.ldz + n * g;
#pragma unroll
  for (int j = 0; j < NB; ++j) w[j] = static_cast<const Raw*>(a.w) + min(n0 + NB * l + j, a.N - 1) * a.ldw + n * g;
  const int units = (a.K + U - 1) / U, shares = kWaves * ra.splits, share = split * kWaves + wave;
  const int first = (int)((long)units * share / shares), last = (int)((long)units * (share + 1) / shares);
  const int whole = min(last, a.K / U);

  f32x4 acc[MB][NB] = {};
  auto multiply = [&](const u32x4 (&zv)[MB][2], const u32x4 (&wv)[NB][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (__is_same(T, F32)) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[i][j] = mfma_f32(__uint_as_float(zv[i][h][q]), __uint_as_float(wv[j][h][q]), acc[i][j]);
          } else {
            acc[i][j] = mfma_16<T>(__builtin_bit_cast(u16x8, zv[i][h]), __builtin_bit_cast(u16x8, wv[j][h]), acc[i][j]);
          }
        }
  };
  auto ahead = [&](int u, auto count) __attribute__((always_inline)) {
    constexpr int c = decltype(count)::value;
    u32x4 zv[c][MB][2], wv[c][NB][2];
#pragma unroll
    for (int e = 0; e < c; ++e) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) wv[e][j][h] = reinterpret_cast<const u32x4*>(w[j] + (size_t)(u + e) * U)[4 * h];
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) zv[e][i][h] = reinterpret_cast<const u32x4*>(z[i] + (size_t)(u + e) * U)[4 * h];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < c; ++e) multiply(zv[e], wv[e]);
  };
  int u = first;
  for (; u + kAhead <= whole; u += kAhead) ahead(u, std::integral_constant<int, kAhead>());
  for (; u < whole; ++u) ahead(u, std::integral_constant<int, 1>());
  if (u < last) {                                                    // (the inputs' rest)
    u32x4 zv[MB][2], wv[NB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool there = u * U + n * (4 * h + g) < a.K;
#pragma unroll
      for (int i = 0; i < MB; ++i) zv[i][h] = there ? reinterpret_cast<const u32x4*>(z[i] + (size_t)u * U)[4 * h] : u32x4{};
#pragma unroll
      for (int j = 0; j < NB; ++j) wv[j][h] = there ? reinterpret_cast<const u32x4*>(w[j] + (size_t)u * U)[4 * h] : u32x4{};
    }
    multiply(zv, wv);
  }
  __syncthreads();
  if (adapters)
    expand_wave<T, false, MB, NB>(
        a, id,
        [&](int i, int r, auto& x) {
#pragma unroll
          for (int q = 0; q < (int)(sizeof(x) / 4); q += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(hl + (16 * i + l) * a.Rp + r + q);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[q + e] = v[e];
          }
        },
        ((size_t)a.f & 15) == 0 && a.R % n == 0, n0, kWaves, wave, acc);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int j = 0; j < NB; ++j) sum[(wave * 16 * MB + 16 * i + 4 * g + v) * kRow + NB * l + j] = acc[i][j][v];
  __syncthreads();
  for (int o = threadIdx.x; o < rows * 16 * NB; o += 64 * kWaves) {
    const int row = o / (16 * NB), col = o % (16 * NB);
    if (n0 + col >= a.N) continue;
    float x = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) x += sum[(k * 16 * MB + row) * kRow + col];
    const size_t at = (size_t)row * a.N + n0 + col;
    if (ra.part) ra.part[(size_t)split * a.T * a.N + at] = x;
    else static_cast<Raw*>(a.y)[at] = T::narrow(a.bias ? x + a.bias[n0 + col] : x);
  }
}

template <class T, int MB>
void launch(const RowsArgs& r, hipStream_t st) {
  rows_kernel<T, MB><<<dim3((r.p.N + 15) / 16, r.splits), 64 * kWaves, 0, st>>>(r);
}
template <class T>
void launch_rows(const RowsArgs& r, hipStream_t st) {
  const int mb = (int)(r.p.T + 15) / 16;
  if (mb == 1) launch<T, 1>(r, st);
  else if (mb == 2) launch<T, 2>(r, st);
  if constexpr (sizeof(typename T::raw) == 2) {
    if (mb == 3) launch<T, 3>(r, st);
    else if (mb == 4) launch<T, 4>(r, st);
  }
}

}  // namespace

RowsPlan rows_plan(size_t T, int K, int N, int dtype) {
  RowsPlan p{};
  if (T > (dtype == CP4_DTYPE_F32 ? 32 : 64)) return p;
  const int units = (K * (dtype == CP4_DTYPE_F32 ? 4 : 2) + 127) / 128, tiles = (N + 15) / 16;
  p.splits = std::max(1, std::min(num_compute_units() / tiles, units / (2 * kWaves)));
  if (p.splits < 4) p.splits = 1;
  return p;
}

hipError_t rows_launch(const ProjectArgs& a, const RowsPlan& plan, float* part, int dtype, hipStream_t st) {
  RowsArgs r{};
  r.p = a;
  r.part = plan.splits > 1 ? part : nullptr;
  r.splits = plan.splits;
  if (dtype == CP4_DTYPE_F32) launch_rows<F32>(r, st);
  else if (dtype == CP4_DTYPE_BF16) launch_rows<BF16>(r, st);
  else launch_rows<F16>(r, st);
  if (const hipError_t e = hipGetLastError()) return e;
  return plan.splits > 1 ? parts_join(part, a.bias, a.y, a.T, a.N, plan.splits, dtype, st) : hipSuccess;
}

}  // namespace adapter
}  // namespace cp4
