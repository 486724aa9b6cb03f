// The shared projection with the adapters' second product beside it (include/cp4/adapter.h): a GEMM
// whose accumulators also take h B_a^T, for the adapters that the tile's rows have, before they are
// rounded and stored.
#include <algorithm>

#include "adapter.h"
#include "adapter_load.h"

namespace cp4 {
namespace adapter {
namespace {

// ---- any strides and alignment ------------------------------------------------------------

constexpr int kTile = 64, kDepth = 32;

// A tile of 64 x 64 outputs, 32 deep through the LDS, element by element; four waves of 32 x 32.
template <class T, bool NN>
__global__ __launch_bounds__(256) void general_kernel(const ProjectArgs a) {
  typedef typename T::raw Raw;
  constexpr int kRow = kDepth + 16 / sizeof(Raw);                    // (rows start on other banks)
  __shared__ Raw lz[kTile][kRow], lw[kTile][kRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const size_t t0 = (size_t)blockIdx.y * kTile;
  const int n0 = blockIdx.x * kTile, wm = 32 * (wave >> 1), wn = 32 * (wave & 1);
  const Raw* const z = static_cast<const Raw*>(a.z);
  const Raw* const w = static_cast<const Raw*>(a.w);
  f32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < a.K; k0 += kDepth) {
    Raw zr[8], wr[8];
    const int kc = threadIdx.x & 31, row0 = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = row0 + 8 * i, k = k0 + kc;
      zr[i] = t0 + row < a.T && k < a.K ? z[(t0 + row) * a.ldz + k] : Raw(0);
      if constexpr (NN) {
        const int kr = k0 + (threadIdx.x >> 6) + 4 * i, n = n0 + (threadIdx.x & 63);
        wr[i] = kr < a.K && n < a.N ? w[(size_t)kr * a.ldw + n] : Raw(0);
      } else {
        wr[i] = n0 + row < a.N && k < a.K ? w[(size_t)(n0 + row) * a.ldw + k] : Raw(0);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lz[row0 + 8 * i][kc] = zr[i];
      if constexpr (NN) lw[threadIdx.x & 63][(threadIdx.x >> 6) + 4 * i] = wr[i];
      else lw[row0 + 8 * i][kc] = wr[i];
    }
    __syncthreads();
    if constexpr (__is_same(T, F32)) {
#pragma unroll
      for (int q = 0; q < 8; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            acc[i][j] = mfma_f32(lz[wm + 16 * i + l][4 * q + g], lw[wn + 2 * l + j][4 * q + g], acc[i][j]);
    } else {
      u16x8 za[2], wb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        za[i] = *reinterpret_cast<const u16x8*>(&lz[wm + 16 * i + l][8 * g]);
        wb[i] = *reinterpret_cast<const u16x8*>(&lw[wn + 2 * l + i][8 * g]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_16<T>(za[i], wb[j], acc[i][j]);
    }
  }
  // the adapters of this wave's 32 rows
  int id = lane < 32 && t0 + wm + lane < a.T ? a.ids[t0 + wm + lane] : -1;
  if (id < 0 || id >= a.G) id = -1;
  expand_wave<T, NN, 2, 2>(a, id, [&](int i, int r, auto& x) { sum_planes(a, t0 + wm + 16 * i + l, r, x); }, false,
                           n0 + wn, 1, 0, acc);
  Raw* const y = static_cast<Raw*>(a.y);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = n0 + wn + 2 * l + j;
    if (n >= a.N) continue;
    const float b = a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const size_t t = t0 + wm + 16 * i + 4 * g + v;
        if (t < a.T) y[t * a.N + n] = T::narrow(acc[i][j][v] + b);
      }
  }
}

template <class T>
void general(const ProjectArgs& a, bool nn, hipStream_t st) {
  ProjectArgs p = a;
  const size_t most = (size_t)65535 * kTile;                         // (rows of one launch's grid)
  for (size_t t = 0; t < a.T; t += most) {
    p.T = std::min(most, a.T - t);
    p.z = static_cast<const typename T::raw*>(a.z) + t * a.ldz;
    p.h = a.h + t * a.Rp;
    p.ids = a.ids + t;
    p.y = static_cast<typename T::raw*>(a.y) + t * a.N;
    const dim3 grid((a.N + kTile - 1) / kTile, (unsigned)((p.T + kTile - 1) / kTile));
    if (nn) general_kernel<T, true><<<grid, 256, 0, st>>>(p);
    else general_kernel<T, false><<<grid, 256, 0, st>>>(p);
  }
}

}  // namespace

// A tile's worth of rows that the last round of tiles would be for can be cheaper on its own.
static size_t main_rows(size_t T, int K, int N, int dtype, bool nn) {
  const TilePlan all = tile_plan(T, K, N, dtype);
  size_t best = T;
  double least = all.cost;
  for (size_t tile : {256, 128}) {
    const size_t rest = T % tile;
    if (!rest || T <= 2 * tile) continue;
    // (the rest's own launches: some microseconds, and W once more)
    const bool rows = !nn && rows_plan(rest, K, N, dtype).splits;
    const double w = (double)K * N * (dtype == CP4_DTYPE_F32 ? 4 : 2) / 3.0e6;
    const double cost = tile_plan(T - rest, K, N, dtype).cost + 4.0 + (rows ? 6.0 + w : std::max(w, tile_plan(rest, K, N, dtype).cost));
    if (cost < least) {
      least = cost;
      best = T - rest;
    }
  }
  return best;
}

static size_t plan_bytes(size_t T, int K, int N, int dtype) {
  const RowsPlan rows = rows_plan(T, K, N, dtype);
  return std::max(tile_part_bytes(tile_plan(T, K, N, dtype), T, N),
                  rows.splits > 1 ? (size_t)rows.splits * T * N * 4 : 0);
}

size_t project_part_bytes(size_t T, int K, int N, int dtype) {
  size_t most = plan_bytes(T, K, N, dtype);
  for (bool nn : {false, true}) {
    const size_t main = main_rows(T, K, N, dtype, nn);
    if (main < T) most = std::max({most, plan_bytes(main, K, N, dtype), plan_bytes(T - main, K, N, dtype)});
  }
  return most;
}

bool project_sums_planes(const ProjectArgs& a, int dtype, bool nn) {
  return !nn && tile_supported(a, dtype, nn) && rows_plan(a.T, a.K, a.N, dtype).splits;
}

hipError_t project_launch(const ProjectArgs& a, float* part, int dtype, bool nn, hipStream_t st) {
  if (tile_supported(a, dtype, nn)) {
    const RowsPlan rows = nn ? RowsPlan{} : rows_plan(a.T, a.K, a.N, dtype);
    if (rows.splits) return rows_launch(a, rows, part, dtype, st);
    const size_t main = main_rows(a.T, a.K, a.N, dtype, nn);
    if (main < a.T) {
      const size_t e = dtype == CP4_DTYPE_F32 ? 4 : 2;
      ProjectArgs p = a, q = a;
      p.T = main;
      q.T = a.T - main;
      q.z = static_cast<const char*>(a.z) + main * a.ldz * e;
      q.h = a.h + main * a.Rp;
      q.ids = a.ids + main;
      q.y = static_cast<char*>(a.y) + main * a.N * e;
      if (const hipError_t err = tile_launch(p, tile_plan(p.T, p.K, p.N, dtype), part, dtype, nn, st)) return err;
      const RowsPlan few = nn ? RowsPlan{} : rows_plan(q.T, q.K, q.N, dtype);
      if (few.splits) return rows_launch(q, few, part, dtype, st);
      return tile_launch(q, tile_plan(q.T, q.K, q.N, dtype), part, dtype, nn, st);
    }
    return tile_launch(a, tile_plan(a.T, a.K, a.N, dtype), part, dtype, nn, st);
  }
  if (dtype == CP4_DTYPE_F32) general<F32>(a, nn, st);
  else if (dtype == CP4_DTYPE_BF16) general<BF16>(a, nn, st);
  else general<F16>(a, nn, st);
  return hipGetLastError();
}

}  // namespace adapter
}  // namespace cp4
