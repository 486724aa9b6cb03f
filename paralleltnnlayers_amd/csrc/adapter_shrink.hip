// h = scale A_a x, token by token (include/cp4/adapter.h): a product with as few columns as the adapters
// have ranks, bound by reading x and the adapters in use once.
#include <algorithm>

#include "adapter.h"

namespace cp4 {
namespace adapter {
namespace {

constexpr int kWaves = 4;

// Any strides and alignment: a workgroup takes 16 tokens; its waves share the inputs in steps of 32 and
// go through the adapters that these tokens have, all sixteen rows against each, so that a batch in which
// every token has its own reads each adapter once and one in which all have the same does a single
// product.
template <class T>
__global__ __launch_bounds__(64 * kWaves) void general_kernel(const ShrinkArgs a) {
  typedef typename T::raw Raw;
  __shared__ float sum[kWaves][16][17];
  __shared__ int own[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const size_t t0 = (size_t)blockIdx.x * 16;
  const int rows = (int)min((size_t)16, a.T - t0);
  int id = lane < rows ? a.ids[t0 + lane] : -1;
  if (id < 0 || id >= a.G) id = -1;
  const Raw* const z = static_cast<const Raw*>(a.z) + (t0 + min(l, rows - 1)) * a.ldz;
  if (threadIdx.x < 16) own[lane] = id;
  __syncthreads();
  for (int i = threadIdx.x; i < rows * a.Rp; i += 64 * kWaves)       // tokens without an adapter
    if (own[i / a.Rp] < 0) a.h[t0 * a.Rp + i] = 0.0f;
  Adapters todo(id);
  int ad;
  unsigned long long whose;
  while (todo.take(ad, whose)) {
    const Raw* const f = static_cast<const Raw*>(a.f) + (size_t)ad * a.R * a.K;
    const float s = a.scale ? a.scale[ad] : 1.0f;
    for (int r0 = 0; r0 < a.Rp; r0 += 16) {
      const int r = r0 + l;
      const Raw* const fr = f + (size_t)min(r, a.R - 1) * a.fr;
      f32x4 acc = {};
      for (int k0 = 32 * wave; k0 < a.K; k0 += 32 * kWaves) {
        if constexpr (__is_same(T, F32)) {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int k = k0 + 4 * q + g;
            const float zv = k < a.K ? z[k] : 0.0f;
            const float fv = k < a.K && r < a.R ? fr[(size_t)k * a.fk] : 0.0f;
            acc = mfma_f32(zv, fv, acc);
          }
        } else {
          u16x8 zv = {}, fv = {};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int k = k0 + 8 * g + j;
            if (k < a.K) zv[j] = z[k];
            if (k < a.K && r < a.R) fv[j] = fr[(size_t)k * a.fk];
          }
          acc = mfma_16<T>(zv, fv, acc);
        }
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < 4; ++v) sum[wave][4 * g + v][l] = acc[v];
      __syncthreads();
      const int row = threadIdx.x >> 4, col = threadIdx.x & 15;      // (256 threads: one sum each)
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) x += sum[w][row][col];
      if (whose >> row & 1) a.h[(t0 + row) * a.Rp + r0 + col] = r0 + col < a.R ? x * s : 0.0f;
    }
  }
}

}  // namespace

hipError_t shrink_launch(const ShrinkArgs& a, int dtype, hipStream_t st) {
  const unsigned grid = (unsigned)((a.T + 15) / 16);
  if (dtype == CP4_DTYPE_F32) general_kernel<F32><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (dtype == CP4_DTYPE_BF16) general_kernel<BF16><<<grid, 64 * kWaves, 0, st>>>(a);
  else general_kernel<F16><<<grid, 64 * kWaves, 0, st>>>(a);
  return hipGetLastError();
}

}  // namespace adapter
}  // namespace cp4
