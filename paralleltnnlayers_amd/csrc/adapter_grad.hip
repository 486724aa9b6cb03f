// The adapters' gradients (include/cp4/adapter.h): for each adapter a sum over its tokens of the outer products
// of an fp32 row of h or dh and a row of dy or x.
#include <algorithm>

#include "adapter.h"

namespace cp4 {
namespace adapter {
namespace {

constexpr int kCols = 64, kList = 2048;

// A workgroup sums 64 columns of one adapter over one range of tokens, 64 ranks at a time: it picks the
// adapter's tokens out of the range, in order, into a list in the LDS and goes through that 32 at a time;
// each wave has 16 columns.  Tokens of other adapters cost a look at their id.
template <class T>
__global__ __launch_bounds__(256) void general_kernel(const GradArgs a) {
  typedef typename T::raw Raw;
  __shared__ int list[kList + 32];
  __shared__ int counts[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const int ad = blockIdx.y % a.G, split = blockIdx.y / a.G, r0 = blockIdx.z * 64;
  const int c = blockIdx.x * kCols + 16 * wave + l, ranks = min(64, a.Rp - r0) / 16;
  const size_t per = (a.T + a.splits - 1) / a.splits;
  const size_t first = min(a.T, split * per), last = min(a.T, first + per);
  const Raw* const z = static_cast<const Raw*>(a.z);
  auto row_of = [&](size_t t, int r) {
    float x = 0.0f;
    for (int s = 0; s < a.planes; ++s) x += a.p[(s * a.T + t) * a.Rp + r];
    return x;
  };
  f32x4 acc[4] = {};
  for (size_t w0 = first; w0 < last; w0 += kList) {
    const int here = (int)min((size_t)kList, last - w0);
    int n = 0;
    __syncthreads();                                                 // (the list is read no more)
    for (int i0 = 0; i0 < here; i0 += 256) {
      const int i = i0 + (int)threadIdx.x;
      const bool mine = i < here && a.ids[w0 + i] == ad;
      const unsigned long long m = __ballot(mine);
      if (lane == 0) counts[wave] = __popcll(m);
      __syncthreads();
      int at = n;
      for (int w = 0; w < 4; ++w) {
        if (w < wave) at += counts[w];
        n += counts[w];
      }
      if (mine) list[at + __popcll(m & ((1ull << lane) - 1))] = i;
      __syncthreads();
    }
    if (threadIdx.x < 32) list[n + threadIdx.x] = -1;
    __syncthreads();
    for (int b = 0; b < n; b += 32) {
      if constexpr (__is_same(T, F32)) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int t = list[b + 4 * q + g];
          const float zv = t >= 0 && c < a.C ? z[(w0 + t) * a.ldz + c] : 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < ranks) acc[i] = mfma_f32(t >= 0 ? row_of(w0 + t, r0 + 16 * i + l) : 0.0f, zv, acc[i]);
        }
      } else {
        u16x8 zv = {};
        int t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t[j] = list[b + 8 * g + j];
          if (t[j] >= 0 && c < a.C) zv[j] = z[(w0 + t[j]) * a.ldz + c];
        }
        u16x8 zh = zv, zl = {};
        if constexpr (__is_same(T, F16)) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = F16::widen(zv[j]);
          two_parts(x, zh, zl);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < ranks) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = t[j] >= 0 ? row_of(w0 + t[j], r0 + 16 * i + l) : 0.0f;
            u16x8 ph, pl;
            two_parts(x, ph, pl);
            if constexpr (__is_same(T, F16)) acc[i] = mfma_bf16(ph, zl, acc[i]);
            acc[i] = mfma_bf16(pl, zh, acc[i]);
            acc[i] = mfma_bf16(ph, zh, acc[i]);
          }
      }
    }
  }
  if (c >= a.C) return;
  const size_t size = (size_t)a.R * a.C;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < ranks)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = r0 + 16 * i + 4 * g + v;
        if (r >= a.R) continue;
        const size_t at = (size_t)ad * size + (size_t)r * a.outr + (size_t)c * a.outc;
        if (a.splits > 1) a.part[(size_t)split * a.G * size + at] = acc[i][v];
        else static_cast<Raw*>(a.out)[at] = T::narrow(acc[i][v]);
      }
}

// The ranges' sums, in their order.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const float* part, void* out, size_t n, int splits) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float x = part[i];
  for (int s = 1; s < splits; ++s) x += part[(size_t)s * n + i];
  static_cast<typename T::raw*>(out)[i] = T::narrow(x);
}

template <class T>
void launch(const GradArgs& a, hipStream_t st) {
  const dim3 grid((a.C + kCols - 1) / kCols, a.G * a.splits, (a.Rp + 63) / 64);
  general_kernel<T><<<grid, 256, 0, st>>>(a);
  if (a.splits > 1) {
    const size_t n = (size_t)a.G * a.R * a.C;
    join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a.part, a.out, n, a.splits);
  }
}

}  // namespace

// Ranges of tokens: enough workgroups for every compute unit to have a few, none of fewer than 256 tokens.
int grad_splits(size_t T, int C, int R, int G) {
  const size_t wgs = (size_t)((C + kCols - 1) / kCols) * G * ((R + 63) / 64);
  const size_t want = (4 * (size_t)num_compute_units() + wgs - 1) / wgs;
  const size_t most = std::min<size_t>((T + 255) / 256, 65535 / G);
  return (int)std::max<size_t>(1, std::min(want, most));
}

hipError_t grad_launch(const GradArgs& a, int dtype, hipStream_t st) {
  if (dtype == CP4_DTYPE_F32) launch<F32>(a, st);
  else if (dtype == CP4_DTYPE_BF16) launch<BF16>(a, st);
  else launch<F16>(a, st);
  return hipGetLastError();
}

}  // namespace adapter
}  // namespace cp4
