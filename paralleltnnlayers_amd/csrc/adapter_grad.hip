// The adapters' gradients (include/cp4/adapter.h): for each adapter a sum over its tokens of the outer products
// of an fp32 row of h or dh and a row of dy or x: a product as deep as the adapter has tokens and as high as
// it has ranks, bound by reading x and dy once.
//
// Both gradients of a call are one launch.  A workgroup takes 128 columns of one adapter.  It picks the adapter's
// tokens out of 8192 ids at a time into a list in the LDS (in order, so that sums do not change from call to call);
// its eight waves share the list, 32 tokens (fp32: 16) a turn, straight from memory: a lane reads eight consecutive
// columns of each of its tokens' rows and turns them in registers into eight column blocks' operands.  The waves' sums
// meet in the LDS at the end.  Rows of h enter as two bfloat16 parts, and so do half-precision rows of dy and x
// (exactly).  Few workgroups (few adapters, short rows): the tokens are split over workgroups too, and a
// second launch adds the parts up in their order.
//
// Measured: 8192 tokens bf16, 4096 and 4096 columns, rank 16, 8 adapters: 46 us, 2.9 TB/s, bound by the loads a wave has
// in flight and by turning them; 1031 tokens f16, 2048 and 2816 columns, rank 64: 22 us, bound by the products of two times two parts.
#include <algorithm>

#include "adapter.h"
#include "adapter_load.h"

namespace cp4 {
namespace adapter {
namespace {

// Both gradients of a call.
struct GradPair {
  GradArgs g[2];
  int tiles;              // workgroups along the first one's columns
};

constexpr int kCols = 128, kWindow = 8192, kWaves = 8, kPad = 4;

template <class T, int RB>
__global__ __launch_bounds__(64 * kWaves, 2) void grad_kernel(const GradPair pair) {
  const GradArgs& a = pair.g[(int)blockIdx.x >= pair.tiles];
  typedef typename T::raw Raw;
  constexpr bool kF32 = __is_same(T, F32);
  constexpr int kTurn = kF32 ? 16 : 32, kOwn = kTurn / 4;            // tokens of a turn, and of a lane
  __shared__ __attribute__((aligned(16))) union {
    unsigned short list[kWindow + 64];
    float sum[kWaves][16][kCols + kPad];
  } lds;
  __shared__ int counts[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const int ad = blockIdx.y % a.G, split = blockIdx.y / a.G, r0 = blockIdx.z * 16 * RB;
  const int c0 = (blockIdx.x - ((int)blockIdx.x >= pair.tiles ? pair.tiles : 0)) * kCols, c = c0 + 8 * l;
  const size_t per = (a.T + a.splits - 1) / a.splits;
  const size_t first = min(a.T, split * per), last = min(a.T, first + per);
  const Raw* const z = static_cast<const Raw*>(a.z) + min(c, a.C - 1);
  const int cols = a.C - c;
  f32x4 acc[RB][8] = {};
  for (size_t w0 = first; w0 < last; w0 += kWindow) {
    // the list: each wave looks through its eighth of the window
    const int here = (int)min((size_t)kWindow, last - w0), share = (here + 8 * 64 - 1) / (8 * 64);   // (64s of a wave)
    unsigned long long mine[kWindow / 512];
    int n_wave = 0;
#pragma unroll
    for (int i = 0; i < kWindow / 512; ++i) {
      const int at = (wave * share + i) * 64 + lane;
      mine[i] = __ballot(i < share && at < here && a.ids[w0 + at] == ad);
      n_wave += __popcll(mine[i]);
    }
    __syncthreads();                                                 // (nobody reads the last list)
    if (lane == 0) counts[wave] = n_wave;
    __syncthreads();
    int at = 0, n = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) at += counts[w];
      n += counts[w];
    }
    if (!n) continue;
#pragma unroll
    for (int i = 0; i < kWindow / 512; ++i) {
      if (mine[i] >> lane & 1)
        lds.list[at + __popcll(mine[i] & ((1ull << lane) - 1))] = (unsigned short)((wave * share + i) * 64 + lane);
      at += __popcll(mine[i]);
    }
    __syncthreads();
    // (a turn's missing tokens are its last one again, times zero)
    const int turns = (n + kTurn - 1) / kTurn, each = (turns + kWaves - 1) / kWaves;
    const int end = min(turns, (wave + 1) * each);
    const bool whole = c0 + kCols <= a.C;
    for (int b = wave * each; b < end; ++b) {
      int t[kOwn];
      float p[RB][kOwn];
      Raw x[kOwn][8];
#pragma unroll
      for (int q = 0; q < kOwn; ++q) {
        const int i = b * kTurn + kOwn * g + q;
        t[q] = lds.list[min(i, n - 1)];
      }
      if (whole) {
#pragma unroll
        for (int q = 0; q < kOwn; ++q) __builtin_memcpy(x[q], z + (w0 + t[q]) * a.ldz, sizeof(x[q]));
      } else {
#pragma unroll
        for (int q = 0; q < kOwn; ++q) load_some(z + (w0 + t[q]) * a.ldz, cols, x[q]);
      }
#pragma unroll
      for (int q = 0; q < kOwn; ++q) {
        const bool there = b * kTurn + kOwn * g + q < n;
        const float* const row = a.p + (w0 + t[q]) * a.Rp + r0 + l;
#pragma unroll
        for (int i = 0; i < RB; ++i) p[i][q] = there && r0 + 16 * i < a.Rp ? row[16 * i] : 0.0f;
      }
      if constexpr (kF32) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < RB; ++i) acc[i][j] = mfma_f32(p[i][q], x[q][j], acc[i][j]);
      } else {
        unsigned in[8][4];
#pragma unroll
        for (int q = 0; q < 8; ++q) __builtin_memcpy(in[q], x[q], 16);
        u16x8 zv[8], ph[RB], pl[RB];
        turn<8>(in, zv);
#pragma unroll
        for (int i = 0; i < RB; ++i) two_parts(p[i], ph[i], pl[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          u16x8 zh = zv[j], zl = {};
          if constexpr (__is_same(T, F16)) {
            float f[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = F16::widen(zv[j][q]);
            two_parts(f, zh, zl);
          }
#pragma unroll
          for (int i = 0; i < RB; ++i) {
            if constexpr (__is_same(T, F16)) acc[i][j] = mfma_bf16(ph[i], zl, acc[i][j]);
            acc[i][j] = mfma_bf16(pl[i], zh, acc[i][j]);
            acc[i][j] = mfma_bf16(ph[i], zh, acc[i][j]);
          }
        }
      }
    }
  }
  const size_t size = (size_t)a.R * a.C;
#pragma unroll
  for (int i = 0; i < RB; ++i) {
    if (r0 + 16 * i >= a.R) break;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int j = 0; j < 8; j += 4)
        *reinterpret_cast<f32x4*>(&lds.sum[wave][4 * g + v][8 * l + j]) =
            f32x4{acc[i][j][v], acc[i][j + 1][v], acc[i][j + 2][v], acc[i][j + 3][v]};
    __syncthreads();
    for (int o = threadIdx.x; o < 16 * kCols; o += 64 * kWaves) {    // (in the output's order)
      const int r = a.outc == 1 ? o / kCols : o % 16, col = a.outc == 1 ? o % kCols : o / 16;
      if (r0 + 16 * i + r >= a.R || c0 + col >= a.C) continue;
      float x = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) x += lds.sum[w][r][col];
      const size_t at = (size_t)ad * size + (size_t)(r0 + 16 * i + r) * a.outr + (size_t)(c0 + col) * a.outc;
      if (a.splits > 1) a.part[(size_t)split * a.G * size + at] = x;
      else static_cast<Raw*>(a.out)[at] = T::narrow(x);
    }
  }
}

// The ranges' sums, in their order.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const GradPair pair, size_t n0, size_t n1) {
  size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const bool second = i >= n0;
  if (second) i -= n0;
  const size_t n = second ? n1 : n0;
  if (i >= n) return;
  const float* const part = second ? pair.g[1].part : pair.g[0].part;
  float x = part[i];
  for (int s = 1; s < pair.g[0].splits; ++s) x += part[(size_t)s * n + i];
  static_cast<typename T::raw*>(second ? pair.g[1].out : pair.g[0].out)[i] = T::narrow(x);
}

template <class T>
void launch(const GradPair& p, hipStream_t st) {
  const GradArgs &a = p.g[0], &b = p.g[1];
  const int rb = a.Rp <= 16 ? 1 : a.Rp <= 32 ? 2 : 4;
  const dim3 grid(p.tiles + (b.C + kCols - 1) / kCols, a.G * a.splits, (a.Rp + 16 * rb - 1) / (16 * rb));
  if (rb == 1) grad_kernel<T, 1><<<grid, 64 * kWaves, 0, st>>>(p);
  else if (rb == 2) grad_kernel<T, 2><<<grid, 64 * kWaves, 0, st>>>(p);
  else grad_kernel<T, 4><<<grid, 64 * kWaves, 0, st>>>(p);
  if (a.splits > 1) {
    const size_t each = (size_t)a.G * a.R, n = each * (a.C + b.C);
    join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(p, each * a.C, each * b.C);
  }
}

}  // namespace

// Ranges of tokens: a workgroup for each compute unit, 256 tokens an adapter and range or more on the average.  (65536
// tokens, one adapter, 1024 + 1024 columns: 604 us in one range, 122 in 16, 132 in 32; 1031 tokens of 8 adapters, 2048 + 2816
// columns, rank 64: 41 us in one, 51 in two.)
int grad_splits(size_t T, int C0, int C1, int R, int G) {
  const size_t wgs = (size_t)((C0 + kCols - 1) / kCols + (C1 + kCols - 1) / kCols) * G * ((R + 63) / 64);
  const size_t want = num_compute_units() / wgs, most = std::min<size_t>(T / G / 256, 65535 / G);
  return (int)std::max<size_t>(1, std::min(want, most));
}

hipError_t grad_launch(const GradArgs& a, const GradArgs& b, int dtype, hipStream_t st) {
  const GradPair p{{a, b}, (a.C + kCols - 1) / kCols};
  if (dtype == CP4_DTYPE_F32) launch<F32>(p, st);
  else if (dtype == CP4_DTYPE_BF16) launch<BF16>(p, st);
  else launch<F16>(p, st);
  return hipGetLastError();
}

}  // namespace adapter
}  // namespace cp4
