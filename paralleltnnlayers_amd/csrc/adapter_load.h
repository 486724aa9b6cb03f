// Device side of the adapters' kernels: operands in registers and the adapters' part of an output tile.
#ifndef CP4_ADAPTER_LOAD_H
#define CP4_ADAPTER_LOAD_H

#include "adapter.h"

namespace cp4 {
namespace adapter {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// 8 rows (depths) of NB columns in 16 bits -> NB columns of 8 depths.
template <int NB>
__device__ __forceinline__ void turn(const unsigned (&in)[8][NB / 2], u16x8 (&out)[NB]) {
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    u32x4 d;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      d[q] = __builtin_amdgcn_perm(in[2 * q + 1][j / 2], in[2 * q][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
    out[j] = __builtin_bit_cast(u16x8, d);
  }
}

// `count` (may be <= 0 or beyond n) values of p, zero behind; vec: p is on a 16-byte boundary.
template <int n, class Raw>
__device__ __forceinline__ void load_some(const Raw* p, int count, bool vec, Raw (&v)[n]) {
  if (vec && count >= n) {
    constexpr int each = 16 / sizeof(Raw);
    if constexpr (n >= each) {
#pragma unroll
      for (int i = 0; i < n / each; ++i) {
        const u32x4 d = reinterpret_cast<const u32x4*>(p)[i];
        __builtin_memcpy(&v[i * each], &d, 16);
      }
      return;
    } else if constexpr (n * sizeof(Raw) == 8) {
      const u32x2 d = *reinterpret_cast<const u32x2*>(p);
      __builtin_memcpy(&v[0], &d, 8);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < n; ++i) v[i] = i < count ? p[i] : Raw(0);
}

// Adds h F_a^T to a wave's MB x NB blocks, for each adapter of its rows.  id: lane i's is row i's adapter (-1:
// none); h(i, r): this lane's pointer to h's values from rank r on of row 16 i + (lane & 15), only asked for
// rows that have an adapter; f: what column n0 + NB * (lane & 15) + j has of rank r lies at n * fn + r * fr of
// each adapter's R * N values.  `mod`, `which`: of the adapters in turn, this wave adds every mod-th.
//
// 16-bit types: depth 0 .. 15 of a product are the first parts of h, 16 .. 31 what they leave, against F_a twice
// (f16: F_a in two parts as well, in two products).  All rows are multiplied with each adapter, and the rows
// that are not its own keep what they had: an infinity or a NaN in one adapter is no other token's.
template <class T, bool NN, int MB, int NB, class H>
__device__ __forceinline__ void expand_wave(const ProjectArgs& a, int id, H h, bool vec, int n0, int mod, int which,
                                            f32x4 (&acc)[MB][NB]) {
  typedef typename T::raw Raw;
  const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4, n = n0 + NB * l;
  constexpr bool kF32 = __is_same(T, F32);
  const unsigned long long have = __ballot(id >= 0);
  if (!have) return;
  for (int r0 = 0; r0 < a.R; r0 += 16) {
    // fp32: depth 4 g + q in product q; 16 bits: ranks 8 (g & 1) + q, first parts for g < 2
    const int rl = r0 + (kF32 ? 4 * g : 8 * (g & 1));
    constexpr int kOwn = kF32 ? 4 : 8;
    float hv[MB][kOwn];
    u16x8 ha[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
      for (int q = 0; q < kOwn; ++q) hv[i][q] = 0.0f;
      if (have >> (16 * i + l) & 1) h(i, rl, hv[i]);
      if constexpr (!kF32) {
        u16x8 hi, lo;
        two_parts(hv[i], hi, lo);
        ha[i] = g < 2 ? hi : lo;
      }
    }
    Adapters todo(id);
    int ad, turn_of = 0;
    unsigned long long whose;
    while (todo.take(ad, whose)) {
      if ((turn_of++ & (mod - 1)) != which) continue;
      const Raw* const f = static_cast<const Raw*>(a.f) + (size_t)ad * a.R * a.N;
      Raw fv[NB][kOwn];                                              // [column][rank]
      if constexpr (NN) {
        Raw fr[kOwn][NB];
#pragma unroll
        for (int q = 0; q < kOwn; ++q)
          load_some<NB>(f + (size_t)(rl + q) * a.fr + n, rl + q < a.R ? a.N - n : 0, vec, fr[q]);
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int q = 0; q < kOwn; ++q) fv[j][q] = fr[q][j];
      } else {
#pragma unroll
        for (int j = 0; j < NB; ++j)
          load_some<kOwn>(f + (size_t)(n + j) * a.fn + rl, n + j < a.N ? a.R - rl : 0, vec, fv[j]);
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        u16x8 fh = {}, fl = {};
        if constexpr (__is_same(T, F16)) {
          float x[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) x[q] = F16::widen(fv[j][q]);
          two_parts(x, fh, fl);
        } else if constexpr (!kF32) {
#pragma unroll
          for (int q = 0; q < 8; ++q) fh[q] = fv[j][q];
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const unsigned rows = (unsigned)(whose >> (16 * i)) & 0xffffu;
          if (!rows) continue;
          f32x4 d = acc[i][j];
          if constexpr (kF32) {
#pragma unroll
            for (int q = 0; q < 4; ++q) d = mfma_f32(hv[i][q], fv[j][q], d);
          } else {
            if constexpr (__is_same(T, F16)) d = mfma_bf16(ha[i], fl, d);
            d = mfma_bf16(ha[i], fh, d);
          }
          if (rows == 0xffffu) {
            acc[i][j] = d;
          } else {
#pragma unroll
            for (int v = 0; v < 4; ++v)
              if (rows >> (4 * g + v) & 1) acc[i][j][v] = d[v];
          }
        }
      }
    }
  }
}
// h's values in memory: the sum of its planes.
template <int n>
__device__ __forceinline__ void sum_planes(const ProjectArgs& a, size_t row, int r, float (&x)[n]) {
  const float* p = a.h + row * a.Rp + r;
  for (int s = 0; s < a.planes; ++s, p += a.plane)
#pragma unroll
    for (int q = 0; q < n; q += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(p + q);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[q + e] += v[e];
    }
}

}  // namespace adapter
}  // namespace cp4
#endif
