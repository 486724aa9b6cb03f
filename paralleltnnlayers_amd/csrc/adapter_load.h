// Device side of the adapters' kernels: operands from memory in registers, at any alignment, and turned there.
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

// 16 bytes from any element's address: one load, whatever the alignment.
template <class Raw>
__device__ __forceinline__ u32x4 load_16(const Raw* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// `count` (may be <= 0 or beyond n) values of p, zero behind.
template <int n, class Raw>
__device__ __forceinline__ void load_some(const Raw* p, int count, Raw (&v)[n]) {
  if (count >= n) {
    __builtin_memcpy(v, p, n * sizeof(Raw));
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = i < count ? p[i] : Raw(0);
  }
}
template <class Raw>
__device__ __forceinline__ u32x4 load_16(const Raw* p, int count) {
  Raw v[16 / sizeof(Raw)];
  load_some(p, count, v);
  return __builtin_bit_cast(u32x4, v);
}

}  // namespace adapter
}  // namespace cp4
#endif
