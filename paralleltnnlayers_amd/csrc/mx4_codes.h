// Device side of microscaled 4-bit floating point (include/cp4/mx4.h): codes to values.
#ifndef CP4_MX4_CODES_H
#define CP4_MX4_CODES_H

#include <hip/hip_runtime.h>

#include "value_types.h"

namespace cp4 {
namespace mx4 {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// A scale's byte as the conversions take it: they read a float's exponent alone, 0 as 2^-127 and 255 as NaN.
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Eight codes to eight values of a type.
template <class T>
__device__ __forceinline__ void values(unsigned codes, float scale, typename T::raw (&v)[8]) {
  if constexpr (__is_same(T, F32)) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1),
                c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
  } else if constexpr (__is_same(T, BF16)) {
    const bf16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)};
    __builtin_memcpy(v, p, 16);
  } else {
    const f16x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1),
                        __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3)};
    __builtin_memcpy(v, p, 16);
  }
}

}  // namespace mx4
}  // namespace cp4
#endif
