// Element types in memory of kernels that compute in fp32.
#ifndef CP4_VALUE_TYPES_H
#define CP4_VALUE_TYPES_H

#include <hip/hip_runtime.h>

namespace cp4 {

struct F32 {
  typedef float raw;
  static __device__ __forceinline__ float widen(float v) { return v; }
  static __device__ __forceinline__ float narrow(float v) { return v; }
};
struct BF16 {
  typedef unsigned short raw;
  static __device__ __forceinline__ float widen(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned short narrow(float v) {
    return __builtin_bit_cast(unsigned short, (__bf16)v);
  }
};
struct F16 {
  typedef unsigned short raw;
  static __device__ __forceinline__ float widen(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ unsigned short narrow(float v) {
    return __builtin_bit_cast(unsigned short, (_Float16)v);
  }
};

}  // namespace cp4
#endif
