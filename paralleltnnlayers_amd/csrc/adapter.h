// Interface between the adapters' C ABI (adapter_capi.hip) and their kernels.
#ifndef CP4_ADAPTER_INTERNAL_H
#define CP4_ADAPTER_INTERNAL_H

#include <hip/hip_runtime.h>

#include "cp4/adapter.h"
#include "cp4_internal.h"
#include "value_types.h"

namespace cp4 {
namespace adapter {

// h[t][r] = scale_a sum_k z[t][k] F_a(r, k), F_a(r, k) at f + a * R * K + r * fr + k * fk.
// h has rows of Rp values (R rounded up to 16s), zero beyond R; those of tokens without an adapter are not
// written.  It is the sum of `planes` planes [T][Rp], one for each part of the inputs.
struct ShrinkArgs {
  const void* z;          // [T][K], rows ldz apart
  const void* f;
  const int* ids;
  const float* scale;     // [G] or null
  float* h;               // [planes][T][Rp]
  size_t T, ldz;
  int K, R, Rp, G;
  int fr, fk;             // K and 1, or 1 and R
  int planes;
};

// y[t][n] = sum_k z[t][k] w(n, k) + bias[n] + sum_r h[t][r] F_a(n, r), F_a(n, r) at
// f + a * R * N + n * fn + r * fr; w(n, k) at w + n * ldw + k, or (nn) at w + k * ldw + n.
struct ProjectArgs {
  const void *z, *w, *f;
  const float *h, *bias;
  const int* ids;
  void* y;                // [T][N]
  size_t T, ldz, ldw;
  int K, N, R, Rp, G;
  int fn, fr;
  int planes;             // h is the sum of so many planes ...
  size_t plane;           // ... so many values apart (more than one: only where project_sums_planes)
  float* keep;            // with planes > 1: where their sum goes as well, or null
};

// out[a][r][c] = sum over tokens with ids[t] = a of p[t][r] z[t][c], at out + a * R * C + r * outr +
// c * outc; with splits > 1 the sums of each range of tokens go to part [splits][G][R][C]
// (in out's order) and are added up by a second launch.
struct GradArgs {
  const float* p;         // [T][Rp]
  const void* z;          // [T][C], rows ldz apart
  const int* ids;
  void* out;
  float* part;
  size_t T, ldz;
  int C, R, Rp, G;
  int outr, outc;
  int splits;
};

int shrink_planes(size_t T, int K, int dtype);
hipError_t shrink_launch(const ShrinkArgs&, int dtype, hipStream_t);
// h [n] = the sum of `planes` planes of n values (n: a multiple of 4), the first of which may be h.
hipError_t planes_join(float* h, const float* from, size_t n, int planes, hipStream_t);
// Whether the projection that these operands get adds up the planes of h itself.
bool project_sums_planes(const ProjectArgs&, int dtype, bool nn);
// part: project_part_bytes of scratch memory.
size_t project_part_bytes(size_t T, int K, int N, int G, int dtype, bool nn);
hipError_t project_launch(const ProjectArgs&, float* part, int dtype, bool nn, hipStream_t);
// What project_launch runs: one launch, or one of whole tiles and one of the rows that are left over.
void project_plan(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, cp4_adapter_launch (&launches)[2]);
// The tiles of a projection on the matrix cores, its depth in `splits` parts of `each` steps, whose partial
// sums take tile_part_bytes.
struct TilePlan {
  int which, splits, each;
  double cost;            // microseconds, about
};
TilePlan tile_plan(size_t T, int K, int N, int dtype, bool nn, bool direct);
size_t tile_part_bytes(const TilePlan&, size_t T, int N);
int tile_rows(const TilePlan&);
int tile_cols(const TilePlan&);
// Whether these operands go from memory to the LDS without passing a register.
bool tile_direct(const ProjectArgs&, int dtype, bool nn);
hipError_t tile_launch(const ProjectArgs&, const TilePlan&, float* part, int dtype, bool nn, hipStream_t);
// y = the sum of [splits][T][N] partial sums, and the bias (may be null).
hipError_t parts_join(const float* part, const float* bias, void* y, size_t T, int N, int splits, int dtype, hipStream_t);
// Up to 64 tokens in 16 bits, 32 in fp32 (w [N][K]).  splits 0: not for this kernel.
struct RowsPlan {
  int splits;
  double cost, adapter;   // microseconds, about, and for each adapter
};
RowsPlan rows_plan(size_t T, int K, int N, int dtype);
hipError_t rows_launch(const ProjectArgs&, const RowsPlan&, float* part, int dtype, hipStream_t);
// Two sums over the same tokens and adapters, their R, G and splits the same.
int grad_splits(size_t T, int C0, int C1, int R, int G);
hipError_t grad_launch(const GradArgs&, const GradArgs&, int dtype, hipStream_t);

// ---- device side ------------------------------------------------------------------------

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// 16 x 16 blocks of products, 32 deep: of a lane's eight values, row (or column) lane & 15 and depth
// 8 * (lane >> 4) + j; the result's column is lane & 15, its row 4 * (lane >> 4) + v.
__device__ __forceinline__ f32x4 mfma_bf16(u16x8 a, u16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <class T>
__device__ __forceinline__ f32x4 mfma_16(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (__is_same(T, BF16)) return mfma_bf16(a, b, c);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// The same 4 deep in fp32: one value a lane, depth lane >> 4.
__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// A value as two bfloat16 parts: to nearest, and what that leaves.
__device__ __forceinline__ void two_parts(float x, unsigned short& hi, unsigned short& lo) {
  hi = BF16::narrow(x);
  lo = BF16::narrow(x - BF16::widen(hi));
}
__device__ __forceinline__ void two_parts(const float (&x)[8], u16x8& hi, u16x8& lo) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    unsigned short h, l;
    two_parts(x[j], h, l);
    hi[j] = h;
    lo[j] = l;
  }
}

// The different adapters of up to 64 tokens, one lane an id (-1: none): take() gives the next
// one and the lanes whose it is.
struct Adapters {
  unsigned long long left;
  int id;
  __device__ __forceinline__ Adapters(int id_) : left(__ballot(id_ >= 0)), id(id_) {}
  __device__ __forceinline__ bool take(int& a, unsigned long long& whose) {
    if (!left) return false;
    a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    whose = __ballot(id == a);
    left &= ~whose;
    return true;
  }
};

}  // namespace adapter
}  // namespace cp4
#endif
