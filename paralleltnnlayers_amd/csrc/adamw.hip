// The AdamW step over many tensors (include/cp4/adamw.h): one pass over parameters, gradients and
// moments, the moments in fp32 or as 8-bit codes with a scale for each block of 256 values.
//
// A value costs its memory traffic alone: 4 + 4 bytes of parameter, 2 or 4 of gradient, 16 of fp32
// moments or 4.06 of 8-bit ones, read and written once.  So the pass is bound by HBM, and everything is
// made to keep many wide loads in flight: a wave takes 1024 consecutive values of a tensor as four
// blocks of 256 (one 16-byte load a lane and array), all of their loads before any arithmetic.  (134 M values with 8-bit
// moments 403 us, 4.7 TB/s, 612 with a branch around each load for a tensor's end; 50 M with fp32 moments and
// bfloat16 copies 246 us, 5.1 TB/s; a large copy reaches 5.1.)  A block of 256 values is one wave's register, so its
// largest magnitude is a reduction inside the wave and a moment is never written before it is rounded for good.  The
// tensors of a launch are a table in the kernel's arguments: no copy to the device that a captured graph would have
// to repeat.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "cp4/adamw.h"
#include "cp4_internal.h"
#include "value_types.h"

// The formula's roundings, one by one: no multiply-add is contracted in this file.
#pragma clang fp contract(off)

namespace {

using cp4::BF16;
using cp4::F16;
using cp4::F32;

constexpr int kBlock = 256;                        // values that share a scale
constexpr int kUnroll = 4;                         // blocks that a wave loads at once
constexpr size_t kChunk = kBlock * kUnroll;        // values of a wave's turn
constexpr int kTensors32 = 75, kTensors8 = 57;     // of a launch: kernel arguments below 4 KB
constexpr int kNormTensors = 192, kMomentTensors = 57;
constexpr unsigned kWaves = 4;                     // of a workgroup
constexpr unsigned kNormWaves = 16;                // of the norm's: fewer that hand in a partial sum
constexpr unsigned kMostParts = 16384;             // partial sums of the norm

struct Item32 {
  void* p;
  const void* g;
  void *m, *v, *copy;
  size_t n;
};
struct Item8 : Item32 {
  float *s, *s2;
};
template <bool Eight>
struct StepArgs {
  typedef std::conditional_t<Eight, Item8, Item32> Item;
  static constexpr int kTensors = Eight ? kTensors8 : kTensors32;
  Item item[kTensors];
  unsigned first[kTensors];                        // each tensor's first chunk
  unsigned chunks, blocks;                         // blocks: of all the group's launches
  int count, copy_dtype;
  double* counter;
  const float* coefficient;                        // {factor of the gradients, 1: go on}; null: `scale`
  double lr, beta1, beta2;
  float b1, c1, b2, c2, decay, eps, scale;
};
static_assert(sizeof(StepArgs<false>) <= 4096 && sizeof(StepArgs<true>) <= 4096, "kernel arguments");
struct NormArgs {
  const void* g[kNormTensors];
  unsigned first[kNormTensors];
  unsigned left[kNormTensors];                     // values in the tensor's last chunk
  unsigned chunks, part, blocks, parts;            // part: where this launch's partial sums start
  int count;
  double *counter, *partial;
  float *coefficient, *norm;
  float scale, max_norm;
};
static_assert(sizeof(NormArgs) <= 4096, "kernel arguments");

// Four consecutive values of an array, as they lie in memory: one load or store at any alignment.  All: they are
// there (a wave's whole turn is; the branch is then the wave's, and nothing lies between its loads).
template <class Raw>
struct Four { Raw v[4]; };
template <bool All, class Raw>
__device__ __forceinline__ Four<Raw> load_four(const Raw* p, size_t at, size_t n) {
  Four<Raw> r{};
  if (All || at + 4 <= n) {
    __builtin_memcpy(r.v, p + at, sizeof(r.v));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j < n) r.v[j] = p[at + j];
  }
  return r;
}
template <bool All, class Raw>
__device__ __forceinline__ void store_four(Raw* p, size_t at, size_t n, const Four<Raw>& r) {
  if (All || at + 4 <= n) {
    __builtin_memcpy(p + at, r.v, sizeof(r.v));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (at + j < n) p[at + j] = r.v[j];
  }
}

// ---- 8-bit moments ------------------------------------------------------------------------

// The largest of the wave's values; as bits, so that infinities and NaN come out on top.  (Shifts within rows of 16
// lanes and from row to row; lanes that nothing is shifted into take 0.)
template <int kControl, int kRows>
__device__ __forceinline__ unsigned max_from(unsigned x) {
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, kControl, kRows, 0xf, false));
}
__device__ __forceinline__ unsigned wave_max(unsigned x) {
  x = max_from<0x111, 0xf>(x);
  x = max_from<0x112, 0xf>(x);
  x = max_from<0x114, 0xf>(x);
  x = max_from<0x118, 0xf>(x);
  x = max_from<0x142, 0xa>(x);
  x = max_from<0x143, 0xc>(x);
  return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
constexpr float kUnitM = (float)(1.0 / (127.0 * 127.0));
constexpr float kUnitV = (float)(1.0 / (255.0 * 255.0 * 255.0 * 255.0));

// What a block's codes are multiplied by.  A small scale times a unit would leave the normal numbers (a second moment's
// from 2^-94 on, where its values are still some): it is taken 2^64 times as large, and the product brought down again.
struct Unit {
  float unit, down;
  unsigned least;                                  // the bits of the smallest value that a code above 0 stands for
};
__device__ __forceinline__ Unit unit_of(float scale, float unit) {
  const bool small = scale < 1.0f;
  return {(small ? scale * 0x1p64f : scale) * unit, small ? 0x1p-64f : 1.0f, scale > 0.0f ? 1u : 0u};
}
__device__ __forceinline__ float decode_m(signed char q, Unit u) {
  const int i = q;
  return (float)(i < 0 ? -i * i : i * i) * u.unit * u.down;
}
__device__ __forceinline__ float decode_v(unsigned char q, Unit u) {
  const float q2 = (float)((unsigned)q * q);
  return __uint_as_float(max(__float_as_uint(q2 * q2 * u.unit * u.down), min((unsigned)q, u.least)));
}
// A block's scale and what its values are multiplied by for their codes.
__device__ __forceinline__ float scale_of(unsigned top, float* over) {
  if (top >= 0x7f800000u) { *over = 0.0f; return __uint_as_float(0x7fc00000u); }
  if (top < 0x00800000u) { *over = 0.0f; return 0.0f; }
  *over = 1.0f / __uint_as_float(top);
  return __uint_as_float(top);
}
__device__ __forceinline__ int signed_code(int q, float m) { return m < 0.0f ? -q : q; }

// Codes and scales of one block of 256 values: four a lane, those beyond the tensor zero.  A code is defined by
// correctly rounded roots; the hardware's, a unit in the last place off, give the same one but near the middle of
// two codes, where the few blocks that have such a value take the long way (134 M values 720 us with
// the long way alone, 622 so).
__device__ __forceinline__ void encode_block(const float (&m)[4], const float (&v)[4], Four<signed char>& qm,
                                             Four<unsigned char>& qv, float& sm, float& sv) {
  unsigned tm = 0, tv = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    tm = max(tm, __float_as_uint(m[j]) & 0x7fffffffu);
    tv = max(tv, __float_as_uint(v[j]) & 0x7fffffffu);
  }
  float om, ov;
  sm = scale_of(wave_max(tm), &om);
  sv = scale_of(wave_max(tv), &ov);
  bool near = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // off by some 2 units in the last place of 127, by 3 of 255
    const float a = __builtin_amdgcn_sqrtf(fabsf(m[j]) * om) * 127.0f;
    const float b = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(v[j] * ov)) * 255.0f;
    const float ra = rintf(a), rb = rintf(b);
    near = near || !(fabsf(a - ra) < 0.5f - 6e-5f) || !(fabsf(b - rb) < 0.5f - 2e-4f);
    qm.v[j] = (signed char)signed_code((int)ra, m[j]);
    qv.v[j] = (unsigned char)(int)rb;
  }
  if (__builtin_expect(__any(near), 0)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      qm.v[j] = (signed char)signed_code((int)rintf(sqrtf(fabsf(m[j]) * om) * 127.0f), m[j]);
      qv.v[j] = (unsigned char)(int)rintf(sqrtf(sqrtf(v[j] * ov)) * 255.0f);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (qv.v[j] == 0 && v[j] > 0.0f && ov > 0.0f) qv.v[j] = 1;
}

// ---- which tensor ---------------------------------------------------------------------------

// The last tensor whose first chunk is not beyond `chunk` (empty tensors are not in the table).
template <class Args>
__device__ __forceinline__ int tensor_of(const Args& a, unsigned chunk) {
  const unsigned lane = threadIdx.x & 63;
  int found = 0;
  for (int base = 0; base < a.count; base += 64) {
    const bool here = base + (int)lane < a.count && a.first[base + lane] <= chunk;
    found += __popcll(__ballot(here));
  }
  return __builtin_amdgcn_readfirstlane(found - 1);
}

// ---- the step ---------------------------------------------------------------------------------

template <class P, class G, bool Eight>
__global__ __launch_bounds__(64 * kWaves, 4) void step_kernel(const StepArgs<Eight> a) {
  typedef typename P::raw RawP;
  typedef typename G::raw RawG;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // (every workgroup has read the counter before the last one of them advances it)
  const double power1 = a.counter[1] * a.beta1, power2 = a.counter[2] * a.beta2;
  const double steps = a.counter[0];
  const float factor = a.coefficient ? a.coefficient[0] : a.scale;
  const bool go = !a.coefficient || a.coefficient[1] != 0.0f;
  if (go) {
    const float rate = (float)(a.lr / (1.0 - power1)), root = (float)(1.0 / sqrt(1.0 - power2));
    for (unsigned c = blockIdx.x * kWaves + wave; c < a.chunks; c += gridDim.x * kWaves) {
      const int t = tensor_of(a, c);
      const auto& it = a.item[t];
      const size_t n = it.n, at0 = (size_t)(c - a.first[t]) * kChunk;
      RawP* const p = static_cast<RawP*>(it.p);
      const RawG* const g = static_cast<const RawG*>(it.g);
      auto turn = [&](auto all) __attribute__((always_inline)) {
        constexpr bool kAll = decltype(all)::value;
        Four<RawP> rp[kUnroll];
        Four<RawG> rg[kUnroll];
        Four<float> m32[kUnroll], v32[kUnroll];
        Four<signed char> m8[kUnroll];
        Four<unsigned char> v8[kUnroll];
        float sm[kUnroll], sv[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const size_t at = at0 + u * kBlock + lane * 4;
          rp[u] = load_four<kAll>(p, at, n);
          rg[u] = load_four<kAll>(g, at, n);
          if constexpr (Eight) {
            m8[u] = load_four<kAll>(static_cast<signed char*>(it.m), at, n);
            v8[u] = load_four<kAll>(static_cast<unsigned char*>(it.v), at, n);
            const size_t b = (at0 + u * kBlock) / kBlock;
            const bool there = kAll || at0 + u * kBlock < n;
            sm[u] = there ? it.s[b] : 0.0f;
            sv[u] = there ? it.s2[b] : 0.0f;
          } else {
            m32[u] = load_four<kAll>(static_cast<float*>(it.m), at, n);
            v32[u] = load_four<kAll>(static_cast<float*>(it.v), at, n);
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const size_t at = at0 + u * kBlock + lane * 4;
          float m[4], v[4];
          Four<RawP> np;
          Four<float> wide;
          const Unit um = Eight ? unit_of(sm[u], kUnitM) : Unit{}, uv = Eight ? unit_of(sv[u], kUnitV) : Unit{};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (Eight) {
              m[j] = decode_m(m8[u].v[j], um);
              v[j] = decode_v(v8[u].v[j], uv);
            } else {
              m[j] = m32[u].v[j];
              v[j] = v32[u].v[j];
            }
            const float x = G::widen(rg[u].v[j]) * factor;
            m[j] = m[j] * a.b1 + x * a.c1;
            v[j] = v[j] * a.b2 + (x * x) * a.c2;
            const float to = m[j] / (sqrtf(v[j]) * root + a.eps);
            wide.v[j] = P::widen(rp[u].v[j]) * a.decay - to * rate;
            np.v[j] = P::narrow(wide.v[j]);
          }
          store_four<kAll>(p, at, n, np);
          if (it.copy) {
            if (a.copy_dtype == CP4_DTYPE_F32) {
              store_four<kAll>(static_cast<float*>(it.copy), at, n, wide);
            } else {
              Four<unsigned short> h;
#pragma unroll
              for (int j = 0; j < 4; ++j)
                h.v[j] = a.copy_dtype == CP4_DTYPE_BF16 ? BF16::narrow(wide.v[j]) : F16::narrow(wide.v[j]);
              store_four<kAll>(static_cast<unsigned short*>(it.copy), at, n, h);
            }
          }
          if constexpr (Eight) {
#pragma unroll
            for (int j = 0; j < 4; ++j)              // (what lies beyond a NaN scale's block is not there)
              if (!kAll && at + j >= n) m[j] = v[j] = 0.0f;
            Four<signed char> qm;
            Four<unsigned char> qv;
            float tm, tv;
            encode_block(m, v, qm, qv, tm, tv);
            store_four<kAll>(static_cast<signed char*>(it.m), at, n, qm);
            store_four<kAll>(static_cast<unsigned char*>(it.v), at, n, qv);
            if (lane == 0 && (kAll || at0 + u * kBlock < n)) {
              it.s[(at0 + u * kBlock) / kBlock] = tm;
              it.s2[(at0 + u * kBlock) / kBlock] = tv;
            }
          } else {
            Four<float> o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o.v[j] = m[j];
            store_four<kAll>(static_cast<float*>(it.m), at, n, o);
#pragma unroll
            for (int j = 0; j < 4; ++j) o.v[j] = v[j];
            store_four<kAll>(static_cast<float*>(it.v), at, n, o);
          }
        }
      };
      if (at0 + kChunk <= n) turn(std::true_type());
      else turn(std::false_type());
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* const ticket = reinterpret_cast<unsigned*>(a.counter + 3);
    if (atomicAdd(ticket, 1u) + 1 == a.blocks) {
      *ticket = 0;
      if (go) {
        a.counter[0] = steps + 1.0;
        a.counter[1] = power1;
        a.counter[2] = power2;
      }
    }
  }
}

// ---- the norm -----------------------------------------------------------------------------------

__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
  for (int s = 32; s; s >>= 1) x += __shfl_xor(x, s);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  double sum = 0.0;
  for (unsigned w = 0; w < kNormWaves; ++w) sum += lds[w];
  return sum;
}

// The squares' sum in 64 bits: a partial sum a workgroup, added up in their order by the workgroup that
// is done last, so that the norm does not depend on which that is.  (50 M bfloat16 gradients 31 us, 3.2 TB/s, with
// 512 workgroups of 16 waves; 52 with 2048 of four, whose partial sums wait for one another at the counter; 92 with a
// fence in each.)
template <class G>
__global__ __launch_bounds__(64 * kNormWaves, 8) void norm_kernel(const NormArgs a) {
  typedef typename G::raw Raw;
  __shared__ double lds[kNormWaves];
  __shared__ bool last;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum = 0.0;
  auto fetch = [&](unsigned c, Four<Raw> (&r)[kUnroll]) __attribute__((always_inline)) {
    const int t = tensor_of(a, c);
    const unsigned end = t + 1 < a.count ? a.first[t + 1] : a.chunks;
    const size_t n = (size_t)(end - 1 - a.first[t]) * kChunk + a.left[t], at0 = (size_t)(c - a.first[t]) * kChunk;
    const Raw* const g = static_cast<const Raw*>(a.g[t]);
    const bool all = at0 + kChunk <= n;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const size_t at = at0 + u * kBlock + lane * 4;
      r[u] = all ? load_four<true>(g, at, n) : load_four<false>(g, at, n);
    }
  };
  // (a turn's loads are on their way while the last one's are summed)
  const unsigned stride = gridDim.x * kNormWaves;
  unsigned c = blockIdx.x * kNormWaves + wave;
  Four<Raw> r[kUnroll];
  if (c < a.chunks) fetch(c, r);
  while (c < a.chunks) {
    Four<Raw> next[kUnroll] = {};
    c += stride;
    if (c < a.chunks) fetch(c, next);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double x = (double)G::widen(r[u].v[j]);
        sum += x * x;
      }
      r[u] = next[u];
    }
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) {
    // (what the workgroups hand over goes past their dies' caches: no write-back of everything else there)
    __hip_atomic_store(a.partial + a.part + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);                                   // (it has arrived)
    unsigned* const ticket = reinterpret_cast<unsigned*>(a.counter + 3) + 1;
    last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == a.blocks;
    if (last) *ticket = 0;
  }
  __syncthreads();
  if (!last) return;
  sum = 0.0;
  for (unsigned i = threadIdx.x; i < a.parts; i += 64 * kNormWaves)
    sum += __hip_atomic_load(a.partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) {
    const float norm = (float)(sqrt(sum) * fabs((double)a.scale));
    const bool finite = fabsf(norm) < __uint_as_float(0x7f800000u);
    a.coefficient[0] = a.scale * fminf(a.max_norm / (norm + 1e-6f), 1.0f);
    a.coefficient[1] = finite ? 1.0f : 0.0f;
    if (a.norm) *a.norm = norm;
  }
}

// ---- codes to values and back -----------------------------------------------------------------------

struct MomentItem {
  void *m, *v;
  float *s, *s2, *to_m, *to_v;
  size_t n;
};
struct MomentArgs {
  MomentItem item[kMomentTensors];
  unsigned first[kMomentTensors];
  unsigned chunks;
  int count;
};
static_assert(sizeof(MomentArgs) <= 4096, "kernel arguments");

// (134 M values out of their codes: 250 us, 5.4 TB/s.)
template <bool Encode>
__global__ __launch_bounds__(64 * kWaves, 4) void moments_kernel(const MomentArgs a) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (unsigned c = blockIdx.x * kWaves + wave; c < a.chunks; c += gridDim.x * kWaves) {
    const int t = tensor_of(a, c);
    const MomentItem& it = a.item[t];
    const size_t n = it.n, at0 = (size_t)(c - a.first[t]) * kChunk;
    signed char* const m8 = static_cast<signed char*>(it.m);
    unsigned char* const v8 = static_cast<unsigned char*>(it.v);
    auto turn = [&](auto all) __attribute__((always_inline)) {
      constexpr bool kAll = decltype(all)::value;
      Four<signed char> qm[kUnroll];
      Four<unsigned char> qv[kUnroll];
      Four<float> fm[kUnroll], fv[kUnroll];
      Unit um[kUnroll], uv[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const size_t at = at0 + u * kBlock + lane * 4, b = at0 / kBlock + u;
        const bool there = kAll || at0 + u * kBlock < n;
        if constexpr (Encode) {
          fm[u] = load_four<kAll>(it.to_m, at, n);
          fv[u] = load_four<kAll>(it.to_v, at, n);
        } else {
          qm[u] = load_four<kAll>(m8, at, n);
          qv[u] = load_four<kAll>(v8, at, n);
          um[u] = unit_of(there ? it.s[b] : 0.0f, kUnitM);
          uv[u] = unit_of(there ? it.s2[b] : 0.0f, kUnitV);
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const size_t at = at0 + u * kBlock + lane * 4, b = at0 / kBlock + u;
        if constexpr (Encode) {
          float tm, tv;
          encode_block(fm[u].v, fv[u].v, qm[u], qv[u], tm, tv);
          store_four<kAll>(m8, at, n, qm[u]);
          store_four<kAll>(v8, at, n, qv[u]);
          if (lane == 0 && (kAll || at0 + u * kBlock < n)) {
            it.s[b] = tm;
            it.s2[b] = tv;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            fm[u].v[j] = decode_m(qm[u].v[j], um[u]);
            fv[u].v[j] = decode_v(qv[u].v[j], uv[u]);
          }
          store_four<kAll>(it.to_m, at, n, fm[u]);
          store_four<kAll>(it.to_v, at, n, fv[u]);
        }
      }
    };
    if (at0 + kChunk <= n) turn(std::true_type());
    else turn(std::false_type());
  }
}

// ---- host ---------------------------------------------------------------------------------------------

using cp4::fail_hip;
using cp4::fail_with;

unsigned grid_for(size_t chunks, unsigned most, unsigned waves = kWaves) {
  return (unsigned)std::max<size_t>(1, std::min<size_t>((chunks + waves - 1) / waves, most));
}
size_t chunks_of(size_t n) { return (n + kChunk - 1) / kChunk; }
bool dtype_ok(int d) { return d == CP4_DTYPE_F32 || d == CP4_DTYPE_BF16 || d == CP4_DTYPE_F16; }

template <class P, bool Eight>
void launch_grad(const StepArgs<Eight>& a, unsigned grid, int g, hipStream_t st) {
  if (g == CP4_DTYPE_F32) step_kernel<P, F32, Eight><<<grid, 64 * kWaves, 0, st>>>(a);
  else if (g == CP4_DTYPE_BF16) step_kernel<P, BF16, Eight><<<grid, 64 * kWaves, 0, st>>>(a);
  else step_kernel<P, F16, Eight><<<grid, 64 * kWaves, 0, st>>>(a);
}
template <bool Eight>
void launch_step(const StepArgs<Eight>& a, unsigned grid, int p, int g, hipStream_t st) {
  if (p == CP4_DTYPE_F32) launch_grad<F32>(a, grid, g, st);
  else if (p == CP4_DTYPE_BF16) launch_grad<BF16>(a, grid, g, st);
  else launch_grad<F16>(a, grid, g, st);
}

// Tensors of a list that one launch takes: the same kernel, at most `most` of them with values, fewer
// than 2^31 chunks.
struct Launch {
  std::vector<size_t> tensors;
  size_t chunks = 0;
  unsigned group = 0;
};
template <class Most, class Same>
std::vector<Launch> launches_of(const cp4_adamw_tensor* t, size_t count, Most most, Same same) {
  std::vector<Launch> out;
  size_t open = 0;                                 // (those before it are full)
  for (size_t i = 0; i < count; ++i) {
    if (!t[i].n) continue;
    const size_t c = chunks_of(t[i].n);
    while (open < out.size() && out[open].tensors.size() == most(t[out[open].tensors[0]])) ++open;
    size_t k = open;
    while (k < out.size() && !(same(t[out[k].tensors[0]], t[i]) && out[k].tensors.size() < most(t[i]) &&
                               out[k].chunks + c < (1u << 31)))
      ++k;
    if (k == out.size()) out.emplace_back();
    out[k].tensors.push_back(i);
    out[k].chunks += c;
  }
  return out;
}

template <bool Eight>
hipError_t step_launch(const cp4_adamw_tensor* t, const Launch& run, const cp4_adamw_group& o, unsigned blocks,
                       unsigned most, const float* coefficient, float grad_scale, hipStream_t st) {
  StepArgs<Eight> a{};
  size_t chunks = 0;
  for (size_t i : run.tensors) {
    a.first[a.count] = (unsigned)chunks;
    auto& item = a.item[a.count++];
    static_cast<Item32&>(item) = Item32{t[i].param, t[i].grad, t[i].exp_avg, t[i].exp_avg_sq, t[i].copy, t[i].n};
    if constexpr (Eight) {
      item.s = t[i].scale;
      item.s2 = t[i].scale_sq;
    }
    chunks += chunks_of(t[i].n);
  }
  const cp4_adamw_tensor none{};
  const cp4_adamw_tensor& x = run.tensors.empty() ? none : t[run.tensors[0]];
  a.copy_dtype = x.copy_dtype;
  a.chunks = (unsigned)chunks;
  a.blocks = blocks;
  a.counter = o.counter;
  a.coefficient = coefficient;
  a.lr = o.lr;
  a.beta1 = o.beta1;
  a.beta2 = o.beta2;
  a.b1 = (float)o.beta1;
  a.c1 = (float)(1.0 - o.beta1);
  a.b2 = (float)o.beta2;
  a.c2 = (float)(1.0 - o.beta2);
  a.decay = (float)(1.0 - o.lr * o.weight_decay);
  a.eps = (float)o.eps;
  a.scale = grad_scale;
  launch_step<Eight>(a, grid_for(chunks, most), x.param_dtype, x.grad_dtype, st);
  return hipGetLastError();
}

cp4_status check_tensors(const cp4_adamw_tensor* t, size_t count, bool step) {
  if (!t && count) return fail_with(CP4_ERR_NULL_POINTER, "tensors is NULL");
  for (size_t i = 0; i < count; ++i) {
    const cp4_adamw_tensor& x = t[i];
    if (step && (x.bits != 32 && x.bits != 8))
      return fail_with(CP4_ERR_SHAPE, "bits of the moments must be 32 or 8");
    if (step && (!dtype_ok(x.param_dtype) || !dtype_ok(x.grad_dtype) || (x.copy && !dtype_ok(x.copy_dtype))))
      return fail_with(CP4_ERR_SHAPE, "unknown dtype of a tensor");
    if (!x.n) continue;
    if (x.n > (size_t)1 << 40) return fail_with(CP4_ERR_SHAPE, "a tensor of more than 2^40 values");
    if (!x.exp_avg || !x.exp_avg_sq || (step && (!x.param || !x.grad)))
      return fail_with(CP4_ERR_NULL_POINTER, "a tensor's pointer is NULL");
    if ((!step || x.bits == 8) && (!x.scale || !x.scale_sq))
      return fail_with(CP4_ERR_NULL_POINTER, "8-bit moments without scales");
  }
  return CP4_OK;
}

cp4_status moments(const cp4_adamw_tensor* t, size_t count, float* const* vm, float* const* vv, bool encode,
                   cp4_stream stream) {
  if (const cp4_status rc = check_tensors(t, count, false)) return rc;
  if (count && (!vm || !vv)) return fail_with(CP4_ERR_NULL_POINTER, "values is NULL");
  for (size_t i = 0; i < count; ++i)
    if (t[i].n && (!vm[i] || !vv[i])) return fail_with(CP4_ERR_NULL_POINTER, "a tensor's values are NULL");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for (const Launch& run : launches_of(t, count, [](auto&) { return (size_t)kMomentTensors; },
                                       [](auto&, auto&) { return true; })) {
    MomentArgs a{};
    size_t chunks = 0;
    for (size_t i : run.tensors) {
      a.first[a.count] = (unsigned)chunks;
      a.item[a.count++] = MomentItem{t[i].exp_avg, t[i].exp_avg_sq, t[i].scale, t[i].scale_sq, vm[i], vv[i], t[i].n};
      chunks += chunks_of(t[i].n);
    }
    a.chunks = (unsigned)chunks;
    const unsigned grid = grid_for(chunks, 8 * cp4::num_compute_units());
    if (encode) moments_kernel<true><<<grid, 64 * kWaves, 0, st>>>(a);
    else moments_kernel<false><<<grid, 64 * kWaves, 0, st>>>(a);
    if (const hipError_t e = hipGetLastError()) return fail_hip(e, "cp4_adamw_moments");
  }
  return CP4_OK;
}

}  // namespace

extern "C" size_t cp4_adamw_workspace_bytes(void) { return 16 + 8 * (size_t)kMostParts; }

extern "C" cp4_status cp4_adamw_step(const cp4_adamw_tensor* t, size_t count, const cp4_adamw_group* group,
                                     size_t n_groups, float grad_scale, float max_norm, float* norm,
                                     void* workspace, size_t workspace_bytes, cp4_stream stream) try {
  if (!group || !n_groups) return fail_with(CP4_ERR_NULL_POINTER, "groups is NULL");
  if (const cp4_status rc = check_tensors(t, count, true)) return rc;
  for (size_t i = 0; i < count; ++i)
    if (t[i].group >= n_groups) return fail_with(CP4_ERR_SHAPE, "a tensor of a group that is not there");
  for (size_t k = 0; k < n_groups; ++k) {
    const cp4_adamw_group& o = group[k];
    if (!o.counter) return fail_with(CP4_ERR_NULL_POINTER, "a group's counter is NULL");
    if ((size_t)o.counter & 7) return fail_with(CP4_ERR_SHAPE, "a counter is not aligned to 8 bytes");
    for (size_t j = 0; j < k; ++j)
      if (group[j].counter == o.counter) return fail_with(CP4_ERR_SHAPE, "two groups share a counter");
    if (!(o.lr >= 0) || !(o.beta1 >= 0 && o.beta1 < 1) || !(o.beta2 >= 0 && o.beta2 < 1) || !(o.eps >= 0) ||
        !(o.weight_decay >= 0) || !std::isfinite(o.lr) || !std::isfinite(o.eps) || !std::isfinite(o.weight_decay))
      return fail_with(CP4_ERR_SHAPE, "lr, eps and weight_decay must be 0 or more, the betas in [0, 1)");
  }
  if (!(max_norm >= 0) || !std::isfinite(grad_scale))
    return fail_with(CP4_ERR_SHAPE, "max_norm must be 0 or more, grad_scale finite");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned most = 8 * cp4::num_compute_units();
  float* coefficient = nullptr;
  if (max_norm > 0) {
    if (!workspace || workspace_bytes < cp4_adamw_workspace_bytes() || ((size_t)workspace & 15))
      return fail_with(CP4_ERR_WORKSPACE, "max_norm needs cp4_adamw_workspace_bytes() of workspace, aligned to 16");
    coefficient = static_cast<float*>(workspace);
    auto runs = launches_of(t, count, [](auto&) { return (size_t)kNormTensors; },
                            [](auto& x, auto& y) { return x.grad_dtype == y.grad_dtype; });
    if (runs.empty()) runs.emplace_back();
    if (runs.size() > kMostParts) return fail_with(CP4_ERR_SHAPE, "too many tensors");
    const unsigned each = std::max(1u, std::min<unsigned>(2 * cp4::num_compute_units(), kMostParts / (unsigned)runs.size()));
    unsigned parts = 0;
    for (const Launch& run : runs) parts += grid_for(run.chunks, each, kNormWaves);
    unsigned part = 0;
    for (const Launch& run : runs) {
      NormArgs a{};
      size_t chunks = 0;
      for (size_t i : run.tensors) {
        a.first[a.count] = (unsigned)chunks;
        a.left[a.count] = (unsigned)(t[i].n - (chunks_of(t[i].n) - 1) * kChunk);
        a.g[a.count++] = t[i].grad;
        chunks += chunks_of(t[i].n);
      }
      a.chunks = (unsigned)chunks;
      a.part = part;
      a.blocks = a.parts = parts;
      a.counter = group[0].counter;
      a.coefficient = coefficient;
      a.partial = reinterpret_cast<double*>(coefficient + 4);
      a.norm = norm;
      a.scale = grad_scale;
      a.max_norm = max_norm;
      const unsigned grid = grid_for(chunks, each, kNormWaves);
      part += grid;
      const int g = run.tensors.empty() ? CP4_DTYPE_F32 : t[run.tensors[0]].grad_dtype;
      if (g == CP4_DTYPE_F32) norm_kernel<F32><<<grid, 64 * kNormWaves, 0, st>>>(a);
      else if (g == CP4_DTYPE_BF16) norm_kernel<BF16><<<grid, 64 * kNormWaves, 0, st>>>(a);
      else norm_kernel<F16><<<grid, 64 * kNormWaves, 0, st>>>(a);
      if (const hipError_t e = hipGetLastError()) return fail_hip(e, "cp4_adamw_step");
    }
  }
  auto runs = launches_of(t, count, [](auto& x) { return (size_t)(x.bits == 8 ? kTensors8 : kTensors32); }, [](auto& x, auto& y) {
    return x.group == y.group && x.param_dtype == y.param_dtype && x.grad_dtype == y.grad_dtype &&
           x.bits == y.bits && (x.copy ? x.copy_dtype : -1) == (y.copy ? y.copy_dtype : -1);
  });
  std::vector<unsigned> blocks(n_groups, 0);
  for (Launch& run : runs) blocks[run.group = t[run.tensors[0]].group] += grid_for(run.chunks, most);
  for (size_t k = 0; k < n_groups; ++k) {                // (a step over nothing counts as well)
    if (blocks[k]) continue;
    blocks[k] = 1;
    runs.emplace_back();
    runs.back().group = (unsigned)k;
  }
  for (const Launch& run : runs) {
    const bool eight = !run.tensors.empty() && t[run.tensors[0]].bits == 8;
    const hipError_t e = eight ? step_launch<true>(t, run, group[run.group], blocks[run.group], most, coefficient, grad_scale, st)
                               : step_launch<false>(t, run, group[run.group], blocks[run.group], most, coefficient, grad_scale, st);
    if (e) return fail_hip(e, "cp4_adamw_step");
  }
  return CP4_OK;
} catch (const std::exception& e) {
  return fail_with(CP4_ERR_HIP, e.what());
}

extern "C" cp4_status cp4_adamw_moments(const cp4_adamw_tensor* t, size_t count, float* const* vm, float* const* vv,
                                        cp4_stream stream) try {
  return moments(t, count, vm, vv, false, stream);
} catch (const std::exception& e) {
  return fail_with(CP4_ERR_HIP, e.what());
}
extern "C" cp4_status cp4_adamw_set_moments(const cp4_adamw_tensor* t, size_t count, const float* const* vm,
                                            const float* const* vv, cp4_stream stream) try {
  return moments(t, count, const_cast<float* const*>(vm), const_cast<float* const*>(vv), true, stream);
} catch (const std::exception& e) {
  return fail_with(CP4_ERR_HIP, e.what());
}
