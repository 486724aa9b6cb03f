// Microscaled 4-bit floating point (include/cp4/mx4.h): rows to it and back, and the product of two operands held in it.
//
// To it: a lane has eight consecutive values, four lanes a block of 32; its largest magnitude's exponent is the scale's, and
// the hardware's conversion divides by that and rounds (to nearest, ties to even, beyond 6 to 6) in one instruction for two
// values.  Bound by reading the values once.
//
// The product runs on the scaled matrix instructions, which take 32 values of each operand with their scale's byte a
// lane, four times bfloat16's rate.  Sums are fp32, products exact.  A tile is fed through the LDS by loads that pass no
// register; a step is 256 of the depth, 128 bytes of every row; the scales of a step, eight bytes a row, go through a
// register of one thread a row, since their rows start anywhere.
//
// Measured: 4096 x 25088 fp32 to 4 bits 83 to 100 us, back 64 to 104 (411 MB of values each way); 8192 x 4096 x 4096 85 us,
// 3.2 PFLOP/s, bound by the LDS: a step of the 256 x 256 tile reads 240 KB and takes in 68, 2.1 us at the 150 bytes a
// nanosecond that a compute unit's LDS gives, twice what the matrix cores need.  (Reads of one half of the waves
// beside the other half's products, 32 x 32 blocks, four steps of 128 under way: 92, 97 and 114 us.  128 x 128 a wave, which reads
// less, does not fit the registers.)
#include <algorithm>
#include <type_traits>

#include "adapter.h"
#include "cp4/mx4.h"
#include "die_order.h"
#include "mx4_codes.h"

namespace {

using namespace cp4;
using adapter::f32x4;
using adapter::u32x4;

typedef int i32x8 __attribute__((ext_vector_type(8)));

// ---- rows to 4 bits and back ----------------------------------------------------------------

struct RowsArgs {
  const void* x;                 // values, or codes
  const unsigned char* scales;   // (from 4 bits)
  void* out;                     // codes, or values
  unsigned char* out_scales;
  size_t ld;                     // of the values
  unsigned rows, K, blocks;
};

// The largest of the bits of four neighbouring lanes.
__device__ __forceinline__ unsigned four_max(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, false));   // (lanes 1 0 3 2)
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, false));   // (lanes 2 3 0 1)
}

// Blocks of a thread, so many threads apart: their loads wait together.
constexpr int kEach = 2;

template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(const RowsArgs a) {
  typedef typename T::raw Raw;
  const unsigned all = a.rows * a.blocks * 4, first = blockIdx.x * (256 * kEach) + threadIdx.x;
  Raw v[kEach][8];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const unsigned i = first + e * 256;
    if (i >= all) continue;
    const unsigned row = i / 4 / a.blocks, c = (i / 4 % a.blocks) * 32 + i % 4 * 8;
    const Raw* const p = static_cast<const Raw*>(a.x) + row * a.ld + c;
    if (c + 8 <= a.K) {
      __builtin_memcpy(v[e], p, sizeof(v[e]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[e][j] = c + j < a.K ? p[j] : Raw(0);
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const unsigned i = first + e * 256;
    if (i >= all) continue;                                          // (whole fours of lanes)
    float x[8];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = T::widen(v[e][j]);
      top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    }
    top = four_max(top);
    const unsigned exponent = top >> 23;                             // (floor(log2) + 127; 255: not finite)
    const unsigned byte = exponent == 255 ? 255 : exponent < 2 ? 0 : exponent - 2;
    const float scale = mx4::scale_of(byte);
    unsigned codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
    static_cast<unsigned*>(a.out)[i] = byte == 255 ? 0u : codes;
    if (i % 4 == 0) a.out_scales[i / 4] = (unsigned char)byte;
  }
}

// 16 bytes of values a store, so that a wave writes whole lines; past the caches what the memory-side one would not hold until
// somebody reads it: 4096 x 25088 fp32 (411 MB) plain 127 us and 244 with a sum over it behind, streamed 64 to 104 and 207;
// 4096 x 16384 84 and 152, 44 and 120; but 196 MB of bf16 54 and 80, 51 and 100, 64 MB of fp32 23 and 41, 13 and 44.
constexpr size_t kStreamFrom = (size_t)224 << 20;  // bytes
template <class T, bool Streamed>
__global__ __launch_bounds__(256) void dequantize_kernel(const RowsArgs a) {
  typedef typename T::raw Raw;
  typedef std::conditional_t<sizeof(Raw) == 4, unsigned short, unsigned> Codes;
  constexpr int n = 16 / (int)sizeof(Raw), kLanes = 32 / n;          // values of a lane, lanes of a block
  const unsigned all = a.rows * a.blocks * kLanes, first = blockIdx.x * (256 * kEach * kLanes / 4) + threadIdx.x;
  constexpr int kTurns = kEach * kLanes / 4;                         // (as many blocks a workgroup for every type)
  Codes codes[kTurns];
  unsigned scale[kTurns];
#pragma unroll
  for (int e = 0; e < kTurns; ++e) {
    const unsigned i = first + e * 256;
    if (i >= all) continue;
    codes[e] = static_cast<const Codes*>(a.x)[i];
    scale[e] = a.scales[i / kLanes];
  }
#pragma unroll
  for (int e = 0; e < kTurns; ++e) {
    const unsigned i = first + e * 256;
    if (i >= all) continue;
    const unsigned row = i / kLanes / a.blocks, c = (i / kLanes % a.blocks) * 32 + i % kLanes * n;
    Raw v[8];
    mx4::values<T>(codes[e], mx4::scale_of(scale[e]), v);            // (fp32: the last four are not used)
    Raw* const p = static_cast<Raw*>(a.out) + row * a.ld + c;
    if (c + n <= a.K) {
      if constexpr (Streamed) {
        typedef u32x4 __attribute__((aligned(2))) Loose;             // (any element's address)
        u32x4 w;
        __builtin_memcpy(&w, v, 16);
        __builtin_nontemporal_store(w, reinterpret_cast<Loose*>(p));
      } else {
        __builtin_memcpy(p, v, 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < n; ++j)
        if (c + j < a.K) p[j] = v[j];
    }
  }
}

template <class T>
void dequantize_launch(const RowsArgs& a, unsigned grid, bool streamed, hipStream_t st) {
  if (streamed) dequantize_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else dequantize_kernel<T, false><<<grid, 256, 0, st>>>(a);
}

size_t value_bytes(int dtype) { return dtype == CP4_DTYPE_F32 ? 4 : 2; }
bool dtype_ok(int d) { return d == CP4_DTYPE_F32 || d == CP4_DTYPE_BF16 || d == CP4_DTYPE_F16; }

// A launch for as many rows as 32-bit places reach.
template <class Launch>
hipError_t in_slabs(size_t T, unsigned K, Launch launch) {
  const unsigned blocks = (K + 31) / 32;
  const size_t most = std::max<size_t>(1, ((size_t)1 << 31) / (8 * (size_t)blocks) - 1);
  for (size_t t = 0; t < T; t += most) {
    const unsigned rows = (unsigned)std::min(T - t, most);
    launch(t, rows, blocks, (unsigned)(((size_t)rows * blocks * 4 + 256 * kEach - 1) / (256 * kEach)));
    if (const hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

cp4_status check_rows(size_t T, unsigned K, int dtype, size_t ld) {
  if (!dtype_ok(dtype)) return fail_with(CP4_ERR_SHAPE, "unknown dtype");
  if (!K || K > 1u << 22) return fail_with(CP4_ERR_SHAPE, "K must be 1 to 2^22");
  if (T > (size_t)1 << 26) return fail_with(CP4_ERR_SHAPE, "more than 2^26 rows");
  if ((ld && ld < K) || ld > (size_t)1 << 30) return fail_with(CP4_ERR_SHAPE, "a row stride smaller than the row or above 2^30");
  return CP4_OK;
}
cp4_status check_codes(const void* codes, const unsigned char* scales) {
  if (!codes || !scales) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  if ((size_t)codes & 15) return fail_with(CP4_ERR_SHAPE, "codes are not aligned to 16 bytes");
  return CP4_OK;
}

// ---- the product of two operands in 4 bits -----------------------------------------------------

struct ProductArgs {
  const char *x, *w;             // codes, rows of `blocks` times 16 bytes
  const unsigned char *xs, *ws;
  const float* bias;
  void* y;                       // [T][N]
  float* part;                   // [splits][T][N], or null: y
  size_t T;
  int N, blocks;
  int mt, nt, splits, steps;     // tiles, and parts of the depth of so many steps (the last one may have fewer)
};

constexpr int wait_for(int loads) { return (loads & 15) | (loads >> 4) << 14 | 7 << 4; }

// WM x WN waves of MB x NB blocks of 16 x 16.  A wave's column block j holds the columns NB l + j, so that a lane has NB
// consecutive values of a row of y.
template <class T, int MB, int NB, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void product_kernel(const ProductArgs a) {
  typedef typename T::raw Raw;
  constexpr int kThreads = 64 * WM * WN, BM = 16 * MB * WM, BN = 16 * NB * WN, B = BM + BN;
  constexpr int kX = BM * 8 / kThreads, kW = BN * 8 / kThreads, kS = (B + kThreads - 1) / kThreads, kRoom = B * 128;
  static_assert(BM * 8 % kThreads == 0 && BN * 8 % kThreads == 0, "whole loads");
  __shared__ __attribute__((aligned(1024))) char lds0[kRoom], lds1[kRoom];
  __shared__ __attribute__((aligned(8))) unsigned long long s0[B], s1[B];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const int place = die_place(blockIdx.x, a.mt * a.nt * a.splits);
  if (place < 0) return;
  const int split = place % a.splits, tile = place / a.splits;
  const int band = tile / (8 * a.mt), in_band = tile % (8 * a.mt), wide = min(8, a.nt - 8 * band);
  const int tm = in_band / wide, tn = 8 * band + in_band % wide;
  const size_t t0 = (size_t)tm * BM, row_bytes = (size_t)a.blocks * 16;
  const int n0 = tn * BN, wm = 16 * MB * (wave / WN), wn = 16 * NB * (wave % WN);
  const int rows = (int)min((size_t)BM, a.T - t0), cols = min(BN, a.N - n0);
  const int first = split * a.steps * 8, last = min(a.blocks, first + a.steps * 8), steps = (last - first) / 8;
  const auto column = [](int slot) __attribute__((always_inline)) {
    const int in = slot % (16 * NB);
    return slot - in + NB * (in & 15) + in / 16;
  };
  const char *xb = a.x + t0 * row_bytes + (size_t)first * 16, *wb = a.w + n0 * row_bytes + (size_t)first * 16;
  unsigned xo[kX], wo[kW];
#pragma unroll
  for (int i = 0; i < kX; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / 8;
    xo[i] = (unsigned)(min(row, rows - 1) * row_bytes) + ((at % 8) ^ (row & 7)) * 16;
  }
#pragma unroll
  for (int i = 0; i < kW; ++i) {
    const int at = i * kThreads + threadIdx.x, slot = at / 8;
    wo[i] = (unsigned)(min(column(slot), cols - 1) * row_bytes) + ((at % 8) ^ (slot & 7)) * 16;
  }
  // the scales of a thread's rows, of x and then of w
  const unsigned char* sp[kS];
#pragma unroll
  for (int i = 0; i < kS; ++i) {
    const int at = i * kThreads + threadIdx.x;
    sp[i] = at < BM ? a.xs + (t0 + min(at, rows - 1)) * a.blocks + first
                    : a.ws + (size_t)(n0 + min(column(min(at, B - 1) - BM), cols - 1)) * a.blocks + first;
  }
  int brought = 0;
  unsigned long long sr[kS];
  auto bring = [&](char* lds) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kS; ++i) __builtin_memcpy(&sr[i], sp[i], 8);
#pragma unroll
    for (int i = 0; i < kX; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(xb + xo[i]),
                                       (__attribute__((address_space(3))) void*)(lds + (i * kThreads + wave * 64) * 16), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < kW; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(wb + wo[i]),
                                       (__attribute__((address_space(3))) void*)(lds + BM * 128 + (i * kThreads + wave * 64) * 16), 16, 0, 0);
    const bool more = ++brought < steps;                             // (beyond the last step that one again)
    xb += more ? 128 : 0;
    wb += more ? 128 : 0;
#pragma unroll
    for (int i = 0; i < kS; ++i) sp[i] += more ? 8 : 0;
  };
  auto put = [&](unsigned long long* s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kS; ++i)
      if (B % kThreads == 0 || i * kThreads + (int)threadIdx.x < B) s[i * kThreads + threadIdx.x] = sr[i];
  };
  f32x4 acc[MB][NB] = {};
  auto multiply = [&](const char* lds, const unsigned long long* s) __attribute__((always_inline)) {
    unsigned long long xs[MB], ws[NB];                               // (byte 8 h + g: the lane's block of half h)
#pragma unroll
    for (int i = 0; i < MB; ++i) xs[i] = s[wm + 16 * i + l] >> (8 * g);
#pragma unroll
    for (int j = 0; j < NB; ++j) ws[j] = s[BM + wn + 16 * j + l] >> (8 * g);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = ((4 * h + g) ^ (l & 7)) * 16;
      i32x8 xv[MB], wv[NB];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(lds + (wm + 16 * i + l) * 128 + at);
        xv[i] = i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(lds + BM * 128 + (wn + 16 * j + l) * 128 + at);
        wv[j] = i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
      }
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xv[i], wv[j], acc[i][j], 4, 4, 0, (int)(xs[i] >> (32 * h)), 0,
                                                                       (int)(ws[j] >> (32 * h)));
    }
  };
  // A step: its own loads have arrived and nobody reads the last one's room any more.
  auto step = [&](const char* lds, const unsigned long long* s, char* into, unsigned long long* s_into) __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_for(0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    bring(into);
    __builtin_amdgcn_sched_barrier(0);
    multiply(lds, s);
    put(s_into);
  };
  if (steps > 0) {
    bring(lds0);
    put(s0);
    int left = steps;
    for (; left >= 2; left -= 2) {
      step(lds0, s0, lds1, s1);
      step(lds1, s1, lds0, s0);
    }
    if (left > 0) step(lds0, s0, lds1, s1);
    __builtin_amdgcn_s_waitcnt(wait_for(0));                         // (the loads beyond the last step)
  }
  if (first + steps * 8 < last) {
    // The depth's rest, through registers: beyond it zero, of the scale 1.
    const int left = last - first - steps * 8;
    const char *const xt = a.x + t0 * row_bytes + (size_t)(last - left) * 16, *const wt = a.w + n0 * row_bytes + (size_t)(last - left) * 16;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kX + kW; ++i) {
      const int at = (i < kX ? i : i - kX) * kThreads + threadIdx.x, row = at / 8, piece = (at % 8) ^ (row & 7);
      u32x4 v = {};
      if (piece < left) v = *reinterpret_cast<const u32x4*>((i < kX ? xt : wt) + (i < kX ? xo[i < kX ? i : 0] : wo[i < kX ? 0 : i - kX]));
      *reinterpret_cast<u32x4*>(lds0 + (i < kX ? 0 : BM * 128) + at * 16) = v;
    }
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      const int at = i * kThreads + threadIdx.x;
      if (at >= B) continue;
      const unsigned char* const p = at < BM ? a.xs + (t0 + min(at, rows - 1)) * a.blocks + last - left
                                             : a.ws + (size_t)(n0 + min(column(at - BM), cols - 1)) * a.blocks + last - left;
      unsigned long long v = 0;
#pragma unroll
      for (int b = 0; b < 8; ++b) v |= (unsigned long long)(b < left ? p[b] : 127) << (8 * b);
      s0[at] = v;
    }
    __syncthreads();
    multiply(lds0, s0);
  }

  const int n = n0 + wn + NB * l;
  if (n >= a.N) return;
  float bias[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) bias[j] = a.bias && n + j < a.N ? a.bias[n + j] : 0.0f;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const size_t t = t0 + wm + 16 * i + 4 * g + v;
      if (t >= a.T) continue;
      if (a.part) {
        float o[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) o[j] = acc[i][j][v];
        float* const p = a.part + ((size_t)split * a.T + t) * a.N + n;
        if (n + NB <= a.N) {
          __builtin_memcpy(p, o, sizeof(o));
        } else {
#pragma unroll
          for (int j = 0; j < NB; ++j)
            if (n + j < a.N) p[j] = o[j];
        }
      } else {
        Raw o[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) o[j] = T::narrow(acc[i][j][v] + bias[j]);
        Raw* const p = static_cast<Raw*>(a.y) + t * a.N + n;
        if (n + NB <= a.N) {
          __builtin_memcpy(p, o, sizeof(o));
        } else {
#pragma unroll
          for (int j = 0; j < NB; ++j)
            if (n + j < a.N) p[j] = o[j];
        }
      }
    }
}

// Tiles of 256 x 256, 128 x 128 and 32 x 128, and the parts of the depth, by the least time of a model of what was measured
// (microseconds a step of 256 and a launch's ends): 256 x 256 2.2 and 8; 128 x 128 one on a compute unit 0.98 and 4, two 1.72
// and 3; 32 x 128 0.36 on few units, 0.83 on most of them or with two each, 1.9 with four.
constexpr int kShapes = 3, kRows[kShapes] = {256, 128, 32}, kCols[kShapes] = {256, 128, 128};
struct Plan {
  int which, splits, steps;
  double cost;                   // microseconds, about
};
Plan plan_of(size_t T, unsigned K, unsigned N) {
  const int steps = std::max(1, (int)(((K + 31) / 32 + 7) / 8));
  const long units = num_compute_units();
  Plan best{};
  for (int w = 0; w < kShapes; ++w) {
    const long tiles = (long)((T + kRows[w] - 1) / kRows[w]) * ((N + kCols[w] - 1) / kCols[w]);
    for (int s = 1; s <= 32 && (s == 1 || (s <= steps / 2 && tiles * s <= 4 * units)); ++s) {
      const int each = (steps + s - 1) / s, parts = (steps + each - 1) / each;
      const long wgs = tiles * parts, once = (wgs + units - 1) / units, twice = (wgs + 2 * units - 1) / (2 * units), fourth = (wgs + 4 * units - 1) / (4 * units);
      double cost = w == 0 ? once * (2.2 * each + 8.0)
                    : w == 1 ? (once == 1 ? 0.98 * each + 4.0 : twice * (1.72 * each + 3.0))
                             : 3.0 + (wgs * 8 <= units ? 0.36 * each : wgs <= 2 * units ? 0.83 * each : fourth * 1.9 * each);
      if (parts > 1) cost += 4.0 + (double)T * N * (parts + 0.5) * 4.0 / 2.5e6;
      if (!best.splits || cost < best.cost) best = {w, parts, each, cost};
    }
  }
  return best;
}

template <class T>
void launch_product(const ProductArgs& a, int which, hipStream_t st) {
  const unsigned grid = die_grid((long)a.mt * a.nt * a.splits);
  if (which == 0) product_kernel<T, 8, 4, 2, 4><<<grid, 512, 0, st>>>(a);
  else if (which == 1) product_kernel<T, 4, 4, 2, 2><<<grid, 256, 0, st>>>(a);
  else product_kernel<T, 2, 2, 1, 4><<<grid, 256, 0, st>>>(a);
}

}  // namespace

extern "C" cp4_status cp4_mx4_quantize(size_t T, unsigned K, int dtype, const void* x, size_t ldx, void* codes,
                                       unsigned char* scales, cp4_stream stream) {
  if (const cp4_status rc = check_rows(T, K, dtype, ldx)) return rc;
  if (!T) return CP4_OK;
  if (!x) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  if (const cp4_status rc = check_codes(codes, scales)) return rc;
  if ((size_t)x % value_bytes(dtype)) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  const size_t ld = ldx ? ldx : K;
  const hipError_t e = in_slabs(T, K, [&](size_t t, unsigned rows, unsigned blocks, unsigned grid) {
    const RowsArgs a{static_cast<const char*>(x) + t * ld * value_bytes(dtype), nullptr, static_cast<char*>(codes) + t * blocks * 16, scales + t * blocks,
                     ld, rows, K, blocks};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == CP4_DTYPE_F32) quantize_kernel<F32><<<grid, 256, 0, st>>>(a);
    else if (dtype == CP4_DTYPE_BF16) quantize_kernel<BF16><<<grid, 256, 0, st>>>(a);
    else quantize_kernel<F16><<<grid, 256, 0, st>>>(a);
  });
  return e ? fail_hip(e, "cp4_mx4_quantize") : CP4_OK;
}

namespace cp4 {
namespace adapter {
hipError_t mx4_unpack(const void* codes, const unsigned char* scales, size_t T, unsigned K, int dtype, void* y, size_t ld, hipStream_t st) {
  const bool streamed = T * ld * value_bytes(dtype) >= kStreamFrom;
  return in_slabs(T, K, [&](size_t t, unsigned rows, unsigned blocks, unsigned grid) {
    const RowsArgs a{static_cast<const char*>(codes) + t * blocks * 16, scales + t * blocks, static_cast<char*>(y) + t * ld * value_bytes(dtype), nullptr,
                     ld, rows, K, blocks};
    if (dtype == CP4_DTYPE_F32) dequantize_launch<F32>(a, grid, streamed, st);
    else if (dtype == CP4_DTYPE_BF16) dequantize_launch<BF16>(a, grid, streamed, st);
    else dequantize_launch<F16>(a, grid, streamed, st);
  });
}
}  // namespace adapter
}  // namespace cp4

extern "C" cp4_status cp4_mx4_dequantize(size_t T, unsigned K, int dtype, const cp4_mx4* q, void* y, cp4_stream stream) {
  if (const cp4_status rc = check_rows(T, K, dtype, 0)) return rc;
  if (!T) return CP4_OK;
  if (!q || !y) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  if (const cp4_status rc = check_codes(q->codes, q->scales)) return rc;
  if ((size_t)y % value_bytes(dtype)) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  const hipError_t e = adapter::mx4_unpack(q->codes, q->scales, T, K, dtype, y, K, static_cast<hipStream_t>(stream));
  return e ? fail_hip(e, "cp4_mx4_dequantize") : CP4_OK;
}

extern "C" size_t cp4_mx4_product_workspace_bytes(size_t T, unsigned K, unsigned N) {
  if (check_rows(T, K, CP4_DTYPE_F32, 0) != CP4_OK || !T || !N || N > 1u << 22) return 0;
  const Plan p = plan_of(T, K, N);
  return p.splits > 1 ? (size_t)p.splits * T * N * 4 : 0;
}

extern "C" cp4_status cp4_mx4_product(size_t T, unsigned K, unsigned N, int dtype, const cp4_mx4* X, const cp4_mx4* W,
                                      const float* bias, void* y, void* workspace, size_t workspace_bytes, cp4_stream stream) {
  if (const cp4_status rc = check_rows(T, K, dtype, 0)) return rc;
  if (!N || N > 1u << 22) return fail_with(CP4_ERR_SHAPE, "N must be 1 to 2^22");
  if (!T) return CP4_OK;
  if (!X || !W || !y) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  for (const cp4_mx4* q : {X, W})
    if (const cp4_status rc = check_codes(q->codes, q->scales)) return rc;
  if ((size_t)y % value_bytes(dtype) || ((size_t)bias & 3)) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  const Plan plan = plan_of(T, K, N);
  if (plan.splits > 1 && (!workspace || ((size_t)workspace & 255) || workspace_bytes < cp4_mx4_product_workspace_bytes(T, K, N)))
    return fail_with(CP4_ERR_WORKSPACE, "workspace missing, too small or not aligned to 256 bytes");
  ProductArgs a{};
  a.x = static_cast<const char*>(X->codes); a.w = static_cast<const char*>(W->codes);
  a.xs = X->scales; a.ws = W->scales;
  a.bias = bias; a.y = y; a.part = plan.splits > 1 ? static_cast<float*>(workspace) : nullptr;
  a.T = T; a.N = (int)N; a.blocks = (int)((K + 31) / 32);
  a.mt = (int)((T + kRows[plan.which] - 1) / kRows[plan.which]);
  a.nt = (int)((N + kCols[plan.which] - 1) / kCols[plan.which]);
  a.splits = plan.splits; a.steps = plan.steps;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == CP4_DTYPE_F32) launch_product<F32>(a, plan.which, st);
  else if (dtype == CP4_DTYPE_BF16) launch_product<BF16>(a, plan.which, st);
  else launch_product<F16>(a, plan.which, st);
  if (const hipError_t e = hipGetLastError()) return fail_hip(e, "cp4_mx4_product");
  if (plan.splits > 1)
    if (const hipError_t e = adapter::parts_join(a.part, bias, y, T, (int)N, plan.splits, dtype, st)) return fail_hip(e, "cp4_mx4_product");
  return CP4_OK;
}
