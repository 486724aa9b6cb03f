// The layer norm of rows, forward and backward (include/cp4/layer_norm.h).
//
// Bound by memory: forward reads x and writes y, backward reads x and dy and writes dx, each once.  A row is held in
// the registers of one wave (up to 1024 values), of four (up to 4096), eight or sixteen, 8 or 16 values a lane (32 from 16384 on), so that
// the mean, the variance about it and the output take one read.  A workgroup goes through many rows with
// its columns of weight and bias in registers (read again for each row they would be more bytes than the
// row), the next row's loads under way while one is reduced.
//
// weight's and bias's gradients: a lane adds up its own columns over all rows of its workgroup in registers; the
// workgroups' sums, [parts][2][D], go to memory and a second launch adds them up in their order.  Rows of more than 16384
// values leave no registers for those sums: a launch by columns reads x and dy once more.
//
// Measured, over so many inputs that no cache holds them: 8192 x 4096 bf16: forward 31 us, 4.3 TB/s (a large copy reaches 4.8 to
// 5.1 on such cards), backward 47 us with the second launch's 4, 4.3 TB/s; fp32 44 and 83 us, 6.1 and 4.9 TB/s.  Over three inputs,
// of which the memory-side cache holds a part, forward 27 us; before its backward pass, with both passes' tensors in that cache by
// turns, 34, and the backward pass 42 + 4.  8192 x 1024 bf16: 10 and 18 us.  1024 x 25088 bf16: 56 and 90 us, where sixteen waves of
// 128 registers hold a row and nothing overlaps its loads.  One row of 4096: 5 us, a launch and three waits for memory.
#include <algorithm>

#include "cp4/layer_norm.h"
#include "cp4_internal.h"
#include "value_types.h"

namespace {

using cp4::BF16;
using cp4::F16;
using cp4::F32;
using cp4::fail_hip;
using cp4::fail_with;

constexpr unsigned kMost = 32768;                  // values of a row

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The sum over the wave, in every lane (shifts within rows of 16 lanes, then from row to row, into lane 63).
template <int kControl, int kRows>
__device__ __forceinline__ float add_from(float x) {
  return x + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kControl, kRows, 0xf, false));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = add_from<0x111, 0xf>(x);
  x = add_from<0x112, 0xf>(x);
  x = add_from<0x114, 0xf>(x);
  x = add_from<0x118, 0xf>(x);
  x = add_from<0x142, 0xa>(x);
  x = add_from<0x143, 0xc>(x);
  return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
// Two sums over the W waves of a row.  room: 2 W floats that nobody reads any more once all are behind another barrier.
template <int W>
__device__ __forceinline__ void row_sums(float& a, float& b, float* room) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      room[2 * wave] = a;
      room[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      a += room[2 * w];
      b += room[2 * w + 1];
    }
  }
}

// Where a lane's values lie: chunk c holds n values from column (c * 64 W + lane) n on.
template <class T, int VPT, int W>
struct Row {
  typedef typename T::raw Raw;
  static constexpr int n = 16 / (int)sizeof(Raw), C = VPT / n, kLanes = 64 * W, kRows = W == 1 ? 4 : 1;
  static constexpr bool kKeep = VPT <= 16;         // whether there are registers for what belongs to a lane's columns
  struct Chunk { Raw v[n]; };

  static __device__ __forceinline__ int column(int c, int lane) { return (c * kLanes + lane) * n; }
  // Columns beyond the row are zero.
  static __device__ __forceinline__ void load(const Raw* p, int D, int lane, Chunk (&r)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = column(c, lane);
      if (at + n <= D) {
        __builtin_memcpy(r[c].v, p + at, sizeof(r[c].v));
      } else {
#pragma unroll
        for (int j = 0; j < n; ++j) r[c].v[j] = at + j < D ? p[at + j] : Raw(0);
      }
    }
  }
  static __device__ __forceinline__ void floats(const float* p, float otherwise, int D, int lane, float (&v)[VPT]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = otherwise;
    if (!p) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = column(c, lane);
      if (at + n <= D) {
        __builtin_memcpy(v + c * n, p + at, n * sizeof(float));
      } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
          if (at + j < D) v[c * n + j] = p[at + j];
      }
    }
  }
  static __device__ __forceinline__ void store(Raw* p, int D, int lane, const float (&v)[VPT]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = column(c, lane);
      Raw o[n];
#pragma unroll
      for (int j = 0; j < n; ++j) o[j] = T::narrow(v[c * n + j]);
      if (at + n <= D) {
        __builtin_memcpy(p + at, o, sizeof(o));
      } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
          if (at + j < D) p[at + j] = o[j];
      }
    }
  }
};

struct ForwardArgs {
  const void* x;
  const float *weight, *bias;
  void* y;
  float* stats;
  size_t T, ldx;
  int D;
  float eps;
};

template <class T, int VPT, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void forward_kernel(const ForwardArgs a) {
  typedef Row<T, VPT, W> R;
  typedef typename T::raw Raw;
  __shared__ float room[2][2 * W];
  const int lane = W == 1 ? threadIdx.x & 63 : threadIdx.x, D = a.D;
  const size_t step = (size_t)gridDim.x * R::kRows;
  size_t t = (size_t)blockIdx.x * R::kRows + (W == 1 ? threadIdx.x >> 6 : 0);
  const float over = 1.0f / (float)D;
  float w[VPT], b[VPT];
  R::floats(a.weight, 1.0f, D, lane, w);
  R::floats(a.bias, 0.0f, D, lane, b);
  typename R::Chunk next[R::C];
  if (t < a.T) R::load(static_cast<const Raw*>(a.x) + t * a.ldx, D, lane, next);
  for (; t < a.T; t += step) {
    float v[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = T::widen(next[i / R::n].v[i % R::n]);
    if (t + step < a.T) R::load(static_cast<const Raw*>(a.x) + (t + step) * a.ldx, D, lane, next);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) s += v[i];
    row_sums<W>(s, q, room[0]);
    const float first = s * over;
    s = q = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const bool there = R::column(i / R::n, lane) + i % R::n < D;
      v[i] = there ? v[i] - first : 0.0f;
      s += v[i];
      q += v[i] * v[i];
    }
    row_sums<W>(s, q, room[1]);
    const float rest = s * over, var = q * over - rest * rest;
    const float r = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + a.eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = (v[i] - rest) * r * w[i] + b[i];
    R::store(static_cast<Raw*>(a.y) + t * D, D, lane, v);
    if (a.stats && lane == 0) {
      a.stats[2 * t] = first + rest;
      a.stats[2 * t + 1] = r;
    }
  }
}

struct BackwardArgs {
  const void *dy, *x;
  const float *weight, *stats;
  void* dx;
  float *dweight, *dbias;        // one workgroup: the gradients (each may be null); more: `part` and part + D, each there
  size_t T, lddy, ldx;
  size_t next;                   // how far one workgroup's sums are from the last one's
  int D;
};

template <class T, int VPT, int W>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void backward_kernel(const BackwardArgs a) {
  typedef Row<T, VPT, W> R;
  typedef typename T::raw Raw;
  __shared__ float room[2][2 * W];
  __shared__ float sums[W == 1 ? 2 * 64 * VPT : 1];
  const int wave = threadIdx.x >> 6, lane = W == 1 ? threadIdx.x & 63 : threadIdx.x, D = a.D;
  const size_t step = (size_t)gridDim.x * R::kRows;
  size_t t = (size_t)blockIdx.x * R::kRows + (W == 1 ? wave : 0);
  const float over = 1.0f / (float)D;
  float w[VPT], dw[R::kKeep ? VPT : 1] = {}, db[R::kKeep ? VPT : 1] = {};
  if constexpr (R::kKeep) R::floats(a.weight, 1.0f, D, lane, w);
  typename R::Chunk x_next[R::C], dy_next[R::C];
  float m_next = 0.0f, r_next = 0.0f;
  auto load = [&](size_t row) __attribute__((always_inline)) {
    R::load(static_cast<const Raw*>(a.x) + row * a.ldx, D, lane, x_next);
    R::load(static_cast<const Raw*>(a.dy) + row * a.lddy, D, lane, dy_next);
    // (by a vector load: a scalar one would be waited for with the LDS's sums of this row)
    size_t at = 2 * row;
    asm volatile("" : "+v"(at));
    m_next = a.stats[at];
    r_next = a.stats[at + 1];
  };
  if (t < a.T) load(t);
  for (int turn = 0; t < a.T; t += step, turn ^= 1) {
    float h[VPT], g[VPT];
    const float m = m_next, r = r_next;
    float s = 0.0f, q = 0.0f;
    if constexpr (!R::kKeep) R::floats(a.weight, 1.0f, D, lane, w);
    // (columns beyond the row: dy and with it all that is summed is zero)
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const float dy = T::widen(dy_next[i / R::n].v[i % R::n]);
      h[i] = (T::widen(x_next[i / R::n].v[i % R::n]) - m) * r;
      g[i] = dy * w[i];
      if constexpr (R::kKeep) {
        db[i] += dy;
        dw[i] += dy * h[i];
      }
      s += g[i];
      q += g[i] * h[i];
    }
    if (t + step < a.T) load(t + step);
    if (!a.dx) continue;
    row_sums<W>(s, q, room[turn]);
    s *= over;
    q *= over;
#pragma unroll
    for (int i = 0; i < VPT; ++i) h[i] = r * (g[i] - s - h[i] * q);
    R::store(static_cast<Raw*>(a.dx) + t * D, D, lane, h);
  }
  if (!R::kKeep || (!a.dweight && !a.dbias)) return;
  if constexpr (W == 1) {
    // the four waves' sums, one after the other
    for (int k = 0; k < R::kRows; ++k) {
      if (wave == k) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          float *const pw = sums + i * 64 + lane, *const pb = pw + VPT * 64;
          *pw = dw[i] = k ? *pw + dw[i] : dw[i];
          *pb = db[i] = k ? *pb + db[i] : db[i];
        }
      }
      __syncthreads();
    }
    if (wave != R::kRows - 1) return;
  }
  if constexpr (R::kKeep) {
    float* const pw = a.dweight ? a.dweight + blockIdx.x * a.next : nullptr;
    float* const pb = a.dbias ? a.dbias + blockIdx.x * a.next : nullptr;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int at = R::column(i / R::n, lane) + i % R::n;
      if (at >= D) continue;
      if (pw) pw[at] = dw[i];
      if (pb) pb[at] = db[i];
    }
  }
}

// The gradients of weight and bias of rows whose columns leave no registers for them above: 512 columns (fp32: 256) and every
// gridDim.y-th row a workgroup, four rows at a time, whose sums meet in the LDS.
template <class T>
__global__ __launch_bounds__(256) void columns_kernel(const BackwardArgs a) {
  typedef typename T::raw Raw;
  constexpr int n = 16 / (int)sizeof(Raw);
  __shared__ float sums[2][64 * n];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (blockIdx.x * 64 + lane) * n;
  float dw[n] = {}, db[n] = {};
  if (c < a.D) {
#pragma unroll 4
    for (size_t t = blockIdx.y * 4 + wave; t < a.T; t += gridDim.y * 4) {
      const Raw *const px = static_cast<const Raw*>(a.x) + t * a.ldx + c, *const pdy = static_cast<const Raw*>(a.dy) + t * a.lddy + c;
      Raw x[n], dy[n];
      if (c + n <= a.D) {
        __builtin_memcpy(x, px, sizeof(x));
        __builtin_memcpy(dy, pdy, sizeof(dy));
      } else {
#pragma unroll
        for (int j = 0; j < n; ++j) {
          x[j] = c + j < a.D ? px[j] : Raw(0);
          dy[j] = c + j < a.D ? pdy[j] : Raw(0);
        }
      }
      const float m = a.stats[2 * t], r = a.stats[2 * t + 1];
#pragma unroll
      for (int j = 0; j < n; ++j) {
        db[j] += T::widen(dy[j]);
        dw[j] += T::widen(dy[j]) * ((T::widen(x[j]) - m) * r);
      }
    }
  }
  for (int k = 0; k < 4; ++k) {
    if (wave == k) {
#pragma unroll
      for (int j = 0; j < n; ++j) {
        float *const pw = &sums[0][lane * n + j], *const pb = &sums[1][lane * n + j];
        *pw = dw[j] = k ? *pw + dw[j] : dw[j];
        *pb = db[j] = k ? *pb + db[j] : db[j];
      }
    }
    __syncthreads();
  }
  if (wave != 3) return;
#pragma unroll
  for (int j = 0; j < n; ++j) {
    if (c + j >= a.D) continue;
    a.dweight[blockIdx.y * a.next + c + j] = dw[j];
    a.dbias[blockIdx.y * a.next + c + j] = db[j];
  }
}


// out[c] = sum over p of part[p][c], c < 2 D: weight's gradient, then bias's.  A workgroup has 64 columns, its waves every
// 16th part.
__global__ __launch_bounds__(1024) void parts_kernel(const float* part, int parts, int D, float* dweight, float* dbias) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const size_t row = 2 * (size_t)D;
  float s = 0.0f;
  if (c < 2 * D) {
    int p = wave;
    for (; p + 16 * 7 < parts; p += 16 * 8) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = part[(p + 16 * e) * row + c];
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[e];
    }
    for (; p < parts; p += 16) s += part[p * row + c];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || c >= 2 * D) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += sums[w][lane];
  if (c < D) {
    if (dweight) dweight[c] = s;
  } else if (dbias) {
    dbias[c - D] = s;
  }
}

__global__ __launch_bounds__(256) void zero_kernel(float* a, float* b, int D) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= D) return;
  if (a) a[i] = 0.0f;
  if (b) b[i] = 0.0f;
}

// Values a lane and waves a row: the fewest that hold it, up to 32 and 16.
struct Split { int vpt, waves; };
Split split_of(unsigned D) {
  if (D <= 512) return {8, 1};
  if (D <= 1024) return {16, 1};
  if (D <= 2048) return {8, 4};
  if (D <= 4096) return {16, 4};
  if (D <= 8192) return {16, 8};
  return {D <= 16384 ? 16 : 32, 16};
}
// Workgroups of a pass: as many as stay on the chip together, or one for each of the rows that it takes at a time.
unsigned grid_of(size_t T, unsigned D, unsigned on_a_unit) {
  const Split s = split_of(D);
  const size_t rows = s.waves == 1 ? 4 : 1, most = (size_t)cp4::num_compute_units() * (s.waves > 4 ? std::max(1u, 4 * on_a_unit / s.waves) : on_a_unit);
  return (unsigned)std::min((T + rows - 1) / rows, most);
}
// Forward from 4 to 16 of them differ by 4 %.  Backward each of them leaves a set of partial sums: 8192 x 4096 bf16 takes 49 us
// with two of them, 53 with three, 58 with four, 80 with eight (fp32 83, 85, 85, 98).
constexpr unsigned kForward = 8, kBackward = 2;
// Partial sums of the gradients of weight and bias: one set a workgroup, or of the kernel that goes by columns.
bool by_columns(unsigned D) { return split_of(D).vpt > 16; }
unsigned parts_of(size_t T, unsigned D) {
  return by_columns(D) ? (unsigned)std::min<size_t>((T + 15) / 16, 64) : grid_of(T, D, kBackward);
}

template <template <class, int, int> class Launch, class T, class Args>
void by_size(const Args& a, unsigned grid, hipStream_t st) {
  const Split s = split_of((unsigned)a.D);
  if (s.waves == 1) {
    s.vpt == 8 ? Launch<T, 8, 1>::run(a, grid, st) : Launch<T, 16, 1>::run(a, grid, st);
  } else if (s.waves == 4) {
    s.vpt == 8 ? Launch<T, 8, 4>::run(a, grid, st) : Launch<T, 16, 4>::run(a, grid, st);
  } else if (s.waves == 8) {
    Launch<T, 16, 8>::run(a, grid, st);
  } else {
    s.vpt == 16 ? Launch<T, 16, 16>::run(a, grid, st) : Launch<T, 32, 16>::run(a, grid, st);
  }
}
template <class T, int VPT, int W>
struct Forward {
  static void run(const ForwardArgs& a, unsigned grid, hipStream_t st) {
    forward_kernel<T, VPT, W><<<grid, W == 1 ? 256 : 64 * W, 0, st>>>(a);
  }
};
template <class T, int VPT, int W>
struct Backward {
  static void run(const BackwardArgs& a, unsigned grid, hipStream_t st) {
    backward_kernel<T, VPT, W><<<grid, W == 1 ? 256 : 64 * W, 0, st>>>(a);
  }
};
template <template <class, int, int> class Launch, class Args>
void by_type(const Args& a, int dtype, unsigned grid, hipStream_t st) {
  if (dtype == CP4_DTYPE_F32) by_size<Launch, F32>(a, grid, st);
  else if (dtype == CP4_DTYPE_BF16) by_size<Launch, BF16>(a, grid, st);
  else by_size<Launch, F16>(a, grid, st);
}

cp4_status check_rows(size_t T, unsigned D, int dtype, size_t ld0, size_t ld1) {
  if (dtype != CP4_DTYPE_F32 && dtype != CP4_DTYPE_BF16 && dtype != CP4_DTYPE_F16)
    return fail_with(CP4_ERR_SHAPE, "unknown dtype");
  if (!D || D > kMost) return fail_with(CP4_ERR_SHAPE, "rows of 1 to 32768 values");
  if (T > (size_t)1 << 40) return fail_with(CP4_ERR_SHAPE, "more than 2^40 rows");
  if ((ld0 && ld0 < D) || (ld1 && ld1 < D)) return fail_with(CP4_ERR_SHAPE, "a row stride is smaller than the row");
  if (std::max(ld0, ld1) > (size_t)1 << 30) return fail_with(CP4_ERR_SHAPE, "a row stride above 2^30");
  return CP4_OK;
}
cp4_status check_aligned(int dtype, std::initializer_list<const void*> values, std::initializer_list<const void*> floats) {
  const size_t bytes = dtype == CP4_DTYPE_F32 ? 4 : 2;
  for (const void* p : values)
    if ((size_t)p % bytes) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  for (const void* p : floats)
    if ((size_t)p & 3) return fail_with(CP4_ERR_SHAPE, "a pointer is not aligned to its element type");
  return CP4_OK;
}

}  // namespace

extern "C" cp4_status cp4_layer_norm_forward(size_t T, unsigned D, int dtype, const void* x, size_t ldx,
                                             const float* weight, const float* bias, float eps, void* y, float* stats,
                                             cp4_stream stream) {
  if (const cp4_status rc = check_rows(T, D, dtype, ldx, 0)) return rc;
  if (!(eps >= 0)) return fail_with(CP4_ERR_SHAPE, "eps must be 0 or more");
  if (!T) return CP4_OK;
  if (!x || !y) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  if (const cp4_status rc = check_aligned(dtype, {x, y}, {weight, bias, stats})) return rc;
  ForwardArgs a{x, weight, bias, y, stats, T, ldx ? ldx : D, (int)D, eps};
  by_type<Forward>(a, dtype, grid_of(T, D, kForward), static_cast<hipStream_t>(stream));
  if (const hipError_t e = hipGetLastError()) return fail_hip(e, "cp4_layer_norm_forward");
  return CP4_OK;
}

extern "C" size_t cp4_layer_norm_backward_workspace_bytes(size_t T, unsigned D) {
  if (check_rows(T, D, CP4_DTYPE_F32, 0, 0) != CP4_OK || !T) return 0;
  const unsigned parts = parts_of(T, D);
  return parts > 1 || by_columns(D) ? (size_t)parts * 2 * D * sizeof(float) : 0;
}

extern "C" cp4_status cp4_layer_norm_backward(size_t T, unsigned D, int dtype, const void* dy, size_t lddy,
                                              const void* x, size_t ldx, const float* weight, const float* stats, void* dx,
                                              float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                                              cp4_stream stream) {
  if (const cp4_status rc = check_rows(T, D, dtype, lddy, ldx)) return rc;
  if (!dx && !dweight && !dbias) return CP4_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (const cp4_status rc = check_aligned(dtype, {dy, x, dx}, {weight, stats, dweight, dbias})) return rc;
  if (!T) {
    if (dweight || dbias) zero_kernel<<<(D + 255) / 256, 256, 0, st>>>(dweight, dbias, (int)D);
    if (const hipError_t e = hipGetLastError()) return fail_hip(e, "cp4_layer_norm_backward");
    return CP4_OK;
  }
  if (!dy || !x || !stats) return fail_with(CP4_ERR_NULL_POINTER, "an operand is NULL");
  const unsigned count = parts_of(T, D);
  const bool sums = dweight || dbias, columns = by_columns(D), parts = sums && (count > 1 || columns);
  if (parts && (!workspace || ((size_t)workspace & 15) || workspace_bytes < cp4_layer_norm_backward_workspace_bytes(T, D)))
    return fail_with(CP4_ERR_WORKSPACE, "workspace missing, too small or not aligned to 16 bytes");
  BackwardArgs a{dy, x, weight, stats, dx, dweight, dbias, T, lddy ? lddy : D, ldx ? ldx : D, 0, (int)D};
  if (parts) {
    a.dweight = static_cast<float*>(workspace);
    a.dbias = a.dweight + D;
    a.next = 2 * (size_t)D;
  }
  if (dx || !columns) by_type<Backward>(a, dtype, grid_of(T, D, kBackward), st);
  if (sums && columns) {
    const unsigned wide = dtype == CP4_DTYPE_F32 ? 256 : 512;
    const dim3 grid((D + wide - 1) / wide, count);
    if (dtype == CP4_DTYPE_F32) columns_kernel<F32><<<grid, 256, 0, st>>>(a);
    else if (dtype == CP4_DTYPE_BF16) columns_kernel<BF16><<<grid, 256, 0, st>>>(a);
    else columns_kernel<F16><<<grid, 256, 0, st>>>(a);
  }
  if (parts)
    parts_kernel<<<(2 * D + 63) / 64, 1024, 0, st>>>(static_cast<const float*>(workspace), (int)count, (int)D, dweight, dbias);
  if (const hipError_t e = hipGetLastError()) return fail_hip(e, "cp4_layer_norm_backward");
  return CP4_OK;
}
