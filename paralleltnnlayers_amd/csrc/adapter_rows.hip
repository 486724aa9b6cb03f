// The shared projection of up to 64 tokens (include/cp4/adapter.h): bound by reading W once, so nothing
// stands between memory and the matrix cores.
//
// A workgroup takes 16 columns (rows of W) of all tokens; its eight waves share the inputs, a cache
// line of every row a turn and four turns' loads ahead of their products, which keeps 64 KB of W under way
// on every compute unit (eight turns ahead: 45 us instead of 43 on the fp32 case below).  x comes from the L2 again for
// every workgroup, which is what bounds it beyond 16 tokens.  Where there are few columns the inputs
// are split over workgroups too.  The adapters' parts are shared out over the waves, h's planes are added up while the first
// turns' loads are on their way, and all sums meet in the LDS.
//
// W in 4 bits: a turn is 128 inputs, and a lane has one block of 32 of its row of W (16 bytes of codes and a scale), which it
// turns into values in its registers; it takes the same 32 inputs of its tokens.  With W a quarter of its bytes x is what bounds
// it: a load of the matrix instructions' operand is 16 bytes from each of 16 rows in a quarter of a wave, 16 cache lines looked
// up one by one, 3.8 us for each 16 tokens of 4096.  So each wave brings its rows of x whole lines at a time into its own part of the
// LDS and reads them there, without a barrier: 4096 x 4096 bf16 16 tokens 7.2 -> 7.0 us, 32 11.0 -> 8.3, 48 15.0 -> 8.6, 64 10.2 (tiles
// 16.5); fp32 16 tokens 13.4 -> 9.8, 32 23 -> 15.6.  Rows off 16-byte boundaries, and more of h than the LDS has room for
// beside them, are read as before.
//
// Measured: 16 tokens fp32, 9216 -> 4096: 43 us, 3.5 TB/s; 48 tokens of 32 adapters bf16, 4096 x 4096: 22 us (9 us without
// adapters and with 16 tokens); one token, 1024 x 1024: 6 us.
#include <algorithm>

#include "adapter.h"
#include "adapter_load.h"
#include "mx4_codes.h"

namespace cp4 {
namespace adapter {
namespace {

constexpr int kWaves = 8;

struct RowsArgs {
  ProjectArgs p;
  float* part;            // [splits][T][N], or null: y
  int splits;
};

// Four of the adapters of a wave's turn at a time, so that their loads wait together.
constexpr int kTogether = 4;

// Adds h B_a^T for every kWaves-th of the rows' adapters, from the wave's own on (16 columns; depths as in
// adapter_tiles.hip).  hl: h [T][Rp] in the LDS.
template <class T, int MB>
__device__ __forceinline__ void expand_rows(const ProjectArgs& a, int id, const float* hl, int n0, int wave, f32x4 (&acc)[MB]) {
  typedef typename T::raw Raw;
  constexpr bool kF32 = __is_same(T, F32);
  constexpr int kOwn = kF32 ? 4 : 8;
  const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const unsigned long long have = __ballot(id >= 0);
  for (int r0 = 0; r0 < a.R; r0 += 16) {
    const int rl = r0 + (kF32 ? 4 * g : 8 * (g & 1));
    float hv[MB][kOwn];
    u16x8 ha[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
#pragma unroll
      for (int q = 0; q < kOwn; ++q) hv[i][q] = 0.0f;
      if (have >> (16 * i + l) & 1) __builtin_memcpy(hv[i], __builtin_assume_aligned(hl + (16 * i + l) * a.Rp + rl, 16), sizeof(hv[i]));
      if constexpr (!kF32) {
        u16x8 hi, lo;
        two_parts(hv[i], hi, lo);
        ha[i] = g < 2 ? hi : lo;
      }
    }
    Adapters todo(id);
    int turn_of = 0;
    for (;;) {
      unsigned long long whose[kTogether];
      Raw f[kTogether][kOwn];
      bool any = false;
#pragma unroll
      for (int e = 0; e < kTogether; ++e) {
        whose[e] = 0;
        int ad = 0;
        unsigned long long w;
        while (!whose[e] && todo.take(ad, w))
          if (turn_of++ % kWaves == wave) whose[e] = w;
        if (!whose[e]) continue;
        any = true;
        const Raw* const p = static_cast<const Raw*>(a.f) + ((size_t)ad * a.N + min(n0 + l, a.N - 1)) * a.R;
        load_some(p + min(rl, a.R - 1), a.R - rl, f[e]);             // (beyond R: zero, and h is as well)
      }
      if (!any) break;
#pragma unroll
      for (int e = 0; e < kTogether; ++e) {
        if (!whose[e]) continue;
        u16x8 fh = {}, fl = {};
        if constexpr (__is_same(T, F16)) {
          float x[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) x[q] = F16::widen(f[e][q]);
          two_parts(x, fh, fl);
        } else if constexpr (!kF32) {
          fh = __builtin_bit_cast(u16x8, f[e]);
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          f32x4 d = {};
          if constexpr (kF32) {
#pragma unroll
            for (int q = 0; q < 4; ++q) d = mfma_f32(hv[i][q], f[e][q], d);
          } else {
            if constexpr (__is_same(T, F16)) d = mfma_bf16(ha[i], fl, d);
            d = mfma_bf16(ha[i], fh, d);
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) acc[i][v] += whose[e] >> (16 * i + 4 * g + v) & 1 ? d[v] : 0.0f;
        }
      }
    }
  }
}

constexpr int kStagedH = 8192;                     // floats of h that the LDS has room for beside the staged rows of x
constexpr int wait_for(int loads) { return (loads & 15) | (loads >> 4) << 14 | 7 << 4; }
constexpr int kWaitLds = 15 | 3 << 14 | 7 << 4;

template <class T, int MB, bool Four, bool Staged>
__global__ __launch_bounds__(64 * kWaves, 2) void rows_kernel(const RowsArgs ra) {
  typedef typename T::raw Raw;
  constexpr int n = 16 / sizeof(Raw), U = Four ? 128 : 128 / sizeof(Raw), kRow = 20;
  // loads of a turn (of a row of x, of W), and how many turns' are under way
  constexpr int kZ = Four ? 32 / n : 2, kW = Four ? 1 : 2, kAhead = !Four ? 4 : kZ * MB > 8 ? 1 : kZ * MB > 4 ? 2 : 4;
  constexpr int kSum = kWaves * 16 * MB * kRow, kH = 16 * MB * 256;
  // (staged) bytes of a row of x in a turn and of all rows, loads of a wave for them, turns that the LDS has room for
  constexpr int kBytes = U * (int)sizeof(Raw), kTurn = 16 * MB * kBytes, kLoads = kTurn / 1024, kRooms = kTurn <= 8192 ? 2 : 1;
  __shared__ __attribute__((aligned(1024))) char stage0[Staged ? kWaves * kTurn : 16], stage1[Staged && kRooms > 1 ? kWaves * kTurn : 16];
  __shared__ __attribute__((aligned(16))) float lds[Staged ? (kH < kStagedH ? kH : kStagedH) : kSum > kH ? kSum : kH];
  float* const hl = lds;                                             // [T][Rp], and then ...
  float* const sum = Staged ? reinterpret_cast<float*>(stage0) : lds;     // ... [kWaves][16 MB][kRow]
  static_assert(!Staged || kSum * 4 <= kWaves * kTurn, "the sums take the staged rows' place");
  const ProjectArgs& a = ra.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const int rows = (int)a.T, n0 = blockIdx.x * 16, split = blockIdx.y;
  int id = lane < rows && a.ids ? a.ids[lane] : -1;
  if (id < 0 || id >= a.G) id = -1;
  const bool adapters = split == 0 && __ballot(id >= 0);
  const size_t w_row = min(n0 + l, a.N - 1) * a.ldw;
  const Raw *z[MB], *const w = static_cast<const Raw*>(a.w) + (Four ? 0 : w_row + n * g);
  const char* const codes = static_cast<const char*>(a.w) + (w_row + g) * 16;
  const unsigned char* const scales = a.scales + w_row + g;
  unsigned sv[kAhead];
#pragma unroll
  for (int i = 0; i < MB; ++i) z[i] = static_cast<const Raw*>(a.z) + min(16 * i + l, rows - 1) * a.ldz + (Four ? 32 : n) * g;
  const int units = (a.K + U - 1) / U, shares = kWaves * ra.splits, share = split * kWaves + wave;
  const int first = (int)((long)units * share / shares), last = (int)((long)units * (share + 1) / shares);
  const int whole = min(last, a.K / U);

  f32x4 acc[MB] = {};
  u32x4 zv[kAhead][MB][kZ], wv[kAhead][kW];
  constexpr int kNext = Four ? n : 4 * n;                            // from one load of a row of x to the next one
  auto load = [&](int u, int e) __attribute__((always_inline)) {
    if constexpr (Four) {
      wv[e][0] = *reinterpret_cast<const u32x4*>(codes + (size_t)u * 64);
      sv[e] = scales[(size_t)u * 4];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) wv[e][h] = load_16(w + (size_t)u * U + 4 * n * h);
    }
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int h = 0; h < kZ; ++h) zv[e][i][h] = load_16(z[i] + (size_t)u * U + kNext * h);
  };
  auto multiply = [&](int e) __attribute__((always_inline)) {
    if constexpr (Four) {
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        Raw v[8];
        mx4::values<T>(wv[e][0][h], mx4::scale_of(sv[e]), v);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (__is_same(T, F32)) {
#pragma unroll
            for (int q = 0; q < 8; ++q) acc[i] = mfma_f32(__uint_as_float(zv[e][i][2 * h + q / 4][q % 4]), v[q], acc[i]);
          } else {
            acc[i] = mfma_16<T>(__builtin_bit_cast(u16x8, zv[e][i][h]), __builtin_bit_cast(u16x8, v), acc[i]);
          }
        }
      }
      return;
    } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (__is_same(T, F32)) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            acc[i] = mfma_f32(__uint_as_float(zv[e][i][h][q]), __uint_as_float(wv[e][h][q]), acc[i]);
        } else {
          acc[i] = mfma_16<T>(__builtin_bit_cast(u16x8, zv[e][i][h]), __builtin_bit_cast(u16x8, wv[e][h]), acc[i]);
        }
      }
    }
  };
  // Staged: a wave brings its own rows of x into its own part of the LDS, so that nobody else is waited for.
  unsigned zo[Staged ? kLoads : 1];
  u32x4 code[kRooms];
  unsigned code_scale[kRooms];
  if constexpr (Staged) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * 64 + lane, row = at / (kBytes / 16), piece = at % (kBytes / 16);
      zo[i] = (unsigned)(min(row, rows - 1) * a.ldz * sizeof(Raw)) + (piece ^ (row & 15)) * 16;
    }
  }
  auto bring = [&](int turn, char* stage, int r) __attribute__((always_inline)) {
    const int t = min(turn, whole - 1);                              // (beyond the last turn that one again)
    const char* const from = static_cast<const char*>(a.z) + (size_t)t * kBytes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + zo[i]),
                                       (__attribute__((address_space(3))) void*)(stage + wave * kTurn + i * 1024), 16, 0, 0);
    code[r] = *reinterpret_cast<const u32x4*>(codes + (size_t)t * 64);
    code_scale[r] = scales[(size_t)t * 4];
    asm volatile("" ::: "memory");                                   // (their order is what the waits count on)
    __builtin_amdgcn_sched_barrier(0);
  };
  auto turn = [&](int t, char* stage, int r) __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_for((kRooms - 1) * (kLoads + 2)));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int h = 0; h < kZ; ++h)
        zv[0][i][h] = *reinterpret_cast<const u32x4*>(stage + wave * kTurn + (16 * i + l) * kBytes + ((kZ * g + h) ^ l) * 16);
    wv[0][0] = code[r];
    sv[0] = code_scale[r];
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(kWaitLds);                            // (the room has been read)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    bring(t + kRooms, stage, r);
    multiply(0);
  };
  // The first turns' loads, h's planes while they are on their way, and then the other turns.
  int u = first;
  const bool head = !Staged && u + kAhead <= whole;
  if constexpr (Staged) {
    if (u < whole) {
      bring(u, stage0, 0);
      if constexpr (kRooms > 1) bring(u + 1, stage1, kRooms - 1);
    }
  }
  if (head) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) load(u + e, e);
  }
  __builtin_amdgcn_sched_barrier(0);
  if (adapters)
    for (int i = threadIdx.x * 4; i < rows * a.Rp; i += 64 * kWaves * 4) {
      f32x4 x = {};
      int s = 0;
      for (; s + 8 <= a.planes; s += 8) {
        f32x4 y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = *reinterpret_cast<const f32x4*>(a.h + (s + e) * a.plane + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) x += y[e];
      }
      for (; s < a.planes; ++s) x += *reinterpret_cast<const f32x4*>(a.h + s * a.plane + i);
      *reinterpret_cast<f32x4*>(hl + i) = x;
      if (a.keep && blockIdx.x == 0) *reinterpret_cast<f32x4*>(a.keep + i) = x;
    }
  if constexpr (Staged) {
    if (u < whole) {
      if constexpr (kRooms > 1) {
        for (; u + 2 <= whole; u += 2) {
          turn(u, stage0, 0);
          turn(u + 1, stage1, 1);
        }
        if (u < whole) turn(u++, stage0, 0);
      } else {
        for (; u < whole; ++u) turn(u, stage0, 0);
      }
      __builtin_amdgcn_s_waitcnt(wait_for(0));                       // (the loads beyond the last turn)
    }
  }
  if (head) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) multiply(e);
    u += kAhead;
  }
  for (; u + kAhead <= whole; u += kAhead) {
#pragma unroll
    for (int e = 0; e < kAhead; ++e) load(u + e, e);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < kAhead; ++e) multiply(e);
  }
  for (; u < whole; ++u) {
    load(u, 0);
    multiply(0);
  }
  if (u < last) {                                                    // (the inputs' rest)
    if constexpr (Four) {
      const bool there = u * U + 32 * g < a.K;
      wv[0][0] = there ? *reinterpret_cast<const u32x4*>(codes + (size_t)u * 64) : u32x4{};
      sv[0] = there ? scales[(size_t)u * 4] : 127u;
    }
#pragma unroll
    for (int h = 0; h < kZ; ++h) {
      const int left = a.K - u * U - (Four ? 32 : n) * g - kNext * h;
      if constexpr (!Four) wv[0][h] = load_16(w + (size_t)u * U + 4 * n * h, left);
#pragma unroll
      for (int i = 0; i < MB; ++i) zv[0][i][h] = load_16(z[i] + (size_t)u * U + kNext * h, left);
    }
    multiply(0);
  }
  __syncthreads();
  if (adapters) expand_rows<T, MB>(a, id, hl, n0, wave, acc);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) sum[(wave * 16 * MB + 16 * i + 4 * g + v) * kRow + l] = acc[i][v];
  __syncthreads();
  for (int o = threadIdx.x; o < rows * 16; o += 64 * kWaves) {
    const int row = o / 16, col = o % 16;
    if (n0 + col >= a.N) continue;
    float x = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) x += sum[(k * 16 * MB + row) * kRow + col];
    const size_t at = (size_t)row * a.N + n0 + col;
    if (ra.part) ra.part[(size_t)split * a.T * a.N + at] = x;
    else static_cast<Raw*>(a.y)[at] = T::narrow(a.bias ? x + a.bias[n0 + col] : x);
  }
}

template <class T, int MB>
void launch(const RowsArgs& r, hipStream_t st) {
  const dim3 grid((r.p.N + 15) / 16, r.splits);
  const ProjectArgs& p = r.p;
  constexpr size_t e = sizeof(typename T::raw);
  const bool staged = !((size_t)p.z & 15) && p.ldz * e % 16 == 0 && p.ldz * e * 64 < (size_t)1 << 31 && (!p.ids || p.T * p.Rp <= (size_t)kStagedH);
  if (!p.scales) rows_kernel<T, MB, false, false><<<grid, 64 * kWaves, 0, st>>>(r);
  else if (staged) rows_kernel<T, MB, true, true><<<grid, 64 * kWaves, 0, st>>>(r);
  else rows_kernel<T, MB, true, false><<<grid, 64 * kWaves, 0, st>>>(r);
}
template <class T>
void launch_rows(const RowsArgs& r, hipStream_t st) {
  const int mb = (int)(r.p.T + 15) / 16;
  if (mb == 1) launch<T, 1>(r, st);
  else if (mb == 2) launch<T, 2>(r, st);
  if constexpr (sizeof(typename T::raw) == 2) {
    if (mb == 3) launch<T, 3>(r, st);
    else if (mb == 4) launch<T, 4>(r, st);
  }
}

}  // namespace

// Few columns: the inputs in as many parts as fill the chip with sixteen turns or more each, if that makes four or
// more (16 tokens, 8192 inputs, 256 outputs: 11.7 us against 20.6 in one part; 1024 x 1024 in four 10.9 against 9.3).
// The cost is what 4096 inputs took: 6, 10, 14, 17 us for up to 16, 32, 48, 64 tokens (fp32: 14, 24) a round of the chip,
// and 0.15 us an adapter; with W in 4 bits and staged rows 7, 8, 9, 10 (fp32: 10, 15).
RowsPlan rows_plan(size_t T, int K, int N, int dtype, bool four, bool direct) {
  RowsPlan p{};
  const bool f32 = dtype == CP4_DTYPE_F32;
  if (T > (f32 ? 32 : 64)) return p;
  const int units = four ? (K + 127) / 128 : (K * (f32 ? 4 : 2) + 127) / 128, tiles = (N + 15) / 16, cus = num_compute_units();
  p.splits = std::max(1, std::min(cus / tiles, units / (2 * kWaves)));
  if (p.splits < 4) p.splits = 1;
  const int rounds = (int)(((long)tiles * p.splits + cus - 1) / cus), blocks = (int)(T + 15) / 16;
  p.cost = 2.0 + rounds * (K / 4096.0 / p.splits) * (four && direct ? (f32 ? 2.5 + 5.3 * blocks : 4.0 + 1.1 * blocks) : f32 ? 5.0 + 9.5 * blocks : 2.5 + 3.7 * blocks) + (p.splits > 1 ? 5.0 : 0.0);
  p.adapter = 0.15 * rounds;
  return p;
}

hipError_t rows_launch(const ProjectArgs& a, const RowsPlan& plan, float* part, int dtype, hipStream_t st) {
  RowsArgs r{};
  r.p = a;
  r.part = plan.splits > 1 ? part : nullptr;
  r.splits = plan.splits;
  if (dtype == CP4_DTYPE_F32) launch_rows<F32>(r, st);
  else if (dtype == CP4_DTYPE_BF16) launch_rows<BF16>(r, st);
  else launch_rows<F16>(r, st);
  if (const hipError_t e = hipGetLastError()) return e;
  return plan.splits > 1 ? parts_join(part, a.bias, a.y, a.T, a.N, plan.splits, dtype, st) : hipSuccess;
}

}  // namespace adapter
}  // namespace cp4
