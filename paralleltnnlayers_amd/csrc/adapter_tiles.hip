// The shared projection on the matrix cores (include/cp4/adapter.h): tiles of 64 to 256 rows x 128 or 256
// columns, fed through the LDS, by loads that never pass a register where rows start on 16-byte boundaries.
//
// A step is RB bytes of depth (64 or 128: 32 or 64 values of 16 bits, half of that in fp32) of all the tile's rows and
// columns.  The LDS has room for two to four steps: while one is multiplied the next ones are on their way, and one
// barrier a step says both that the next one has arrived and that the last one's room is free.  A wave has 64 rows and
// 32 to 128 columns in registers.  Two workgroups of the 64-row and the 128 x 256 tile share a compute unit and keep its
// matrix cores busy over each other's barriers; the 256 x 256 tile is alone there and reads one half of a step's
// operands while the other half's are multiplied (8192 x 4096 x 4096 243 -> 216 us; nn: the turned operands' registers
// do not fit beside it, 255 us with it and 240 without).
//
// fp32 is multiplied as three bfloat16 parts of each value, six of the nine products (148 -> 95 us at 64 x 25088 x
// 4096 against the fp32 instructions), which is nearer to 64 bits than an fp32 sum in one go.
//
// A wave's column block j holds the columns n0 + NB * l + j (l: lane & 15), not 16 j + l: a lane then
// has NB consecutive values of every output row (one or two 16-byte stores), and where w is [K][N] (nn)
// the same order lets one load bring NB blocks' values, which are turned in registers (one byte permute
// for two values).
//
// The adapters: when a tile's sum is done, h F_a^T is added for each adapter that the tile's rows have (a
// 16-deep product a rank block against a sum over thousands of inputs), so y is written once.
//
// Little work for the chip is split over the depth: the partial tiles go to the workspace in
// fp32 (the first one with the adapters' part) and a second launch adds them up in their order.
//
// Measured: 8192 x 4096 x 4096 bf16 with adapters of rank 16: 212 us, 1.30 PFLOP/s (nn 239; the library's product
// alone 179), bound by the LDS's bandwidth beside the matrix cores; 2048 x 4096 x 8192 121 us; 1031 x 2048 x 2816 f16, rank 64:
// 30 us (nn 42), one workgroup a compute unit (three rooms of 32 KB leave as little place for a second one as four, and are as
// fast), so that nothing overlaps its barriers and the adapters' loads behind the depth; 64 x 25088 x 4096 fp32 93 us, 4.4 TB/s of W.
#include <algorithm>
#include <type_traits>

#include "adapter.h"
#include "adapter_load.h"
#include "die_order.h"
#include "mx4_codes.h"
#include "split_bf16.h"

namespace cp4 {
namespace adapter {

struct TileArgs {
  ProjectArgs p;
  float* part;            // [splits][T][N], or null: y
  int mt, nt, splits;     // tiles, and parts of the depth
  int steps;              // of a part (the last one may have fewer)
};

namespace {

// This file is built twice: for w in the operands' type, and for w in 4 bits.
#ifndef CP4_TILE_FOUR
#define CP4_TILE_FOUR 0
#endif
constexpr bool kFour = CP4_TILE_FOUR;

template <class T>
constexpr int kVec = 16 / sizeof(typename T::raw);                   // values of a 16-byte load

// s_waitcnt's operand: all but `loads` memory loads done, and all of the LDS's.
constexpr int wait_for(int loads) { return (loads & 15) | (loads >> 4) << 14 | 7 << 4; }

// The first `count` of n consecutive values, whatever p's alignment.
template <int n, class Raw>
__device__ __forceinline__ void store_some(Raw* p, const Raw (&o)[n], int count) {
  if (count >= n) {
    __builtin_memcpy(p, o, n * sizeof(Raw));
  } else {
#pragma unroll
    for (int j = 0; j < n; ++j)
      if (j < count) p[j] = o[j];
  }
}

__device__ __forceinline__ f32x4 mfma_parts(u32x4 a, u32x4 b, f32x4 c) {
  return mfma_bf16(__builtin_bit_cast(u16x8, a), __builtin_bit_cast(u16x8, b), c);
}

// Adds h F_a^T to a tile.  h's rows come into one room of the LDS once, 32 or 64 ranks at a time, and the ranks of the
// tile's adapters into another, 16 of one adapter a unit and up to kE units between two barriers, whatever their strides and
// alignment; each wave multiplies them with its own rows.  (64 tokens of 64 adapters, 1024 x 1024: 97 us with one adapter
// at a time, 56 with four.  h in registers instead, 32 ranks a pass: 1024 tokens of 4 adapters of rank 256, 4096 x 4096, 109 us
// instead of 83.  Straight from memory to the matrix cores the loads' addresses spill: 60 to 80 us more a large tile.)
//
// 16-bit types: depth 0 .. 15 of a product are the first parts of h, 16 .. 31 what they leave, against F_a twice
// (f16: F_a in two parts as well, in two products).  Ranks beyond R are zero in h and read F_a's last one
// again; columns beyond N read its last ones and are not stored.  A product is added only to the rows that are the
// adapter's: an infinity or a NaN in one adapter is no other token's.
template <class T, bool NN, int MB, int NB, int WM, int WN, int RB>
__device__ __forceinline__ void expand_tile(const ProjectArgs& a, size_t t0, int n0, char* lds0, char* lds1,
                                            f32x4 (&acc)[MB][NB]) {
  typedef typename T::raw Raw;
  constexpr bool kF32 = __is_same(T, F32);
  constexpr int kThreads = 64 * WM * WN, BM = 16 * MB * WM, BN = 16 * NB * WN, kRoom = (BM + BN) * RB;
  constexpr int kUnits = (2 * BN + kThreads - 1) / kThreads;         // 8 ranks of a column each
  constexpr int kBlock = BN * (__is_same(T, BF16) ? 32 : 64);        // bytes of a unit in the LDS
  constexpr int kFit = kRoom / kBlock, kMost = NB == 8 || NN ? 4 : 8, kE = kFit < kMost ? kFit : kMost;
  // (nn: eight units of strided loads gain nothing, 91 us for rank 256 instead of 86)
  constexpr int kC = BM * 256 <= kRoom ? 4 : 2;                      // blocks of ranks of h in the LDS: 64 bytes a row each
  constexpr int kI = (BM * kC * 2 + kThreads - 1) / kThreads;        // 8 ranks of a row each
  static_assert(MB == 4 && kE >= 1 && BM * kC * 64 <= kRoom, "a wave's rows are a ballot");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const int wm = wave / WN, wn = 16 * NB * (wave % WN);
  int id[WM];
  unsigned long long have[WM], any = 0;
#pragma unroll
  for (int w = 0; w < WM; ++w) {
    const size_t row = t0 + 64 * w + lane;
    id[w] = row < a.T && a.ids ? a.ids[row] : -1;
    if (id[w] < 0 || id[w] >= a.G) id[w] = -1;
    any |= have[w] = __ballot(id[w] >= 0);
  }
  if (!any) return;
  for (int c0 = 0; c0 < a.R; c0 += 16 * kC) {
    const int blocks = min(kC, (a.R - c0 + 15) / 16);
    unsigned long long left[WM];
#pragma unroll
    for (int w = 0; w < WM; ++w) left[w] = have[w];
    // The next units, which of this wave's rows are each one's own, and their ranks on their way.
    int ad = -1, block = 0, of[kE];
    unsigned long long own = 0, mine[kE];
    Raw x[kE][kUnits][8];
    auto next = [&]() __attribute__((always_inline)) {
      int count = 0;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        if (ad < 0) {
#pragma unroll
          for (int w = 0; w < WM; ++w)
            if (ad < 0 && left[w]) ad = __builtin_amdgcn_readlane(id[w], __builtin_ctzll(left[w]));
          if (ad >= 0)
#pragma unroll
            for (int w = 0; w < WM; ++w) {
              const unsigned long long whose = __ballot(id[w] == ad);
              left[w] &= ~whose;
              if (w == wm) own = whose;
            }
        }
        mine[e] = 0;
        of[e] = block;
        if (ad < 0) continue;
        ++count;
        mine[e] = own;
        const Raw* const f = static_cast<const Raw*>(a.f) + (size_t)ad * a.R * a.N;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int at = u * kThreads + threadIdx.x, r = c0 + 16 * block + at / BN * 8;
          if (at >= 2 * BN) continue;
          const Raw* const p = f + (size_t)min(n0 + at % BN, a.N - 1) * a.fn;
          if (!NN && r + 8 <= a.R) {
            __builtin_memcpy(x[e][u], p + r, sizeof(x[e][u]));
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) x[e][u][q] = p[(size_t)min(r + q, a.R - 1) * a.fr];
          }
        }
        if (++block == blocks) {
          block = 0;
          ad = -1;
        }
      }
      return count;
    };
    int count = next();
    {
      f32x4 hv[kI][2];
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        const int at = i * kThreads + threadIdx.x, row = at % BM, r = at / BM * 8;
        hv[i][0] = hv[i][1] = f32x4{};
        if (r >= 16 * blocks || t0 + row >= a.T) continue;
        const float* const p = a.h + (t0 + row) * a.Rp + c0 + r;
        hv[i][0] = *reinterpret_cast<const f32x4*>(p);
        hv[i][1] = *reinterpret_cast<const f32x4*>(p + 4);
      }
      __syncthreads();                                               // (nobody reads what was there)
      // [block of ranks][piece][row]: 16 bytes that a lane multiplies, piece g of its row
#pragma unroll
      for (int i = 0; i < kI; ++i) {
        const int at = i * kThreads + threadIdx.x, row = at % BM, r = at / BM * 8, half = r / 8 & 1;
        if (r >= 16 * blocks) continue;
        char* const to = lds1 + ((size_t)(r / 16) * 4 * BM + row) * 16;
        if constexpr (kF32) {
          *reinterpret_cast<f32x4*>(to + (2 * half) * BM * 16) = hv[i][0];
          *reinterpret_cast<f32x4*>(to + (2 * half + 1) * BM * 16) = hv[i][1];
        } else {
          float y[8];
          __builtin_memcpy(y, &hv[i][0], 32);
          u16x8 hi, lo;
          two_parts(y, hi, lo);
          *reinterpret_cast<u16x8*>(to + half * BM * 16) = hi;
          *reinterpret_cast<u16x8*>(to + (2 + half) * BM * 16) = lo;
        }
      }
    }
    while (count) {
      unsigned long long rows[kE];
      int part[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        rows[e] = mine[e];
        part[e] = of[e];
      }
#pragma unroll
      for (int e = 0; e < kE; ++e)
        if (e < count)
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            const int at = u * kThreads + threadIdx.x, col = at % BN, half = at / BN;
            if (at >= 2 * BN) continue;
            const int in = col % (16 * NB), slot = col - in + 16 * (in % NB) + in / NB;    // block j's columns side by side
            char* const to = lds0 + e * kBlock;
            if constexpr (kF32) {
              __builtin_memcpy(__builtin_assume_aligned(to + slot * 64 + half * 32, 16), x[e][u], 32);
            } else if constexpr (__is_same(T, F16)) {
              float y[8];
#pragma unroll
              for (int q = 0; q < 8; ++q) y[q] = F16::widen(x[e][u][q]);
              u16x8 hi, lo;
              two_parts(y, hi, lo);
              *reinterpret_cast<u16x8*>(to + slot * 64 + half * 16) = hi;
              *reinterpret_cast<u16x8*>(to + slot * 64 + 32 + half * 16) = lo;
            } else {
              __builtin_memcpy(__builtin_assume_aligned(to + slot * 32 + half * 16, 16), x[e][u], 16);
            }
          }
      count = next();
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        if (!rows[e]) continue;
        const char* const hp = lds1 + ((size_t)(part[e] * 4 + g) * BM + 64 * wm + l) * 16;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if (!(rows[e] >> (16 * i) & 0xffff)) continue;
          const u32x4 hv = *reinterpret_cast<const u32x4*>(hp + 16 * i * 16);
          // (a product's bits where the row is the adapter's, none elsewhere)
          const unsigned bits = (unsigned)(rows[e] >> (16 * i)) >> (4 * g);
          unsigned keep[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) keep[v] = (unsigned)__builtin_amdgcn_sbfe((int)bits, v, 1);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            const char* const at = lds0 + e * kBlock + (wn + 16 * j + l) * (__is_same(T, BF16) ? 32 : 64);
            f32x4 d = {};
            if constexpr (kF32) {
              const f32x4 fv = *reinterpret_cast<const f32x4*>(at + g * 16);
#pragma unroll
              for (int q = 0; q < 4; ++q) d = mfma_f32(__uint_as_float(hv[q]), fv[q], d);
            } else {
              const u16x8 hb = __builtin_bit_cast(u16x8, hv);
              if constexpr (__is_same(T, F16)) d = mfma_bf16(hb, *reinterpret_cast<const u16x8*>(at + 32 + (g & 1) * 16), d);
              d = mfma_bf16(hb, *reinterpret_cast<const u16x8*>(at + (g & 1) * 16), d);
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] += __uint_as_float(__float_as_uint(d[v]) & keep[v]);
          }
        }
      }
      __syncthreads();                                               // (nobody reads what was there)
    }
  }
}

// One wave of a tile: MB x NB blocks of 16 x 16.
template <class T, bool NN, bool Direct, int MB, int NB, int WM, int WN, int RB, int Rooms>
__global__ __launch_bounds__(64 * WM * WN, 2) void tile_kernel(const TileArgs ta) {
  typedef typename T::raw Raw;
  constexpr int kThreads = 64 * WM * WN, BM = 16 * MB * WM, BN = 16 * NB * WN, KS = RB / (int)sizeof(Raw);
  constexpr int RC = RB / 16;                                        // a row's bytes of a step: 16-byte pieces
  constexpr int kZ = BM * RC / kThreads, kW = BN * RC / kThreads;    // 16-byte loads of a thread and step
  static_assert(BM * RC % kThreads == 0 && BN * RC % kThreads == 0, "whole loads");
  // (variables of their own, so that the compiler knows a load into one from a read of another)
  constexpr int kRoom = (BM + BN) * RB;
  __shared__ __attribute__((aligned(1024))) char lds0[kRoom], lds1[kRoom], lds2[Rooms > 2 ? kRoom : 16], lds3[Rooms > 3 ? kRoom : 16];
  const ProjectArgs& a = ta.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  // the place of this workgroup: each die a contiguous run of tiles, up to eight columns of tiles wide
  const int place = die_place(blockIdx.x, ta.mt * ta.nt * ta.splits);
  if (place < 0) return;
  const int split = place % ta.splits, tile = place / ta.splits;
  const int band = tile / (8 * ta.mt), in_band = tile % (8 * ta.mt), wide = min(8, ta.nt - 8 * band);
  const int tm = in_band / wide, tn = 8 * band + in_band % wide;
  const size_t t0 = (size_t)tm * BM;
  const int n0 = tn * BN, wm = 16 * MB * (wave / WN), wn = 16 * NB * (wave % WN);
  const int rows = (int)min((size_t)BM, a.T - t0), cols = min(BN, a.N - n0);
  const int k_first = split * ta.steps * KS, k_last = min(a.K, k_first + ta.steps * KS);
  const int steps = (k_last - k_first) / KS;

  const char* zb = reinterpret_cast<const char*>(static_cast<const Raw*>(a.z) + t0 * a.ldz + k_first);
  const char* wb = reinterpret_cast<const char*>(static_cast<const Raw*>(a.w) +
                                                 (NN ? (size_t)k_first * a.ldw + n0 : (size_t)n0 * a.ldw + k_first));
  const size_t w_next = NN ? (size_t)KS * a.ldw * sizeof(Raw) : RB;
  // (a row's pieces in another order in each row, so that a column of them lies in all banks)
  auto piece = [](int slot, int row) __attribute__((always_inline)) { return RC == 4 ? slot ^ (row >> 1 & 3) : slot ^ (row & 7); };
  // What each thread brings: the LDS is filled in the threads' order; which 16 bytes come there is theirs to choose.
  // Rows beyond the operand's are read again from its last one: what they give is not stored.
  typedef std::conditional_t<Direct, unsigned, size_t> Offset;       // (bytes)
  Offset zo[kZ], wo[kFour ? 1 : kW];
  int w_count[kFour ? 1 : kW];                                       // values there of a piece of w's row (nn)
  // w in 4 bits: blocks of 32 values, their codes and scales in registers for a step until put_four() turns them into values in the
  // LDS.  (Registers for several steps' gain nothing: 512 tokens of 4096 x 4096 36 us with one step's, 39 with four.  What
  // bounds w [N][K] is that 64 lanes' blocks lie in 64 rows.)
  constexpr int kBlocks = BN * KS / 32, kC = (kBlocks + kThreads - 1) / kThreads;
  unsigned co[kFour ? kC : 1], at_lds[kFour ? kC : 1];               // a thread's blocks: where, from the step's first one on, ...
  int depth_of[kFour ? kC : 1];                                      // ... whither, and the depth of their first value
  u32x4 codes[kFour ? kC : 1];
  unsigned scale[kFour ? kC : 1];
  int fetched = 0;
  size_t w_block = NN ? (size_t)k_first * a.ldw + n0 / 32 : (size_t)n0 * a.ldw + k_first / 32;
  const size_t w_blocks = NN ? (size_t)KS * a.ldw : KS / 32;
  if constexpr (kFour) {
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      // (threads beyond the last block read others' again: the waits count the same loads in every wave)
      const int at = (i * kThreads + threadIdx.x) % kBlocks;
      if constexpr (NN) {
        constexpr int kRow = BN / 32;
        const int block = at % kRow;
        depth_of[i] = at / kRow;
        co[i] = (unsigned)(depth_of[i] * a.ldw) + min(block, (cols - 1) / 32);
        at_lds[i] = BM * RB + (unsigned)(depth_of[i] * BN + 32 * block) * sizeof(Raw);
      } else {
        // (a row's blocks of a step side by side: half the lines that 64 lanes touch otherwise)
        const int slot = at / (KS / 32), block = at % (KS / 32), in = slot % (16 * NB), col = slot - in + NB * (in & 15) + in / 16;
        depth_of[i] = 32 * block;
        co[i] = (unsigned)(min(col, cols - 1) * a.ldw) + block;
        at_lds[i] = BM * RB + slot * RB;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kZ; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / RC, chunk = piece(at % RC, row);
    zo[i] = (Offset)(min(row, rows - 1) * a.ldz * sizeof(Raw)) + chunk * 16;
  }
#pragma unroll
  for (int i = 0; i < (kFour ? 0 : kW); ++i) {
    const int at = i * kThreads + threadIdx.x;
    if constexpr (NN) {
      constexpr int kRow = BN / kVec<T>;                             // 16-byte pieces of a row
      const int last = min(at % kRow, (cols - 1) / kVec<T>);
      wo[i] = (Offset)(at / kRow * a.ldw * sizeof(Raw)) + last * 16;
      w_count[i] = cols - last * kVec<T>;
    } else {
      const int slot = at / RC, chunk = piece(at % RC, slot), in = slot % (16 * NB);
      const int col = slot - in + NB * (in & 15) + in / 16;
      wo[i] = (Offset)(min(col, cols - 1) * a.ldw * sizeof(Raw)) + chunk * 16;
      w_count[i] = kVec<T>;
    }
  }
  int brought = 0;
  auto advance = [&]() __attribute__((always_inline)) {
    const bool more = ++brought < steps;                             // (beyond the last step that one again)
    zb += more ? RB : 0;
    if constexpr (!kFour) wb += more ? w_next : 0;
  };
  // the codes of the next step of which none are under way
  auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < (kFour ? kC : 0); ++i) {
      codes[i] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.w) + (w_block + co[i]) * 16);
      scale[i] = a.scales[w_block + co[i]];
    }
    w_block += ++fetched < steps ? w_blocks : 0;
  };
  // Operands on 16-byte boundaries go from memory to the LDS by themselves; others through registers, which put()
  // writes when the step that hid their way is multiplied.
  u32x4 zr[Direct ? 1 : kZ], wr[Direct || kFour ? 1 : kW];
  auto bring = [&](char* lds) __attribute__((always_inline)) {
    if constexpr (Direct) {
#pragma unroll
      for (int i = 0; i < kZ; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(zb + zo[i]),
                                         (__attribute__((address_space(3))) void*)(lds + (i * kThreads + wave * 64) * 16), 16, 0, 0);
#pragma unroll
      for (int i = 0; i < (kFour ? 0 : kW); ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(wb + wo[i]),
                                         (__attribute__((address_space(3))) void*)(lds + BM * RB + (i * kThreads + wave * 64) * 16), 16, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < kZ; ++i) zr[i] = load_16(reinterpret_cast<const Raw*>(zb + zo[i]));
#pragma unroll
      for (int i = 0; i < (kFour ? 0 : kW); ++i) wr[i] = load_16(reinterpret_cast<const Raw*>(wb + wo[i]), NN ? w_count[i] : kVec<T>);
    }
    advance();
  };
  auto put_four = [&](char* lds) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < (kFour ? kC : 0); ++i) {
      const int at = i * kThreads + threadIdx.x;
      if (kBlocks % kThreads && at >= kBlocks) continue;
      // (nn: neighbouring threads' blocks lie 64 bytes apart, and begin with another part each, so that eight are in all banks)
      const int turn = NN ? at % (BN / 32) >> 1 : 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int word = (q + turn) & 3;
        unsigned c = codes[i][q];
        if constexpr (NN) c = word & 2 ? (word & 1 ? codes[i][3] : codes[i][2]) : word & 1 ? codes[i][1] : codes[i][0];
        Raw v[8];
        mx4::values<T>(c, mx4::scale_of(scale[i]), v);
#pragma unroll
        for (int h = 0; h < (int)sizeof(v) / 16; ++h) {
          const int part = word * ((int)sizeof(v) / 16) + h;         // 16 bytes of the block's
          char* to = lds + at_lds[i];
          if constexpr (NN) to += part * 16;
          else to += piece(depth_of[i] / kVec<T> + part, at / (KS / 32)) * 16;
          __builtin_memcpy(__builtin_assume_aligned(to, 16), reinterpret_cast<const char*>(v) + 16 * h, 16);
        }
      }
    }
  };
  auto put = [&](char* lds) __attribute__((always_inline)) {
    if constexpr (!Direct) {
#pragma unroll
      for (int i = 0; i < kZ; ++i) *reinterpret_cast<u32x4*>(lds + (i * kThreads + threadIdx.x) * 16) = zr[i];
#pragma unroll
      for (int i = 0; i < (kFour ? 0 : kW); ++i) *reinterpret_cast<u32x4*>(lds + BM * RB + (i * kThreads + threadIdx.x) * 16) = wr[i];
    }
  };

  f32x4 acc[MB][NB] = {};
  // (16-bit: piece g of a row; fp32: pieces 2 g and 2 g + 1)
  const int z_at = (wm + l) * RB, w_at = BM * RB + (NN ? 0 : (wn + l) * RB);
  // (16 bits) the operands of 32 of a step's depths, and their products
  auto read = [&](const char* lds, int kk, u16x8 (&zf)[MB], u16x8 (&wf)[NB]) __attribute__((always_inline)) {
    const int at = piece(4 * kk + g, l) * 16;
#pragma unroll
    for (int i = 0; i < MB; ++i) zf[i] = *reinterpret_cast<const u16x8*>(lds + z_at + at + i * 16 * RB);
    if constexpr (NN) {
      unsigned in[8][NB / 2];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const char* const p = lds + w_at + ((32 * kk + 8 * g + q) * BN + wn + NB * l) * 2;
        if constexpr (NB == 2) {
          in[q][0] = *reinterpret_cast<const unsigned*>(p);
        } else if constexpr (NB == 8) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) in[q][e] = x[e];
        } else {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p);
          in[q][0] = x[0];
          in[q][1] = x[1];
        }
      }
      turn<NB>(in, wf);
    } else {
#pragma unroll
      for (int j = 0; j < NB; ++j) wf[j] = *reinterpret_cast<const u16x8*>(lds + w_at + at + j * 16 * RB);
    }
  };
  auto products = [&](const u16x8 (&zf)[MB], const u16x8 (&wf)[NB]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i][j] = mfma_16<T>(zf[i], wf[j], acc[i][j]);
  };
  auto multiply = [&](const char* lds) __attribute__((always_inline)) {
    if constexpr (__is_same(T, F32)) {
      // fp32 values as three bfloat16 parts, a product as the six largest partial products
      const int p0 = piece(2 * g, l) * 16, p1 = piece(2 * g + 1, l) * 16;
      u32x4 zh[MB], zm[MB], zl[MB];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        float x[8];
        __builtin_memcpy(x, __builtin_assume_aligned(lds + z_at + i * 16 * RB + p0, 16), 16);
        __builtin_memcpy(x + 4, __builtin_assume_aligned(lds + z_at + i * 16 * RB + p1, 16), 16);
        split::split8(x, zh[i], zm[i], zl[i]);
      }
      typedef float Row __attribute__((ext_vector_type(NB)));
      Row in[8];
      if constexpr (NN) {
#pragma unroll
        for (int q = 0; q < 8; ++q) in[q] = *reinterpret_cast<const Row*>(lds + w_at + ((8 * g + q) * BN + wn + NB * l) * 4);
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float x[8];
        if constexpr (NN) {
#pragma unroll
          for (int q = 0; q < 8; ++q) x[q] = in[q][j];
        } else {
          __builtin_memcpy(x, __builtin_assume_aligned(lds + w_at + j * 16 * RB + p0, 16), 16);
          __builtin_memcpy(x + 4, __builtin_assume_aligned(lds + w_at + j * 16 * RB + p1, 16), 16);
        }
        u32x4 wh, wmid, wl;
        if constexpr (kFour) {                                       // (a 4-bit value is its first part alone)
#pragma unroll
          for (int q = 0; q < 4; ++q) wh[q] = split::pack_hi16(x[2 * q], x[2 * q + 1]);
#pragma unroll
          for (int i = 0; i < MB; ++i) {
            acc[i][j] = mfma_parts(zl[i], wh, acc[i][j]);
            acc[i][j] = mfma_parts(zm[i], wh, acc[i][j]);
            acc[i][j] = mfma_parts(zh[i], wh, acc[i][j]);
          }
          continue;
        }
        split::split8(x, wh, wmid, wl);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          acc[i][j] = mfma_parts(zl[i], wh, acc[i][j]);
          acc[i][j] = mfma_parts(zm[i], wmid, acc[i][j]);
          acc[i][j] = mfma_parts(zh[i], wl, acc[i][j]);
          acc[i][j] = mfma_parts(zm[i], wh, acc[i][j]);
          acc[i][j] = mfma_parts(zh[i], wmid, acc[i][j]);
          acc[i][j] = mfma_parts(zh[i], wh, acc[i][j]);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < RB / 64; ++kk) {
        u16x8 zf[MB], wf[NB];
        read(lds, kk, zf, wf);
        products(zf, wf);
      }
    }
  };
  // A step: its own loads have arrived (with more than two rooms those of the next ones may still be on their way),
  // and nobody reads the last one's room any more.  Every step brings one, so that no branch keeps the
  // compiler from counting the loads under way.
  auto step = [&](const char* lds, char* into) __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    // (w in 4 bits: the codes under way are waited for where they are used, behind the older of these loads)
    if constexpr (Direct) __builtin_amdgcn_s_waitcnt(wait_for((Rooms - 2) * (kZ + (kFour ? 2 * kC : kW))));
    else __builtin_amdgcn_s_waitcnt(wait_for(63));                   // (the LDS alone)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    bring(into);
    __builtin_amdgcn_sched_barrier(0);
    multiply(lds);
    put(into);
    if constexpr (kFour) {
      put_four(into);
      fetch();
    }
  };
  if constexpr (Direct && !NN && NB == 8 && RB == 128 && !kFour) {
    // A half step's operands are read while the other half's are multiplied, so that the LDS and the matrix cores
    // work at the same time.  In the middle of a step its room is free - all have read the second half - and
    // the next one's has arrived.  (8192x4096x4096 bf16: 216 us, 243 one after the other.  With w [K][N] the turned
    // operands of 128 columns do not fit beside: 255 us with what spills, 243.)
    u16x8 za[MB], wa[NB], zc[MB], wc[NB];
    static_assert(Rooms == 2, "the loop below");
    auto turns = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < MB + NB; ++e) {                            // (a read, two products)
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
      }
    };
    auto both = [&](char* lds, const char* then) __attribute__((always_inline)) {
      read(lds, 1, zc, wc);
      products(za, wa);
      turns();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(wait_for(0));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      bring(lds);
      __builtin_amdgcn_sched_barrier(0);
      read(then, 0, za, wa);
      products(zc, wc);
      turns();
      __builtin_amdgcn_sched_barrier(0);
    };
    if (steps > 0) {
      bring(lds0);
      asm volatile("" ::: "memory");                                 // (their order is what the wait counts on)
      __builtin_amdgcn_sched_barrier(0);
      bring(lds1);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(wait_for(kZ + kW));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      read(lds0, 0, za, wa);
      int left = steps;
      for (; left >= 2; left -= 2) {
        both(lds0, lds1);
        both(lds1, lds0);
      }
      if (left > 0) both(lds0, lds1);
      __builtin_amdgcn_s_waitcnt(wait_for(0));                       // (the loads beyond the last step)
    }
  } else if (steps > 0) {
    auto ahead = [&](char* lds) __attribute__((always_inline)) {
      bring(lds);
      put(lds);
      asm volatile("" ::: "memory");                                 // (their order is what the waits count on)
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (kFour) fetch();
    ahead(lds0);
    if constexpr (Rooms > 2) ahead(lds1);
    if constexpr (Rooms > 3) ahead(lds2);
    if constexpr (kFour) {
      put_four(lds0);
      fetch();
      if constexpr (Rooms > 2) {
        put_four(lds1);
        fetch();
      }
      if constexpr (Rooms > 3) {
        put_four(lds2);
        fetch();
      }
    }
    int left = steps;                                                // (no way out in the middle: the same reason)
    for (; left >= Rooms; left -= Rooms) {
      if constexpr (Rooms == 2) {
        step(lds0, lds1);
        step(lds1, lds0);
      } else if constexpr (Rooms == 3) {
        step(lds0, lds2);
        step(lds1, lds0);
        step(lds2, lds1);
      } else {
        step(lds0, lds3);
        step(lds1, lds0);
        step(lds2, lds1);
        step(lds3, lds2);
      }
    }
    if (left > 0) step(lds0, Rooms == 2 ? lds1 : Rooms == 3 ? lds2 : lds3);
    if constexpr (Rooms > 2)
      if (left > 1) step(lds1, lds0);
    if constexpr (Rooms > 3)
      if (left > 2) step(lds2, lds1);
    __builtin_amdgcn_s_waitcnt(wait_for(0));                         // (the loads beyond the last step)
  }
  if (k_first + steps * KS < k_last) {
    // The depth's rest, through registers, zero behind it.
    const int left = k_last - k_first - steps * KS;
    zb = reinterpret_cast<const char*>(static_cast<const Raw*>(a.z) + t0 * a.ldz + k_last - left);
    wb = reinterpret_cast<const char*>(static_cast<const Raw*>(a.w) + (NN ? (size_t)(k_last - left) * a.ldw + n0
                                                                          : (size_t)n0 * a.ldw + k_last - left));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kZ; ++i) {
      const int at = i * kThreads + threadIdx.x, depth = piece(at % RC, at / RC) * kVec<T>;
      u32x4 x = {};
      if (depth < left) x = load_16(reinterpret_cast<const Raw*>(zb + zo[i]), left - depth);
      *reinterpret_cast<u32x4*>(lds0 + at * 16) = x;
    }
    if constexpr (kFour) {
      w_block = NN ? (size_t)(k_last - left) * a.ldw + n0 / 32 : (size_t)n0 * a.ldw + (k_last - left) / 32;
#pragma unroll
      for (int i = 0; i < kC; ++i) {
        const bool there = depth_of[i] < left;
        codes[i] = there ? *reinterpret_cast<const u32x4*>(static_cast<const char*>(a.w) + (w_block + co[i]) * 16) : u32x4{};
        scale[i] = there ? a.scales[w_block + co[i]] : 127u;
      }
      put_four(lds0);
    }
#pragma unroll
    for (int i = 0; i < (kFour ? 0 : kW); ++i) {
      const int at = i * kThreads + threadIdx.x;
      const int depth = NN ? at / (BN / kVec<T>) : piece(at % RC, at / RC) * kVec<T>;
      u32x4 x = {};
      if (depth < left) x = load_16(reinterpret_cast<const Raw*>(wb + wo[i]), NN ? w_count[i] : left - depth);
      *reinterpret_cast<u32x4*>(lds0 + BM * RB + at * 16) = x;
    }
    __syncthreads();
    multiply(lds0);
  }

  if (split == 0) expand_tile<T, NN, MB, NB, WM, WN, RB>(a, t0, n0, lds0, lds1, acc);
  const int n = n0 + wn + NB * l;
  if (n >= a.N) return;
  if (ta.part) {
    float* const y = ta.part + ((size_t)split * a.T + t0 + wm) * a.N + n;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int row = 16 * i + 4 * g + v;
        if (t0 + wm + row >= a.T) continue;
        float* const p = y + (size_t)row * a.N;
        float o[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) o[j] = acc[i][j][v];
        store_some(p, o, a.N - n);
      }
    return;
  }
  float bias[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) bias[j] = a.bias && n + j < a.N ? a.bias[n + j] : 0.0f;
  Raw* const y = static_cast<Raw*>(a.y) + (t0 + wm) * a.N + n;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int row = 16 * i + 4 * g + v;
      if (t0 + wm + row >= a.T) continue;
      Raw o[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) o[j] = T::narrow(acc[i][j][v] + bias[j]);
      store_some(y + (size_t)row * a.N, o, a.N - n);
    }
}

#if !CP4_TILE_FOUR
// The depth's parts, in their order, and the bias.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const float* part, const float* bias, void* y, size_t n, int N, int splits) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  typename T::raw* const o = static_cast<typename T::raw*>(y) + i;
  if (n % 4 == 0 && N % 4 == 0) {
    f32x4 x = {};
    int s = 0;
    for (; s + 8 <= splits; s += 8) {
      f32x4 y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = *reinterpret_cast<const f32x4*>(part + (s + e) * n + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) x += y[e];
    }
    for (; s < splits; ++s) x += *reinterpret_cast<const f32x4*>(part + s * n + i);
    if (bias) {
      const int c = (int)(i % N);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] += bias[c + j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = T::narrow(x[j]);
    return;
  }
  for (int j = 0; j < 4 && i + j < n; ++j) {
    float x = part[i + j];
    for (int s = 1; s < splits; ++s) x += part[s * n + i + j];
    if (bias) x += bias[(i + j) % N];
    o[j] = T::narrow(x);
  }
}

#endif

template <class T, bool NN, bool Direct, int MB, int NB, int WM, int WN, int RB, int Rooms>
void launch(const TileArgs& t, hipStream_t st) {
  tile_kernel<T, NN, Direct, MB, NB, WM, WN, RB, Rooms><<<die_grid((long)t.mt * t.nt * t.splits), 64 * WM * WN, 0, st>>>(t);
}
// (fp32: its parts take the registers of 128 columns a wave; through registers and w in 4 bits: the two smaller shapes)
template <class T, bool NN, bool Direct>
void launch_shape(const TileArgs& t, int which, hipStream_t st) {
  if constexpr (Direct && !__is_same(T, F32) && !kFour) {
    if (which == 0) return launch<T, NN, true, 4, 8, 2, 2, 64, 3>(t, st);
    if (which == 3) return launch<T, NN, true, 4, 8, 4, 2, 128, 2>(t, st);
  }
  if (which == 1) return launch<T, NN, Direct, 4, 2, 2, 4, 128, Direct ? 4 : 2>(t, st);
  launch<T, NN, Direct, 4, 4, 1, 4, 128, 2>(t, st);
}
template <class T>
void launch_type(const TileArgs& t, int which, bool nn, bool direct, hipStream_t st) {
  if (direct) nn ? launch_shape<T, true, true>(t, which, st) : launch_shape<T, false, true>(t, which, st);
  else nn ? launch_shape<T, true, false>(t, which, st) : launch_shape<T, false, false>(t, which, st);
}

#if !CP4_TILE_FOUR
constexpr int kShapes = 4, kRows[kShapes] = {128, 128, 64, 256}, kCols[kShapes] = {256, 128, 256, 256};
#endif

template <class... Args>
void launch_dtype(const TileArgs& t, int dtype, Args... args) {
  if (dtype == CP4_DTYPE_F32) launch_type<F32>(t, args...);
  else if (dtype == CP4_DTYPE_BF16) launch_type<BF16>(t, args...);
  else launch_type<F16>(t, args...);
}

}  // namespace

#if CP4_TILE_FOUR
void four_launch(const TileArgs& t, int dtype, int which, bool nn, bool direct, hipStream_t st) {
  launch_dtype(t, dtype, which, nn, direct, st);
}
#else
void four_launch(const TileArgs& t, int dtype, int which, bool nn, bool direct, hipStream_t st);

// Which shape of tile, and in how many parts its depth: the least time by a model of what was measured at a depth of
// 4096 (microseconds; 16-bit types, fp32 in brackets), one tile on a compute unit and two of them, whose waits
// overlap where the LDS has room for both:
//   128 x 256: 74, 132 (nn 74, 116)
//   128 x 128: 37, 75 (nn 42, 88)  [192, 390; nn 190, 376]
//    64 x 256: 51, 69 (nn 55, 76)  [218, 340; nn 213, 293]
//   256 x 256: 97, 194, with up to 5 of 8 units busy 80 (nn 102, 204)
// The parts of a split depth cost their way to memory and back at 2.5 TB/s and a launch of 5 us.  At 50 sizes of
// 64 .. 8192 tokens the choice was 3 % from the best of all shapes and splits on the average and 15 % at worst; the shapes
// differ by up to 3 times: 100 tokens of 4096 x 4096 take 25 us (128 x 128 in four parts) and 82 (256 x 256), 8192 tokens
// 223 us (256 x 256) and 331 (128 x 128), 6000 tokens nn 206 us (128 x 256), 224 (256 x 256) and 239 (64 x 256).  Parts other
// than powers of two fill the chip where those leave a round half empty: 300 tokens fp32 4096 x 4096 97 -> 87 us (nn 103 -> 84).
TilePlan tile_plan(size_t T, int K, int N, int dtype, bool nn, bool aligned, bool four) {
  static constexpr float k16[2][kShapes][2] = {{{74, 132}, {37, 75}, {51, 69}, {97, 194}}, {{74, 116}, {42, 88}, {55, 76}, {102, 204}}};
  static constexpr float k32[2][kShapes][2] = {{{}, {192, 390}, {218, 340}, {}}, {{}, {190, 376}, {213, 293}, {}}};
  // (w in 4 bits)
  static constexpr float k16_four[2][kShapes][2] = {{{}, {48, 90}, {64, 88}, {}}, {{}, {45, 86}, {62, 84}, {}}};
  static constexpr float k32_four[2][kShapes][2] = {{{}, {134, 230}, {142, 218}, {}}, {{}, {125, 223}, {138, 200}, {}}};
  const long units = num_compute_units();
  const bool f32 = dtype == CP4_DTYPE_F32, some = f32 || !aligned || four;
  TilePlan best{};
  for (int w = some ? 1 : 0; w < (some ? 3 : kShapes); ++w) {
    const int KS = f32 || w == 0 ? 32 : 64, steps = (K + KS - 1) / KS;
    const long tiles = (long)((T + kRows[w] - 1) / kRows[w]) * ((N + kCols[w] - 1) / kCols[w]);
    const float* const us = four ? (f32 ? k32_four[nn][w] : k16_four[nn][w]) : f32 ? k32[nn][w] : k16[nn][w];
    for (int s = 1; s <= 64 && s <= std::max(1, steps / 4) && (s == 1 || tiles * s <= 4 * units); s += s < 8 ? 1 : s < 16 ? 2 : s < 32 ? 4 : 8) {
      const int each = (steps + s - 1) / s, parts = (steps + each - 1) / each;
      const long wgs = tiles * parts, most = (wgs + units - 1) / units;
      const double deep = KS * each / 4096.0;
      double cost = 3.0 + deep * (most / 2 * us[1] + most % 2 * (w == 3 && !nn && wgs <= units * 5 / 8 ? 80.0 : us[0]));
      if (s > 1) cost += 5.0 + (double)T * N * (parts + 0.5) * 4.0 / 2.5e6;
      if (!best.splits || cost < best.cost) best = {w, parts, each, cost};
    }
  }
  return best;
}
int tile_rows(const TilePlan& p) { return kRows[p.which]; }
int tile_cols(const TilePlan& p) { return kCols[p.which]; }

// Whether the LDS can be filled directly: 16-byte boundaries, and a thread's places in a tile as 32-bit byte offsets.
bool tile_direct(const ProjectArgs& a, int dtype, bool nn) {
  const size_t e = dtype == CP4_DTYPE_F32 ? 4 : 2, vec = 16 / e;
  if (a.scales) return !((size_t)a.z & 15) && a.ldz % vec == 0 && a.ldz * e * 256 < (size_t)1 << 31;
  if (((size_t)a.z & 15) || ((size_t)a.w & 15) || a.ldz % vec || a.ldw % vec || (nn ? a.N : a.K) % vec) return false;
  return a.ldz * e * 256 < (size_t)1 << 31 && a.ldw * e * 256 < (size_t)1 << 31;
}

hipError_t parts_join(const float* part, const float* bias, void* y, size_t T, int N, int splits, int dtype, hipStream_t st) {
  const size_t n = T * (size_t)N;
  const unsigned grid = (unsigned)((n + 1023) / 1024);
  if (dtype == CP4_DTYPE_F32) join_kernel<F32><<<grid, 256, 0, st>>>(part, bias, y, n, N, splits);
  else if (dtype == CP4_DTYPE_BF16) join_kernel<BF16><<<grid, 256, 0, st>>>(part, bias, y, n, N, splits);
  else join_kernel<F16><<<grid, 256, 0, st>>>(part, bias, y, n, N, splits);
  return hipGetLastError();
}

hipError_t tile_launch(const ProjectArgs& a, const TilePlan& plan, float* part, int dtype, bool nn, hipStream_t st) {
  TileArgs t{};
  t.p = a;
  t.part = plan.splits > 1 ? part : nullptr;
  t.mt = (int)((a.T + kRows[plan.which] - 1) / kRows[plan.which]);
  t.nt = (a.N + kCols[plan.which] - 1) / kCols[plan.which];
  t.splits = plan.splits;
  t.steps = plan.each;
  const bool d = tile_direct(a, dtype, nn);
  if (a.scales) four_launch(t, dtype, plan.which, nn, d, st);
  else launch_dtype(t, dtype, plan.which, nn, d, st);
  if (const hipError_t e = hipGetLastError()) return e;
  return plan.splits > 1 ? parts_join(part, a.bias, a.y, a.T, a.N, plan.splits, dtype, st) : hipSuccess;
}

#endif

}  // namespace adapter
}  // namespace cp4
