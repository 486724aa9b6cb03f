// Products of matrices in two float16 parts for the Muon step (muon.h): C = alpha E + beta P Q^T of many matrices in one
// launch, on the matrix cores.
//
// A value is hi + lo, 22 bits, a product hi hi + hi lo + lo hi: what is dropped is below 2^-22 of it, so three
// float16 instructions stand for an fp32 product (16 times an fp32 matrix instruction's work a cycle each; bfloat16 would need
// six for as many bits, and two of its parts leave an orthogonalised 1024 x 1024 matrix 2.4e-5 off 64 bits
// where these leave 1.8e-6 and fp32 1.7e-6; of updates of few directions, cp4/muon.h).  Newton-Schulz keeps its matrices' values below 3, so float16's range is no
// limit.
//
// A tile is 256 x 256 (eight waves of 128 x 64), 128 x 128 (four of 64 x 64, two workgroups a compute unit) or 64 x 64 (four
// of 32 x 32, seven steps under way); a step is 32 of the depth, one cache line of every row, from memory to the LDS without
// passing a register.  The larger two read an operand's second parts and the next step's first ones while the others are
// multiplied.  A wave's column block j holds the columns NB l + j, so that a lane has NB consecutive values
// of a row; its four rows of a block are consecutive too, so C and C transposed leave in wide stores both.
// Symmetric products (two of the three of an iteration) have the tiles on and below the diagonal alone, the others are
// mirrored: 4 instead of 6 m^3 for a square matrix.  a X is no addition but a on the diagonal of b A + c A A, 134 MB less to
// read of 2048 x 4096 by four.
//
// Measured (traced): four matrices of 2048 x 4096, a launch each: A 247 us, b A + c A A 143, X 333, which is 0.89, 0.77 and 1.24 PFLOP/s
// of float16 (the library's float16 product of 8192^3 reaches 1.1 on the card): bound by the matrix cores' clock under
// load, A and its square by 144 tiles on 256 compute units.  777 x 1001: 12 us each, which is seven steps' latency and the
// launch's ends.
#include <algorithm>
#include <type_traits>

#include "die_order.h"
#include "muon.h"

namespace cp4 {
namespace muon {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum Kind { kParts, kFinal, kPartial };

struct TileArgs {
  Product p[kProducts];
  unsigned first[kProducts];                       // each entry's first workgroup; ~0: no entry
  unsigned tiles[kProducts];                       // of a matrix
  unsigned total;
  int splits, steps;                               // steps: of a part of the depth (the last one may have fewer)
};
static_assert(sizeof(TileArgs) <= 4096, "kernel arguments");

constexpr int wait_for(int loads) { return (loads & 15) | (loads >> 4) << 14 | 7 << 4; }

// A wave has MB x NB blocks of 16 x 16, a workgroup 2 x WN waves; the LDS has room for so many steps.
template <int MB, int NB, int WN, int Rooms, int What>
__global__ __launch_bounds__(128 * WN, Rooms > 2 ? 1 : 2) void product_kernel(const TileArgs a) {
  constexpr int kThreads = 128 * WN, B = 32 * MB, kLoads = B * 8 / kThreads, kRoom = 2 * B * 128;
  static_assert(B == 16 * NB * WN && B * 8 % kThreads == 0, "a square tile, in whole loads");
  // (variables of their own, so that the compiler knows a load into one from a read of another)
  __shared__ __attribute__((aligned(1024))) char lds0[kRoom], lds1[kRoom], lds2[Rooms > 2 ? kRoom : 16], lds3[Rooms > 2 ? kRoom : 16],
      lds4[Rooms > 4 ? kRoom : 16], lds5[Rooms > 4 ? kRoom : 16], lds6[Rooms > 4 ? kRoom : 16], lds7[Rooms > 4 ? kRoom : 16];
  const int place = die_place(blockIdx.x, a.total);
  if (place < 0) return;
  const int entry = entry_of(a.first, place);
  const Product& p = a.p[entry];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
  const unsigned in_entry = place - a.first[entry];
  const unsigned split = in_entry % a.splits, matrix = in_entry / a.splits / a.tiles[entry];
  const int tile = in_entry / a.splits % a.tiles[entry];
  int tm, tn;
  if (p.symmetric) {
    tm = (int)((__builtin_sqrtf(8.0f * tile + 1.0f) - 1.0f) * 0.5f);
    while (tm * (tm + 1) / 2 > tile) --tm;
    while ((tm + 1) * (tm + 2) / 2 <= tile) ++tm;
    tn = tile - tm * (tm + 1) / 2;
  } else {                                         // up to eight columns of tiles wide, then the next ones
    const int mt = (p.R + B - 1) / B, nt = (p.N + B - 1) / B, band = tile / (8 * mt), in_band = tile % (8 * mt), wide = min(8, nt - 8 * band);
    tm = in_band / wide;
    tn = 8 * band + in_band % wide;
  }
  const int R = p.R, N = p.N, m0 = tm * B, n0 = tn * B, wm = 16 * MB * (wave / WN), wn = 16 * NB * (wave % WN);
  const size_t ldk = padded(p.K) * 4, ldn = padded(p.N) * 4, ldr = padded(p.R) * 4;
  const int depth = (int)(ldk / 128), k_first = split * a.steps, steps = min(depth - k_first, a.steps);
  const char* pb = p.P + (size_t)matrix * p.R * ldk + m0 * ldk + (size_t)k_first * 128;
  const char* qb = p.Q + (size_t)matrix * p.N * ldk + n0 * ldk + (size_t)k_first * 128;
  // A thread's places: the LDS is filled in the threads' order; rows beyond the operand's are read again from its
  // last one (what they give is not stored), and a row's pieces lie in another order in each row, so that a column of
  // them is in all banks.
  unsigned po[kLoads], qo[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = i * kThreads + threadIdx.x, row = at / 8, piece = (at % 8) ^ (row & 7);
    const int in = row % (16 * NB), col = row - in + NB * (in & 15) + in / 16;
    po[i] = (unsigned)(min(row, R - 1 - m0) * ldk) + piece * 16;
    qo[i] = (unsigned)(min(col, N - 1 - n0) * ldk) + piece * 16;
  }
  // (by a vector load, older than all others, so that nobody waits for it; a product without them: 1)
  float t0 = 1.0f;
  if (What != kPartial && p.t0) {
    unsigned at = matrix;
    asm volatile("" : "+v"(at));
    t0 = p.t0[at];
  }
  int brought = 0;
  auto bring = [&](char* lds) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(pb + po[i]),
                                       (__attribute__((address_space(3))) void*)(lds + (i * kThreads + wave * 64) * 16), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(qb + qo[i]),
                                       (__attribute__((address_space(3))) void*)(lds + B * 128 + (i * kThreads + wave * 64) * 16), 16, 0, 0);
    const bool more = ++brought < steps;           // (beyond the last step that one again)
    pb += more ? 128 : 0;
    qb += more ? 128 : 0;
  };
  f32x4 acc[MB][NB] = {};
  const int p_at = (wm + l) * 128, q_at = B * 128 + (wn + l) * 128;
  const int first_part = (g ^ (l & 7)) * 16, second_part = ((4 + g) ^ (l & 7)) * 16;
  auto read_p = [&](const char* lds, int part, f16x8 (&x)[MB]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MB; ++i) x[i] = *reinterpret_cast<const f16x8*>(lds + p_at + part + i * 16 * 128);
  };
  auto read_q = [&](const char* lds, int part, f16x8 (&x)[NB]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j) x[j] = *reinterpret_cast<const f16x8*>(lds + q_at + part + j * 16 * 128);
  };
  auto products = [&](const f16x8 (&x)[MB], const f16x8 (&y)[NB]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i], y[j], acc[i][j], 0, 0, 0);
  };
  auto ahead = [&](char* lds) __attribute__((always_inline)) {
    bring(lds);
    asm volatile("" ::: "memory");                 // (their order is what the waits count on)
    __builtin_amdgcn_sched_barrier(0);
  };
  if constexpr (Rooms == 2) {
    // The next operands are read while the last ones are multiplied.  Behind
    // two of a step's three products its room has been read, the next step's has arrived, and the third product covers the
    // reads of that one.
    f16x8 ph[MB], pl[MB], q0[NB], q1[NB];
    auto interleave = [&](auto reads) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < decltype(reads)::value; ++e) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, MB * NB / decltype(reads)::value, 0);
      }
    };
    auto step = [&](char* lds, const char* then, f16x8 (&qh)[NB], f16x8 (&ql)[NB]) __attribute__((always_inline)) {
      read_q(lds, second_part, ql);
      products(ph, qh);
      interleave(std::integral_constant<int, NB>());
      read_p(lds, second_part, pl);
      products(ph, ql);
      interleave(std::integral_constant<int, MB>());
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(wait_for(0));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      bring(lds);
      __builtin_amdgcn_sched_barrier(0);
      read_p(then, first_part, ph);
      read_q(then, first_part, ql);
      products(pl, qh);
      interleave(std::integral_constant<int, MB + NB>());
      __builtin_amdgcn_sched_barrier(0);
    };
    if (steps > 0) {
      ahead(lds0);
      ahead(lds1);
      __builtin_amdgcn_s_waitcnt(wait_for(2 * kLoads));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      read_p(lds0, first_part, ph);
      read_q(lds0, first_part, q0);
      int left = steps;
      for (; left >= 2; left -= 2) {
        step(lds0, lds1, q0, q1);
        step(lds1, lds0, q1, q0);
      }
      if (left > 0) step(lds0, lds1, q0, q1);
      __builtin_amdgcn_s_waitcnt(wait_for(0));     // (the loads beyond the last step)
    }
  } else if (steps > 0) {
    // A step: its own loads have arrived (those of later ones may still be on their way), and nobody reads the last
    // one's room any more.
    auto step = [&](const char* lds, char* into) __attribute__((always_inline)) {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(wait_for((Rooms - 2) * 2 * kLoads));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      bring(into);
      __builtin_amdgcn_sched_barrier(0);
      f16x8 ph[MB], pl[MB], qh[NB], ql[NB];
      read_p(lds, first_part, ph);
      read_q(lds, first_part, qh);
      read_q(lds, second_part, ql);
      read_p(lds, second_part, pl);
      products(ph, qh);
      products(ph, ql);
      products(pl, qh);
    };
    char* const last = Rooms == 4 ? lds3 : lds7;
    ahead(lds0);
    ahead(lds1);
    ahead(lds2);
    if constexpr (Rooms > 4) {
      ahead(lds3);
      ahead(lds4);
      ahead(lds5);
      ahead(lds6);
    }
    int left = steps;                              // (no way out in the middle, so that the loads under way can be counted)
    for (; left >= Rooms; left -= Rooms) {
      step(lds0, last);
      step(lds1, lds0);
      step(lds2, lds1);
      step(lds3, lds2);
      if constexpr (Rooms > 4) {
        step(lds4, lds3);
        step(lds5, lds4);
        step(lds6, lds5);
        step(lds7, lds6);
      }
    }
    if (left > 0) step(lds0, last);
    if (left > 1) step(lds1, lds0);
    if (left > 2) step(lds2, lds1);
    if constexpr (Rooms > 4) {
      if (left > 3) step(lds3, lds2);
      if (left > 4) step(lds4, lds3);
      if (left > 5) step(lds5, lds4);
      if (left > 6) step(lds6, lds5);
    }
    __builtin_amdgcn_s_waitcnt(wait_for(0));       // (the loads beyond the last step)
  }

  const int n = n0 + wn + NB * l;
  if constexpr (What == kPartial) {
    float* const out = p.part + ((size_t)matrix * a.splits + split) * R * N;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = m0 + wm + 16 * i + 4 * g + v;
        float x[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) x[j] = acc[i][j][v];
        if (r < R) store_values<NB>(out, CP4_DTYPE_F32, (size_t)r * N + n, N - n, x);
      }
    return;
  }
  const float t = scale_at(t0, p.four_to_step), next = scale_at(t, 4.0f), over = What == kParts ? t / next : 1.0f;
  const float alpha = p.alpha * (over * (t * t)), beta = p.beta * (1.0f / kScale) * (What == kFinal ? next : over * (t * t) * (t * t));
  const float diagonal = p.diagonal * kScale * over;
  const char* const E = p.E ? p.E + (size_t)matrix * R * ldn : nullptr;
  char* const C = p.C + (size_t)matrix * R * ldn;
  char* Ct = nullptr;
  if constexpr (What == kParts) {
    if (p.symmetric && tm != tn) Ct = C;           // (R is N)
    else if (p.Ct) Ct = p.Ct + (size_t)matrix * N * ldr;
  }
  Outputs o;
  Rates rates;
  if constexpr (What == kFinal) {
    o = p.o;
    rates = p.rates;
    const size_t at = (size_t)matrix * R * N;
    const auto shift = [&](void* q, int dtype) { return q ? (char*)q + at * (dtype == CP4_DTYPE_F32 ? 4 : 2) : nullptr; };
    o.param = shift(o.param, o.param_dtype);
    o.copy = shift(o.copy, o.copy_dtype);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int row = m0 + wm + 16 * i + 4 * g;
    float es[4][NB] = {};
    if (E) {                                       // (four rows at once; what is outside is not used)
#pragma unroll
      for (int v = 0; v < 4; ++v) load_parts<NB>(E + (size_t)min(row + v, R - 1) * ldn, min(n, (int)padded(N) - NB), es[v]);
    }
    if (row >= (int)padded(R)) continue;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = row + v;
      float x[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        x[j] = beta * acc[i][j][v];
        x[j] += alpha * es[v][j];
        if (r == n + j) x[j] += diagonal;
        if (r >= R || n + j >= N) x[j] = 0.0f;     // (what fills up the last block of 32)
        acc[i][j][v] = x[j];
      }
      if (r >= R || n >= (int)padded(N)) continue;
      if constexpr (What == kParts) {
        store_parts<NB>(C + (size_t)r * ldn, n, x);
      } else {
#pragma unroll
        for (int j = 0; j < NB; ++j) x[j] *= 1.0f / kScale;
        put_out<NB>(o, rates, (size_t)r * N + n, N - n, x);
      }
    }
    if constexpr (What == kParts)
      if (Ct)
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          float x[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) x[v] = acc[i][j][v];
          if (n + j < N) store_parts<4>(Ct + (size_t)(n + j) * ldr, row, x);
        }
  }
}

// A symmetric C from the parts of its depth: four columns of a row a thread; what lies above the diagonal's tiles (of
// `edge` rows) is read from below it.
__global__ __launch_bounds__(256) void join_kernel(const TileArgs a, int edge) {
  const int entry = entry_of(a.first, blockIdx.x);
  const Product& p = a.p[entry];
  const unsigned fours = (unsigned)padded(p.N) / 4;
  const size_t at = (size_t)(blockIdx.x - a.first[entry]) * 256 + threadIdx.x;
  if (at >= (size_t)p.count * p.R * fours) return;
  const unsigned c = at % fours * 4, r = at / fours % p.R;
  const size_t matrix = at / fours / p.R, size = (size_t)p.R * p.N;
  const float* const part = p.part + matrix * a.splits * size;
  float x[4] = {};
  const bool below = r / edge >= c / edge;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c + j >= p.N) continue;
    const float* const q = part + (below ? (size_t)r * p.N + c + j : (size_t)(c + j) * p.N + r);
    for (int s = 0; s < a.splits; ++s) x[j] += q[s * size];
    x[j] *= p.beta * (1.0f / kScale);
  }
  store_parts<4>(p.C + (matrix * p.R + r) * padded(p.N) * 4, c, x);
}

size_t tiles_of(const Product& p, int edge) {
  const size_t mt = (p.R + edge - 1) / edge, nt = (p.N + edge - 1) / edge;
  return p.symmetric ? mt * (mt + 1) / 2 : mt * nt;
}
size_t all_tiles(const Product* p, int n, int edge) {
  size_t t = 0;
  for (int i = 0; i < n; ++i) t += p[i].count * tiles_of(p[i], edge);
  return t;
}
int depth_of(const Product* p, int n) {
  size_t d = 0;
  for (int i = 0; i < n; ++i) d = std::max(d, padded(p[i].K) / 32);
  return (int)d;
}

constexpr int kEdges[3] = {256, 128, 64};
// The tiles' edge and the parts of the depth by the least time of a model of what was measured (microseconds a step and for the
// launch's ends): 64 x 64 0.225 and 5.5; 128 x 128 one on a compute unit 0.63 and 7.5, two 1.3 and 14; 256 x 256 1.58 and 21 where
// they leave a good part of the units free, 2.2 where all are at work.  (The last product's outputs leave the largest one no
// registers.)
struct Choice {
  int which, splits;
};
Choice choose(const Product* p, int n, bool may_split) {
  const int depth = depth_of(p, n);
  const size_t units = num_compute_units();
  Choice best{2, 1};
  double least = 0.0;
  for (int w = p[0].final; w < 3; ++w) {
    const size_t tiles = all_tiles(p, n, kEdges[w]);
    for (int s = 1; s <= 32 && (s == 1 || (may_split && depth / s >= 16)); ++s) {
      const size_t wgs = tiles * s, once = (wgs + units - 1) / units, twice = (wgs + 2 * units - 1) / (2 * units);
      const int steps = (depth + s - 1) / s;
      double cost = w == 2 ? once * (0.225 * steps + 5.5)
                    : w == 1 ? (once == 1 ? 0.63 * steps + 7.5 : twice * (1.3 * steps + 14.0))
                             : once * ((wgs * 5 <= units * 3 ? 1.58 : 2.2) * steps + 21.0);
      if (s > 1) {
        cost += 6.0;
        for (int i = 0; i < n; ++i) cost += (double)p[i].count * p[i].R * p[i].N * (s + 0.5) * 4.0 / 2.0e6;
      }
      if (least == 0.0 || cost < least) {
        least = cost;
        best = {w, s};
      }
    }
  }
  return best;
}

template <int MB, int NB, int WN, int Rooms>
hipError_t launch(const TileArgs& t, Kind kind, hipStream_t st) {
  const unsigned grid = die_grid((long)t.total);
  if (kind == kParts) {
    product_kernel<MB, NB, WN, Rooms, kParts><<<grid, 128 * WN, 0, st>>>(t);
  } else if (kind == kPartial) {
    product_kernel<MB, NB, WN, Rooms, kPartial><<<grid, 128 * WN, 0, st>>>(t);
  } else {
    if constexpr (MB == 8) return hipErrorInvalidValue;            // (choose() takes the others)
    else product_kernel<MB, NB, WN, Rooms, kFinal><<<grid, 128 * WN, 0, st>>>(t);
  }
  return hipGetLastError();
}

}  // namespace

int product_splits(const Product* p, int n) { return choose(p, n, true).splits; }

hipError_t product_launch(const Product* p, int n, int splits, hipStream_t st) {
  TileArgs t{};
  const Choice c = choose(p, n, splits > 1);
  const int edge = kEdges[c.which], depth = depth_of(p, n);
  t.steps = (depth + splits - 1) / splits;
  t.splits = splits;
  for (int i = 0; i < kProducts; ++i) {
    t.first[i] = ~0u;
    if (i >= n) continue;
    t.p[i] = p[i];
    t.first[i] = t.total;
    t.tiles[i] = (unsigned)tiles_of(p[i], edge);
    t.total += p[i].count * t.tiles[i] * splits;
  }
  const Kind kind = splits > 1 ? kPartial : p[0].final ? kFinal : kParts;
  const hipError_t e = c.which == 0 ? launch<8, 4, 4, 2>(t, kind, st) : c.which == 1 ? launch<4, 4, 2, 2>(t, kind, st) : launch<2, 2, 2, 8>(t, kind, st);
  if (e || splits == 1) return e;
  unsigned grid = 0;
  for (int i = 0; i < n; ++i) {
    t.first[i] = grid;
    grid += (unsigned)(((size_t)p[i].count * p[i].R * (padded(p[i].N) / 4) + 255) / 256);
  }
  join_kernel<<<grid, 256, 0, st>>>(t, edge);
  return hipGetLastError();
}

}  // namespace muon
}  // namespace cp4
