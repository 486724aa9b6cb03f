// Which kernel a shared projection runs on (include/cp4/adapter.h).
#include <algorithm>

#include "adapter.h"

namespace cp4 {
namespace adapter {
namespace {

// The rows kernel or tiles, for tokens that both take.  A tile takes its adapters a few at a time, some 0.6 us each
// (fp32: 1.2), the rows kernel's waves share them; how many different ones there are only the device knows: at most G.
// (bf16, 4096 x 4096, rank 16, rows kernel and tiles: 20 tokens of 2 adapters 17 us and 21, of 20 adapters 26 and 40; 64 tokens of
// 2 adapters 26 and 22, of 64 adapters 42 and 55; 4096 x 14336, 20 tokens of 2 adapters 50 and 33.)
bool by_rows(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four) {
  const RowsPlan rows = nn ? RowsPlan{} : rows_plan(T, K, N, dtype, four, direct);
  if (!rows.splits || T <= 16) return rows.splits;                   // (up to 16 tokens: within 8 % of the tiles at worst)
  const double adapters = (double)std::min<size_t>(T, G);
  return rows.cost + rows.adapter * adapters <=
         tile_plan(T, K, N, dtype, nn, direct, four).cost + (dtype == CP4_DTYPE_F32 ? 1.2 : 0.6) * adapters;
}

// Rows of the tiles' launch; the rest, less than a tile's, is cheaper on its own where it would take a round of
// tiles of its own.
size_t main_rows(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four) {
  if (T <= 256) return T;
  size_t best = T;
  double least = tile_plan(T, K, N, dtype, nn, direct, four).cost;
  for (size_t tile : {256, 128}) {
    const size_t rest = T % tile;
    if (!rest || T <= 2 * tile) continue;
    const double other = by_rows(rest, K, N, G, dtype, nn, direct, four) ? rows_plan(rest, K, N, dtype, four, direct).cost
                                                                   : tile_plan(rest, K, N, dtype, nn, direct, four).cost;
    const double cost = tile_plan(T - rest, K, N, dtype, nn, direct, four).cost + other + 6.0;    // (a launch and its start)
    if (cost < least) {
      least = cost;
      best = T - rest;
    }
  }
  return best;
}

hipError_t launch(const ProjectArgs& a, float* part, int dtype, bool nn, bool direct, hipStream_t st) {
  const bool four = a.scales;
  if (by_rows(a.T, a.K, a.N, a.G, dtype, nn, direct, four)) return rows_launch(a, rows_plan(a.T, a.K, a.N, dtype, four, direct), part, dtype, st);
  return tile_launch(a, tile_plan(a.T, a.K, a.N, dtype, nn, direct, four), part, dtype, nn, st);
}

}  // namespace

namespace {
// The operands of a projection with W as values in memory.
size_t unpacked_row(int cols) { return ((size_t)cols + 7) / 8 * 8; }
double cost_of(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four) {
  const size_t main = main_rows(T, K, N, G, dtype, nn, direct, four);
  double cost = 0.0;
  for (size_t rows : {main, T - main}) {
    if (!rows) continue;
    cost += by_rows(rows, K, N, G, dtype, nn, direct, four) ? rows_plan(rows, K, N, dtype, four, direct).cost
                                                            : tile_plan(rows, K, N, dtype, nn, direct, four).cost;
  }
  return cost;
}
// Whether W is unpacked: in 16 bits from some 600 tokens on, where the larger tiles take whole cache lines of W (4096 x 4096:
// 512 tokens 34 us from codes, 35 through memory; 1024 tokens 50 and 45; 8192 tokens 337 and 195).  fp32 reads codes with three
// matrix instructions where values take six (8192 tokens 929 us, values 1212).
bool unpacks(size_t T, int K, int N, int G, int dtype, bool nn) {
  if (dtype == CP4_DTYPE_F32 || K % 8 || N % 8 || T <= 64) return false;
  return cost_of(T, K, N, G, dtype, nn, true, false) + 3.0 + (double)K * N * 2.53 / 5.0e6 < cost_of(T, K, N, G, dtype, nn, true, true);
}
}  // namespace

size_t unpack_bytes(size_t T, int K, int N, int G, int dtype, bool nn) {
  return unpacks(T, K, N, G, dtype, nn) ? (size_t)(nn ? K : N) * unpacked_row(nn ? N : K) * 2 : 0;
}
hipError_t unpack_launch(ProjectArgs& a, void* room, int dtype, bool nn, hipStream_t st) {
  if (!a.scales || !tile_direct(a, dtype, nn) || !unpacks(a.T, a.K, a.N, a.G, dtype, nn)) return hipSuccess;
  const int rows = nn ? a.K : a.N, cols = nn ? a.N : a.K;
  const size_t ld = unpacked_row(cols);
  if (const hipError_t e = mx4_unpack(a.w, a.scales, rows, cols, dtype, room, ld, st)) return e;
  a.w = room;
  a.ldw = ld;
  a.scales = nullptr;
  return hipSuccess;
}

// Enough for each choice that the operands' alignment makes.
size_t project_part_bytes(size_t T, int K, int N, int G, int dtype, bool nn, bool four) {
  size_t most = 0;
  const auto part = [&](size_t rows, bool direct) {
    const RowsPlan few = rows_plan(rows, K, N, dtype, four, direct);
    if (by_rows(rows, K, N, G, dtype, nn, direct, four)) most = std::max(most, few.splits > 1 ? few.splits * rows * N * 4 : 0);
    else most = std::max(most, tile_part_bytes(tile_plan(rows, K, N, dtype, nn, direct, four), rows, N));
  };
  if (four && unpacks(T, K, N, G, dtype, nn)) most = project_part_bytes(T, K, N, G, dtype, nn, false);
  for (bool direct : {false, true}) {
    if (direct && dtype == CP4_DTYPE_F32) break;                     // (the same plans)
    const size_t main = main_rows(T, K, N, G, dtype, nn, direct, four);
    part(T, direct);
    if (main == T) continue;
    part(main, direct);
    part(T - main, direct);
  }
  return most;
}

void project_plan(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four, cp4_adapter_launch (&launches)[2]) {
  const auto one = [&](size_t rows) {
    if (!rows) return cp4_adapter_launch{};
    if (by_rows(rows, K, N, G, dtype, nn, direct, four)) return cp4_adapter_launch{rows, 0, 0, rows_plan(rows, K, N, dtype, four, direct).splits};
    const TilePlan p = tile_plan(rows, K, N, dtype, nn, direct, four);
    return cp4_adapter_launch{rows, tile_rows(p), tile_cols(p), p.splits};
  };
  const size_t main = main_rows(T, K, N, G, dtype, nn, direct, four);
  launches[0] = one(main);
  launches[1] = one(T - main);
}

bool project_sums_planes(const ProjectArgs& a, int dtype, bool nn) {
  return by_rows(a.T, a.K, a.N, a.G, dtype, nn, tile_direct(a, dtype, nn), a.scales);
}

hipError_t project_launch(const ProjectArgs& a, float* part, int dtype, bool nn, hipStream_t st) {
  const bool direct = tile_direct(a, dtype, nn), four = a.scales;
  const size_t main = main_rows(a.T, a.K, a.N, a.G, dtype, nn, direct, four);
  if (main == a.T) return launch(a, part, dtype, nn, direct, st);
  const size_t e = dtype == CP4_DTYPE_F32 ? 4 : 2;
  ProjectArgs first = a, rest = a;
  first.T = main;
  rest.T = a.T - main;
  rest.z = static_cast<const char*>(a.z) + main * a.ldz * e;
  if (a.h) rest.h = a.h + main * a.Rp;
  if (a.ids) rest.ids = a.ids + main;
  rest.y = static_cast<char*>(a.y) + main * a.N * e;
  if (const hipError_t err = launch(first, part, dtype, nn, direct, st)) return err;
  return launch(rest, part, dtype, nn, direct, st);
}

}  // namespace adapter
}  // namespace cp4
