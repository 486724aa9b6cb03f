// Which kernel a shared projection runs on (include/cp4/adapter.h).
#include <algorithm>

#include "adapter.h"

namespace cp4 {
namespace adapter {
namespace {

// What a launch runs on.
struct Choice {
  bool by_rows;
  RowsPlan rows;
  TilePlan tile;
  double cost() const { return by_rows ? rows.cost : tile.cost; }
  int splits() const { return by_rows ? rows.splits : tile.splits; }
  size_t part_bytes(size_t T, int N) const { return splits() > 1 ? (size_t)splits() * T * N * 4 : 0; }
};
// The rows kernel or tiles, for tokens that both take.  A tile takes its adapters a few at a time, some 0.6 us each
// (fp32: 1.2), the rows kernel's waves share them; how many different ones there are only the device knows: at most G.
// (bf16, 4096 x 4096, rank 16, rows kernel and tiles: 20 tokens of 2 adapters 17 us and 21, of 20 adapters 26 and 40; 64 tokens of
// 2 adapters 26 and 22, of 64 adapters 42 and 55; 4096 x 14336, 20 tokens of 2 adapters 50 and 33.)
Choice choose(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four) {
  Choice c{};
  if (!nn) c.rows = rows_plan(T, K, N, dtype, four, direct);
  c.by_rows = c.rows.splits;
  if (c.by_rows && T <= 16) return c;                                // (up to 16 tokens: within 8 % of the tiles at worst)
  c.tile = tile_plan(T, K, N, dtype, nn, direct, four);
  const double adapters = (double)std::min<size_t>(T, G);
  c.by_rows = c.by_rows && c.rows.cost + c.rows.adapter * adapters <= c.tile.cost + (dtype == CP4_DTYPE_F32 ? 1.2 : 0.6) * adapters;
  return c;
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
    const double other = choose(rest, K, N, G, dtype, nn, direct, four).cost();
    const double cost = tile_plan(T - rest, K, N, dtype, nn, direct, four).cost + other + 6.0;    // (a launch and its start)
    if (cost < least) {
      least = cost;
      best = T - rest;
    }
  }
  return best;
}

hipError_t launch(const ProjectArgs& a, const Choice& c, float* part, int dtype, bool nn, hipStream_t st) {
  return c.by_rows ? rows_launch(a, c.rows, part, dtype, st) : tile_launch(a, c.tile, part, dtype, nn, st);
}

// The operands of a projection with W as values in memory.
size_t unpacked_row(int cols) { return ((size_t)cols + 7) / 8 * 8; }
double cost_of(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four) {
  const size_t main = main_rows(T, K, N, G, dtype, nn, direct, four);
  const double cost = choose(main, K, N, G, dtype, nn, direct, four).cost();
  return main == T ? cost : cost + choose(T - main, K, N, G, dtype, nn, direct, four).cost();
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

// Enough for each choice that the operands' alignment makes: of the tiles in 16 bits, of the few rows in every type where W is
// in 4 bits.
size_t project_part_bytes(size_t T, int K, int N, int G, int dtype, bool nn, bool four) {
  size_t most = 0;
  const auto part = [&](size_t rows, bool direct) {
    most = std::max(most, choose(rows, K, N, G, dtype, nn, direct, four).part_bytes(rows, N));
  };
  if (four && unpacks(T, K, N, G, dtype, nn)) most = project_part_bytes(T, K, N, G, dtype, nn, false);
  for (bool direct : {false, true}) {
    if (direct && dtype == CP4_DTYPE_F32 && !four) break;            // (the same plans)
    const size_t main = main_rows(T, K, N, G, dtype, nn, direct, four);
    part(main, direct);
    if (main != T) part(T - main, direct);
  }
  return most;
}

void project_plan(size_t T, int K, int N, int G, int dtype, bool nn, bool direct, bool four, cp4_adapter_launch (&launches)[2]) {
  const auto one = [&](size_t rows) {
    if (!rows) return cp4_adapter_launch{};
    const Choice c = choose(rows, K, N, G, dtype, nn, direct, four);
    return cp4_adapter_launch{rows, c.by_rows ? 0 : tile_rows(c.tile), c.by_rows ? 0 : tile_cols(c.tile), c.splits()};
  };
  const size_t main = main_rows(T, K, N, G, dtype, nn, direct, four);
  launches[0] = one(main);
  launches[1] = one(T - main);
}

bool project_sums_planes(const ProjectArgs& a, int dtype, bool nn) {
  return choose(a.T, a.K, a.N, a.G, dtype, nn, tile_direct(a, dtype, nn), a.scales).by_rows;
}

hipError_t project_launch(const ProjectArgs& a, float* part, size_t part_bytes, int dtype, bool nn, hipStream_t st) {
  const bool direct = tile_direct(a, dtype, nn), four = a.scales;
  const size_t main = main_rows(a.T, a.K, a.N, a.G, dtype, nn, direct, four), e = dtype == CP4_DTYPE_F32 ? 4 : 2;
  const Choice of_main = choose(main, a.K, a.N, a.G, dtype, nn, direct, four);
  if (of_main.part_bytes(main, a.N) > part_bytes) return hipErrorInvalidValue;
  if (main == a.T) return launch(a, of_main, part, dtype, nn, st);
  const Choice of_rest = choose(a.T - main, a.K, a.N, a.G, dtype, nn, direct, four);
  if (of_rest.part_bytes(a.T - main, a.N) > part_bytes) return hipErrorInvalidValue;
  ProjectArgs first = a, rest = a;
  first.T = main;
  rest.T = a.T - main;
  rest.z = static_cast<const char*>(a.z) + main * a.ldz * e;
  if (a.h) rest.h = a.h + main * a.Rp;
  if (a.ids) rest.ids = a.ids + main;
  rest.y = static_cast<char*>(a.y) + main * a.N * e;
  if (const hipError_t err = launch(first, of_main, part, dtype, nn, st)) return err;
  return launch(rest, of_rest, part, dtype, nn, st);
}

}  // namespace adapter
}  // namespace cp4
