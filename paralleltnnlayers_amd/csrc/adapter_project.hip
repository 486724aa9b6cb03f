// Which kernel a shared projection runs on (include/cp4/adapter.h).
#include <algorithm>

#include "adapter.h"

namespace cp4 {
namespace adapter {
namespace {

// Rows of the tiles' launch; the rest, less than a tile's, is cheaper on its own where it would take a round of
// tiles of its own.
size_t main_rows(size_t T, int K, int N, int dtype, bool nn, bool direct) {
  const TilePlan all = tile_plan(T, K, N, dtype, direct);
  size_t best = T;
  double least = all.cost;
  for (size_t tile : {256, 128}) {
    const size_t rest = T % tile;
    if (!rest || T <= 2 * tile) continue;
    // (the rest's own launches: some microseconds, and W once more)
    const bool rows = !nn && rows_plan(rest, K, N, dtype).splits;
    const double w = (double)K * N * (dtype == CP4_DTYPE_F32 ? 4 : 2) / 3.0e6;
    const double cost = tile_plan(T - rest, K, N, dtype, direct).cost + 4.0 +
                        (rows ? 6.0 + w : std::max(w, tile_plan(rest, K, N, dtype, direct).cost));
    if (cost < least) {
      least = cost;
      best = T - rest;
    }
  }
  return best;
}

size_t plan_bytes(size_t T, int K, int N, int dtype, bool direct) {
  const RowsPlan rows = rows_plan(T, K, N, dtype);
  return std::max(tile_part_bytes(tile_plan(T, K, N, dtype, direct), T, N),
                  rows.splits > 1 ? (size_t)rows.splits * T * N * 4 : 0);
}

hipError_t launch(const ProjectArgs& a, float* part, int dtype, bool nn, bool direct, hipStream_t st) {
  const RowsPlan rows = nn ? RowsPlan{} : rows_plan(a.T, a.K, a.N, dtype);
  if (rows.splits) return rows_launch(a, rows, part, dtype, st);
  return tile_launch(a, tile_plan(a.T, a.K, a.N, dtype, direct), part, dtype, nn, st);
}

}  // namespace

size_t project_part_bytes(size_t T, int K, int N, int dtype) {
  size_t most = 0;
  for (bool direct : {false, true}) {
    most = std::max(most, plan_bytes(T, K, N, dtype, direct));
    for (bool nn : {false, true}) {
      const size_t main = main_rows(T, K, N, dtype, nn, direct);
      if (main < T)
        most = std::max({most, plan_bytes(main, K, N, dtype, direct), plan_bytes(T - main, K, N, dtype, direct)});
    }
  }
  return most;
}

bool project_sums_planes(const ProjectArgs& a, int dtype, bool nn) {
  return !nn && rows_plan(a.T, a.K, a.N, dtype).splits;
}

hipError_t project_launch(const ProjectArgs& a, float* part, int dtype, bool nn, hipStream_t st) {
  const bool direct = tile_direct(a, dtype, nn);
  const size_t main = project_sums_planes(a, dtype, nn) ? a.T : main_rows(a.T, a.K, a.N, dtype, nn, direct);
  if (main == a.T) return launch(a, part, dtype, nn, direct, st);
  const size_t e = dtype == CP4_DTYPE_F32 ? 4 : 2;
  ProjectArgs first = a, rest = a;
  first.T = main;
  rest.T = a.T - main;
  rest.z = static_cast<const char*>(a.z) + main * a.ldz * e;
  rest.h = a.h + main * a.Rp;
  rest.ids = a.ids + main;
  rest.y = static_cast<char*>(a.y) + main * a.N * e;
  if (const hipError_t err = launch(first, part, dtype, nn, direct, st)) return err;
  return launch(rest, part, dtype, nn, direct, st);
}

}  // namespace adapter
}  // namespace cp4
