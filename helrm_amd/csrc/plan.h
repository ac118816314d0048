// plan.h -- the tiles of the products of products.hip: which of the two sizes,
// how many pieces of k, and the launches of the loss's.  Host code alone.
#pragma once
#include <algorithm>
#include <initializer_list>

namespace clr {

constexpr int STEP = 64;                 // k of a step
struct Shape { long M, N; };
inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

// The tile and the splits of products in one launch: the least time of their
// rounds over the 256 CUs, which hold one 256 x 256 tile or two 128 x 128 ones
// (whose steps and ends overlap).  Microseconds, measured: a step 1.6 and 1.0,
// the end of a tile 8.5 and 6, a small tile alone on its CU 0.55 of that.  The
// large tile has half the traffic for each product, the small one fills the
// GPU with a quarter of the rows.  8192 x 4096 over 4096, gate gradient: 323 us
// large, 349 small; 2048 x 8192 over 512, gate: 67 us large, 54 small.
struct Plan {
  bool big;
  int splits;
  int tile() const { return big ? 256 : 128; }      // rows and columns
  int threads() const { return big ? 512 : 256; }   // of its workgroup
};
inline Plan plan_of(std::initializer_list<Shape> shapes, long steps, bool gate, bool may_split) {
  Plan best{};
  double least = 1e30;
  for (int big = 0; big < 2; big++) {
    const long size = big ? 256 : 128;
    long tiles = 0;
    double results = 0;
    for (const Shape& s : shapes) {
      tiles += ceil_div(s.M, size) * ceil_div(s.N, gate ? size / 2 : size);
      results += (double)s.M * s.N * (gate ? 2 : 1);
    }
    for (int s = 1; s <= (may_split ? 16 : 1); s++) {
      if (s > 1 && steps / s < 4) break;
      const double sums = s > 1 ? 4.0 + (s + 1) * results * 4 / 3e6 : 0.0;   // of a kernel more, and its traffic
      const long rounds = ceil_div(tiles * s, 256), each = ceil_div(steps, s);
      const double t = (big ? rounds * (each * 1.6 + 8.5) : (rounds + 1) / 2 * (each * 1.0 + 6) * (rounds == 1 ? 0.55 : 1.0)) + sums;
      if (t < least) { least = t; best = {big != 0, s}; }
    }
  }
  return best;
}
inline long steps_of(long K, int pairs) { return ceil_div(K, STEP) * pairs; }

// M rows against N rows of a table, each row's softmax left in `parts` pieces, a
// tile's columns each.  One choice of the tile for the whole product, which
// goes in launches of `columns` table rows, a multiple of the tile: a launch has
// less than 2^32 threads (2^22 tiles and those of one column more).
struct SoftmaxPlan {
  Plan plan;
  int parts;
  long columns;
};
inline SoftmaxPlan softmax_plan(long M, long N, long K, int pairs) {
  const Plan plan = plan_of({{M, N}}, steps_of(K, pairs), false, false);
  const long size = plan.tile(), parts = ceil_div(N, size);
  const long launches = ceil_div(ceil_div(M, size) * parts, 1L << 22);
  return {plan, (int)parts, ceil_div(parts, launches) * size};
}

}  // namespace clr
