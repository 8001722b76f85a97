// Products of nn.GroupedLinear: all groups in one launch.
//
//   forward       D(o, r) = sum_i w[e](o, i) x(r, i)      rows r of group e
//   gradInput     D(i, r) = sum_o w[e](o, i) gz(r, o)
//   gradWeight    D[e](i, o) += sum_r x(r, i) gz(r, o)     over the rows of group e
//
// A launch per group, as gemm() would have it, leaves most of the device idle behind each (37 groups of some 40 rows, 333 -> 515: three products
// took 785 us); here the pieces of all groups are a launch's work items.  The 64-row (or 256-row) side of a tile is the features', so that a weight
// that meets few rows is read once, in tiles as narrow as the rows.
#include "mm_launch.cuh"
#include "nn_linear.h"

namespace thc {

using namespace mm;

// Entries that do not travel with a launch.
static __global__ void __launch_bounds__(256) group_list_kernel(const __grid_constant__ GroupList piece, GroupEntry *to) {
  pdl_begin();
  for (int i = threadIdx.x; i < piece.count; i += 256) to[i] = piece.few[i];
}
static GroupList make_list(const GroupEntry *e, int n) {
  GroupList l;
  l.count = n;
  l.more = nullptr;
  if (n <= kGroupEntries) {
    std::copy(e, e + n, l.few);
    return l;
  }
  GroupEntry *to = (GroupEntry *)ws_alloc(sizeof(GroupEntry) * n);
  for (int i = 0; i < n; i += kGroupEntries) {
    GroupList piece;
    piece.count = std::min(n - i, kGroupEntries);
    piece.more = nullptr;
    std::copy(e + i, e + i + piece.count, piece.few);
    pdl_launch(group_list_kernel, 1, 256, 0, piece, to + i);
    check_launch("group_list");
  }
  l.more = to;
  return l;
}
// Pieces of at most `width` rows of each group.
static std::vector<GroupEntry> row_tiles(const Groups &g, int width) {
  std::vector<GroupEntry> v;
  long r = 0;
  for (int e = 0; e < g.n; r += g.counts[e++])
    for (long i = 0; i < g.counts[e]; i += width) v.push_back(GroupEntry{e, (int)(r + i), (int)(r + std::min<long>(g.counts[e], i + width))});
  return v;
}
static std::vector<GroupEntry> whole_groups(const Groups &g) {
  std::vector<GroupEntry> v;
  long r = 0;
  for (int e = 0; e < g.n; r += g.counts[e++])
    if (g.counts[e]) v.push_back(GroupEntry{e, (int)r, (int)(r + g.counts[e])});
  return v;
}
// The width of the warp-level engine's tiles that takes the groups' rows in the least time: a tile's cost by width, from the times that
// small_product_us() goes by.
static int small_group_width(const Groups &g) {
  const int widths[4] = {64, 32, 16, 8};
  const double cost[4] = {2.9, 1.9, 1.2, 1.0};
  int best = 64;
  double least = 0;
  for (int i = 0; i < 4; i++) {
    double t = 0;
    for (int e = 0; e < g.n; e++) t += cost[i] * (double)((g.counts[e] + widths[i] - 1) / widths[i]);
    if (!i || t < least) { best = widths[i]; least = t; }
  }
  return best;
}

// The warp-level engine over the groups: any size, pitch and alignment.
static void small_groups(SmallGroups p, const std::vector<GroupEntry> &entries, int bn, bool a_k, bool b_k) {
  p.stalled = stall_ctl().dev_flag;
  const int most = std::max(1, 65535 / p.column_tiles);
  for (size_t i = 0; i < entries.size(); i += most) {
    const int n = (int)std::min(entries.size() - i, (size_t)most);
    p.list = make_list(entries.data() + i, n);
    p.slices = 1;
    p.tiles_per_slice = INT_MAX;
    p.ws = nullptr;
    if (p.kind == kGroupRows) {
      const long tiles = (long)ceil_div(p.M, 64) * n, ktiles = ceil_div(p.K, TC_BK);
      const long slices = small_slices(tiles, ktiles, bn);
      p.tiles_per_slice = ceil_div(ktiles, slices);
      p.slices = ceil_div(ktiles, p.tiles_per_slice);
      if (p.slices > 1) {
        p.ws = (float *)ws_alloc(sizeof(float) * tiles * p.slices * 64 * bn);
        p.tickets = zero_words();
      }
    }
    launch_small_width(p, bn, a_k, b_k);
  }
}

// The "simt" math mode: a product of the FP32 engine for each group.
template <class F> static bool each_group(const Groups &g, F f) {
  THC_CHECK(g.rows <= 1l << 30, "more rows than a launch counts");
  if (ctx().math_mode != 1) return false;
  long r = 0;
  for (int e = 0; e < g.n; r += g.counts[e++])
    if (g.counts[e]) f(e, r, g.counts[e]);
  return true;
}

void group_forward(const Groups &g, const float *x, long ldx, long in, long out, const float *w, const float *b, float *y, int act, float *z) {
  if (each_group(g, [&](int e, long r, long n) {
        LinearTail tail;
        tail.act = act;
        tail.z = z ? z + r * out : nullptr;
        linear_product(x + r * ldx, ldx, n, in, out, w + e * out * in, b ? b + e * out : nullptr, y + r * out, tail);
      }))
    return;
  SmallGroups p = {};
  p.a = small_operand(w, in); p.b = small_operand(x, ldx);
  p.M = (int)out; p.N = 0; p.K = (int)in;
  p.c = y; p.sm = 1; p.sn = out;
  p.alpha = 1.f;
  p.bias = b; p.bias_m = 1;
  p.act = act; p.z = z;
  p.kind = kGroupRows; p.column_tiles = 1;
  p.at = GroupPlaces{out * in, 0, ldx, 0, out, out};
  const int bn = small_group_width(g);
  small_groups(p, row_tiles(g, bn), bn, true, true);
}
void group_grad_input(const Groups &g, const float *gz, long ldg, long in, long out, const float *w, float *gx) {
  if (each_group(g, [&](int e, long r, long n) { gemm('n', 'n', in, n, out, 1.f, w + e * out * in, in, gz + r * ldg, ldg, 0.f, gx + r * in, in); })) return;
  SmallGroups p = {};
  p.a = small_operand(w, in); p.b = small_operand(gz, ldg);
  p.M = (int)in; p.N = 0; p.K = (int)out;
  p.c = gx; p.sm = 1; p.sn = in;
  p.alpha = 1.f;
  p.kind = kGroupRows; p.column_tiles = 1;
  p.at = GroupPlaces{out * in, 0, ldg, 0, in, 0};
  const int bn = small_group_width(g);
  small_groups(p, row_tiles(g, bn), bn, false, true);
}
void group_grad_weight(const Groups &g, const float *x, long ldx, const float *gz, long ldg, long in, long out, float *gw, float scale) {
  if (each_group(g, [&](int e, long r, long n) { gemm('n', 't', in, out, n, scale, x + r * ldx, ldx, gz + r * ldg, ldg, 1.f, gw + e * out * in, in); })) return;
  SmallGroups p = {};
  p.a = small_operand(x, ldx); p.b = small_operand(gz, ldg);
  p.M = (int)in; p.N = (int)out; p.K = 0;
  p.c = gw; p.sm = 1; p.sn = in;
  p.alpha = scale; p.beta = 1.f;
  p.kind = kGroupSums;
  const int bn = small_tile_width(out);
  p.column_tiles = ceil_div(out, bn);
  p.at = GroupPlaces{0, ldx, ldg, out * in, 0, 0};
  small_groups(p, whole_groups(g), bn, false, false);
}

}  // namespace thc
