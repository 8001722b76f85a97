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
// The warp-level engine's time, by small_product_us()'s figures: `features` tiles of 64, times `tiles` along the groups' rows (or the other features), which
// take `steps` k tiles in all.  A tile's start and end cost as much as three k tiles.
static double small_groups_us(double features, double tiles, double steps, int bn, bool aligned) {
  const double blocks = features * tiles / ctx().sm_count, depth = bn == 64 ? 3 : bn == 8 ? 5 : 4, resident = std::min(std::max(blocks, 1.0), depth);
  const double step = bn == 64 ? 1.35 + 0.4 * resident : bn == 32 ? 1.3 + 0.15 * resident : bn == 16 ? 0.6 + 0.15 * resident : 0.45 + 0.15 * resident;
  return 5 + (aligned ? 1.0 : 1.3) * step * features * (steps + 3 * tiles) / ctx().sm_count / resident;
}
// The two-SM engine's k tile over FP32 values: 16 groups of 512 rows, 1024 -> 4096, 298 / 342 / 336 / 495 us with tiles of 256 / 192 / 128 / 64 columns.
static double group_tile_us(int width) { return width == 256 ? 1.25 : width == 192 ? 0.91 : width == 128 ? 0.71 : 0.52; }
static long tiles_of(const Groups &g, long width) {
  long t = 0;
  for (int e = 0; e < g.n; e++) t += (g.counts[e] + width - 1) / width;
  return t;
}
struct Choice { bool engine; int width; };
// For kGroupRows: the engine and the width of its tiles along the rows that finish first.  The two-SM engine takes all tiles round by round, with two k
// tiles for a tile's epilogue and, where its operands have to be copied, `pack` bytes at 2 TB/s.
static Choice choose_rows(const Groups &g, long features, long K, bool small_aligned, double pack, bool tma) {
  Choice best{false, 64};
  double least = 0;
  const long ktiles = (K + 31) / 32;
  for (int w : {64, 32, 16, 8}) {
    const double n = (double)tiles_of(g, w), us = small_groups_us((double)((features + 63) / 64), n, n * (double)ktiles, w, small_aligned);
    if (!least || us < least) { best = Choice{false, w}; least = us; }
  }
  if (!tma) return best;
  for (int w : {256, 192, 128, 64}) {
    const double tiles = (double)((features + 255) / 256) * (double)tiles_of(g, w);
    const double us = 10 + std::ceil(tiles / (ctx().sm_count / 2)) * (double)(ktiles + 2) * group_tile_us(w) + (pack ? 5 + pack / 2e6 : 0);
    if (us < least) { best = Choice{true, w}; least = us; }
  }
  return best;
}

// A handful of rows in each group, K-major operands in whole 16-byte pieces: the weights' bytes are the bound (few_rows_kernel).
static bool few_rows_groups(SmallGroups p, const Groups &g) {
  if (!p.a.vec4 || !p.b.vec4 || p.K % 4) return false;
  long most = 0;
  for (int e = 0; e < g.n; e++) most = std::max(most, g.counts[e]);
  if (most > 4) return false;
  const std::vector<GroupEntry> entries = row_tiles(g, 4);
  for (size_t i = 0; i < entries.size(); i += 65535) {
    p.list = make_list(entries.data() + i, (int)std::min(entries.size() - i, (size_t)65535));
    p.stalled = stall_ctl().dev_flag;
    launch_few_rows_kernel(p, (int)most, dim3(1, (unsigned)p.list.count));
    check_launch("few_rows");
  }
  return true;
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

// ---- the two-SM engine ----------------------------------------------------------------------------------------------
// An operand's lines at a pitch that TMA takes: as they are, or copied.
struct Lines {
  const float *p;
  long lines, run, ld;
  bool ok() const { return raw_matrix_ok(p, ld); }
};
static double pack_bytes(const Lines &a, const Lines &b) {
  return (a.ok() ? 0 : 8. * (double)a.lines * (double)a.run) + (b.ok() ? 0 : 8. * (double)b.lines * (double)b.run);
}
static void pack(Lines &a, Lines &b) {
  PackJob jobs[2] = {};
  Lines *l[2] = {&a, &b};
  bool any = false;
  for (int i = 0; i < 2; i++) {
    if (l[i]->ok()) continue;
    any = true;
    const long ld = (l[i]->run + 3) / 4 * 4;
    float *to = (float *)ws_alloc(sizeof(float) * l[i]->lines * ld);
    jobs[i] = PackJob{l[i]->p, to, l[i]->lines, l[i]->run, l[i]->ld, ld};
    l[i]->p = to; l[i]->ld = ld;
  }
  if (any) launch_pack(jobs[0], jobs[1]);
}
template <class P, class Attach>
static void launch_groups(P p, int bn2, const std::vector<GroupEntry> &entries, long tiles_of_entry, Attach attach) {
  p.list = make_list(entries.data(), (int)entries.size());
  p.ws = nullptr; p.k_per_split = 0;
  p.items = (long)entries.size() * tiles_of_entry;
  THC_CHECK(p.items < (1l << 31) - 4096, "grouped product with too many tiles for one launch");
  attach(p, bn2);
  auto go = [&](auto w) { launch_tc2r_kernel<P, decltype(w)::value>(p, p.items, false); };
  if (bn2 == 256) go(std::integral_constant<int, 256>());
  else if (bn2 == 192) go(std::integral_constant<int, 192>());
  else if (bn2 == 128) go(std::integral_constant<int, 128>());
  else go(std::integral_constant<int, 64>());
  ctx().products[kTf32]++;
}

// D(f, r) = sum_k A[e](f, k) B(r, k): the forward pass (the features are w's rows) and gradInput (its columns, MN).
template <bool MN, bool FUSED>
static void engine_rows(const Groups &g, Lines a, Lines b, long features, long K, int width, const Epilogue &epi, long bias_group, const LinearEpilogue &tail) {
  pack(a, b);
  GroupProblem<GroupOperand<MN>, RawOperand<false>, kGroupRows, FUSED> p;
  p.epi = epi;
  p.M = features; p.N = g.rows; p.K = K;
  p.bias_group = bias_group;
  p.tail = tail;
  launch_groups(p, width, row_tiles(g, width), (features + 255) / 256, [&](auto &q, int bn2) {
    encode_groups(&q.a.tmap, a.p, MN, g.n, features, K, a.ld, TC_BM);
    attach_raw_map<kTf32>(q.b, b.p, g.rows, K, b.ld, bn2 / 2);
  });
}

// ---- the passes -------------------------------------------------------------------------------------------------------
void group_forward(const Groups &g, const float *x, long ldx, long in, long out, const float *w, const float *b, float *y, int act, float *z) {
  if (each_group(g, [&](int e, long r, long n) {
        LinearTail tail;
        tail.act = act;
        tail.z = z ? z + r * out : nullptr;
        linear_product(x + r * ldx, ldx, n, in, out, w + e * out * in, b ? b + e * out : nullptr, y + r * out, tail);
      }))
    return;
  WsScope scope;
  SmallGroups p = {};
  p.a = small_operand(w, in); p.b = small_operand(x, ldx);
  p.M = (int)out; p.N = 0; p.K = (int)in;
  p.c = y; p.sm = 1; p.sn = out;
  p.alpha = 1.f;
  p.bias = b; p.bias_m = 1;
  p.act = act; p.z = z;
  p.kind = kGroupRows; p.column_tiles = 1;
  p.at = GroupPlaces{out * in, 0, ldx, 0, out, out};
  if (few_rows_groups(p, g)) return;
  const Lines ws{w, (long)g.n * out, in, in}, xs{x, g.rows, in, ldx};
  const Choice c = choose_rows(g, out, in, ws.ok() && xs.ok(), pack_bytes(ws, xs), encode_tiled_fn() != nullptr);
  if (c.engine) {
    Epilogue epi{y, nullptr, 1.f, 0.f, LONG_MAX, 0, out};
    epi.row_bias = b;
    LinearEpilogue tail;
    tail.act = act; tail.z = z;
    engine_rows<false, true>(g, ws, xs, out, in, c.width, epi, out, tail);
    return;
  }
  small_groups(p, row_tiles(g, c.width), c.width, true, true);
}
void group_grad_input(const Groups &g, const float *gz, long ldg, long in, long out, const float *w, float *gx) {
  if (each_group(g, [&](int e, long r, long n) { gemm('n', 'n', in, n, out, 1.f, w + e * out * in, in, gz + r * ldg, ldg, 0.f, gx + r * in, in); })) return;
  WsScope scope;
  const Lines ws{w, (long)g.n * out, in, in}, gs{gz, g.rows, out, ldg};
  const Choice c = choose_rows(g, in, out, ws.ok() && gs.ok(), pack_bytes(ws, gs), encode_tiled_fn() != nullptr);
  if (c.engine) {
    engine_rows<true, false>(g, ws, gs, in, out, c.width, Epilogue{gx, nullptr, 1.f, 0.f, LONG_MAX, 0, in}, 0, {});
    return;
  }
  SmallGroups p = {};
  p.a = small_operand(w, in); p.b = small_operand(gz, ldg);
  p.M = (int)in; p.N = 0; p.K = (int)out;
  p.c = gx; p.sm = 1; p.sn = in;
  p.alpha = 1.f;
  p.kind = kGroupRows; p.column_tiles = 1;
  p.at = GroupPlaces{out * in, 0, ldg, 0, in, 0};
  small_groups(p, row_tiles(g, c.width), c.width, false, true);
}
void group_grad_weight(const Groups &g, const float *x, long ldx, const float *gz, long ldg, long in, long out, float *gw, float scale) {
  if (each_group(g, [&](int e, long r, long n) { gemm('n', 't', in, out, n, scale, x + r * ldx, ldx, gz + r * ldg, ldg, 1.f, gw + e * out * in, in); })) return;
  WsScope scope;
  Lines xs{x, g.rows, in, ldx}, gs{gz, g.rows, out, ldg};
  const int bn2 = tc2_tile_width(out), bn = small_tile_width(out);
  long ktiles = 0, most = 0;
  std::vector<GroupEntry> entries = whole_groups(g);
  for (const GroupEntry &e : entries) {
    const long t = (e.end - e.first + 31) / 32;
    ktiles += t;
    most = std::max(most, t);
  }
  const double bytes = pack_bytes(xs, gs), tiles = (double)((in + 255) / 256) * (double)((out + bn2 - 1) / bn2);
  const double engine = 10 + std::max(tiles * (double)(ktiles + 2 * (long)entries.size()) / (ctx().sm_count / 2), (double)(most + 2)) * group_tile_us(bn2) +
                        (bytes ? 5 + bytes / 2e6 : 0);
  const double columns = (double)((out + bn - 1) / bn);
  if (encode_tiled_fn() && engine < small_groups_us((double)((in + 63) / 64), columns * (double)entries.size(), columns * (double)ktiles, bn, xs.ok() && gs.ok())) {
    pack(xs, gs);
    // the largest first: the clusters take items as they finish, and short ones level the end
    std::stable_sort(entries.begin(), entries.end(), [](const GroupEntry &a, const GroupEntry &b) { return a.end - a.first > b.end - b.first; });
    GroupProblem<RawOperand<true>, RawOperand<true>, kGroupSums, false> p;
    p.epi = Epilogue{gw, nullptr, scale, 1.f, LONG_MAX, 0, in};
    p.M = in; p.N = out; p.K = g.rows;
    p.out_group = out * in;
    launch_groups(p, bn2, entries, ((in + 255) / 256) * ((out + bn2 - 1) / bn2), [&](auto &q, int) {
      attach_raw_map<kTf32>(q.a, xs.p, in, g.rows, xs.ld, TC_BM);
      attach_raw_map<kTf32>(q.b, gs.p, out, g.rows, gs.ld, bn2 / 2);
    });
    return;
  }
  SmallGroups p = {};
  p.a = small_operand(x, ldx); p.b = small_operand(gz, ldg);
  p.M = (int)in; p.N = (int)out; p.K = 0;
  p.c = gw; p.sm = 1; p.sn = in;
  p.alpha = scale; p.beta = 1.f;
  p.kind = kGroupSums;
  p.column_tiles = ceil_div(out, bn);
  p.at = GroupPlaces{0, ldx, ldg, out * in, 0, 0};
  small_groups(p, entries, bn, false, false);
}

}  // namespace thc
