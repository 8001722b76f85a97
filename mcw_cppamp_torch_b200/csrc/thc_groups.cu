// Products of nn.GroupedLinear: all groups in one launch.
//
//   forward       D(o, r) = sum_i w[e](o, i) x(r, i)      rows r of group e
//   gradInput     D(i, r) = sum_o w[e](o, i) gz(r, o)
//   gradWeight    D[e](i, o) += sum_r x(r, i) gz(r, o)     over the rows of group e
//
// A launch per group, as gemm() would have it, leaves most of the device idle behind each (37 groups of some 40 rows, 333 -> 515: three products
// took 785 us); here the pieces of all groups are a launch's work items.  The 64-row (or 256-row) side of a tile is the features', so that a weight
// that meets few rows is read once, in tiles as narrow as the rows.
//
// What each way measured (forward; a product of FP32 accuracy is three of halves, 555 TFLOP/s at the rate of library products):
//   few rows        64 groups, 24 rows, 1024 -> 2048: 35 us, 168 MB of weights at 4.8 TB/s; the warp-level engine took 129
//   warp-level      37 groups, 1537 rows, gradInput of 333 -> 515: 42 us, 12 TFLOP/s; operands of odd pitch come in 4-byte pieces, 17 k tiles in turn
//   two-SM, FP32    16 groups, 8192 rows, 1024 -> 4096: 382 us with gelu, 180 TFLOP/s; 8 groups, 6000 rows, 2048 -> 1408: 190, 182.  The splitters and
//                   the MMAs (tensor pipe 57 - 63 %) share the SM's memory
//   two-SM, pairs   at twice that rate, but the weights are read twice and written once to make them: for the first of these 454 us in all against 429,
//                   for gradWeight of the second 2 % less, with both gradients in pairs 3 %; they pay where rows are many for each weight
#include <map>

#include "mm_launch.cuh"
#include "nn_linear.h"

namespace thc {

using namespace mm;

// Entries that do not travel with a launch go ahead of it, as many at a time as a kernel's 32 KB of parameters hold: by value, so that a recording has
// its own.
struct GroupUpload {
  static constexpr int kMost = 2000;
  int count;
  GroupEntry at[kMost];
};
static __global__ void __launch_bounds__(256) group_list_kernel(const __grid_constant__ GroupUpload piece, GroupEntry *to) {
  pdl_begin();
  for (int i = threadIdx.x; i < piece.count; i += 256) to[i] = piece.at[i];
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
  GroupUpload piece;
  for (int i = 0; i < n; i += GroupUpload::kMost) {
    piece.count = std::min(n - i, GroupUpload::kMost);
    std::copy(e + i, e + i + piece.count, piece.at);
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
    for (long i = 0; i < g.counts[e]; i += width) v.push_back(GroupEntry{e, (int)(r + i), (int)(r + std::min<long>(g.counts[e], i + width)), 0});
  return v;
}
// The same with the pieces that are not full behind those that are, the largest first: the clusters take items as they finish, and short ones level
// the end.
static std::vector<GroupEntry> largest_first(std::vector<GroupEntry> v) {
  std::stable_sort(v.begin(), v.end(), [](const GroupEntry &a, const GroupEntry &b) { return a.end - a.first > b.end - b.first; });
  return v;
}
static std::vector<GroupEntry> whole_groups(const Groups &g) {
  std::vector<GroupEntry> v;
  long r = 0;
  for (int e = 0; e < g.n; r += g.counts[e++])
    if (g.counts[e]) v.push_back(GroupEntry{e, (int)r, (int)(r + g.counts[e]), 0});
  return v;
}
// The warp-level engine's time, by small_product_us()'s figures: `features` tiles of 64, times `tiles` along the groups' rows (or the other features), which
// take `steps` k tiles in all.  A tile's start and end cost as much as three k tiles.
static double small_groups_us(double features, double tiles, double steps, int bn, bool aligned) {
  const double blocks = features * tiles / ctx().sm_count, depth = bn == 64 ? 3 : bn == 8 ? 5 : 4, resident = std::min(std::max(blocks, 1.0), depth);
  const double step = bn == 64 ? 1.35 + 0.4 * resident : bn == 32 ? 1.3 + 0.15 * resident : bn == 16 ? 0.6 + 0.15 * resident : 0.45 + 0.15 * resident;
  return 5 + (aligned ? 1.0 : 1.3) * step * features * (steps + 3 * tiles) / ctx().sm_count / resident;
}
// The two-SM engine's k tile of `columns` columns in tiles of up to `width`.  FP32 values: 16 groups of 512 rows, 1024 -> 4096, 298 / 342 / 336 / 495 us
// with tiles of 256 / 192 / 128 / 64 columns; fewer columns spare the MMAs, but the loads and most of the splitting go on (32 groups of
// some 16 rows, 1024 -> 2048: 145 / 121 / 99 / 92 us).
static double group_tile_us(int columns, int width, bool pairs) {
  if (pairs) return std::max(tc2_tile_us(columns, kPairs), 0.75 * tc2_tile_us(width, kPairs));
  const double mma = columns == 256 ? 1.25 : columns == 192 ? 0.91 : columns == 128 ? 0.71 : 0.52;
  return std::max(mma, width == 256 ? 0.95 : width == 192 ? 0.8 : width == 128 ? 0.65 : 0.58);
}
// Work items of a launch, the longest first: how many take how long.
struct Items {
  double us[5] = {};
  long n[5] = {};
};
// When the last cluster is done if each takes the next item as it finishes one.
static double makespan_us(const Items &items) {
  std::map<double, long> done;     // clusters by the time they are free
  done[0] = ctx().sm_count / 2;
  for (int i = 0; i < 5; i++)
    for (long n = items.n[i]; n > 0;) {
      const auto first = *done.begin();
      const long take = std::min(first.second, n);
      done.erase(done.begin());
      if (take < first.second) done[first.first] = first.second - take;
      done[first.first + items.us[i]] += take;
      n -= take;
    }
  return 10 + done.rbegin()->first;
}
// Adds the tiles along `n` columns, at most `width` each, the last as wide as it has to be, `features` times; k tiles of one of them.
static void add_tiles(Items &items, long n, int width, int step, long features, double k, bool pairs) {
  items.us[0] = k * group_tile_us(width, width, pairs);
  items.n[0] += n / width * features;
  const int rest = (int)((n % width + step - 1) / step * step);
  if (!rest) return;
  const int i = rest == width ? 0 : 5 - rest / 64;
  items.us[i] = k * group_tile_us(rest, width, pairs);
  items.n[i] += features;
}
static double columns_us(long n, int width, int step, bool pairs) {
  const long rest = (n % width + step - 1) / step * step;
  return (double)(n / width) * group_tile_us(width, width, pairs) + (rest ? group_tile_us((int)rest, width, pairs) : 0);
}
static long tiles_of(const Groups &g, long width) {
  long t = 0;
  for (int e = 0; e < g.n; e++) t += (g.counts[e] + width - 1) / width;
  return t;
}
enum Way { kSmall, kEngine, kEnginePairs };   // the warp-level engine; the two-SM one over FP32 values; over FP16 pairs
struct Choice { Way way; int width; };
// Passes over `values` values that make pairs of them, as pairs_are_faster() has it; value by value where 16-byte accesses do not fit (15 M values of
// 1653 columns: 62 us).
static double pair_passes_us(double values, bool aligned) { return 14 + 4e-6 * values * (1 / 5.5 + 2 / 5.0) * (aligned ? 1 : 1.4); }
// Copies of operands whose pitch TMA cannot take, `bytes` read and written (the same 15 M values: 10 us).
static double pack_us(double bytes) { return bytes ? 4 + bytes / 8e6 : 0; }
static bool pairs_fit(const Groups &g, double values) { return ctx().math_mode == 0 && g.n <= kPaddedGroups && g.rows < 1l << 28 && 4 * values < 16e9 && encode_tiled_fn(); }
// For kGroupRows: the way and the width of its tiles along the rows that finish first.  The two-SM engine takes two k
// tiles' time for a tile's epilogue, and more where that has exponentials; copies of `pack` bytes, and pairs of the `values` of both operands, take their passes.
static Choice choose_rows(const Groups &g, long features, long K, bool small_aligned, double pack, double values, int act = kActNone) {
  Choice best{kSmall, 64};
  double least = 0;
  const long ktiles = (K + 31) / 32, ktiles_half = (K + 63) / 64;
  for (int w : {64, 32, 16, 8}) {
    const double n = (double)tiles_of(g, w), us = small_groups_us((double)((features + 63) / 64), n, n * (double)ktiles, w, small_aligned);
    if (!least || us < least) { best = Choice{kSmall, w}; least = us; }
  }
  if (!encode_tiled_fn()) return best;
  for (bool pairs : {false, true}) {
    if (pairs && !pairs_fit(g, values)) break;
    for (int w : {256, 192, 128, 64}) {
      Items items;
      const double k = (double)(pairs ? ktiles_half : ktiles) + 2 + (act >= kActGelu ? w / 64 : 0);
      for (int e = 0; e < g.n; e++) add_tiles(items, g.counts[e], w, 64, (features + 255) / 256, k, pairs);
      const double us = makespan_us(items) + (pairs ? pair_passes_us(values, pack == 0) : pack_us(pack));
      if (us < least) { best = Choice{pairs ? kEnginePairs : kEngine, w}; least = us; }
    }
  }
  return best;
}

// A handful of rows in each group, K-major operands in whole 16-byte pieces: the weights' bytes are the bound (few_rows_kernel).  Up to four rows at
// a time; a group of more reads its weight again, from L2, so that few may have more.
static bool few_rows_groups(SmallGroups p, const Groups &g) {
  if (!p.a.vec4 || !p.b.vec4 || p.K % 4) return false;
  long most = 0, live = 0;
  for (int e = 0; e < g.n; e++) { most = std::max(most, g.counts[e]); live += g.counts[e] > 0; }
  if (4 * tiles_of(g, 4) > 5 * live) return false;
  const std::vector<GroupEntry> entries = row_tiles(g, 4);
  for (size_t i = 0; i < entries.size(); i += 65535) {
    p.list = make_list(entries.data() + i, (int)std::min(entries.size() - i, (size_t)65535));
    p.stalled = stall_ctl().dev_flag;
    launch_few_rows_kernel(p, (int)std::min(most, 4l), dim3(1, (unsigned)p.list.count));
    check_launch("few_rows");
  }
  return true;
}
// gradWeight where no group has more than sixteen rows: gw[e] is read and written once, which is the bound, and FP32 multiply-adds keep up.  A thread
// has four columns (VEC: neighbours, else T apart) with their inputs in registers, and eight rows of gw, four on their way at a time; a block has 4 T
// columns and 8 * (256 / T) rows.  7 rows, 5716 -> 5630 (257 MB): the two-SM engine, whose epilogue is all there is to that product, took
// 79 us, a backward call 144 where it now takes 112.
constexpr int kFewSums = 16;
template <int R, bool VEC>
static __global__ void __launch_bounds__(256) few_rows_sums_kernel(const float *__restrict__ x, long ldx, const float *__restrict__ gz, long ldg, long in, long out,
                                                                   float *__restrict__ gw, float scale, int T, const int *stalled_flag,
                                                                   const __grid_constant__ GroupList list) {
  pdl_begin();
  const int stalled = *reinterpret_cast<const volatile int *>(stalled_flag);   // as SmallProblem::stalled
  constexpr int U = 4, ROWS = 8;
  __shared__ __align__(16) float g[8 * ROWS][R];
  const GroupEntry e = list.at(blockIdx.z);
  const int tx = threadIdx.x % T, ty = threadIdx.x / T, rows = ROWS * (256 / T), n = e.end - e.first;
  const long c0 = (long)blockIdx.x * 4 * T, o0 = (long)blockIdx.y * rows;
  for (int i = threadIdx.x; i < rows * R; i += 256) {
    const int r = i / rows, o = i % rows;
    g[o][r] = r < n && o0 + o < out ? scale * __ldg(gz + (e.first + r) * ldg + o0 + o) : 0.f;
  }
  auto column = [&](int j) { return c0 + (VEC ? 4 * tx + j : tx + (long)T * j); };
  float v[R][4];
#pragma unroll
  for (int r = 0; r < R; r++) {
    const float *row = x + (e.first + r) * ldx;
    if constexpr (VEC) {
      const float4 q = r < n && column(0) < in ? __ldg(reinterpret_cast<const float4 *>(row + column(0))) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[r][0] = q.x; v[r][1] = q.y; v[r][2] = q.z; v[r][3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) v[r][j] = r < n && column(j) < in ? __ldg(row + column(j)) : 0.f;
    }
  }
  __syncthreads();
  if (column(0) >= in || stalled) return;
  float *to = gw + e.group * out * in;
#pragma unroll
  for (int u0 = 0; u0 < ROWS; u0 += U) {
    float old[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const long o = o0 + ty * ROWS + u0 + u;
      const float *p = to + o * in;
      if constexpr (VEC) {
        const float4 q = o < out ? *reinterpret_cast<const float4 *>(p + column(0)) : make_float4(0.f, 0.f, 0.f, 0.f);
        old[u][0] = q.x; old[u][1] = q.y; old[u][2] = q.z; old[u][3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) old[u][j] = o < out && column(j) < in ? p[column(j)] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int lo = ty * ROWS + u0 + u;
      const long o = o0 + lo;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] = fmaf(g[lo][r], v[r][j], s[j]);
      if (o >= out) continue;
      float *p = to + o * in;
      if constexpr (VEC) {
        *reinterpret_cast<float4 *>(p + column(0)) = make_float4(old[u][0] + s[0], old[u][1] + s[1], old[u][2] + s[2], old[u][3] + s[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (column(j) < in) p[column(j)] = old[u][j] + s[j];
      }
    }
  }
}
// f(R as a constant, list) for the groups with rows, as many as a launch has blocks for along z.
template <int MOST, class F> static void each_few(const Groups &g, long most, F f) {
  const std::vector<GroupEntry> entries = whole_groups(g);
  for (size_t i = 0; i < entries.size(); i += 65535) {
    const GroupList list = make_list(entries.data() + i, (int)std::min(entries.size() - i, (size_t)65535));
    if (most <= 1) f(std::integral_constant<int, 1>(), list);
    else if (most <= 2) f(std::integral_constant<int, 2>(), list);
    else if (most <= 4) f(std::integral_constant<int, 4>(), list);
    else if (MOST == 8 || most <= 8) f(std::integral_constant<int, 8>(), list);
    else f(std::integral_constant<int, MOST>(), list);
  }
}
static long most_rows(const Groups &g) { return *std::max_element(g.counts, g.counts + g.n); }
bool few_rows_sums(const Groups &g, const float *x, long ldx, const float *gz, long ldg, long in, long out, float *gw, float scale) {
  const long most = most_rows(g);
  if (most > kFewSums) return false;
  const bool vec = in % 4 == 0 && ldx % 4 == 0 && (((uintptr_t)x | (uintptr_t)gw) & 15) == 0;
  int T = 32;
  while (T < 256 && 4 * T < in) T *= 2;
  const long columns = (in + 4 * T - 1) / (4 * T), rows = 8 * (256 / T), tiles = (out + rows - 1) / rows;
  if (tiles > 65535) return false;
  WsScope scope;
  const int *stalled = stall_ctl().dev_flag;
  each_few<kFewSums>(g, most, [&](auto r, const GroupList &list) {
    const dim3 grid((unsigned)columns, (unsigned)tiles, (unsigned)list.count);
    if (vec) pdl_launch(few_rows_sums_kernel<decltype(r)::value, true>, grid, 256, 0, x, ldx, gz, ldg, in, out, gw, scale, T, stalled, list);
    else pdl_launch(few_rows_sums_kernel<decltype(r)::value, false>, grid, 256, 0, x, ldx, gz, ldg, in, out, gw, scale, T, stalled, list);
    check_launch("few_rows_sums");
  });
  return true;
}

// gradInput of eight groups and more where none has more than eight rows: w[e] is read once, along its rows, and multiply-adds in FP32 keep up.  A warp has 128 columns (VEC: four neighbours a lane, else 32
// apart) and eight rows of w on their way; the eight warps of a block take eight rows each in turn of the block's `run` rows of w and meet in shared memory,
// the blocks of a column tile in memory, where the last one adds their sums up in their order.  kFewRun rows' gradients lie in shared memory at a time.
// A backward call of 64 groups, 1024 -> 2048 with 24 rows, 333 -> 515 with 100: 174 and 64 us, with the warp-level engine 208 and 76.  One
// matrix, which has to be cut along its rows for blocks enough, stays with that engine (7 rows, 5716 -> 5630: 131 and 112).  gradInput alone, this way / that
// engine: 8 groups of four rows 13.8 / 21.0 us (1024 -> 2048), 132 / 150 (4096 -> 4096), 7.0 / 9.5 (333 -> 515), 16 groups 38 / 44, 174 / 208, 9.9 / 11.6; with
// eight rows the shared memory's reads show: 22.6 / 21.1, 168 / 150, 10.4 / 9.6, and 50 / 43, 329 / 209, 14.0 / 11.7.  Below eight groups, four rows:
// four groups 8.8 / 12.9, 70 / 76, 6.3 / 8.1, two 8.2 / 10.6, 39 / 37, 6.3 / 7.3.
constexpr int kFewRun = 512, kFewBack = 8;
template <int R, bool VEC>
static __global__ void __launch_bounds__(256) few_rows_back_kernel(const float *__restrict__ w, const float *__restrict__ gz, long ldg, long in, long out, float *__restrict__ gx,
                                                                   int run, float *part, unsigned *tickets, const int *stalled_flag,
                                                                   const __grid_constant__ GroupList list) {
  pdl_begin();
  const int stalled = *reinterpret_cast<const volatile int *>(stalled_flag);   // as SmallProblem::stalled
  constexpr int U = 8, Q = R < 4 ? R : 4;
  __shared__ __align__(16) float sm[R * kFewRun > 8 * Q * 128 ? R * kFewRun : 8 * Q * 128];
  __shared__ bool last;
  const GroupEntry e = list.at(blockIdx.z);
  const int n = e.end - e.first, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long c0 = blockIdx.x * 128l, o0 = (long)blockIdx.y * run;
  const int all_rows = (int)min((long)run, out - o0);
  w += (e.group * out + o0) * in;
  auto column = [&](int j) { return c0 + (VEC ? 4 * lane + j : lane + 32 * j); };
  float acc[R][4];
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int j = 0; j < 4; j++) acc[r][j] = 0.f;
  for (int from = 0; from < all_rows; from += kFewRun) {
    const int rows = min(kFewRun, all_rows - from);
    __syncthreads();
    for (int i = threadIdx.x; i < R * kFewRun; i += 256) {
      const int r = i / kFewRun, o = i % kFewRun;
      if (o < (rows + 7) / 8 * 8) sm[i] = r < n && o < rows ? __ldg(gz + (e.first + r) * ldg + o0 + from + o) : 0.f;
    }
    __syncthreads();
    for (int o = warp * U; o < rows; o += 8 * U) {
      float v[U][4];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const float *p = w + (long)(o + u) * in;
        if constexpr (VEC) {
          const float4 q = o + u < rows && column(0) < in ? __ldg(reinterpret_cast<const float4 *>(p + column(0))) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[u][0] = q.x; v[u][1] = q.y; v[u][2] = q.z; v[u][3] = q.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) v[u][j] = o + u < rows && column(j) < in ? __ldg(p + column(j)) : 0.f;
        }
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float4 g0 = *reinterpret_cast<const float4 *>(sm + r * kFewRun + o), g1 = *reinterpret_cast<const float4 *>(sm + r * kFewRun + o + 4);
        const float gs[U] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int j = 0; j < 4; j++) acc[r][j] = fmaf(gs[u], v[u][j], acc[r][j]);
      }
    }
    w += (long)kFewRun * in;
  }
  if (stalled) return;   // (all blocks: no ticket is taken)
  const long tile = (long)blockIdx.z * gridDim.x + blockIdx.x;
  float *mine = part + (tile * gridDim.y + blockIdx.y) * (R * 128);
#pragma unroll
  for (int r0 = 0; r0 < R; r0 += Q) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; q++)
#pragma unroll
      for (int j = 0; j < 4; j++) sm[(warp * Q + q) * 128 + (VEC ? 4 * lane + j : lane + 32 * j)] = acc[r0 + q][j];
    __syncthreads();
    for (int i = threadIdx.x; i < Q * 128; i += 256) {
      float s = sm[i];
#pragma unroll
      for (int k = 1; k < 8; k++) s += sm[k * Q * 128 + i];
      const int r = r0 + i / 128;
      if (gridDim.y > 1) mine[r * 128 + i % 128] = s;
      else if (r < n && c0 + i % 128 < in) gx[(e.first + r) * in + c0 + i % 128] = s;
    }
  }
  if (gridDim.y == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(tickets + tile, 1u) == gridDim.y - 1;
    if (last) tickets[tile] = 0;   // ready for the next launch on this stream
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float *all = part + tile * gridDim.y * (R * 128);
  for (int i = threadIdx.x; i < n * 128; i += 256) {
    if (c0 + i % 128 >= in) continue;
    float s = 0.f;
#pragma unroll 8
    for (int z = 0; z < (int)gridDim.y; z++) s += __ldcg(all + (long)z * (R * 128) + i);
    gx[(e.first + i / 128) * in + c0 + i % 128] = s;
  }
}
static bool few_rows_back(const Groups &g, const float *gz, long ldg, long in, long out, const float *w, float *gx) {
  const long most = most_rows(g);
  if (most > kFewBack || g.n - std::count(g.counts, g.counts + g.n, 0l) < 8) return false;
  const bool vec = in % 4 == 0 && ((uintptr_t)w & 15) == 0;
  const long columns = (in + 127) / 128;
  const int *stalled = stall_ctl().dev_flag;
  WsScope scope;
  each_few<kFewBack>(g, most, [&](auto r, const GroupList &list) {
    constexpr int R = decltype(r)::value;
    // as many blocks as are resident at once, rows of w in whole eights for each warp
    constexpr long kResident = R <= 2 ? 4 : 2;
    const long tiles = columns * list.count, wanted = std::max(1l, ctx().sm_count * kResident / tiles);
    const long run = std::max(64l, ((out + wanted - 1) / wanted + 63) / 64 * 64), splits = (out + run - 1) / run;
    const dim3 grid((unsigned)columns, (unsigned)splits, (unsigned)list.count);
    float *part = splits > 1 ? (float *)ws_alloc(sizeof(float) * tiles * splits * R * 128) : nullptr;
    if (vec) pdl_launch(few_rows_back_kernel<R, true>, grid, 256, 0, w, gz, ldg, in, out, gx, (int)run, part, zero_words(), stalled, list);
    else pdl_launch(few_rows_back_kernel<R, false>, grid, 256, 0, w, gz, ldg, in, out, gx, (int)run, part, zero_words(), stalled, list);
    check_launch("few_rows_back");
  });
  return true;
}
// Entries of sums with the groups of more than `most` k tiles cut into slices, those first.  `cut`: how many entries they are.
static std::vector<GroupEntry> cut_groups(const std::vector<GroupEntry> &groups, int most, long &cut) {
  std::vector<GroupEntry> v;
  for (GroupEntry e : groups) {
    const int slices = SmallGroups::slices_of(e.end - e.first, most);
    for (e.shift = 0; slices > 1 && e.shift < slices; e.shift++) v.push_back(e);
  }
  cut = (long)v.size();
  for (const GroupEntry &e : groups)
    if (SmallGroups::slices_of(e.end - e.first, most) <= 1) v.push_back(e);
  return v;
}
// The warp-level engine over the groups: any size, pitch and alignment.
static void small_groups(SmallGroups p, std::vector<GroupEntry> entries, int bn, bool a_k, bool b_k) {
  p.stalled = stall_ctl().dev_flag;
  p.tile_floats = 64 * bn;
  const int most = std::max(1, 65535 / p.column_tiles);
  const long tiles = (long)ceil_div(p.M, 64) * p.column_tiles;   // of an entry
  long cut = 0;
  if (p.kind == kGroupSums) {
    // no slice longer than a block's share of all k tiles (three blocks an SM), or than sixteen, but no more than 32 slices.  So fewer than six tiles an SM
    // keep partial sums (15 MB), however uneven the groups are.  128 groups, 256 -> 256, 13800 rows in one and 20 in each of the others: 88 us; with all
    // of them in as many slices as the longest, 528 us and 738 MB.
    long all = 0, longest = 1;
    for (const GroupEntry &e : entries) {
      const long t = ceil_div(e.end - e.first, TC_BK);
      all += t * tiles;
      longest = std::max(longest, t);
    }
    const long share = 3l * ctx().sm_count;
    p.tiles_per_slice = (int)std::max(std::max(16l, (all + share - 1) / share), (longest + 31) / 32);
    entries = cut_groups(entries, p.tiles_per_slice, cut);
    THC_CHECK(cut <= most && cut * tiles <= kZeroWords, "internal: grouped sums cut into too many slices");
  }
  for (size_t i = 0; i < entries.size(); i += most) {
    const int n = (int)std::min(entries.size() - i, (size_t)most);
    p.list = make_list(entries.data() + i, n);
    p.ws = nullptr;
    p.slices = 1;
    if (p.kind == kGroupRows) {
      const long ktiles = std::max(1, ceil_div(p.K, TC_BK)), slices = n * tiles <= 2 * ctx().sm_count ? small_slices(n * tiles, ktiles, bn) : 1;
      p.tiles_per_slice = ceil_div(ktiles, slices);
      p.slices = ceil_div(ktiles, p.tiles_per_slice);
    }
    const long slots = p.kind == kGroupRows ? (p.slices > 1 ? n * p.slices : 0) : i ? 0 : cut;
    if (slots) {
      p.ws = (float *)ws_alloc(sizeof(float) * slots * tiles * p.tile_floats);
      p.tickets = zero_words();
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
static void pack(Lines &a, Lines &b, Lines *c = nullptr) {
  PackJob jobs[3] = {};
  int n = 0;
  for (Lines *l : {&a, &b, c}) {
    if (!l || l->ok()) continue;
    const long ld = (l->run + 3) / 4 * 4;
    float *to = (float *)ws_alloc(sizeof(float) * l->lines * ld);
    jobs[n++] = PackJob{l->p, to, l->lines, l->run, l->ld, ld};
    l->p = to; l->ld = ld;
  }
  if (n) launch_pack(jobs[0], jobs[1], jobs[2]);
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
  else if (bn2 == 128) go(std::integral_constant<int, 128>());
  else if constexpr (P::PREC == kTf32 || !P::OpB::MN_MAJOR) {
    if (bn2 == 192) go(std::integral_constant<int, 192>());
    else go(std::integral_constant<int, 64>());
  } else {
    fail("internal: tile width %d for a problem that has none", bn2);
  }
  ctx().products[P::PREC]++;
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
  launch_groups(p, width, largest_first(row_tiles(g, width)), (features + 255) / 256, [&](auto &q, int bn2) {
    attach_group_map<MN, kTf32>(q.a, a.p, g.n, features, K, a.ld, TC_BM);
    attach_raw_map<kTf32>(q.b, b.p, g.rows, K, b.ld, bn2 / 2);
  });
}

// ---- the two-SM engine over pairs ------------------------------------------------------------------------------------
// An operand as FP16 pairs (mm_problem.cuh): weights as they lie, rows with each group padded by zeros to whole k tiles, so that no k tile has two
// groups' rows.
struct GroupSide {
  const float *p;
  long lines, run, ld;
  bool grouped;
  Measured m;
  void *dst;
  long ldp;
  float *wide = nullptr;   // (PairJob)
};
static Ranges ranges_of(const GroupSide &own, const GroupSide &other) {
  Ranges r;
  r.rec[0] = own.m.rec; r.rec[1] = other.m.rec;
  return r;
}
struct GroupPairs {
  GroupRows rows;
  long padded() const { return rows.padded[rows.n]; }
};
// Both operands of a product, or of two, with the first operand in each, whose forms are decided product by product.  False: there is no room for the
// pairs, and nothing has been done.
static bool make_pairs(GroupPairs &gp, const Groups &g, std::initializer_list<GroupSide *> list) {
  const int n = (int)list.size();
  GroupSide *const *sides = list.begin();
  gp.rows.n = g.n;
  gp.rows.real[0] = gp.rows.padded[0] = 0;
  for (int e = 0; e < g.n; e++) {
    gp.rows.real[e + 1] = gp.rows.real[e] + (int)g.counts[e];
    gp.rows.padded[e + 1] = gp.rows.padded[e] + (int)((g.counts[e] + 63) / 64 * 64);
  }
  double need = 96e6;
  for (int i = 0; i < n; i++) need += 4.1 * (double)(sides[i]->grouped ? gp.padded() : sides[i]->lines) * (double)(sides[i]->run + 64) * (n > 2 && i == 0 ? 2 : 1);
  if (!ws_reserve((size_t)need)) return false;
  RangeJob ranges[3];
  GroupPairJob jobs[3] = {};
  long pieces = 0;
  for (int i = 0; i < n; i++) sides[i]->m = new_measured();
  for (int i = 0; i < n; i++) {
    GroupSide &s = *sides[i];
    s.ldp = (s.run + 63) / 64 * 64;
    const long lines = s.grouped ? gp.padded() : s.lines;
    s.dst = ws_alloc(sizeof(float) * lines * s.ldp);
    ranges[i] = range_job(s.p, s.lines, s.run, s.ld, s.m);
    GroupPairJob &j = jobs[i];
    static_cast<PairJob &>(j) = PairJob{s.p, s.dst, s.lines, s.run, s.ld, s.ldp, ((uintptr_t)s.p & 15) == 0 && s.ld % 4 == 0, {}};
    j.grouped = s.grouped;
    j.ranges = ranges_of(s, *sides[i ? 0 : 1]);
    if (n > 2 && i == 0) {
      j.wide = s.wide = (float *)ws_alloc(sizeof(float) * lines * s.ldp);
      j.other = ranges_of(s, *sides[2]);
    }
    pieces = std::max(pieces, lines * ((s.ldp + 511) / 512));
  }
  launch_ranges(ranges[0], &ranges[1]);
  if (n > 2) launch_ranges(ranges[2], nullptr);
  pdl_launch(split_groups_kernel, dim3((unsigned)std::min<long>((pieces + 7) / 8, ctx().sm_count * 8l), (unsigned)n), 256, 0, jobs[0], jobs[1], jobs[2], gp.rows);
  check_launch("split_groups");
  return true;
}
static std::vector<GroupEntry> padded(std::vector<GroupEntry> v, const GroupRows &rows) {
  for (GroupEntry &e : v) {
    e.shift = rows.padded[e.group] - rows.real[e.group];
    e.first += e.shift; e.end += e.shift;
  }
  return v;
}
// As engine_rows, over the pairs of w and of the rows; what they leave out is added to `sums`.
template <bool MN, bool FUSED>
static void pairs_rows(const Groups &g, const GroupPairs &gp, const GroupSide &w, const GroupSide &x, long in, long out, int width, const Epilogue &epi, float *sums,
                       const LinearEpilogue &tail) {
  const long features = MN ? in : out, K = MN ? out : in;
  GroupProblem<GroupOperand<MN, kPairs>, RawOperand<false, kPairs>, kGroupRows, FUSED, kPairs> p;
  p.epi = epi;
  p.M = features; p.N = gp.padded(); p.K = K;
  p.bias_group = out;
  p.tail = tail;
  p.range_a = w.m.rec; p.range_b = x.m.rec; p.ranges = ranges_of(w, x);
  launch_groups(p, width, padded(largest_first(row_tiles(g, width)), gp.rows), (features + 255) / 256, [&](auto &q, int bn2) {
    attach_group_map<MN, kPairs>(q.a, w.dst, g.n, features, K, w.ldp, TC_BM);
    attach_raw_map<kPairs>(q.b, x.dst, gp.padded(), K, x.ldp, bn2 / 2, x.wide);
  });
  pdl_launch(group_row_strays_kernel, (unsigned)std::min<long>(g.rows, ctx().sm_count), 256, 0, GroupStrays{w.p, in, out, x.p, x.ld, x.run, w.m, x.m}, !MN, sums, p.ranges,
             gp.rows);
  check_launch("group_strays");
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
  const Choice c = choose_rows(g, out, in, ws.ok() && xs.ok(), pack_bytes(ws, xs), (double)in * (double)(g.n * out + g.rows), act);
  if (c.way != kSmall) {
    Epilogue epi{y, nullptr, 1.f, 0.f, LONG_MAX, 0, out};
    epi.row_bias = b;
    LinearEpilogue tail;
    tail.act = act; tail.z = z;
    if (c.way == kEnginePairs) {
      GroupSide wp{w, (long)g.n * out, in, in, false}, xp{x, g.rows, in, ldx, true};
      GroupPairs gp;
      if (make_pairs(gp, g, {&wp, &xp})) {
        tail.a = wp.m.rec; tail.b = xp.m.rec; tail.ranges = ranges_of(wp, xp);
        float *sums = z ? z : y;
        pairs_rows<false, true>(g, gp, wp, xp, in, out, c.width, epi, sums, tail);
        LinearTail after;
        after.act = act;
        if (act != kActNone || z) linear_tail(sums, y, g.rows, out, after, tail);
        return;
      }
    }
    engine_rows<false, true>(g, ws, xs, out, in, c.width, epi, out, tail);
    return;
  }
  small_groups(p, row_tiles(g, c.width), c.width, true, true);
}
static Choice choose_grad_input(const Groups &g, long ldg, const float *gz, long in, long out, const float *w) {
  const Lines ws{w, (long)g.n * out, in, in}, gs{gz, g.rows, out, ldg};
  return choose_rows(g, in, out, ws.ok() && gs.ok(), pack_bytes(ws, gs), (double)out * (double)(g.n * in + g.rows));
}
static void grad_input(const Groups &g, const Choice &c, const Lines &gz, long in, long out, const Lines &w, float *gx) {
  WsScope scope;
  if (c.way != kSmall) {
    engine_rows<true, false>(g, w, gz, in, out, c.width, Epilogue{gx, nullptr, 1.f, 0.f, LONG_MAX, 0, in}, 0, {});
    return;
  }
  SmallGroups p = {};
  p.a = small_operand(w.p, w.ld); p.b = small_operand(gz.p, gz.ld);
  p.M = (int)in; p.N = 0; p.K = (int)out;
  p.c = gx; p.sm = 1; p.sn = in;
  p.alpha = 1.f;
  p.kind = kGroupRows; p.column_tiles = 1;
  p.at = GroupPlaces{out * w.ld, 0, gz.ld, 0, in, 0};
  small_groups(p, row_tiles(g, c.width), c.width, false, true);
}
static Choice choose_grad_weight(const Groups &g, const Lines &xs, const Lines &gs) {
  const long in = xs.run, out = gs.run;
  long ktiles = 0, halves = 0, most = 0, live = 0;
  for (int e = 0; e < g.n; e++) {
    const long t = (g.counts[e] + 31) / 32;
    ktiles += t; halves += (g.counts[e] + 63) / 64; live += t > 0;
    most = std::max(most, t);
  }
  const int bn = small_tile_width(out);
  const double columns = (double)((out + bn - 1) / bn), bytes = pack_bytes(xs, gs), values = (double)g.rows * (double)(in + out);
  Choice best{kSmall, bn};
  double least = small_groups_us((double)((in + 63) / 64), columns * (double)live, columns * (double)ktiles, bn, xs.ok() && gs.ok());
  if (!encode_tiled_fn()) return best;
  if (columns > 65535) least = 1e30;   // more tiles than a launch of that engine has
  for (bool pairs : {false, true}) {
    if (pairs && !pairs_fit(g, values)) break;
    for (int w : {256, 192, 128, 64}) {
      if (pairs && w % 128) continue;
      const long tiles = (in + 255) / 256 * ((out + w - 1) / w);
      const double per = (double)((in + 255) / 256), total = per * columns_us(out, w, pairs ? 128 : 64, pairs) * ((double)(pairs ? halves : ktiles) + (pairs ? 6 : 2) * (double)live);
      const double longest = ((double)(pairs ? (most + 1) / 2 : most) + 2) * group_tile_us(w, w, pairs);
      // items of many lengths, the longest first: level but for what the last are long.  (Accumulating a tile takes as long as six k tiles of pairs.)
      const double us = 10 + std::max(total / (ctx().sm_count / 2) + 0.25 * total / (double)(tiles * std::max(live, 1l)), longest) +
                        (pairs ? pair_passes_us(values, bytes == 0) : pack_us(bytes));
      if (us < least) { best = Choice{pairs ? kEnginePairs : kEngine, w}; least = us; }
    }
  }
  return best;
}
template <class P> static void set_sums(P &p, long in, long out, float *gw, float scale) {
  p.epi = Epilogue{gw, nullptr, scale, 1.f, LONG_MAX, 0, in};
  p.M = in; p.N = out;
  p.out_group = out * in;
}
static void grad_weight(const Groups &g, const Choice &c, Lines xs, Lines gs, float *gw, float scale) {
  WsScope scope;
  const long in = xs.run, out = gs.run;
  if (c.way != kSmall) {
    pack(xs, gs);
    GroupProblem<RawOperand<true>, RawOperand<true>, kGroupSums, false> p;
    set_sums(p, in, out, gw, scale);
    p.K = g.rows;
    const int bn2 = c.width;
    launch_groups(p, bn2, largest_first(whole_groups(g)), ((in + 255) / 256) * ((out + bn2 - 1) / bn2), [&](auto &q, int) {
      attach_raw_map<kTf32>(q.a, xs.p, in, g.rows, xs.ld, TC_BM);
      attach_raw_map<kTf32>(q.b, gs.p, out, g.rows, gs.ld, bn2 / 2);
    });
    return;
  }
  SmallGroups p = {};
  p.a = small_operand(xs.p, xs.ld); p.b = small_operand(gs.p, gs.ld);
  p.M = (int)in; p.N = (int)out; p.K = 0;
  p.c = gw; p.sm = 1; p.sn = in;
  p.alpha = scale; p.beta = 1.f;
  p.kind = kGroupSums;
  p.column_tiles = ceil_div(out, c.width);
  p.at = GroupPlaces{0, xs.ld, gs.ld, out * in, 0, 0};
  small_groups(p, whole_groups(g), c.width, false, false);
}
static void pairs_sums(const Groups &g, const GroupPairs &gp, int w, const GroupSide &x, const GroupSide &gz, float *gw, float scale) {
  const long in = x.run, out = gz.run;
  GroupProblem<RawOperand<true, kPairs>, RawOperand<true, kPairs>, kGroupSums, false, kPairs> p;
  set_sums(p, in, out, gw, scale);
  p.K = gp.padded();
  p.range_a = x.m.rec; p.range_b = gz.m.rec; p.ranges = ranges_of(x, gz);
  launch_groups(p, w, largest_first(padded(whole_groups(g), gp.rows)), ((in + 255) / 256) * ((out + w - 1) / w), [&](auto &q, int bn2) {
    attach_raw_map<kPairs>(q.a, x.dst, in, gp.padded(), x.ldp, TC_BM);
    attach_raw_map<kPairs>(q.b, gz.dst, out, gp.padded(), gz.ldp, bn2 / 2, gz.wide);
  });
  pdl_launch(group_sum_strays_kernel, (unsigned)std::min<long>(out, ctx().sm_count), 256, 0, x.p, x.ld, in, gz.p, gz.ld, out, gw, scale, x.m, gz.m, p.ranges, gp.rows);
  check_launch("group_strays");
}

// Which way a gradient takes, and over pairs its form, depends on it and its operands alone, not on whether the other is asked for too; where both take pairs,
// gz is measured and split once.
void group_backward(const Groups &g, const float *x, long ldx, const float *gz, long ldg, long in, long out, const float *w, float *gx, float *gw, float scale) {
  if (each_group(g, [&](int e, long r, long n) {
        if (gx) gemm('n', 'n', in, n, out, 1.f, w + e * out * in, in, gz + r * ldg, ldg, 0.f, gx + r * in, in);
        if (gw) gemm('n', 't', in, out, n, scale, x + r * ldx, ldx, gz + r * ldg, ldg, 1.f, gw + e * out * in, in);
      }))
    return;
  WsScope scope;
  if (gx && few_rows_back(g, gz, ldg, in, out, w, gx)) gx = nullptr;
  if (gw && few_rows_sums(g, x, ldx, gz, ldg, in, out, gw, scale)) gw = nullptr;
  Lines xs{x, g.rows, in, ldx}, gs{gz, g.rows, out, ldg};
  const Choice ci = gx ? choose_grad_input(g, ldg, gz, in, out, w) : Choice{kSmall, 64}, cw = gw ? choose_grad_weight(g, xs, gs) : Choice{kSmall, 64};
  const bool pi = gx && ci.way == kEnginePairs, pw = gw && cw.way == kEnginePairs;
  if (pi || pw) {
    GroupSide wp{w, (long)g.n * out, in, in, false}, xp{x, g.rows, in, ldx, true}, gp{gz, g.rows, out, ldg, true};
    GroupPairs pairs;
    const bool made = pi && pw ? make_pairs(pairs, g, {&gp, &wp, &xp}) : pi ? make_pairs(pairs, g, {&gp, &wp}) : make_pairs(pairs, g, {&gp, &xp});
    if (made) {
      if (pi) {
        pairs_rows<true, false>(g, pairs, wp, gp, in, out, ci.width, Epilogue{gx, nullptr, 1.f, 0.f, LONG_MAX, 0, in}, gx, {});
        gx = nullptr;
      }
      if (pw) {
        pairs_sums(g, pairs, cw.width, xp, gp, gw, scale);
        gw = nullptr;
      }
    }
  }
  Lines ws{w, (long)g.n * out, in, in};
  if (gx && gw && ci.way != kSmall && cw.way != kSmall) pack(gs, ws, &xs);   // once for both
  if (gx) grad_input(g, ci, gs, in, out, ws, gx);
  if (gw) grad_weight(g, cw, xs, gs, gw, scale);
}

}  // namespace thc
