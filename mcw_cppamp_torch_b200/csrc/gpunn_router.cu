// nn.Router: the k largest of a row's E scores and softmax weights over them, or over all open ones.
//
//   order: descending, equal scores by their place; a score of minus infinity is a closed expert's and is never chosen; a NaN counts as the largest
//   w_i = exp(s_i - max) / sum exp(s_j - max), j over the chosen (normalize) or over all
//   ds_j = w_j (g_j - sum_i g_i w_i) on the chosen and zero elsewhere (normalize), else p_j ([j chosen] g_j - sum_i g_i w_i) with p the whole softmax
//
// A row is read once, by a warp or eight lanes of one, and stays in registers: 4 E bytes a row and 8 k out.  Work on the scores and its latency bind it, not bytes: 36 MB in 11.4 us
// are half of what HBM gives.
#include <type_traits>

#include "nn_args.h"

namespace thc {

constexpr int kRouterScores = 1024, kRouterChosen = 32;   // most scores a row, most of them chosen: what a warp's registers and lanes hold

// ---- a row in a warp's registers: V values a lane, in pieces of four where lengths and addresses allow it
template <int V, bool VEC> struct WarpRow {
  static __device__ __forceinline__ int at(int j, int lane) { return VEC ? ((j >> 2) * 32 + lane) * 4 + (j & 3) : j * 32 + lane; }
  static __device__ __forceinline__ void load(const float *__restrict__ p, int lane, int n, float (&v)[V]) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at(j, lane) < n) q = __ldg(reinterpret_cast<const float4 *>(p + at(j, lane)));
        v[j] = q.x; v[j + 1] = q.y; v[j + 2] = q.z; v[j + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < V; j++) v[j] = at(j, lane) < n ? __ldg(p + at(j, lane)) : -INFINITY;
    }
  }
  static __device__ __forceinline__ void store(float *__restrict__ p, int lane, int n, const float (&v)[V]) {
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < V; j += 4)
        if (at(j, lane) < n) *reinterpret_cast<float4 *>(p + at(j, lane)) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < V; j++)
        if (at(j, lane) < n) p[at(j, lane)] = v[j];
    }
  }
};
static __device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Whole numbers in the order of the scores they stand for (both zeros alike, a NaN above all), and back.
static __device__ __forceinline__ unsigned score_key(float s) {
  const unsigned u = __float_as_uint(s + 0.f);
  if (s != s) return 0xffffffffu;
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
static __device__ __forceinline__ float key_score(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);     // (all ones: a NaN)
}
constexpr unsigned kClosedKey = 0x007fffffu;    // of minus infinity

static __device__ __forceinline__ float larger_score(float a, float b) {      // a NaN if there is one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
static __device__ __forceinline__ float warp_max(float v) {      // a NaN if there is one
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The chosen score of a lane, if it has one.
struct Chosen {
  float score;
  int expert, slot;      // expert from 1, 0: none
};
// The k largest one after the other: the largest of each lane's, of the warp's, its first place; lane i has the i-th.
template <int V> static __device__ __forceinline__ Chosen choose_in_turn(const float (&v)[V], int lane, int k) {
  unsigned key[V];
#pragma unroll
  for (int j = 0; j < V; j++) key[j] = score_key(v[j]);
  Chosen c{-INFINITY, 0, lane};
  for (int i = 0; i < k; i++) {
    unsigned best = 0;
#pragma unroll
    for (int j = 0; j < V; j++) best = max(best, key[j]);
    best = __reduce_max_sync(0xffffffffu, best);
    if (best <= kClosedKey) break;
    unsigned mine = 0xffffffffu;
#pragma unroll
    for (int j = V - 1; j >= 0; j--)
      if (key[j] == best) mine = j * 32 + lane;
    const unsigned place = __reduce_min_sync(0xffffffffu, mine);
#pragma unroll
    for (int j = 0; j < V; j++)
      if ((unsigned)(j * 32 + lane) == place) key[j] = 0;
    if (lane == i) { c.score = key_score(best); c.expert = (int)place + 1; }
  }
  return c;
}
// The k largest at once.  The k-th largest of the lanes' largest is no more than the k-th of all, so that those from it on, some 32 log(32 / (32 - k)) of scores in
// random order, are all that is left to rank: each is compared with each.  False where they are more than the lanes, with nothing done.
// With k above 16 too many are left (22 on average, 31 at 20); with few chosen of few scores, the rounds are shorter.  16384 rows, us in turn and at once: 64 scores, 4 chosen 4.7 and 4.8,
// 8 chosen 6.5 and 5.7; 128 scores, 2 chosen 4.7 and 5.2, 3 chosen 5.4 and 5.3; 256 scores, 1 chosen 5.3 and 5.8, 2 chosen 6.6 and 6.0; 1024 scores, 1 chosen 16.0 and 18.2, 2 chosen 20.2 and 18.4.
constexpr int kFewChosen = 16;
static __host__ __device__ __forceinline__ constexpr bool at_once(int V, int k) { return k <= kFewChosen && k > 1 && k * (V + 2) >= 16; }
struct Candidates {
  float score[32];
  unsigned short place[32];
};
template <int V> static __device__ __forceinline__ bool choose_at_once(const float (&v)[V], float most, float top, Candidates &left, int lane, int k, Chosen &c) {
  float bound = top;
  auto next = [&] {
    most = most == bound ? -INFINITY : most;
    bound = warp_max(most);
  };
  int rounds = k - 1;
  for (; rounds >= 4; rounds -= 4) { next(); next(); next(); next(); }
  for (; rounds > 0; rounds--) next();
  bound = fmaxf(bound, -3.402823466e+38f);      // (an open score)
  unsigned in[V];
  int n = 0;
#pragma unroll
  for (int j = 0; j < V; j++) {
    in[j] = __ballot_sync(0xffffffffu, v[j] >= bound);
    n += __popc(in[j]);
  }
  if (n > 32) return false;
  left.score[lane] = -INFINITY;                 // behind the last one
  __syncwarp();
  const unsigned lower = (1u << lane) - 1;
  n = 0;
#pragma unroll
  for (int j = 0; j < V; j++) {
    const int at = n + __popc(in[j] & lower);
    if (v[j] >= bound) {
      left.score[at] = v[j];
      left.place[at] = (unsigned short)(j * 32 + lane);
    }
    n += __popc(in[j]);
  }
  __syncwarp();
  // the place of a score among all: how many are larger, or as large and before it
  c = Chosen{left.score[lane] + 0.f, 0, 0};     // (both zeros alike)
  for (int i = 0; i < n; i += 4) {
    const float4 o = *reinterpret_cast<const float4 *>(&left.score[i]);
    c.slot += (o.x > c.score) + (o.y > c.score) + (o.z > c.score) + (o.w > c.score);
  }
  c.slot += __popc(__match_any_sync(0xffffffffu, __float_as_uint(c.score)) & lower);
  if (lane < n && c.slot < k) c.expert = left.place[lane] + 1;
  return true;
}

// A row by a warp.
template <int V>
static __device__ __forceinline__ void route_row(const float *__restrict__ x, float *__restrict__ weights, float *__restrict__ experts, int E, int k, bool normalize,
                                                 Candidates &left, int lane) {
  float v[V];
  const float *mine = x + lane;
  if (E == 32 * V) {
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = __ldg(mine + j * 32);
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) v[j] = j * 32 + lane < E ? __ldg(mine + j * 32) : -INFINITY;
  }
  float most = v[0];
#pragma unroll
  for (int j = 1; j < V; j++) most = larger_score(most, v[j]);
  const float top = warp_max(most);
  Chosen c;
  bool done = false;
  if (at_once(V, k) && top == top) done = choose_at_once<V>(v, most, top, left, lane, k, c);
  if (!done) c = choose_in_turn<V>(v, lane, k);
  const float e = c.expert ? expf(c.score - top) : 0.f;
  float total = 0.f;
  if (normalize) total = e;
  else if (top != -INFINITY) {
#pragma unroll
    for (int j = 0; j < V; j++) total += expf(v[j] - top);
  }
  total = warp_total(total);
  if (c.slot < k) {
    weights[c.slot] = c.expert ? e / total : 0.f;
    experts[c.slot] = (float)c.expert;
  }
}
template <int V>
static __global__ void __launch_bounds__(256) router_forward_kernel(const float *__restrict__ x, long ld, float *__restrict__ weights, float *__restrict__ experts,
                                                                    long rows, int E, int k, bool normalize) {
  pdl_begin();
  __shared__ __align__(16) Candidates left[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long row = blockIdx.x * 8l + warp;
  if (row < rows) route_row<V>(x + row * ld, weights + row * k, experts + row * k, E, k, normalize, left[warp], lane);
}

// Many rows: four by a warp, eight lanes each, so that what a row costs apart from its scores is shared.  A lane has 4 V scores, which with V a place make 32 sets a
// row whose largest give the bound as above.  The candidates' places in the lane's registers are bits of a word; they are read again, from L1, on their way to
// shared memory.  A warp that meets a NaN or more candidates than there is room for takes its rows one after the other.
// 32768 x 256, 8 chosen: 11.6 us against 13.3 by warps for a row, 4 chosen 9.3 against 11.9; 24000 rows 9.3 against 10.1.  With fewer rows the longer way of a warp shows (16384:
// 7.7 against 7.1), with 16 chosen the rounds of the bound, which take three exchanges where a whole warp takes one instruction (18.1 against 16.2).
constexpr long kManyRows = 24000;
constexpr int kManyChosen = 8;
struct FourRows {
  float score[4][36];                 // (rows 16 bytes apart modulo 128: read without conflicts)
  unsigned short place[4][32];
};
static __device__ __forceinline__ float eighth_max(float v) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int V, bool VEC>
static __global__ void __launch_bounds__(64) router_forward_rows_kernel(const float *__restrict__ x, long ld, float *__restrict__ weights, float *__restrict__ experts,
                                                                         long rows, int E, int k, bool normalize) {
  pdl_begin();
  constexpr int C = 4 * V;
  __shared__ __align__(16) FourRows shared[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = lane >> 3, l = lane & 7;
  FourRows &left = shared[warp];
  const long first = blockIdx.x * 8l + warp * 4, row = first + group;
  if (first >= rows) return;
  const bool live = row < rows;
  const float *mine = x + row * ld;
  auto place = [&](int b) { return VEC ? ((b >> 2) * 8 + l) * 4 + (b & 3) : b * 8 + l; };
  float v[C];
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < V; j++) {
      float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (live && place(4 * j) < E) q = __ldg(reinterpret_cast<const float4 *>(mine + place(4 * j)));
      v[4 * j] = q.x; v[4 * j + 1] = q.y; v[4 * j + 2] = q.z; v[4 * j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < C; j++) v[j] = live && place(j) < E ? __ldg(mine + place(j)) : -INFINITY;
  }
  *reinterpret_cast<float4 *>(&left.score[group][4 * l]) = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  // the largest of the 32 sets, and the k-th largest of those
  float set[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    set[i] = v[i];
#pragma unroll
    for (int j = 1; j < V; j++) set[i] = larger_score(set[i], v[4 * j + i]);
  }
  const float lane_top = larger_score(larger_score(set[0], set[1]), larger_score(set[2], set[3]));
  bool odd = lane_top != lane_top;
  const float top = eighth_max(lane_top);
  float bound = top;
  for (int i = 1; i < k; i++) {
#pragma unroll
    for (int j = 0; j < 4; j++) set[j] = set[j] == bound ? -INFINITY : set[j];
    bound = eighth_max(fmaxf(fmaxf(set[0], set[1]), fmaxf(set[2], set[3])));
  }
  bound = fmaxf(bound, -3.402823466e+38f);      // (an open score)
  unsigned in = 0;
#pragma unroll
  for (int b = 0; b < C; b++)
    if (v[b] >= bound) in |= 1u << b;
  int at = __popc(in);
  const int own = at;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, at, o, 8);
    if (l >= o) at += up;
  }
  const int n = __shfl_sync(0xffffffffu, at, 7, 8);      // the row's candidates
  at -= own;
  odd |= n > 32;
  if (__any_sync(0xffffffffu, odd)) {
    static_assert(sizeof(Candidates) <= sizeof(FourRows), "the same memory");
    for (int r = 0; r < 4 && first + r < rows; r++) {
      __syncwarp();
      route_row<V>(x + (first + r) * ld, weights + (first + r) * k, experts + (first + r) * k, E, k, normalize, *reinterpret_cast<Candidates *>(&left), lane);
    }
    return;
  }
  float total = 0.f;
  if (!normalize && top != -INFINITY) {
#pragma unroll
    for (int b = 0; b < C; b++) total += expf(v[b] - top);
  }
  __syncwarp();
  while (__any_sync(0xffffffffu, in != 0)) {
    if (in) {
      const int p = place(__ffs(in) - 1);
      in &= in - 1;
      left.score[group][at] = __ldg(mine + p);
      left.place[group][at++] = (unsigned short)p;
    }
  }
  __syncwarp();
  // the place of each candidate among its row's: a lane has the l-th, the (l + 8)-th ...
  const int most = __reduce_max_sync(0xffffffffu, n);
  float score[4];
  int rank[4], sum = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    rank[i] = 0;
    score[i] = 8 * i < most ? left.score[group][8 * i + l] : -INFINITY;
  }
  for (int j = 0; j < most; j += 4) {
    const float4 o = *reinterpret_cast<const float4 *>(&left.score[group][j]);
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (8 * i < most) rank[i] += (o.x > score[i]) + (o.y > score[i]) + (o.z > score[i]) + (o.w > score[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) sum += 8 * i + l < n ? rank[i] : 0;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (__any_sync(0xffffffffu, 2 * sum != n * (n - 1))) {      // equal scores: by their place
    for (int j = 0; j < most; j++) {
      const float o = left.score[group][j];
      const int p = left.place[group][j];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (8 * i + l < n) rank[i] += o == score[i] && j < n && p < left.place[group][8 * i + l];
    }
  }
  float e[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    e[i] = 0.f;
    if (8 * i < most) {
      if (8 * i + l < n && rank[i] < k) e[i] = expf(score[i] - top);
      if (normalize) total += e[i];
    }
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (!live) return;
  weights += row * k;
  experts += row * k;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int c = 8 * i + l;
    if (c < n) {
      if (rank[i] < k) {
        weights[rank[i]] = e[i] / total;
        experts[rank[i]] = (float)(left.place[group][c] + 1);
      }
    } else if (c < k) weights[c] = experts[c] = 0.f;
  }
}

// The gradient of a row's scores.  x is read where the weights are of the whole softmax, and may else be null.  32768 x 256, 8 chosen: 6.2 us without x (5.5 TB/s of what it
// writes) and 15.3 with it; 7001 x 77: 3.9 with it.
template <int V, bool VEC>
static __global__ void __launch_bounds__(256) router_backward_kernel(const float *__restrict__ x, long ldx, const float *__restrict__ g, long ldg,
                                                                     const float *__restrict__ weights, const float *__restrict__ experts, float *__restrict__ gx,
                                                                     long rows, int E, int k) {
  pdl_begin();
  typedef WarpRow<V, VEC> Row;
  __shared__ __align__(16) float share[8][32 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long row = blockIdx.x * 8l + warp;
  if (row >= rows) return;
  float w = 0.f, d = 0.f, v[V];
  int expert = -1;
  if (lane < k) {
    expert = (int)experts[row * k + lane] - 1;
    w = weights[row * k + lane];
    d = g[row * ldg + lane];
  }
  if (x) Row::load(x + row * ldx, lane, E, v);
  if (expert < 0) w = d = 0.f;                  // (whatever lay there)
  // each expert's share to its place, through shared memory
  float out[V], *mine = share[warp];
#pragma unroll
  for (int j = 0; j < V; j++) mine[j * 32 + lane] = 0.f;
  const float spread = warp_total(w * d);
  __syncwarp();
  if (expert >= 0 && expert < E) mine[expert] = x ? d : w * (d - spread);
  __syncwarp();
  if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const float4 q = *reinterpret_cast<const float4 *>(mine + Row::at(j, lane));
      out[j] = q.x; out[j + 1] = q.y; out[j + 2] = q.z; out[j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; j++) out[j] = mine[j * 32 + lane];
  }
  if (x) {
    float top = -INFINITY, total = 0.f;
#pragma unroll
    for (int j = 0; j < V; j++) top = fmaxf(top, v[j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int j = 0; j < V; j++) {
      v[j] = v[j] == -INFINITY ? 0.f : expf(v[j] - top);
      total += v[j];
    }
    total = warp_total(total);
#pragma unroll
    for (int j = 0; j < V; j++) out[j] = v[j] == 0.f ? 0.f : v[j] / total * (out[j] - spread);
  }
  Row::store(gx + row * E, lane, E, out);
}

// f(integral constant V, bool constant VEC) for rows of E scores
template <class F> static void with_row(int E, bool vec, F f) {
  const int v = (E + 31) / 32;
  auto go = [&](auto V) {
    if constexpr (decltype(V)::value >= 4) {
      if (vec) return f(V, std::true_type());
    }
    f(V, std::false_type());
  };
  if (v <= 1) go(std::integral_constant<int, 1>());
  else if (v <= 2) go(std::integral_constant<int, 2>());
  else if (v <= 4) go(std::integral_constant<int, 4>());
  else if (v <= 8) go(std::integral_constant<int, 8>());
  else if (v <= 16) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 32>());
}
static bool in_pieces(const float *p, long ld, int E) { return ((uintptr_t)p & 15) == 0 && ld % 4 == 0 && E % 4 == 0; }

}  // namespace thc

using namespace thc;

THC_API int THGPUNN_Router_updateOutput(THGPUTensor *input, THGPUTensor *weights, THGPUTensor *experts, int k, int normalize) {
  THC_BEGIN
  THC_ARG(input && weights && experts, 1, "tensors expected");
  check_here({input, weights, experts});
  const long rows = nelem(input) ? input->size[0] : 0;
  if (rows) THC_ARG(input->nDimension == 2, 1, "batch of rows of scores expected");
  const long E = rows ? input->size[1] : kRouterScores;
  THC_ARG(E <= kRouterScores, 1, "at most 1024 scores a row");
  THC_ARG(k >= 1 && k <= kRouterChosen && k <= E, 4, "between 1 and 32 experts a row, and no more than there are, expected");
  const long s[2] = {rows, k};
  size_result(weights, 2, s, {input, experts}, 2);
  size_result(experts, 2, s, {input, weights}, 3);
  if (rows == 0) return 0;
  DenseRows x(input);
  const bool vec = in_pieces(x.p, x.ld, (int)E);
  with_row((int)E, vec, [&](auto V, auto VEC) {
    constexpr int v = decltype(V)::value;
    if constexpr (v <= 8) {
      if (rows >= kManyRows && k <= kManyChosen) {
        auto go = [&](auto PIECES) {
          pdl_launch(router_forward_rows_kernel<v, decltype(PIECES)::value>, (unsigned)ceil_div(rows, 8), 64, 0, x.p, x.ld, data_ptr(weights), data_ptr(experts), rows,
                     (int)E, k, normalize != 0);
        };
        if (vec) go(std::true_type());
        else go(std::false_type());
        return;
      }
    }
    pdl_launch(router_forward_kernel<v>, (unsigned)ceil_div(rows, 8), 256, 0, x.p, x.ld, data_ptr(weights), data_ptr(experts), rows, (int)E, k, normalize != 0);
  });
  check_launch("Router_updateOutput");
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_Router_updateGradInput(THGPUTensor *input, THGPUTensor *gradWeights, THGPUTensor *gradInput, THGPUTensor *weights, THGPUTensor *experts,
                                           int normalize) {
  THC_BEGIN
  THC_ARG(input && gradWeights && gradInput && weights && experts, 1, "tensors expected");
  check_here({input, gradWeights, gradInput, weights, experts});
  const long rows = nelem(input) ? input->size[0] : 0;
  if (rows) THC_ARG(input->nDimension == 2, 1, "batch of rows of scores expected");
  const long E = rows ? input->size[1] : 0;
  THC_ARG(E <= kRouterScores, 1, "at most 1024 scores a row");
  const long k = rows && weights->nDimension == 2 ? weights->size[1] : 0;
  auto fits = [&](const THGPUTensor *t) { return rows ? t->nDimension == 2 && t->size[0] == rows && t->size[1] == k : nelem(t) == 0; };
  THC_ARG(fits(weights) && is_contiguous(weights) && k <= kRouterChosen, 4, "weights of this input, as updateOutput left them, expected");
  THC_ARG(fits(experts) && is_contiguous(experts), 5, "experts of this input, as updateOutput left them, expected");
  THC_ARG(fits(gradWeights), 2, "gradWeights has the wrong size");
  const long s[2] = {rows, E};
  size_result(gradInput, 2, s, {input, gradWeights, weights, experts}, 3);
  if (rows == 0) return 0;
  DenseRows g(gradWeights);
  auto run = [&](const float *x, long ldx) {
    const bool vec = in_pieces(data_ptr(gradInput), E, (int)E) && (!x || in_pieces(x, ldx, (int)E));
    with_row((int)E, vec, [&](auto V, auto VEC) {
      pdl_launch(router_backward_kernel<decltype(V)::value, decltype(VEC)::value>, (unsigned)ceil_div(rows, 8), 256, 0, x, ldx, g.p, g.ld, data_ptr(weights),
                 data_ptr(experts), data_ptr(gradInput), rows, (int)E, (int)k);
    });
  };
  if (normalize) run(nullptr, 0);
  else {
    DenseRows x(input);
    run(x.p, x.ld);
  }
  check_launch("Router_updateGradInput");
  return 0;
  THC_END(1)
}
