// nn.Dispatch and nn.Combine: rows copied to the experts they go to, sorted by expert, and each token's rows summed again.
//
//   slot (t, i) of T tokens with k slots each names an expert, from 1, or none: 0.  Slots sorted by expert, then by t k + i, are the rows; pos(t, i) is
//   the place of the slot's row, from 1, 0 where it has none.
//   Dispatch  rows[pos(t, i)] = x[t];                    dx[t] = sum_i drows[pos(t, i)]
//   Combine   y[t] = residual[t] + sum_i w(t, i) rows[pos(t, i)];  drows[pos(t, i)] = w(t, i) dy[t],  dw(t, i) = <dy[t], rows[pos(t, i)]>
//
// A row is D values of 4 bytes and is read or written once: all of it is bound by HBM, in small calls by launches.  Each thread of a token's team takes the
// same columns of all its rows, so that nothing but the dot products crosses threads, and every result has one writer and one order
// (in Combine's gradient of rows of which each has one slot; rows without one are zero).
#include <cstring>
#include <type_traits>
#include <vector>

#include "nn_args.h"
#include "per_device.h"

namespace thc {

constexpr long kMostSlots = 1l << 24;     // positions are floats
constexpr int kMostGroups = 4096;
constexpr long kMostValues = 1l << 23;    // of a row: its pieces are a dimension of the grid
// Three ways to rank the slots, us a call with 64 groups: by every block of the copy for its own token, in a launch of its own, in two.  The first reads all slots in each of its
// blocks, one for a token and 1024 of its columns, or 256 without 16-byte pieces: where blocks times slots are 2^20 or fewer.  Blocks x slots, first and second way: 96 x 192 9.1 and
// 9.7; 512 x 1024 9.5 and 10.6; 256 x 2048 9.9 and 10.9; 2048 x 512 9.5 and 9.8; 1024 x 1024 9.8 and 10.6; 1024 x 2048 11 to 14 and 11; 2048 x 2048 15 and 11; 32768 x 2048 108 and 14.
// The second and the third, rows of 16 values: 16384 slots 11.7 and 11.9, 32768 13.7 and 12.2, 65536 17.2 and 12.8.  With rows of 1024 values the line lies
// at 32768 as well (34.3 and 34.7; 65536: 62.4 and 60.0); with 1024 groups further on (36.5 and 42.1; 64.5 and 72.5).
constexpr long kFewSlots = 2048, kFewReads = 1l << 20, kRankedSlots = 32768;
constexpr int kRankedGroups = 1024;       // of the second way: a thread each

// The expert of a slot, from 1; 0: none; -1: the number stands for no expert.
static __device__ __forceinline__ int slot_expert(float e, int groups) {
  return e >= 0.f && e <= (float)groups && e == truncf(e) ? (int)e : -1;
}
// The row at a place, or -1: a place that stands for none of the `rows` is passed over.
static __device__ __forceinline__ int row_at(float place, long rows) {
  const int r = (int)place;               // (of an infinity the last number there is, of a NaN none above zero; places beyond 2^24 are none of Dispatch's)
  return r >= 1 && r <= kMostSlots && r <= rows ? r - 1 : -1;
}

// ---- where the rows go -------------------------------------------------------------------------------------------------
// The first block tells the host the rows of each group, and as one more group the slots whose number stands for no expert.
// Many slots: in pieces of `per`, a block each.  The first launch counts: hist[group][chunk], the bad numbers as one more group.  In the second one
// a block adds up what lies before its own piece, counts its warps' shares of it, and each warp goes through its share 32 slots at a time.
static __global__ void __launch_bounds__(256) slots_count_kernel(const float *__restrict__ experts, long slots, int per, int groups, int *__restrict__ hist) {
  pdl_begin();
  extern __shared__ int count[];   // [groups + 1]
  for (int g = threadIdx.x; g <= groups; g += 256) count[g] = 0;
  __syncthreads();
  const long from = blockIdx.x * (long)per, to = min(slots, from + per);
  for (long s = from + threadIdx.x; s < to; s += 256) {
    const int e = slot_expert(experts[s], groups);
    if (e != 0) atomicAdd(&count[e > 0 ? e - 1 : groups], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g <= groups; g += 256) hist[(long)g * gridDim.x + blockIdx.x] = count[g];
}

static __global__ void __launch_bounds__(1024) slots_place_kernel(const float *__restrict__ experts, long slots, int per, int groups, const int *__restrict__ hist,
                                                                  float *__restrict__ positions, CountStage tell) {
  pdl_begin();
  extern __shared__ int place[];                   // [8 warps][groups]: rows before the warp's next one of a group
  int *before = place + 8 * groups, *total = before + groups;   // [groups]: a group's rows in the pieces before this one, and in all; [groups + 1] with the bad numbers
  __shared__ int sums[32];
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, chunks = gridDim.x;
  const long from = blockIdx.x * (long)per, to = min(slots, from + per);
  const int share = (per / 8 + 31) & ~31;          // of the first eight warps; the others help with the sums
  const long mine = warp < 8 ? from + (long)warp * share : to, end = min(to, mine + share);
  for (int g = t; g < 8 * groups; g += 1024) place[g] = 0;
  __syncthreads();
  for (long s = mine + lane; s < end; s += 32) {
    const int e = slot_expert(experts[s], groups);
    if (e > 0) atomicAdd(&place[warp * groups + e - 1], 1);
  }
  for (int g = 4 * warp; g <= groups; g += 128) {     // (four groups at a time: what comes from L2 is on its way together)
    int all[4] = {}, ahead[4] = {};
#pragma unroll 5
    for (int c = lane; c < chunks; c += 32) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int n = g + i <= groups ? hist[(long)(g + i) * chunks + c] : 0;
        all[i] += n;
        if (c < (int)blockIdx.x) ahead[i] += n;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      all[i] = __reduce_add_sync(0xffffffffu, all[i]);
      ahead[i] = __reduce_add_sync(0xffffffffu, ahead[i]);
      if (lane == i && g + i <= groups) {
        total[g + i] = all[i];
        if (g + i < groups) before[g + i] = ahead[i];
      }
    }
  }
  __syncthreads();
  if (blockIdx.x == 0)                             // (neighbours together: each store is a message to the host)
    for (int g = t; g <= groups; g += 1024) count_deliver(tell, g, total[g]);
  // the groups' first rows: each thread has some neighbouring groups
  const int some = (groups + 1023) / 1024, g0 = min(groups, t * some), g1 = min(groups, g0 + some);
  int own = 0;
  for (int g = g0; g < g1; g++) own += total[g];
  int run = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  int first = run - own + __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);
  for (int g = g0; g < g1; g++) {
    int at = first + before[g];
    for (int w = 0; w < 8; w++) {
      const int n = place[w * groups + g];
      place[w * groups + g] = at;
      at += n;
    }
    first += total[g];
  }
  __syncthreads();
  for (long s = mine; s < end; s += 32) {
    const int e = s + lane < end ? max(0, slot_expert(experts[s + lane], groups)) : 0;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    int at = 0;
    if (e > 0) at = place[warp * groups + e - 1];
    __syncwarp();
    if (e > 0 && lane == __ffs(same) - 1) place[warp * groups + e - 1] = at + __popc(same);
    __syncwarp();
    if (s + lane < end) positions[s + lane] = e > 0 ? (float)(at + __popc(same & ((1u << lane) - 1)) + 1) : 0.f;
  }
}

// In one launch, where every block can as well count all slots by itself: 1024 threads with a slot each.
static __global__ void __launch_bounds__(1024) slots_rank_kernel(const float *__restrict__ experts, int slots, int groups, float *__restrict__ positions,
                                                                 CountStage tell) {
  pdl_begin();
  extern __shared__ int ahead[];                                  // [32 warps][groups]: rows of a group in the warps, then before them
  int *before = ahead + 32 * groups, *after = before + groups;    // [groups]: rows of the slots before the block's, and behind them
  __shared__ int sums[32], wrong;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, from = blockIdx.x * 1024, mine = from + t;
  for (int g = t; g < 34 * groups; g += 1024) ahead[g] = 0;
  if (t == 0) wrong = 0;
  const int e = mine < slots ? slot_expert(experts[mine], groups) : 0;
  __syncthreads();
  const unsigned same = __match_any_sync(0xffffffffu, e);
  const bool leads = lane == __ffs(same) - 1;
  if (leads && e > 0) ahead[warp * groups + e - 1] = __popc(same);
  if (leads && e < 0) atomicAdd(&wrong, __popc(same));
  // the others' four at a time, of one block each
  const bool whole = ((uintptr_t)experts & 15) == 0;
#pragma unroll 4
  for (int s = 4 * t; s < slots; s += 4096) {
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (whole && s + 4 <= slots) {
      const float4 q = __ldg(reinterpret_cast<const float4 *>(experts + s));
      x[0] = q.x; x[1] = q.y; x[2] = q.z; x[3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (s + j < slots) x[j] = __ldg(experts + s + j);
    }
    if (s >= from && s < from + 1024) continue;
    int *count = s < from ? before : after;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int o = slot_expert(x[j], groups);
      if (o > 0) atomicAdd(&count[o - 1], 1);
      else if (o < 0) atomicAdd(&wrong, 1);
    }
  }
  __syncthreads();
  int total = 0;                                                  // thread g: group g, at most 1024 of them
  if (t < groups) {
    int n[32], at = before[t];
#pragma unroll
    for (int w = 0; w < 32; w++) n[w] = ahead[w * groups + t];
#pragma unroll
    for (int w = 0; w < 32; w++) {
      ahead[w * groups + t] = at;
      at += n[w];
    }
    total = at + after[t];
    if (blockIdx.x == 0) count_deliver(tell, t, total);
  }
  if (blockIdx.x == 0 && t == 0) count_deliver(tell, groups, wrong);
  int run = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += up;
  }
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  const int base = run - total + __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0);
  if (t < groups) before[t] = base;
  __syncthreads();
  if (mine < slots) positions[mine] = e > 0 ? (float)(before[e - 1] + ahead[warp * groups + e - 1] + __popc(same & ((1u << lane) - 1)) + 1) : 0.f;
}

// ---- copying and summing rows ------------------------------------------------------------------------------------------
// Blocks of 256 threads in teams of T, a team for each token (blockIdx.x) and T U W of its columns (blockIdx.y): U pieces of W = 4 values, or one where
// lengths or addresses do not allow it, a thread.
template <int T, int U, bool VEC> struct Columns {
  static constexpr int W = VEC ? 4 : 1;
  float v[U * W];
  int c;                                              // the thread's first column; its u-th piece is u T W further on
  Columns() = default;
  __device__ __forceinline__ explicit Columns(long piece) : c((int)(piece * (T * U * W)) + (int)(threadIdx.x % T) * W) {}
  static __device__ __forceinline__ long token(int before = 0) { return (blockIdx.x - before) * (long)(256 / T) + threadIdx.x / T; }     // (blocks before its own)
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < U * W; j++) v[j] = 0.f;
  }
  __device__ __forceinline__ void load(const float *__restrict__ row, int n) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = c + u * T * W;
      if constexpr (VEC) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at < n) q = __ldg(reinterpret_cast<const float4 *>(row + at));
        v[4 * u] = q.x; v[4 * u + 1] = q.y; v[4 * u + 2] = q.z; v[4 * u + 3] = q.w;
      } else v[u] = at < n ? __ldg(row + at) : 0.f;
    }
  }
  // to L2, a lane for each line
  __device__ __forceinline__ void bring(const float *row, int n) const {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = c + u * T * W;
      if (at < n && (threadIdx.x * W) % 32 == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + at));
    }
  }
  __device__ __forceinline__ void store(float *__restrict__ row, int n) const {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int at = c + u * T * W;
      if (at >= n) continue;
      if constexpr (VEC) *reinterpret_cast<float4 *>(row + at) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
      else row[at] = v[u];
    }
  }
};

// Rows on their way at once: eight with one piece of each a thread, else two, with four pieces of 16 bytes or eight of 4.  (Eight rows by four pieces of 4 bytes took more
// registers and twice the time: 19056 x 333, 2 rows a token, 22.6 us against 11.4, backward 69 against 25; two rows by four pieces 11.4 and 33.)
template <int U> static __host__ __device__ constexpr int rows_at_once() { return U == 1 ? 8 : 2; }

struct Rows {            // a matrix of rows at a distance
  const float *p;
  long ld;
};

// rows[pos(t, i)] = x[t].  8192 x 4096, two rows a token: 60 us, 6.7 TB/s.
template <int T, int U, bool VEC>
static __global__ void __launch_bounds__(256) rows_out_kernel(Rows x, const float *__restrict__ positions, float *__restrict__ rows, long tokens, int k, int D, long most) {
  typedef Columns<T, U, VEC> Cols;
  const long t = Cols::token();
  Cols a(blockIdx.y);
  if (t < tokens) a.bring(x.p + t * x.ld, D);      // while the slots are still being ranked: 3 of 68 us for 8192 x 4096
  pdl_begin();
  if (t >= tokens) return;
  a.load(x.p + t * x.ld, D);
  for (int i = 0; i < k; i++) {
    const int r = row_at(__ldg(positions + t * k + i), most);
    if (r >= 0) a.store(rows + (long)r * D, D);
  }
}

// The same for few slots, with the ranking: a block for a token and 256 U W of its columns.  A slot's place is the number of slots that name a lower expert,
// or the same and come before it.  One more block counts for the host, behind those of the tokens' first columns: at most 1024 of them (each reads as many slots or more), which find room at
// once, so that it waits for no copy.  24 x 4096, 8 of 64 experts: 8.6 us from the call to the counts, most of them on the way to the GPU and back; with that block in front 0.1 to 0.5 longer.
template <int U, bool VEC>
static __global__ void __launch_bounds__(256) few_rows_out_kernel(Rows x, const float *__restrict__ experts, float *__restrict__ positions, float *__restrict__ rows, int k,
                                                                  int D, int slots, int groups, CountStage tell) {
  pdl_begin();
  extern __shared__ int expert[];       // [slots] and the token's rows [k], or the counts [groups + 1]
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  if (blockIdx.x == gridDim.x - 1) {
    if (blockIdx.y) return;
    for (int g = t; g <= groups; g += 256) expert[g] = 0;
    __syncthreads();
    for (int s = t; s < slots; s += 256) {
      const int e = slot_expert(experts[s], groups);
      if (e != 0) atomicAdd(&expert[e > 0 ? e - 1 : groups], 1);
    }
    __syncthreads();
    for (int g = t; g <= groups; g += 256) count_deliver(tell, g, expert[g]);
    return;
  }
  int *mine = expert + slots;
  const long token = blockIdx.x;
  Columns<256, U, VEC> a(blockIdx.y);
  a.load(x.p + token * x.ld, D);
  for (int s = t; s < slots; s += 256) expert[s] = slot_expert(experts[s], groups);
  __syncthreads();
  for (int i = warp; i < k; i += 8) {
    const int at = (int)token * k + i, e = expert[at];
    int before = 0;
    for (int s = lane; s < slots; s += 32) before += expert[s] > 0 && (expert[s] < e || (expert[s] == e && s < at));
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) {
      mine[i] = e > 0 ? before : -1;
      if (blockIdx.y == 0) positions[at] = e > 0 ? (float)(before + 1) : 0.f;
    }
  }
  __syncthreads();
  for (int i = 0; i < k; i++)
    if (mine[i] >= 0) a.store(rows + mine[i] * (long)D, D);
}

// y[t] = residual[t] + sum_i w(t, i) rows[pos(t, i)]; w and the residual may be null.  8192 x 4096, two rows a token: 58.7 us, 6.9 TB/s; 24 x 4096, eight rows and a
// residual: 3.3 us a call; 19056 x 333, two rows: 11.4 us, 6.7 TB/s, from L2 in part.
template <int T, int U, bool VEC>
static __global__ void __launch_bounds__(256) rows_sum_kernel(Rows rows, const float *__restrict__ w, const float *__restrict__ positions, Rows residual,
                                                              float *__restrict__ y, long tokens, int k, int D, long most) {
  pdl_begin();
  typedef Columns<T, U, VEC> Cols;
  const long t = Cols::token();
  if (t >= tokens) return;
  Cols a(blockIdx.y);
  if (residual.p) a.load(residual.p + t * residual.ld, D);
  else a.zero();
  constexpr int B = rows_at_once<U>();
  for (int i0 = 0; i0 < k; i0 += B) {
    int r[B];
    float f[B];
    Cols b[B];
#pragma unroll
    for (int i = 0; i < B; i++) {
      r[i] = i0 + i < k ? row_at(__ldg(positions + t * k + i0 + i), most) : -1;
      f[i] = r[i] < 0 ? 0.f : w ? __ldg(w + t * k + i0 + i) : 1.f;
    }
#pragma unroll
    for (int i = 0; i < B; i++) {
      b[i].c = a.c;
      b[i].zero();
      if (r[i] >= 0) b[i].load(rows.p + r[i] * rows.ld, D);
    }
#pragma unroll
    for (int i = 0; i < B; i++) {
#pragma unroll
      for (int j = 0; j < U * Cols::W; j++) a.v[j] = fmaf(f[i], b[i].v[j], a.v[j]);
    }
  }
  a.store(y + t * D, D);
}

// Rows that no slot names, which Combine's gradient makes zero: blocks of their own look for them, each among some rows, in all slots, whose places they read in 16-byte
// pieces ahead.  A place stands for the row that row_at gives: its distance from the block's first row's place is exact, and in the sum with 2^23, rounded down, the low bits are
// its whole part; distances below zero, beyond the rows and no numbers become words that are too large.
constexpr int kClearRows = 32768;         // of a block at most: a bit each
constexpr int kClearBlocks = 64;
static __device__ __noinline__ void clear_rows(unsigned *named, const float *__restrict__ positions, long slots, float *__restrict__ rows, long first, int n, int D) {
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  for (int w = t; w * 32 < n; w += 256) named[w] = 0;
  __syncthreads();
  const unsigned words = (unsigned)__cvta_generic_to_shared(named), valid = first < kMostSlots ? (unsigned)min((long)n, kMostSlots - first) : 0;
  const float from = (float)(first + 1);               // (exact where rows are valid)
  auto name = [&](float place) {
    const unsigned r = __float_as_uint(__fadd_rd(place - from, 8388608.f)) - 0x4b000000u;
    asm volatile("{ .reg .pred p; setp.lt.u32 p, %0, %1; @p red.shared.or.b32 [%2], %3; }" ::"r"(r), "r"(valid), "r"(words + (r >> 5) * 4), "r"(1u << (r & 31)) : "memory");
  };
  const long head = min(slots, (long)((16 - ((uintptr_t)positions & 15)) & 15) / 4), quads = (slots - head) / 4;
  if (t < head) name(__ldg(positions + t));
  if (t < slots - head - 4 * quads) name(__ldg(positions + head + 4 * quads + t));
  const float4 *p = reinterpret_cast<const float4 *>(positions + head);
  float4 q[4], next[4];
  auto load = [&](float4 (&v)[4], long s) {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = s + 256 * i < quads ? __ldg(p + s + 256 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  load(q, t);
  for (long s = t; s < quads; s += 1024) {
    load(next, s + 1024);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      name(q[i].x); name(q[i].y); name(q[i].z); name(q[i].w);
      q[i] = next[i];
    }
  }
  __syncthreads();
  const bool vec = D % 4 == 0 && ((uintptr_t)rows & 15) == 0;
  for (int w = warp; w * 32 < n; w += 8) {
    unsigned none = ~named[w];
    if (n - w * 32 < 32) none &= (1u << (n - w * 32)) - 1;
    for (; none; none &= none - 1) {
      float *row = rows + (first + w * 32 + __ffs(none) - 1) * D;
      if (vec)
        for (int c = 4 * lane; c < D; c += 128) *reinterpret_cast<float4 *>(row + c) = make_float4(0.f, 0.f, 0.f, 0.f);
      else
        for (int c = lane; c < D; c += 32) row[c] = 0.f;
    }
  }
}

// All rows zero.  (A memory operation between kernels takes 2 us more than one that starts as a programmatic dependent.)
static __global__ void __launch_bounds__(256) clear_all_kernel(float *__restrict__ p, long n) {
  pdl_begin();
  const long head = min(n, (long)((16 - ((uintptr_t)p & 15)) & 15) / 4), quads = (n - head) / 4, step = gridDim.x * 256l;
  const long t = blockIdx.x * 256l + threadIdx.x;
  if (t < head) p[t] = 0.f;
  if (t < n - head - 4 * quads) p[head + 4 * quads + t] = 0.f;
  float4 *q = reinterpret_cast<float4 *>(p + head);
  for (long i = t; i < quads; i += step) q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
}

// drows[pos(t, i)] = w(t, i) dy[t] and dw(t, i) = <dy[t], rows[pos(t, i)]>, either of them unless null; w may be null.  A team has all columns of its token.
// 8192 x 2048, eight rows a token: 173 us, 6.6 TB/s; 19056 x 333, two rows: 25 us, 5.0 TB/s.
constexpr int kDotSlots = 32;
template <int T, int U, bool VEC>
static __global__ void __launch_bounds__(256) rows_sum_backward_kernel(Rows rows, const float *__restrict__ w, const float *__restrict__ positions, Rows dy,
                                                                       float *__restrict__ drows, float *__restrict__ dw, long tokens, int k, int D, long most,
                                                                       int clears, int each) {
  pdl_begin();
  typedef Columns<T, U, VEC> Cols;
  constexpr int WARPS = T > 32 ? T / 32 : 1;       // of a team
  __shared__ union {
    float dots[256 / T][WARPS][kDotSlots];
    unsigned named[kClearRows / 32];
  } shared;
  if ((int)blockIdx.x < clears) {
    const long first = blockIdx.x * (long)each;
    clear_rows(shared.named, positions, tokens * k, drows, first, (int)min((long)each, most - first), D);
    return;
  }
  auto &dots = shared.dots;
  const long t = Cols::token(clears);
  const int team = threadIdx.x / T, member = threadIdx.x % T, pieces = (D + T * U * Cols::W - 1) / (T * U * Cols::W);
  const bool live = t < tokens;                    // (teams of a warp stay together: the others take part in its exchanges)
  constexpr int B = U == 1 ? 4 : 2;                // as rows_at_once, with gradOutput's row in registers as well
  Cols g(0);
  if (live && pieces == 1) g.load(dy.p + t * dy.ld, D);
  for (int i0 = 0; i0 < k; i0 += kDotSlots) {
    const int n = min(kDotSlots, k - i0);
    for (int i = 0; i < n; i += B) {
      int r[B];
      float f[B], dot[B];
#pragma unroll
      for (int b = 0; b < B; b++) {
        const long slot = t * k + i0 + i + b;
        r[b] = live && i + b < n ? row_at(__ldg(positions + slot), most) : -1;
        f[b] = r[b] < 0 ? 0.f : w ? __ldg(w + slot) : 1.f;
        dot[b] = 0.f;
      }
      for (int p = 0; p < pieces; p++) {
        Cols row[B];
#pragma unroll
        for (int b = 0; b < B; b++) {
          row[b] = Cols(p);
          row[b].zero();
          if (dw && r[b] >= 0) row[b].load(rows.p + r[b] * rows.ld, D);
        }
        if (live && pieces > 1) {
          g = Cols(p);
          g.load(dy.p + t * dy.ld, D);
        }
#pragma unroll
        for (int b = 0; b < B; b++) {
#pragma unroll
          for (int j = 0; j < U * Cols::W; j++) {
            dot[b] = fmaf(row[b].v[j], g.v[j], dot[b]);
            row[b].v[j] = f[b] * g.v[j];
          }
          if (drows && r[b] >= 0) row[b].store(drows + (long)r[b] * D, D);
        }
      }
      if (!dw) continue;
#pragma unroll
      for (int b = 0; b < B; b++) {
#pragma unroll
        for (int o = (T < 32 ? T : 32) / 2; o > 0; o >>= 1) dot[b] += __shfl_xor_sync(0xffffffffu, dot[b], o);
        if (member % 32 == 0 && i + b < n) dots[team][member / 32][i + b] = r[b] < 0 ? 0.f : dot[b];     // (0 times a NaN of gradOutput)
      }
    }
    if (!dw) continue;
    if constexpr (T > 32) __syncthreads();
    else __syncwarp();
    for (int i = member; live && i < n; i += T) {
      float s = dots[team][0][i];
#pragma unroll
      for (int o = 1; o < WARPS; o++) s += dots[team][o][i];
      dw[t * k + i0 + i] = s;
    }
    if constexpr (T > 32) __syncthreads();
    else __syncwarp();
  }
}

// f(integral constants T, U, VEC) for rows of D values, k of which come to a token.  T: for rows that half a warp or less covers, and where a team has to have all of its row
// (whole), the narrowest team that does, at most a block; else the widest that leaves the fewest columns over.  U: one piece a thread, and up to eight rows at a time, for few
// rows, which that spreads over more SMs, and for narrow ones, both where k is more than two; else more pieces of two rows at a time.
// Combine, 8 rows a token, us with one piece and with four: 24 x 4096 3.1 and 4.5, 128 x 4096 3.6 and 4.6, 256 x 4096 5.3 and 4.4, 4096 x 64 3.7 and 5.5; backward 128 x 1024
// 3.6 and 5.7, 512 x 1024 6.9 and 6.0, 4096 x 64 6.5 and 9.2.  2 rows a token: 8192 x 64 4.5 and 3.5.  Teams of a warp and of eight lanes, 22024 x 20, 6 rows a token: 10.8 and 4.0.
template <class F> static void with_columns(long tokens, int D, int k, bool vec, bool whole, F f) {
  auto go = [&](auto VEC, auto U) {
    constexpr int per = (decltype(VEC)::value ? 4 : 1) * decltype(U)::value;
    int team = 256;
    if (whole || D <= 32 * per) {
      while (team > 8 && D <= team / 2 * per) team /= 2;
    } else if (D <= 16 * 256 * per) {
      auto width = [&](int t) { return (long)ceil_div(D, t * per) * t; };
      for (int t = 128; t >= 32; t /= 2)
        if (width(t) < width(team)) team = t;
    }
    if (team == 8) f(std::integral_constant<int, 8>(), U, VEC);
    else if (team == 16) f(std::integral_constant<int, 16>(), U, VEC);
    else if (team == 32) f(std::integral_constant<int, 32>(), U, VEC);
    else if (team == 64) f(std::integral_constant<int, 64>(), U, VEC);
    else if (team == 128) f(std::integral_constant<int, 128>(), U, VEC);
    else f(std::integral_constant<int, 256>(), U, VEC);
  };
  const int w = vec ? 4 : 1;
  const bool few = tokens * (long)D <= ctx().sm_count * (whole ? 512l : 1024l) * w, narrow = vec && D <= 128;
  const bool one = k > 2 && (few || narrow) && (!whole || D <= 256 * w);
  auto with_u = [&](auto VEC) {
    if (one) go(VEC, std::integral_constant<int, 1>());
    else go(VEC, std::integral_constant<int, decltype(VEC)::value ? 4 : 8>());
  };
  if (vec) with_u(std::true_type());
  else with_u(std::false_type());
}

static bool pieces_of_four(std::initializer_list<Rows> all, int D) {
  bool ok = D % 4 == 0;
  for (const Rows &r : all) ok = ok && ((uintptr_t)r.p & 15) == 0 && r.ld % 4 == 0;
  return ok;
}

// ---- launches
// Whether slots may be ranked block by block.
static bool are_few(long slots, int k, long blocks) { return slots <= kFewSlots && k <= 64 && slots * blocks <= kFewReads; }

static void dispatch(Rows x, const float *experts, long tokens, int k, int D, int groups, float *positions, float *rows, const CountStage &tell) {
  const long slots = tokens * k;
  const bool vec = pieces_of_four({x, Rows{rows, D}}, D);
  if (are_few(slots, k, tokens * ceil_div(D, vec ? 1024 : 256))) {
    const size_t smem = sizeof(int) * std::max(slots + k, groups + 1l);
    if (vec) pdl_launch(few_rows_out_kernel<1, true>, dim3((unsigned)tokens + 1, (unsigned)ceil_div(D, 1024)), 256, smem, x, experts, positions, rows, k, D, (int)slots, groups, tell);
    else pdl_launch(few_rows_out_kernel<1, false>, dim3((unsigned)tokens + 1, (unsigned)ceil_div(D, 256)), 256, smem, x, experts, positions, rows, k, D, (int)slots, groups, tell);
    check_launch("Dispatch_updateOutput");
    return;
  }
  const int sms = ctx().sm_count;
  if (slots <= kRankedSlots && groups <= kRankedGroups) {
    static PerDevice allowed;
    allowed.get(ctx().device, [&] {
      THC_CUDA(cudaFuncSetAttribute(slots_rank_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(int) * 34 * kRankedGroups));
      return 1;
    });
    pdl_launch(slots_rank_kernel, (unsigned)ceil_div(slots, 1024), 1024, sizeof(int) * 34 * groups, experts, (int)slots, groups, positions, tell);
    check_launch("Dispatch_updateOutput");
  } else {
    const int per = (int)std::max(1024l, (slots + sms * 256l - 1) / (sms * 256l) * 256), chunks = ceil_div(slots, per);
    int *hist = (int *)ws_alloc(sizeof(int) * (groups + 1) * chunks);
    pdl_launch(slots_count_kernel, (unsigned)chunks, 256, sizeof(int) * (groups + 1), experts, slots, per, groups, hist);
    check_launch("Dispatch_updateOutput");
    constexpr size_t most = sizeof(int) * (10 * kMostGroups + 1);
    static PerDevice allowed;
    allowed.get(ctx().device, [&] {
      THC_CUDA(cudaFuncSetAttribute(slots_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
      return 1;
    });
    pdl_launch(slots_place_kernel, (unsigned)chunks, 1024, sizeof(int) * (10 * groups + 1), experts, slots, per, groups, hist, positions, tell);
    check_launch("Dispatch_updateOutput");
  }
  with_columns(tokens, D, 1, vec, false, [&](auto T, auto U, auto VEC) {      // (reads a row a token)
    constexpr int t = decltype(T)::value, u = decltype(U)::value, width = t * u * (decltype(VEC)::value ? 4 : 1);
    pdl_launch(rows_out_kernel<t, u, decltype(VEC)::value>, dim3((unsigned)ceil_div(tokens, 256 / t), (unsigned)ceil_div(D, width)), 256, 0, x, positions, rows, tokens, k,
               D, slots);
  });
  check_launch("Dispatch_updateOutput");
}

static void sum_rows(Rows rows, long most, const float *w, const float *positions, Rows residual, float *y, long tokens, int k, int D, const char *what) {
  const bool vec = pieces_of_four({rows, residual, Rows{y, D}}, D);
  with_columns(tokens, D, k, vec, false, [&](auto T, auto U, auto VEC) {
    constexpr int t = decltype(T)::value, u = decltype(U)::value, width = t * u * (decltype(VEC)::value ? 4 : 1);
    pdl_launch(rows_sum_kernel<t, u, decltype(VEC)::value>, dim3((unsigned)ceil_div(tokens, 256 / t), (unsigned)ceil_div(D, width)), 256, 0, rows, w, positions, residual,
               y, tokens, k, D, most);
  });
  check_launch(what);
}

// ---- checks
// Slots of `tokens` tokens: [tokens][k]
static bool slots_fit(const THGPUTensor *t, long tokens, long k) {
  return tokens ? t->nDimension == 2 && t->size[0] == tokens && t->size[1] == k : nelem(t) == 0;
}
static void check_slots(const THGPUTensor *t, int argn) {
  THC_ARG(nelem(t) == 0 || t->nDimension == 2, argn, "matrix of a row of slots for each token expected");
  THC_ARG(nelem(t) <= kMostSlots, argn, "at most 2^24 slots");
}
static void check_rows(const THGPUTensor *t, int argn) {
  THC_ARG(nelem(t) == 0 || t->nDimension == 2, argn, "matrix of rows expected");
  THC_ARG(nelem(t) == 0 || t->size[1] <= kMostValues, argn, "at most 2^23 values a row expected");
}

}  // namespace thc

using namespace thc;

THC_API int THGPUNN_Dispatch_updateOutput(THGPUTensor *input, THGPUTensor *experts, THGPUTensor *output, THGPUTensor *positions, long *counts, int groups) {
  THC_BEGIN
  THC_ARG(input && experts && output && positions, 1, "tensors expected");
  THC_ARG(counts, 5, "room for a count of each group expected");
  THC_ARG(groups >= 1 && groups <= kMostGroups, 6, "between 1 and 4096 groups expected");
  check_here({input, experts, output, positions});
  check_rows(input, 1);
  check_slots(experts, 2);
  const long tokens = nelem(input) ? input->size[0] : 0, D = tokens ? input->size[1] : 0, k = nelem(experts) ? experts->size[1] : 0;
  THC_ARG(slots_fit(experts, tokens, k), 2, "a row of slots for each row of the input expected");
  check_apart(output, {input, experts, positions}, 3);
  check_apart(positions, {input, experts}, 4);
  if (tokens) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    THC_CUDA(cudaStreamIsCapturing(stream(), &capture));
    THC_CHECK(capture == cudaStreamCaptureStatusNone, "Dispatch hands its counts to the host, which cannot be recorded: call it before, and record what follows");
  }
  const long ps[2] = {tokens, k}, room[2] = {tokens * k, D};
  size_result(positions, 2, ps, {input, experts}, 4);
  size_result(output, 2, room, {input, experts, positions}, 3);
  std::memset(counts, 0, sizeof(long) * groups);
  if (tokens == 0) return 0;
  WsScope scope;
  DenseRows x(input);
  TensorRef e(tensor_new_contiguous(experts));
  static_assert(kMostGroups < kCountStage, "a word for each group and one more");
  const CountStage tell = counts_expect();
  dispatch(Rows{x.p, x.ld}, data_ptr(e), tokens, (int)k, (int)D, groups, data_ptr(positions), data_ptr(output), tell);
  std::vector<int> told(groups + 1);
  counts_wait(tell, told.data(), groups + 1);
  long rows = 0;
  for (int g = 0; g < groups; g++) rows += counts[g] = told[g];
  const long s[2] = {rows, D};
  resize_nd(output, 2, s, nullptr);
  if (told[groups]) fail("Invalid argument 2: %d slots hold something else than a whole number from 0 to %d", told[groups], groups);
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_Dispatch_updateGradInput(THGPUTensor *input, THGPUTensor *gradOutput, THGPUTensor *gradInput, THGPUTensor *positions) {
  THC_BEGIN
  THC_ARG(input && gradOutput && gradInput && positions, 1, "tensors expected");
  check_here({input, gradOutput, gradInput, positions});
  check_rows(input, 1);
  check_slots(positions, 4);
  check_rows(gradOutput, 2);
  const long tokens = nelem(input) ? input->size[0] : 0, D = tokens ? input->size[1] : 0, k = nelem(positions) ? positions->size[1] : 0;
  const long rows = nelem(gradOutput) ? gradOutput->size[0] : 0;
  THC_ARG(slots_fit(positions, tokens, k), 4, "positions of this input, as updateOutput left them, expected");
  THC_ARG(rows == 0 || (gradOutput->size[1] == D && rows <= tokens * k), 2, "gradOutput has the wrong size");
  const long s[2] = {tokens, D};
  size_result(gradInput, 2, s, {input, gradOutput, positions}, 3);
  if (tokens == 0) return 0;
  TensorRef p(tensor_new_contiguous(positions));
  auto run = [&](Rows g) { sum_rows(g, rows, nullptr, data_ptr(p), Rows{nullptr, 0}, data_ptr(gradInput), tokens, (int)k, (int)D, "Dispatch_updateGradInput"); };
  if (rows == 0) run(Rows{nullptr, 0});
  else {
    DenseRows g(gradOutput);
    run(Rows{g.p, g.ld});
  }
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_Combine_updateOutput(THGPUTensor *input, THGPUTensor *weights, THGPUTensor *positions, THGPUTensor *residual, THGPUTensor *output, long size) {
  THC_BEGIN
  THC_ARG(input && positions && output, 1, "tensors expected");
  THC_ARG(size >= 1 && size <= kMostValues, 6, "size must be positive and at most 2^23");
  check_here({input, weights, positions, residual, output});
  check_rows(input, 1);
  check_slots(positions, 3);
  const long rows = nelem(input) ? input->size[0] : 0, tokens = nelem(positions) ? positions->size[0] : 0, k = tokens ? positions->size[1] : 0;
  THC_ARG(rows == 0 || input->size[1] == size, 1, "rows of the given size expected");
  if (weights) THC_ARG(slots_fit(weights, tokens, k), 2, "a weight for each slot expected");
  if (residual) THC_ARG(tokens ? residual->nDimension == 2 && residual->size[0] == tokens && residual->size[1] == size : nelem(residual) == 0, 4,
                        "residual of the output's size expected");
  const long s[2] = {tokens, size};
  size_result(output, 2, s, {input, weights, positions, residual}, 5);
  if (tokens == 0) return 0;
  TensorRef p(tensor_new_contiguous(positions)), w(weights ? tensor_new_contiguous(weights) : nullptr);
  THGPUTensor *some = rows ? input : output;      // (without rows nothing is read through it)
  DenseRows x(some);
  auto run = [&](Rows r) {
    sum_rows(Rows{x.p, x.ld}, rows, weights ? data_ptr(w) : nullptr, data_ptr(p), r, data_ptr(output), tokens, (int)k, (int)size, "Combine_updateOutput");
  };
  if (residual) {
    DenseRows r(residual);
    run(Rows{r.p, r.ld});
  } else run(Rows{nullptr, 0});
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_Combine_backward(THGPUTensor *input, THGPUTensor *weights, THGPUTensor *positions, THGPUTensor *gradOutput, THGPUTensor *gradInput,
                                     THGPUTensor *gradWeights) {
  THC_BEGIN
  THC_ARG(input && positions && gradOutput, 1, "tensors expected");
  THC_ARG(weights || !gradWeights, 6, "weights have a gradient where there are weights");
  check_here({input, weights, positions, gradOutput, gradInput, gradWeights});
  check_rows(input, 1);
  check_slots(positions, 3);
  check_rows(gradOutput, 4);
  const long rows = nelem(input) ? input->size[0] : 0, tokens = nelem(positions) ? positions->size[0] : 0, k = tokens ? positions->size[1] : 0;
  const long D = nelem(gradOutput) ? gradOutput->size[1] : rows ? input->size[1] : 0;
  if (weights) THC_ARG(slots_fit(weights, tokens, k), 2, "a weight for each slot expected");
  THC_ARG(tokens ? nelem(gradOutput) && gradOutput->size[0] == tokens : nelem(gradOutput) == 0, 4, "gradOutput has the wrong size");
  THC_ARG(rows == 0 || input->size[1] == D, 1, "rows of gradOutput's size expected");
  const long xs[2] = {rows, D}, ws[2] = {tokens, k};
  if (gradInput) size_result(gradInput, 2, xs, {input, weights, positions, gradOutput, gradWeights}, 5);
  if (gradWeights) size_result(gradWeights, 2, ws, {input, weights, positions, gradOutput, gradInput}, 6);
  // Rows that no slot names: looked for by blocks in front of the tokens', unless these would read more than a twelfth of what the others move, or take longer, as with many narrow
  // rows.  Then all rows are zero first.  us a call without either, searched, and cleared: 8192 x 2048, 8 rows a token 172.1, 172.1; 1537 x 333, 4 rows 5.8, 5.9; 19056 x 333, 2 rows
  // 25.1, 25.2; 512 x 1024, 8 rows 5.9 to 7.1, 6.0 to 7.2; 4096 x 64, 8 rows 4.8, 7.6, 8.1; 32768 x 64, 2 rows 6.7, 12.8, 10.4; 32768 x 128, 8 rows 55.0, 56.9.
  int clears = 0, each = 0;
  if (gradInput && rows) {
    clears = (int)std::min((rows + 255) / 256, std::min((long)kClearBlocks, std::max(1l, D / 4)));
    clears = std::max(clears, ceil_div(rows, kClearRows));
    const bool search = tokens * k <= kClearRows || (D >= 128 && clears <= D / 4);
    if (!tokens || !search) {
      const long blocks = std::min((rows * D + 4095) / 4096, ctx().sm_count * 8l);
      pdl_launch(clear_all_kernel, (unsigned)blocks, 256, 0, data_ptr(gradInput), rows * D);
      check_launch("Combine_backward");
      clears = 0;
    } else each = ceil_div(rows, clears);
  }
  if (tokens == 0 || (!gradInput && !gradWeights)) return 0;
  TensorRef p(tensor_new_contiguous(positions)), w(weights ? tensor_new_contiguous(weights) : nullptr);
  DenseRows g(gradOutput);
  auto run = [&](Rows x) {
    float *gx = gradInput && rows ? data_ptr(gradInput) : nullptr, *gw = gradWeights ? data_ptr(gradWeights) : nullptr;
    const bool vec = pieces_of_four({x, Rows{g.p, g.ld}, Rows{gx, D}}, (int)D);
    with_columns(tokens, (int)D, (int)k, vec, true, [&](auto T, auto U, auto VEC) {
      constexpr int t = decltype(T)::value, u = decltype(U)::value;
      pdl_launch(rows_sum_backward_kernel<t, u, decltype(VEC)::value>, (unsigned)(ceil_div(tokens, 256 / t) + clears), 256, 0, x, weights ? data_ptr(w) : nullptr, data_ptr(p),
                 Rows{g.p, g.ld}, gx, gw, tokens, (int)k, (int)D, rows, clears, each);
    });
    check_launch("Combine_backward");
  };
  if (rows == 0) run(Rows{nullptr, 0});
  else {
    DenseRows x(input);
    run(Rows{x.p, x.ld});
  }
  return 0;
  THC_END(1)
}
