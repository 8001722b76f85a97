// nn.LayerNorm: rows normalised to mean zero and variance one, times a weight plus a bias.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  inv = 1 / sqrt(var + eps),  u = (x - mean) inv,  y = u w + b
//   dx = inv (g w - mean(g w) - u mean(g w u)),  dw += scale sum_rows g u,  db += scale sum_rows g
//
// The least traffic is 8 bytes a value forward and 12 backward: everything here is bound by HBM.  So rows of up to 8192 values are read once and
// stay in registers, those of up to 512 in a warp's, the others in a block's.  Longer ones are cut into pieces: a launch sums over the pieces of all
// rows and a second one, which reads them again (from L2 where they fit), joins a row's sums and finishes it.
// The variance is taken around the mean, not as a difference of two sums: rows whose mean is large against their spread keep their bits.
// With s1 = sum (x - m) left over from the rounding of m, mean = m + s1 / D and var = sum (x - m)^2 / D - (s1 / D)^2.
#include <type_traits>

#include "nn_args.h"
#include "per_device.h"

namespace thc {

// ---- rows in registers ------------------------------------------------------------------------------------------------
// The share of a thread in a row (or a piece of one): 4 V of the T threads' 4 V T values, in 16-byte pieces where lengths and addresses
// allow it (VEC), else T apart.
template <int T, int V, bool VEC> struct Share {
  float v[4 * V];
  static __device__ __forceinline__ int at(int j, int t) { return VEC ? ((j >> 2) * T + t) * 4 + (j & 3) : j * T + t; }
  static __device__ __forceinline__ bool in(int j, int t, int n) { return at(j, t) < n; }
  // what lies past the row's end reads as zero; STREAM: passes by the L1, which the weights are left in
  template <bool STREAM> __device__ __forceinline__ void load(const float *p, int t, int n) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in(4 * i, t, n)) {
          const float *a = p + at(4 * i, t);
          if constexpr (STREAM)
            asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(q.x), "=f"(q.y), "=f"(q.z), "=f"(q.w) : "l"(a));
          else q = __ldg(reinterpret_cast<const float4 *>(a));
        }
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4 * V; j++) {
        v[j] = 0.f;
        if (in(j, t, n)) {
          if constexpr (STREAM) asm volatile("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(v[j]) : "l"(p + at(j, t)));
          else v[j] = __ldg(p + at(j, t));
        }
      }
    }
  }
  __device__ __forceinline__ void store(float *p, int t, int n) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < V; i++)
        if (in(4 * i, t, n)) *reinterpret_cast<float4 *>(p + at(4 * i, t)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4 * V; j++)
        if (in(j, t, n)) p[at(j, t)] = v[j];
    }
  }
};

// Two sums over the T threads of a row.  T == 32: its warp; else the block, through one of two sets of places in shared memory in turn, so that
// one barrier a sum is enough.
template <int T> struct RowSums {
  float2 *sm;
  int turn = 0;
  __device__ __forceinline__ float2 operator()(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (T > 32) {
      float2 *s = sm + turn * (T / 32);
      turn ^= 1;
      if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
      __syncthreads();
      v = s[0];
#pragma unroll
      for (int i = 1; i < T / 32; i++) { v.x += s[i].x; v.y += s[i].y; }
    }
    return v;
  }
};

// The row's sums of the block's (or warp's) values: mean = base + off, and the sum of the squares around it.
struct RowStats { float base, off, square; };
template <int T, int V, bool VEC> __device__ __forceinline__ RowStats row_stats(const Share<T, V, VEC> &a, RowSums<T> &sums, int t, int n) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 4 * V; j++) s += a.v[j];
  const float m0 = sums(make_float2(s, 0.f)).x / (float)n;
  float2 q = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < 4 * V; j++) {
    if (!a.in(j, t, n)) continue;
    const float c = a.v[j] - m0;
    q.x += c;
    q.y = fmaf(c, c, q.y);
  }
  q = sums(q);
  const float off = q.x / (float)n;
  return RowStats{m0, off, fmaf(-off, q.x, q.y)};
}
// y = u w + b over a share, in place of x
template <int T, int V, bool VEC>
__device__ __forceinline__ void apply_norm(Share<T, V, VEC> &a, const RowStats &s, float inv, const float *w, const float *b, int t, int n) {
  if (w) {
    Share<T, V, VEC> p, c;
    p.template load<false>(w, t, n);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) p.v[j] *= inv;      // (u w = (x - mean) (inv w))
    c.template load<false>(b, t, n);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) a.v[j] = fmaf((a.v[j] - s.base) - s.off, p.v[j], c.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4 * V; j++) a.v[j] = ((a.v[j] - s.base) - s.off) * inv;
  }
}

// Forward.  A row by T threads (BLOCK / T rows a block).  One row of 4096: 3.1 us a call, a launch and one round trip to memory; 30011 x 333, in 4-byte
// pieces: 19 us, 4.3 TB/s.
template <int T, int V, bool VEC>
static __global__ void __launch_bounds__(T < 128 ? 256 : T) norm_forward_kernel(const float *__restrict__ x, float *__restrict__ y, const float *__restrict__ w,
                                                                              const float *__restrict__ b, float *mean, float *inv, long rows, int D, float eps) {
  pdl_begin();
  constexpr int BLOCK = T < 128 ? 256 : T;
  __shared__ float2 sm[2 * (BLOCK / 32)];
  const int t = threadIdx.x % T;
  const long row = blockIdx.x * (long)(BLOCK / T) + threadIdx.x / T;
  if (T == 32 && row >= rows) return;
  RowSums<T> sums{sm};
  Share<T, V, VEC> a;
  a.template load<true>(x + row * D, t, D);
  const RowStats s = row_stats(a, sums, t, D);
  const float i = 1.f / sqrtf(s.square / (float)D + eps);
  if (mean && t == 0) { mean[row] = s.base + s.off; inv[row] = i; }
  apply_norm(a, s, i, w, b, t, D);
  a.store(y + row * D, t, D);
}

// Backward.  The blocks stay, each with the rows team, team + teams, ... (a team: T threads), the next row on its way while one is worked on, and
// with the sums of its columns for the weight's and the bias's gradient in registers, which part[block][2][D] gets.  gx or part may be null.
// gx is summed without fused multiply-adds: of a row of two values the formula leaves eps / (var + eps) of its terms, which then is the same
// whatever else evaluates it step by step in FP32.
// 16384 x 4096: 120 us, 6.7 TB/s; 30011 x 333: 22 us, 5.6 TB/s.
template <int T, int V, bool VEC>
static __global__ void __launch_bounds__(T < 128 ? 256 : T, T < 512 ? 2 : 1) norm_backward_kernel(const float *__restrict__ x, const float *__restrict__ g, float *__restrict__ gx,
                                                                               const float *__restrict__ w, const float *__restrict__ mean,
                                                                               const float *__restrict__ inv, long rows, int D, float *part) {
  pdl_begin();
  constexpr int BLOCK = T < 128 ? 256 : T, TEAMS = BLOCK / T;
  __shared__ float2 sm[2 * (BLOCK / 32)];
  const int t = threadIdx.x % T;
  const long team = blockIdx.x * (long)TEAMS + threadIdx.x / T, teams = gridDim.x * (long)TEAMS;
  RowSums<T> sums{sm};
  float gw[4 * V], gb[4 * V];
#pragma unroll
  for (int j = 0; j < 4 * V; j++) gw[j] = gb[j] = 0.f;
  Share<T, V, VEC> xn, gn;
  float mn = 0.f, in = 0.f;
  auto fetch = [&](long r) {
    xn.template load<true>(x + r * D, t, D);
    gn.template load<true>(g + r * D, t, D);
    mn = __ldg(mean + r);
    in = __ldg(inv + r);
  };
  if (team < rows) fetch(team);
  for (long r = team; r < rows; r += teams) {
    Share<T, V, VEC> a = xn, c = gn;
    const float m = mn, i = in;
    if (r + teams < rows) fetch(r + teams);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) {
      a.v[j] = a.in(j, t, D) ? (a.v[j] - m) * i : 0.f;
      gw[j] = fmaf(c.v[j], a.v[j], gw[j]);
      gb[j] += c.v[j];
    }
    if (!gx) continue;
    if (w) {
      Share<T, V, VEC> p;
      p.template load<false>(w, t, D);
#pragma unroll
      for (int j = 0; j < 4 * V; j++) c.v[j] *= p.v[j];
    }
#pragma unroll
    for (int j = 0; j < 4 * V; j++) {
      s.x += c.v[j];
      s.y = __fadd_rn(s.y, __fmul_rn(c.v[j], a.v[j]));
    }
    s = sums(s);
    const float one = s.x / (float)D, two = s.y / (float)D;
#pragma unroll
    for (int j = 0; j < 4 * V; j++) a.v[j] = i * __fsub_rn(c.v[j] - one, __fmul_rn(a.v[j], two));
    a.store(gx + r * D, t, D);
  }
  if (!part) return;
  if constexpr (TEAMS > 1) {   // the block's warps one after the other
    extern __shared__ float columns[];   // [2][T * 4 * V]
    constexpr int N = T * 4 * V;
    for (int k = 0; k < TEAMS; k++) {
      if ((int)(threadIdx.x / T) == k) {
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
          const int at = Share<T, V, VEC>::at(j, t);
          columns[at] = (k ? columns[at] : 0.f) + gw[j];
          columns[N + at] = (k ? columns[N + at] : 0.f) + gb[j];
        }
      }
      __syncthreads();
    }
    for (int d = threadIdx.x; d < D; d += BLOCK) {
      part[(2l * blockIdx.x) * D + d] = columns[d];
      part[(2l * blockIdx.x + 1) * D + d] = columns[N + d];
    }
  } else {
    Share<T, V, VEC> o;
#pragma unroll
    for (int j = 0; j < 4 * V; j++) o.v[j] = gw[j];
    o.store(part + 2 * team * D, t, D);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) o.v[j] = gb[j];
    o.store(part + (2 * team + 1) * D, t, D);
  }
}

// ---- rows cut into pieces ---------------------------------------------------------------------------------------------
// 256 threads, up to 16 values each.  Block (a, b) has piece a of row b, b + gridDim.y, ...  A cluster for each row, its values in its blocks' registers,
// reads them once, but a block waits for the slowest of its cluster at each sum: forward and backward of 200 x 43264 took 109 us that way and 68 this
// way.  Of those the launches take 12 + 17 us forward and 16 + 20 + 7 backward from cold caches, 35 MB of values each (2.2 - 4.5 TB/s): with one to
// two blocks' worth of loads a thread their starts and ends show.
constexpr int kPiece = 4096;
// part[row][piece] = mean and sum of squares around it
template <bool VEC>
static __global__ void __launch_bounds__(256) norm_pieces_kernel(const float *__restrict__ x, long rows, long D, float2 *part) {
  pdl_begin();
  __shared__ float2 sm[2 * 8];
  RowSums<256> sums{sm};
  const long c0 = blockIdx.x * (long)kPiece;
  const int n = (int)min((long)kPiece, D - c0), t = threadIdx.x;
  for (long r = blockIdx.y; r < rows; r += gridDim.y) {
    Share<256, 4, VEC> a;
    a.template load<true>(x + r * D + c0, t, n);
    const RowStats s = row_stats(a, sums, t, n);
    if (t == 0) part[r * gridDim.x + blockIdx.x] = make_float2(s.base + s.off, s.square);
  }
}
// The row's mean and squares from its pieces': mean = m_0 + sum n (m - m_0) / D, squares = sum q + n (m - mean)^2, by the threads of a block.
static __device__ __forceinline__ RowStats join_pieces(const float2 *part, int pieces, long D, RowSums<256> &sums) {
  auto size = [&](int k) { return (float)min((long)kPiece, D - k * (long)kPiece); };
  const float base = part[0].x;
  float2 s = make_float2(0.f, 0.f);
  for (int k = threadIdx.x; k < pieces; k += 256) s.x = fmaf(size(k), part[k].x - base, s.x);
  const float off = sums(s).x / (float)D;
  s = make_float2(0.f, 0.f);
  for (int k = threadIdx.x; k < pieces; k += 256) {
    const float e = (part[k].x - base) - off;
    s.x += fmaf(size(k) * e, e, part[k].y);
  }
  return RowStats{base, off, sums(s).x};
}
template <bool VEC>
static __global__ void __launch_bounds__(256) norm_apply_kernel(const float *__restrict__ x, float *__restrict__ y, const float *__restrict__ w,
                                                                const float *__restrict__ b, float *mean, float *inv, long rows, long D, float eps,
                                                                const float2 *__restrict__ part) {
  pdl_begin();
  __shared__ float2 sm[2 * 8];
  RowSums<256> sums{sm};
  const long c0 = blockIdx.x * (long)kPiece;
  const int n = (int)min((long)kPiece, D - c0), t = threadIdx.x;
  for (long r = blockIdx.y; r < rows; r += gridDim.y) {
    Share<256, 4, VEC> a;
    a.template load<true>(x + r * D + c0, t, n);
    const RowStats s = join_pieces(part + r * gridDim.x, gridDim.x, D, sums);
    const float i = 1.f / sqrtf(s.square / (float)D + eps);
    if (mean && blockIdx.x == 0 && t == 0) { mean[r] = s.base + s.off; inv[r] = i; }
    apply_norm(a, s, i, w ? w + c0 : nullptr, b ? b + c0 : nullptr, t, n);
    a.store(y + r * D + c0, t, n);
  }
}
// part[row][piece] = sums of g w and of g w u
template <bool VEC>
static __global__ void __launch_bounds__(256) norm_piece_sums_kernel(const float *__restrict__ x, const float *__restrict__ g, const float *__restrict__ w,
                                                                     const float *__restrict__ mean, const float *__restrict__ inv, long rows, long D,
                                                                     float2 *part) {
  pdl_begin();
  __shared__ float2 sm[2 * 8];
  RowSums<256> sums{sm};
  const long c0 = blockIdx.x * (long)kPiece;
  const int n = (int)min((long)kPiece, D - c0), t = threadIdx.x;
  for (long r = blockIdx.y; r < rows; r += gridDim.y) {
    Share<256, 4, VEC> a, c;
    a.template load<true>(x + r * D + c0, t, n);
    c.template load<true>(g + r * D + c0, t, n);
    const float m = mean[r], i = inv[r];
    if (w) {
      Share<256, 4, VEC> p;
      p.template load<false>(w + c0, t, n);
#pragma unroll
      for (int j = 0; j < 16; j++) c.v[j] *= p.v[j];
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 16; j++) {
      if (!a.in(j, t, n)) continue;
      s.x += c.v[j];
      s.y = fmaf(c.v[j], (a.v[j] - m) * i, s.y);
    }
    s = sums(s);
    if (t == 0) part[r * gridDim.x + blockIdx.x] = s;
  }
}
// The gradients of 1024 columns (blockIdx.x) over the rows [per * blockIdx.y, + per): gx, and the columns' sums in columns[blockIdx.y][2][D].
// No thread waits for another: four rows are on the way.  The rows' sums over their pieces come first, kRowSums rows at a time.
constexpr int kRowSums = 64;
template <bool VEC>
static __global__ void __launch_bounds__(256) norm_columns_kernel(const float *__restrict__ x, const float *__restrict__ g, float *__restrict__ gx,
                                                                  const float *__restrict__ w, const float *__restrict__ mean, const float *__restrict__ inv,
                                                                  long rows, long D, long per, const float2 *__restrict__ part, int pieces, float *columns) {
  pdl_begin();
  __shared__ float4 row_sums[kRowSums];   // mean, inv, mean of g w, mean of g w u
  const long c0 = blockIdx.x * 1024l, end = min(rows, (blockIdx.y + 1) * per);
  const int n = (int)min(1024l, D - c0), t = threadIdx.x, warp = t >> 5, lane = t & 31;
  float gw[4] = {0.f, 0.f, 0.f, 0.f}, gb[4] = {0.f, 0.f, 0.f, 0.f};
  Share<256, 1, VEC> p;
#pragma unroll
  for (int j = 0; j < 4; j++) p.v[j] = 1.f;
  if (w) p.template load<false>(w + c0, t, n);
  for (long r0 = blockIdx.y * per; r0 < end; r0 += kRowSums) {
    const int some = (int)min((long)kRowSums, end - r0);
    __syncthreads();
    for (int k = warp; k < some; k += 8) {
      float2 s = make_float2(0.f, 0.f);
      if (gx)
        for (int q = lane; q < pieces; q += 32) {
          const float2 v = part[(r0 + k) * pieces + q];
          s.x += v.x; s.y += v.y;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
        s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
      }
      if (lane == 0) row_sums[k] = make_float4(mean[r0 + k], inv[r0 + k], s.x / (float)D, s.y / (float)D);
    }
    __syncthreads();
    constexpr int U = 4;
    for (int k0 = 0; k0 < some; k0 += U) {
      Share<256, 1, VEC> a[U], c[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (k0 + u < some) {
          a[u].template load<true>(x + (r0 + k0 + u) * D + c0, t, n);
          c[u].template load<true>(g + (r0 + k0 + u) * D + c0, t, n);
        }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (k0 + u < some) {
          const float4 q = row_sums[k0 + u];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const float z = (a[u].v[j] - q.x) * q.y;
            gw[j] = fmaf(c[u].v[j], z, gw[j]);
            gb[j] += c[u].v[j];
            a[u].v[j] = q.y * (c[u].v[j] * p.v[j] - q.z - z * q.w);
          }
          if (gx) a[u].store(gx + (r0 + k0 + u) * D + c0, t, n);
        }
    }
  }
  if (!columns) return;
  Share<256, 1, VEC> o;
#pragma unroll
  for (int j = 0; j < 4; j++) o.v[j] = gw[j];
  o.store(columns + 2l * blockIdx.y * D + c0, t, n);
#pragma unroll
  for (int j = 0; j < 4; j++) o.v[j] = gb[j];
  o.store(columns + (2l * blockIdx.y + 1) * D + c0, t, n);
}

// gw += scale * sum of part[.][0], gb += scale * sum of part[.][1]: LANES threads a column, which take every LANES-th part and meet in the order of
// their places.  296 parts of 2 x 4096 sums (10 MB): 8 us.
template <int LANES>
static __global__ void __launch_bounds__(256) norm_fold_kernel(const float *__restrict__ part, int parts, long D, float *gw, float *gb, float scale) {
  pdl_begin();
  constexpr int COLS = 256 / LANES;
  __shared__ float sm[LANES][COLS];
  const int tx = threadIdx.x % COLS, ty = threadIdx.x / COLS;
  const long c = blockIdx.x * (long)COLS + tx;
  float s = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int p = ty; p < parts; p += LANES) s += part[p * 2l * D + c];
  }
  if constexpr (LANES > 1) {
    sm[ty][tx] = s;
    __syncthreads();
    if (ty) return;
#pragma unroll
    for (int i = 1; i < LANES; i++) s += sm[i][tx];
  }
  if (c >= 2 * D) return;
  float *o = c < D ? gw + c : gb + (c - D);
  *o = fmaf(scale, s, *o);
}

template <int T, int V> struct NormConfig { static constexpr int kT = T, kV = V; };
constexpr long kRowMost = 8192;
// f(config) for the narrowest threads' share that holds a row
template <class F> static void with_norm_config(long D, F f) {
  if (D <= 128) f(NormConfig<32, 1>());
  else if (D <= 256) f(NormConfig<32, 2>());
  else if (D <= 384) f(NormConfig<32, 3>());
  else if (D <= 512) f(NormConfig<32, 4>());
  else if (D <= 1024) f(NormConfig<128, 2>());
  else if (D <= 2048) f(NormConfig<256, 2>());
  else if (D <= 4096) f(NormConfig<256, 4>());
  else f(NormConfig<512, 4>());
}
template <class F> static void with_vec(bool vec, F f) {
  if (vec) f(std::true_type()); else f(std::false_type());
}
template <int T, int V, bool VEC> static int resident_blocks() {
  static PerDevice resident;
  constexpr int BLOCK = T < 128 ? 256 : T;
  return resident.get(ctx().device, [] {
    int n = 0;
    THC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_backward_kernel<T, V, VEC>, BLOCK, T < 128 ? 2 * T * 4 * V * 4 : 0));
    return std::max(n, 1);
  });
}
static bool aligned(std::initializer_list<const float *> ps) {
  for (const float *p : ps)
    if ((uintptr_t)p & 15) return false;
  return true;
}

// Rows of `size` values: how many, or a refusal when no trailing dimensions come to `size`.
static long rows_of(const THGPUTensor *t, long size, int argn) {
  long inner = 1;
  int d = t->nDimension;
  while (d > 0 && inner < size) inner *= t->size[--d];
  THC_ARG(inner == size, argn, "the trailing dimensions do not come to the normalised size");
  return nelem(t) / size;
}

static void norm_backward(THGPUTensor *input, THGPUTensor *gradOutput, THGPUTensor *gradInput, THGPUTensor *weight, THGPUTensor *gradWeight,
                          THGPUTensor *gradBias, THGPUTensor *mean, THGPUTensor *invStd, long size, float scale) {
  THC_ARG(input && gradOutput && mean && invStd, 1, "tensors expected");
  THC_ARG(size > 0, 9, "size must be positive");
  THC_ARG(THGPUTensor_isSameSizeAs(input, gradOutput), 2, "gradOutput has the wrong size");
  THC_ARG(!weight || (nelem(weight) == size && is_contiguous(weight)), 4, "contiguous weight of the normalised size expected");
  THC_ARG(!gradWeight == !gradBias, 6, "both or neither of gradWeight and gradBias expected");
  if (gradWeight) {
    THC_ARG(nelem(gradWeight) == size && is_contiguous(gradWeight), 5, "contiguous gradWeight of the normalised size expected");
    THC_ARG(nelem(gradBias) == size && is_contiguous(gradBias), 6, "contiguous gradBias of the normalised size expected");
  }
  check_here({input, gradOutput, gradInput, weight, gradWeight, gradBias, mean, invStd});
  if (nelem(input) == 0) {
    if (gradInput) tensor_resize_as(gradInput, input);
    return;
  }
  const long rows = rows_of(input, size, 1);
  THC_ARG(nelem(mean) == rows && nelem(invStd) == rows && is_contiguous(mean) && is_contiguous(invStd), 7, "the statistics are not this input's");
  if (gradInput) size_result(gradInput, input->nDimension, input->size, {input, gradOutput, weight, mean, invStd, gradWeight, gradBias}, 3);
  check_apart(gradWeight, {input, gradOutput, weight, mean, invStd, gradBias}, 5);
  check_apart(gradBias, {input, gradOutput, weight, mean, invStd}, 6);
  if (!gradInput && !gradWeight) return;
  WsScope scope;
  TensorRef x(tensor_new_contiguous(input)), g(tensor_new_contiguous(gradOutput));
  const float *w = weight ? data_ptr(weight) : nullptr, *xp = data_ptr(x), *gp = data_ptr(g), *mp = data_ptr(mean), *ip = data_ptr(invStd);
  float *gx = gradInput ? data_ptr(gradInput) : nullptr, *part = nullptr;
  long parts = 0;
  const bool vec = size % 4 == 0 && aligned({xp, gp, gx, w});
  if (size <= kRowMost) {
    with_norm_config(size, [&](auto c) {
      with_vec(vec, [&](auto v) {
        constexpr bool VEC = decltype(v)::value;
        constexpr int T = decltype(c)::kT, V = decltype(c)::kV, BLOCK = T < 128 ? 256 : T, TEAMS = BLOCK / T;
        parts = std::min((rows + TEAMS - 1) / TEAMS, ctx().sm_count * (long)resident_blocks<T, V, VEC>());   // as many as are resident at once
        if (gradWeight) part = (float *)ws_alloc(sizeof(float) * 2 * size * parts);
        pdl_launch(norm_backward_kernel<T, V, VEC>, (unsigned)parts, BLOCK, TEAMS > 1 ? sizeof(float) * 2 * T * 4 * V : 0, xp, gp, gx, w, mp, ip, rows, (int)size,
                   part);
      });
    });
    check_launch("LayerNorm_backward");
  } else {
    const long pieces = (size + kPiece - 1) / kPiece, columns = (size + 1023) / 1024;
    // rows enough in each of the column sums' blocks, and eight blocks an SM
    parts = std::max(1l, std::min(std::min((rows + 3) / 4, (ctx().sm_count * 8l + columns - 1) / columns), 65535l));
    const long per = (rows + parts - 1) / parts;
    parts = (rows + per - 1) / per;
    float2 *sums = nullptr;
    if (gradWeight) part = (float *)ws_alloc(sizeof(float) * 2 * size * parts);
    with_vec(vec, [&](auto v) {
      constexpr bool VEC = decltype(v)::value;
      if (gx) {
        sums = (float2 *)ws_alloc(sizeof(float2) * rows * pieces);
        pdl_launch(norm_piece_sums_kernel<VEC>, dim3((unsigned)pieces, (unsigned)std::min(rows, 65535l)), 256, 0, xp, gp, w, mp, ip, rows, size, sums);
        check_launch("LayerNorm_backward");
      }
      pdl_launch(norm_columns_kernel<VEC>, dim3((unsigned)columns, (unsigned)parts), 256, 0, xp, gp, gx, w, mp, ip, rows, size, per, sums, (int)pieces, part);
    });
    check_launch("LayerNorm_backward");
  }
  if (gradWeight) {
    // a thread a column where that fills the device or there is little to add up
    if (parts <= 8 || size >= 32768)
      pdl_launch(norm_fold_kernel<1>, ceil_div(2 * size, 256), 256, 0, part, (int)parts, size, data_ptr(gradWeight), data_ptr(gradBias), scale);
    else
      pdl_launch(norm_fold_kernel<16>, ceil_div(2 * size, 16), 256, 0, part, (int)parts, size, data_ptr(gradWeight), data_ptr(gradBias), scale);
    check_launch("LayerNorm_backward");
  }
}

}  // namespace thc

using namespace thc;

THC_API int THGPUNN_LayerNorm_updateOutput(THGPUTensor *input, THGPUTensor *output, THGPUTensor *weight, THGPUTensor *bias, THGPUTensor *mean,
                                           THGPUTensor *invStd, long size, double eps) {
  THC_BEGIN
  THC_ARG(input && output, 1, "tensors expected");
  THC_ARG(size > 0, 7, "size must be positive");
  THC_ARG(eps >= 0, 8, "eps must not be negative");
  THC_ARG(!weight == !bias, 4, "both or neither of weight and bias expected");
  THC_ARG(!mean == !invStd, 6, "both or neither of mean and invStd expected");
  if (weight) {
    THC_ARG(nelem(weight) == size && is_contiguous(weight), 3, "contiguous weight of the normalised size expected");
    THC_ARG(nelem(bias) == size && is_contiguous(bias), 4, "contiguous bias of the normalised size expected");
  }
  check_here({input, output, weight, bias, mean, invStd});
  if (nelem(input) == 0) {
    tensor_resize_as(output, input);
    return 0;
  }
  const long rows = rows_of(input, size, 1);
  size_result(output, input->nDimension, input->size, {input, weight, bias, mean, invStd}, 2);
  if (mean) {
    size_result(mean, 1, &rows, {input, weight, bias, output, invStd}, 5);
    size_result(invStd, 1, &rows, {input, weight, bias, output, mean}, 6);
  }
  TensorRef x(tensor_new_contiguous(input));
  const float *xp = data_ptr(x), *w = weight ? data_ptr(weight) : nullptr, *bp = bias ? data_ptr(bias) : nullptr;
  float *y = data_ptr(output), *mp = mean ? data_ptr(mean) : nullptr, *ip = mean ? data_ptr(invStd) : nullptr;
  const bool vec = size % 4 == 0 && aligned({xp, y, w, bp});
  WsScope scope;
  with_vec(vec, [&](auto v) {
    constexpr bool VEC = decltype(v)::value;
    if (size <= kRowMost) {
      with_norm_config(size, [&](auto c) {
        constexpr int T = decltype(c)::kT, BLOCK = T < 128 ? 256 : T, TEAMS = BLOCK / T;
        // (a launch has less than 2^31 blocks)
        for (long r = 0; r < rows; r += 1l << 30) {
          const long n = std::min(rows - r, 1l << 30);
          pdl_launch(norm_forward_kernel<T, decltype(c)::kV, VEC>, (unsigned)((n + TEAMS - 1) / TEAMS), BLOCK, 0, xp + r * size, y + r * size, w, bp, mp ? mp + r : nullptr,
                     ip ? ip + r : nullptr, n, (int)size, (float)eps);
        }
      });
      return;
    }
    const long pieces = (size + kPiece - 1) / kPiece;
    const dim3 grid((unsigned)pieces, (unsigned)std::min(rows, 65535l));
    float2 *part = (float2 *)ws_alloc(sizeof(float2) * rows * pieces);
    pdl_launch(norm_pieces_kernel<VEC>, grid, 256, 0, xp, rows, size, part);
    check_launch("LayerNorm_updateOutput");
    pdl_launch(norm_apply_kernel<VEC>, grid, 256, 0, xp, y, w, bp, mp, ip, rows, size, (float)eps, part);
  });
  check_launch("LayerNorm_updateOutput");
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_LayerNorm_backward(THGPUTensor *input, THGPUTensor *gradOutput, THGPUTensor *gradInput, THGPUTensor *weight, THGPUTensor *gradWeight,
                                       THGPUTensor *gradBias, THGPUTensor *mean, THGPUTensor *invStd, long size, float scale) {
  THC_BEGIN
  norm_backward(input, gradOutput, gradInput, weight, gradWeight, gradBias, mean, invStd, size, scale);
  return 0;
  THC_END(1)
}
