// nn.LayerNorm: rows normalised to mean zero and variance one, times a weight plus a bias.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  inv = 1 / sqrt(var + eps),  u = (x - mean) inv,  y = u w + b
//   dx = inv (g w - mean(g w) - u mean(g w u)),  dw += scale sum_rows g u,  db += scale sum_rows g
//
// The least traffic is 8 bytes a value forward and 12 backward: everything here is bound by HBM.  So a row is read once and stays in
// registers, whatever its length up to 65536 values: a warp has the rows of up to 512, a block those of up to 8192, and a cluster of two,
// four or eight blocks the longer ones, each block a slice, whose sums meet through distributed shared memory.
// The variance is taken around the mean, not as a difference of two sums: rows whose mean is large against their spread keep their bits.
// With s1 = sum (x - m) left over from the rounding of m, mean = m + s1 / D and var = sum (x - m)^2 / D - (s1 / D)^2.
#include <type_traits>

#include "nn_args.h"
#include "per_device.h"

namespace thc {

// ---- rows in registers ------------------------------------------------------------------------------------------------
// The share of a thread in a row (or a block's slice of one): 4 V of the T threads' 4 V T values, in 16-byte pieces where lengths and addresses
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

constexpr int kMostBlocks = 8;   // of a cluster
__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned cluster_blocks() { unsigned n; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n)); return n; }
// Every block of the cluster gets every block's two values, in the order of their ranks.  Two sets of places in turn: a block writes into one only
// after the barrier of the other, which all have come to with the first one read.
struct ClusterValues {
  float2 (*sm)[kMostBlocks];
  int turn = 0;
  // Before the first exchange: a block may write into another's shared memory once that has started.
  static __device__ __forceinline__ void begin() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  }
  __device__ __forceinline__ const float2 *exchange(float2 mine, unsigned rank, unsigned blocks) {
    float2 *s = sm[turn];
    turn ^= 1;
    if (threadIdx.x < blocks) {
      unsigned there;
      const unsigned here = (unsigned)__cvta_generic_to_shared(s + rank);
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(threadIdx.x));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(mine.x), "f"(mine.y) : "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    return s;
  }
};
// Forward.  A row by T threads of this block (BLOCK / T rows a block), or by all threads of a cluster's blocks.
template <int T, int V, bool VEC, bool CLUSTER>
static __global__ void __launch_bounds__(T < 128 ? 256 : T) norm_forward_kernel(const float *__restrict__ x, float *__restrict__ y, const float *__restrict__ w,
                                                                              const float *__restrict__ b, float *mean, float *inv, long rows, int D, int slice,
                                                                              float eps) {
  pdl_begin();
  constexpr int BLOCK = T < 128 ? 256 : T;
  __shared__ float2 sm[2 * (BLOCK / 32)];
  __shared__ float2 shared_values[2][kMostBlocks];
  const int t = threadIdx.x % T;
  const unsigned rank = CLUSTER ? cluster_rank() : 0, blocks = CLUSTER ? cluster_blocks() : 1;
  const int first = (int)rank * slice, n = min(slice, D - first);
  const long row = CLUSTER ? blockIdx.x / blocks : blockIdx.x * (long)(BLOCK / T) + threadIdx.x / T;
  if (T == 32 && row >= rows) return;
  RowSums<T> sums{sm};
  Share<T, V, VEC> a;
  a.template load<true>(x + row * D + first, t, n);
  if constexpr (CLUSTER) ClusterValues::begin();
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
  float base = m0, off = q.x / (float)n, square = fmaf(-off, q.x, q.y);   // mean = base + off; square: sum (x - mean)^2
  if constexpr (CLUSTER) {
    // of the slices' means m and squares q: mean = m_0 + sum n (m - m_0) / D, square = sum q + n (m - mean)^2
    ClusterValues values{shared_values};
    const float2 *all = values.exchange(make_float2(m0 + off, square), rank, blocks);
    base = all[0].x;
    float d = 0.f;
    for (unsigned k = 1; k < blocks; k++) d = fmaf((float)min(slice, D - (int)k * slice), all[k].x - base, d);
    off = d / (float)D;
    square = 0.f;
    for (unsigned k = 0; k < blocks; k++) {
      const float e = (all[k].x - base) - off;
      square += fmaf((float)min(slice, D - (int)k * slice) * e, e, all[k].y);
    }
  }
  const float i = 1.f / sqrtf(square / (float)D + eps);
  if (mean && rank == 0 && t == 0) { mean[row] = base + off; inv[row] = i; }
  if (w) {
    Share<T, V, VEC> p;
    p.template load<false>(w + first, t, n);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) p.v[j] *= i;      // (u w = (x - mean) (inv w))
    Share<T, V, VEC> c;
    c.template load<false>(b + first, t, n);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) a.v[j] = fmaf((a.v[j] - base) - off, p.v[j], c.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4 * V; j++) a.v[j] = ((a.v[j] - base) - off) * i;
  }
  a.store(y + row * D + first, t, n);
}

// Backward.  The blocks stay, each with the rows team, team + teams, ... (a team: T threads, or a cluster), the next row on its way while one is
// worked on, and with the sums of its columns for the weight's and the bias's gradient in registers, which part[block or cluster][2][D] gets.
// gx or part may be null.
template <int T, int V, bool VEC, bool CLUSTER>
static __global__ void __launch_bounds__(T < 128 ? 256 : T, T < 512 ? 2 : 1) norm_backward_kernel(const float *__restrict__ x, const float *__restrict__ g, float *__restrict__ gx,
                                                                               const float *__restrict__ w, const float *__restrict__ mean,
                                                                               const float *__restrict__ inv, long rows, int D, int slice, float *part) {
  pdl_begin();
  constexpr int BLOCK = T < 128 ? 256 : T, TEAMS = BLOCK / T;
  __shared__ float2 sm[2 * (BLOCK / 32)];
  __shared__ float2 shared_values[2][kMostBlocks];
  const int t = threadIdx.x % T;
  const unsigned rank = CLUSTER ? cluster_rank() : 0, blocks = CLUSTER ? cluster_blocks() : 1;
  const int first = (int)rank * slice, n = min(slice, D - first);
  const long team = CLUSTER ? blockIdx.x / blocks : blockIdx.x * (long)TEAMS + threadIdx.x / T, teams = CLUSTER ? gridDim.x / blocks : gridDim.x * (long)TEAMS;
  RowSums<T> sums{sm};
  ClusterValues values{shared_values};
  float gw[4 * V], gb[4 * V];
#pragma unroll
  for (int j = 0; j < 4 * V; j++) gw[j] = gb[j] = 0.f;
  Share<T, V, VEC> xn, gn;
  float mn = 0.f, in = 0.f;
  auto fetch = [&](long r) {
    xn.template load<true>(x + r * D + first, t, n);
    gn.template load<true>(g + r * D + first, t, n);
    mn = __ldg(mean + r);
    in = __ldg(inv + r);
  };
  if (team < rows) fetch(team);
  if constexpr (CLUSTER) ClusterValues::begin();
  for (long r = team; r < rows; r += teams) {
    Share<T, V, VEC> a = xn, c = gn;
    const float m = mn, i = in;
    if (r + teams < rows) fetch(r + teams);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) {
      a.v[j] = a.in(j, t, n) ? (a.v[j] - m) * i : 0.f;
      gw[j] = fmaf(c.v[j], a.v[j], gw[j]);
      gb[j] += c.v[j];
    }
    if (!gx) continue;
    if (w) {
      Share<T, V, VEC> p;
      p.template load<false>(w + first, t, n);
#pragma unroll
      for (int j = 0; j < 4 * V; j++) c.v[j] *= p.v[j];
    }
#pragma unroll
    for (int j = 0; j < 4 * V; j++) {
      s.x += c.v[j];
      s.y = fmaf(c.v[j], a.v[j], s.y);
    }
    s = sums(s);
    if constexpr (CLUSTER) {
      const float2 *all = values.exchange(s, rank, blocks);
      s = all[0];
      for (unsigned k = 1; k < blocks; k++) { s.x += all[k].x; s.y += all[k].y; }
    }
    const float one = s.x / (float)D, two = s.y / (float)D;
#pragma unroll
    for (int j = 0; j < 4 * V; j++) a.v[j] = i * (c.v[j] - one - a.v[j] * two);
    a.store(gx + r * D + first, t, n);
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
    o.store(part + 2 * team * D + first, t, n);
#pragma unroll
    for (int j = 0; j < 4 * V; j++) o.v[j] = gb[j];
    o.store(part + (2 * team + 1) * D + first, t, n);
  }
}

// ---- rows of more than 65536 values -----------------------------------------------------------------------------------
// Two sums over a block; every thread gets both.
static __device__ __forceinline__ float2 block_sum2(float2 v, float2 *sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); i++) { v.x += sm[i].x; v.y += sm[i].y; }
  __syncthreads();
  return v;
}

// Rows of any length, a block each, from memory three times.
static __global__ void __launch_bounds__(256) norm_rows_kernel(const float *__restrict__ x, float *y, const float *__restrict__ w, const float *__restrict__ b,
                                                               float *mean, float *inv, long rows, long D, float eps) {
  pdl_begin();
  __shared__ float2 sm[8];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float *xr = x + r * D;
    float2 s = make_float2(0.f, 0.f);
    for (long d = threadIdx.x; d < D; d += 256) s.x += xr[d];
    const float m0 = block_sum2(s, sm).x / (float)D;
    s = make_float2(0.f, 0.f);
    for (long d = threadIdx.x; d < D; d += 256) {
      const float c = xr[d] - m0;
      s.x += c;
      s.y = fmaf(c, c, s.y);
    }
    s = block_sum2(s, sm);
    const float off = s.x / (float)D, m = m0 + off, i = 1.f / sqrtf(fmaf(-off, off, s.y / (float)D) + eps);
    if (threadIdx.x == 0 && mean) { mean[r] = m; inv[r] = i; }
    for (long d = threadIdx.x; d < D; d += 256) {
      const float u = (xr[d] - m) * i;
      y[r * D + d] = w ? fmaf(u, w[d], b[d]) : u;
    }
  }
}
static __global__ void __launch_bounds__(256) norm_rows_grad_kernel(const float *__restrict__ x, const float *__restrict__ g, float *gx, const float *__restrict__ w,
                                                                    const float *__restrict__ mean, const float *__restrict__ inv, long rows, long D) {
  pdl_begin();
  __shared__ float2 sm[8];
  for (long r = blockIdx.x; r < rows; r += gridDim.x) {
    const float *xr = x + r * D, *gr = g + r * D;
    const float m = mean[r], i = inv[r];
    float2 s = make_float2(0.f, 0.f);
    for (long d = threadIdx.x; d < D; d += 256) {
      const float gw = w ? gr[d] * w[d] : gr[d];
      s.x += gw;
      s.y = fmaf(gw, (xr[d] - m) * i, s.y);
    }
    s = block_sum2(s, sm);
    const float a = s.x / (float)D, c = s.y / (float)D;
    for (long d = threadIdx.x; d < D; d += 256) {
      const float gw = w ? gr[d] * w[d] : gr[d], u = (xr[d] - m) * i;
      gx[r * D + d] = i * (gw - a - u * c);
    }
  }
}
// Sums over a part of the rows (blockIdx.y) of 32 columns: part[blockIdx.y][2][D].
static __global__ void __launch_bounds__(256) norm_columns_kernel(const float *__restrict__ x, const float *__restrict__ g, const float *__restrict__ mean,
                                                                  const float *__restrict__ inv, long rows, long D, long per, float *part) {
  pdl_begin();
  __shared__ float2 sm[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long end = min(rows, (blockIdx.y + 1) * per);
  for (long d0 = blockIdx.x * 32l; d0 < D; d0 += gridDim.x * 32l) {
    const long d = d0 + tx;
    float2 s = make_float2(0.f, 0.f);
    if (d < D)
      for (long r = blockIdx.y * per + ty; r < end; r += 8) {
        const float gv = g[r * D + d];
        s.x = fmaf(gv, (x[r * D + d] - mean[r]) * inv[r], s.x);
        s.y += gv;
      }
    sm[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && d < D) {
      for (int i = 1; i < 8; i++) { s.x += sm[i][tx].x; s.y += sm[i][tx].y; }
      part[(2l * blockIdx.y) * D + d] = s.x;
      part[(2l * blockIdx.y + 1) * D + d] = s.y;
    }
    __syncthreads();
  }
}
// gw += scale * sum of part[.][0], gb += scale * sum of part[.][1]: LANES threads a column, which take every LANES-th part and meet in the order of
// their places.
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

// How rows of D values are shared out.
struct NormShape {
  int blocks = 1, slice = 0;   // blocks of a cluster, values of a block's slice
};
constexpr long kRowMost = 65536;
static NormShape norm_shape(long D) {
  NormShape s;
  while (s.blocks < kMostBlocks && (D + s.blocks - 1) / s.blocks > 8192) s.blocks *= 2;
  s.slice = (int)((D + 4l * s.blocks - 1) / (4l * s.blocks) * 4);
  return s;
}
template <int T, int V, bool CLUSTER> struct NormConfig {
  static constexpr int kT = T, kV = V;
  static constexpr bool kCluster = CLUSTER;
};
// f(config) for the narrowest threads' share that holds a row, or a slice of one
template <class F> static void with_norm_config(long D, const NormShape &s, F f) {
  if (s.blocks > 1) f(NormConfig<512, 4, true>());
  else if (D <= 128) f(NormConfig<32, 1, false>());
  else if (D <= 256) f(NormConfig<32, 2, false>());
  else if (D <= 384) f(NormConfig<32, 3, false>());
  else if (D <= 512) f(NormConfig<32, 4, false>());
  else if (D <= 1024) f(NormConfig<128, 2, false>());
  else if (D <= 2048) f(NormConfig<256, 2, false>());
  else if (D <= 4096) f(NormConfig<256, 4, false>());
  else f(NormConfig<512, 4, false>());
}
template <class... P, class... A>
static void launch_rows(void (*kernel)(P...), long grid, int block, size_t smem, int cluster, A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(block); cfg.dynamicSmemBytes = smem; cfg.stream = stream();
  cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);   // check_launch() picks an error up
}
template <int T, int V, bool VEC, bool CLUSTER> static int resident_blocks() {
  static PerDevice resident;
  constexpr int BLOCK = T < 128 ? 256 : T;
  return resident.get(ctx().device, [] {
    int n = 0;
    THC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_backward_kernel<T, V, VEC, CLUSTER>, BLOCK, T < 128 ? 2 * T * 4 * V * 4 : 0));
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
  WsScope scope;
  TensorRef x(tensor_new_contiguous(input)), g(tensor_new_contiguous(gradOutput));
  const float *w = weight ? data_ptr(weight) : nullptr, *xp = data_ptr(x), *gp = data_ptr(g), *mp = data_ptr(mean), *ip = data_ptr(invStd);
  float *gx = gradInput ? data_ptr(gradInput) : nullptr, *part = nullptr;
  long parts = 0;
  if (size <= kRowMost) {
    const NormShape s = norm_shape(size);
    const bool vec = size % 4 == 0 && aligned({xp, gp, gx, w});
    with_norm_config(size, s, [&](auto c) {
      typedef decltype(c) Cfg;
      auto go = [&](auto v) {
        constexpr bool VEC = decltype(v)::value;
        constexpr int T = Cfg::kT, V = Cfg::kV, BLOCK = T < 128 ? 256 : T, TEAMS = BLOCK / T;
        // as many teams as are resident at once
        const long blocks = std::min((rows + TEAMS - 1) / TEAMS * s.blocks, ctx().sm_count * (long)resident_blocks<T, V, VEC, Cfg::kCluster>() / s.blocks * s.blocks);
        if (gradWeight) {
          parts = blocks / s.blocks;
          part = (float *)ws_alloc(sizeof(float) * 2 * size * parts);
        }
        launch_rows(norm_backward_kernel<T, V, VEC, Cfg::kCluster>, blocks, BLOCK, TEAMS > 1 ? sizeof(float) * 2 * T * 4 * V : 0, s.blocks, xp, gp, gx, w, mp, ip, rows,
                    size, s.slice, part);
      };
      if (vec) go(std::true_type()); else go(std::false_type());
    });
    check_launch("LayerNorm_backward");
  } else {
    if (gx) {
      pdl_launch(norm_rows_grad_kernel, (unsigned)std::min(rows, ctx().sm_count * 64l), 256, 0, xp, gp, gx, w, mp, ip, rows, size);
      check_launch("LayerNorm_backward");
    }
    if (gradWeight) {
      const long columns = std::min<long>((size + 31) / 32, 1l << 20);
      parts = std::max(1l, std::min(std::min((rows + 31) / 32, (ctx().sm_count * 8l + columns - 1) / columns), 65535l));
      const long per = (rows + parts - 1) / parts;
      part = (float *)ws_alloc(sizeof(float) * 2 * size * parts);
      pdl_launch(norm_columns_kernel, dim3((unsigned)columns, (unsigned)parts), 256, 0, xp, gp, mp, ip, rows, size, per, part);
      check_launch("LayerNorm_backward");
    }
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
  if (size <= kRowMost && rows <= 1l << 27) {
    const NormShape s = norm_shape(size);
    const bool vec = size % 4 == 0 && aligned({xp, y, w, bp});
    with_norm_config(size, s, [&](auto c) {
      typedef decltype(c) Cfg;
      auto go = [&](auto v) {
        constexpr int T = Cfg::kT, BLOCK = T < 128 ? 256 : T, TEAMS = BLOCK / T;
        launch_rows(norm_forward_kernel<T, Cfg::kV, decltype(v)::value, Cfg::kCluster>, (rows + TEAMS - 1) / TEAMS * s.blocks, BLOCK, 0, s.blocks, xp, y, w, bp, mp, ip,
                    rows, size, s.slice, (float)eps);
      };
      if (vec) go(std::true_type()); else go(std::false_type());
    });
  } else {
    pdl_launch(norm_rows_kernel, (unsigned)std::min(rows, ctx().sm_count * 64l), 256, 0, xp, y, w, bp, mp, ip, rows, size, (float)eps);
  }
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
