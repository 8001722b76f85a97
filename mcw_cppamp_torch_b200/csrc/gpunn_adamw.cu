// optim.AdamW: a step of Adam with decoupled weight decay over many tensors in one launch.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// 28 bytes a value with m and v in 32 bits, 16.06 with both in 8: bound by HBM.  The number t of the step lies in device memory, so that a recorded step counts on
// when it is replayed.
//
// In 8 bits m and r = sqrt v are kept as codes, each with a scale for 256 values.  A code c stands for (f(B + c 2^s) - f(B)) scale, f(i) the float of the bits i
// and f(B) = 2^-16: even steps from zero to 2^-16 and steps that double with the value beyond, over 16 powers of two.  m: a sign and 7 bits, s = 20, eight steps a
// power; r: 8 bits, s = 19, sixteen.  The root is kept because its span is half of v's.  A value is rounded up or down at random, by the distance: v moves by
// 1 - b2, a thousandth of itself or less, where codes are 6 to 13 % apart, and rounded to the nearest it would stay where it is for good.  Random bits are a
// hash of the value's place, the tensor's number, the step's and a seed, and every operation on the way to a code is a rounded one of its own, in the order
// written here: the same state, gradients and seed give the same codes.
//
// A value below the least codes, 2^-19 of its block's largest m and 2^-20 of the largest r, is mostly rounded to zero and now and then up, and an m that was rounded up
// over an r that was rounded down would move its weight by hundreds of learning rates.  So what the step divides by has two bounds.  It is no less than 2^-19 of the
// scale that r was decoded with, from where a gradient's share of v, (1 - b2) / (1 - b2^t), is a sixteenth at most; before that one gradient over its own root moves a
// weight by less than half a rate.  And it is no less than |m| over the most that any gradients could make it: by Cauchy's inequality |m| <= C sqrt(v) with
// C = (1 - b1) / sqrt((1 - b2) (1 - b1^2 / b2)), 7.3 at 0.9 and 0.999, which the bias corrections make less; C at least 2, for the codes' noise about a steady
// gradient's 1.  Of a block with one value whose gradients are of size 1 the others, with 1e-6 (1e-7): steps of up to 183 (213) rates, 1.8 (7.4) in the mean, without
// bounds, and with them 7.3 in the first sixteen steps, 1.8 behind them, 0.22 (0.09) in the mean.  Exact moments give 1.1 and 0.23.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "nn_args.h"

namespace thc {

constexpr int kAdamBlock = 256;                                // values under one scale
constexpr int kAdamTurn = 2048;                                // values of a block's turn: a warp has 256
constexpr unsigned kCodeBits = 0x37800000u;                    // of 2^-16
constexpr int kMeanShift = 20, kRootShift = 19;
constexpr float kCodeFloor = 0x1p-16f, kMeanTop = 0.9375f - 0x1p-16f, kRootTop = 0.96875f - 0x1p-16f;   // f(B), and what the largest codes stand for

// A tensor: weights, gradients, and m and v, or the codes of m and r and their scales in turn.
struct AdamTensor {
  float *w;
  const float *g;
  void *m, *v;
  float *scales;
  long n;
};
// As many as fit a launch's parameters; first[i]: the number of tensor i's first chunk.  The smaller table is for the usual few tensors: parameters are copied with
// every launch.
template <int N> struct AdamTable {
  int count;
  unsigned first[N + 1];
  AdamTensor t[N];
};
constexpr int kFewTensors = 24, kSomeTensors = 64, kMoreTensors = 160, kManyTensors = 512;
struct AdamStep {
  float *step;               // steps taken, and the count of blocks that are done (zero between launches)
  bool last;                 // the launch that counts the step
  float lr, beta1, beta2, rest1, rest2, eps, keep;    // rest: 1 - beta, keep: 1 - lr decay
  float log1, log2;          // of the betas
  float most;                // learning rates a step in 8 bits is at most
  unsigned seed;
  int number;                // of the table's first tensor
};
// What a step's number t decides: lr / (1 - b1^t) and 1 / sqrt(1 - b2^t).  1 - b^t = -expm1(t log b): t log b carries its rounding to the result at most as it is,
// where a power of b near one would lose it.
// In 8 bits also what of m, and of a scale, the step's divisor is at least.
struct AdamFactors {
  float rate, root, share, least;
  unsigned step;
};
// By threads 0 and 1 into shared memory; a barrier has to follow.
static __device__ __forceinline__ void adam_factors(const AdamStep &s, AdamFactors &f) {
  if (threadIdx.x > 1) return;
  const float step = truncf(s.step[0]) + 1.f, rest = -expm1f(step * (threadIdx.x ? s.log2 : s.log1));
  if (threadIdx.x == 0) {
    f.rate = s.lr / rest;
    f.share = 1.f / (s.most * rest);
    f.step = (unsigned)step;
  } else {
    f.root = 1.f / sqrtf(rest);
    f.least = rest >= 16.f * s.rest2 ? 0x1p-19f : 0.f;
  }
}
// The last block of the last launch counts the step: by then every block has read, and used, its number.  Nothing else passes between blocks here, so that there is
// no fence to wait for.
static __device__ __forceinline__ void adam_count(const AdamStep &s, unsigned step) {
  if (!s.last) return;
  __syncthreads();
  if (threadIdx.x != 0) return;
  unsigned *done = reinterpret_cast<unsigned *>(s.step + 1);
  if (atomicAdd(done, 1u) == gridDim.x - 1) {
    s.step[0] = (float)step;
    *done = 0;
  }
}
// The tensor of a chunk.
template <int N> static __device__ __forceinline__ int tensor_of(const AdamTable<N> &table, unsigned chunk) {
  int lo = 0, hi = table.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

static __device__ __forceinline__ void load_four(float *v, const float *p) {
  const float4 q = *reinterpret_cast<const float4 *>(p);
  v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
static __device__ __forceinline__ void store_four(float *p, const float *v) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }

// ---- moments in 32 bits
static __device__ __forceinline__ float reciprocal(float v) {     // within a step
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
static __device__ __forceinline__ float square_root(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
static __device__ __forceinline__ float adam_weight(float w, float m, float root, const AdamStep &s, const AdamFactors &f) {
  return fmaf(-f.rate, m * reciprocal(fmaf(root, f.root, s.eps)), w * s.keep);      // (epsilon is no subnormal)
}
static __device__ __forceinline__ void adam_value(float &w, float g, float &m, float &v, const AdamStep &s, const AdamFactors &f) {
  m = fmaf(s.beta1, m, s.rest1 * g);
  v = fmaf(s.beta2, v, s.rest2 * (g * g));
  w = adam_weight(w, m, square_root(v), s, f);
}
// Eight values a thread, in pieces of four where addresses allow it.  The step's factors are made while the loads are on their way.  A block for each 2048 values: the
// scheduler's blocks come and go at different times, so that loads and stores mix; blocks that stay and take turns took 282 us for 61 M values, these 248, 6.9 TB/s.
template <int N>
static __global__ void __launch_bounds__(256) adam_kernel(const __grid_constant__ AdamTable<N> table, const AdamStep s) {
  pdl_begin();
  __shared__ AdamFactors f;
  const int i = tensor_of(table, blockIdx.x), t = threadIdx.x;
  const AdamTensor &a = table.t[i];
  const long from = (blockIdx.x - table.first[i]) * (long)kAdamTurn;      // (t[0] of an empty table is not set, and then not used)
  const int n = blockIdx.x < table.first[table.count] ? (int)min((long)kAdamTurn, a.n - from) : 0;      // none: a step of no values counts all the same
  float *w = a.w + from, *m = (float *)a.m + from, *v = (float *)a.v + from;
  const float *g = a.g + from;
  const bool vec = n == kAdamTurn && (((uintptr_t)w | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15) == 0;
  float ww[8], gg[8], mm[8], vv[8];
  if (vec) {
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const int at = j * 256 + t * 4;
      load_four(gg + j, g + at); load_four(ww + j, w + at); load_four(mm + j, m + at); load_four(vv + j, v + at);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int at = j * 256 + t;
      ww[j] = gg[j] = mm[j] = vv[j] = 0.f;
      if (at < n) { gg[j] = g[at]; ww[j] = w[at]; mm[j] = m[at]; vv[j] = v[at]; }
    }
  }
  adam_factors(s, f);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; j++) adam_value(ww[j], gg[j], mm[j], vv[j], s, f);
  if (vec) {
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      const int at = j * 256 + t * 4;
      store_four(w + at, ww + j); store_four(m + at, mm + j); store_four(v + at, vv + j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const int at = j * 256 + t;
      if (at < n) { w[at] = ww[j]; m[at] = mm[j]; v[at] = vv[j]; }
    }
  }
  adam_count(s, f.step);
}

// ---- moments in 8 bits
// Two values side by side: sm_100a multiplies, or adds, both in one instruction, which this kernel is short of.  A sum of two products of pairs is made a fused one
// by the assembler, whatever its rounding says (12.9), and so would not be the sum that codes are defined by: those are added one by one.
struct Pair {
  unsigned long long v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ Pair(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
  __device__ __forceinline__ void get(float &x, float &y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
};
static __device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
static __device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
static __device__ __forceinline__ Pair fused(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
static __device__ __forceinline__ void add_singly(Pair a, Pair b, float &x, float &y) {
  float ax, ay, bx, by;
  a.get(ax, ay);
  b.get(bx, by);
  x = __fadd_rn(ax, bx);
  y = __fadd_rn(ay, by);
}
static __device__ __forceinline__ float code_float(unsigned code, int shift) { return __uint_as_float(kCodeBits + (code << shift)); }      // f(B) more than it stands for
static __device__ __forceinline__ Pair code_pair(unsigned codes, int j, int shift, Pair scale) {      // of bytes j and j + 1
  return (Pair(code_float(__byte_perm(codes, 0, 0x4440 + j), shift), code_float(__byte_perm(codes, 0, 0x4441 + j), shift)) + Pair(-kCodeFloor, -kCodeFloor)) * scale;
}
// The code of x >= 0, times 1 / scale, with `noise` below 2^shift on its bits.  The largest value of a block needs no bound: on the way to its code, whose fraction
// is zero, are at most three roundings of 2^-24 after that of the constant 1 / top, which is -0.32 of that for m and 0.68 for r, and the sum's half: 3.6 and 2.8 of the last bit
// in all, where the noise leaves 8 (m) and 4 (r) to the next code.  In a block that is not finite codes do not matter.
static __device__ __forceinline__ unsigned value_code(float x, int shift, unsigned noise) {
  return (__float_as_uint(__fadd_rn(x, kCodeFloor)) + noise - (kCodeBits - (1u << (shift - 17)))) >> shift;
}
// 32 random bits of a place, but for the last step of the hash, h ^ h >> 16, which is taken along with the halves: products with odd numbers (the fractions of
// the golden ratio, of e and of 2 e as words) between shifts
static __device__ __forceinline__ unsigned place_bits(unsigned h) {
  h = (h ^ (h >> 16)) * 0xb7e15163u;
  return (h ^ (h >> 15)) * 0xadf85459u;
}
constexpr unsigned kPlaceStep = 0x9e3779b9u;
static __device__ __forceinline__ unsigned mean_noise(unsigned h) { return ((h << 4) ^ (h >> 12)) & 0xffff0u; }     // 16 bits below 2^kMeanShift
static __device__ __forceinline__ unsigned root_noise(unsigned h) { return (h >> 13) & 0x7fff8u; }                  // and below 2^kRootShift
static __device__ __forceinline__ unsigned step_key(unsigned seed, unsigned step, unsigned number) { return (seed ^ step * kPlaceStep) + number * 0x6a09e667u; }
// The larger size of two values, with a sign that says nothing; a NaN is the largest.
static __device__ __forceinline__ float larger_size(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The largest size of three; a NaN if there is one.
static __device__ __forceinline__ float largest_size(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
static __device__ __forceinline__ float warp_largest(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Four values of a warp's 256: those from 4 lane on, in either half.
static __device__ __forceinline__ void load_four(float (&v)[4], const float *p, int n, bool vec) {
  if (vec) load_four(v, p);
  else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = j < n ? p[j] : 0.f;
  }
}
static __device__ __forceinline__ void store_four(float *p, const float (&v)[4], int n, bool vec) {
  if (vec) store_four(p, v);
  else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (j < n) p[j] = v[j];
  }
}

// The words of codes of a block's places: those behind its values are zero.
static __device__ __forceinline__ unsigned codes_of(const unsigned *codes, int h, int lane, int n) {
  unsigned q = codes[h * 32 + lane];
  const int left = n - (h * 128 + lane * 4);
  if (left < 4) q = left > 0 ? q & ((1u << (8 * left)) - 1) : 0;
  return q;
}
// Brings what a warp reads of a block to L2, 20 lines.
static __device__ __forceinline__ void bring(const AdamTensor &a, long block, int lane) {
  if (lane >= 20 || (block + 1) * kAdamBlock > a.n) return;
  const char *line = lane < 8 ? (const char *)(a.w + block * kAdamBlock) + lane * 128 : lane < 16 ? (const char *)(a.g + block * kAdamBlock) + (lane - 8) * 128 :
                     lane < 18 ? (const char *)((const unsigned *)a.m + block * 64) + (lane - 16) * 128 : (const char *)((const unsigned *)a.v + block * 64) + (lane - 18) * 128;
  asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
}
// A warp for a block of 256 values, eight a lane, and for others at the same distance, the next of which is brought to L2 meanwhile.  46 M values: 154 us, 4.8 TB/s; what
// holds it back is the work on codes, 88 instructions a value and lane, half of them on whole numbers, which issue at half rate, and the roots, which have to be exact for the
// codes and branch.  Tried before the step's bounds, with a tensor looked up for four turns at a time (143): a block for each chunk, which does not stay, 156; five blocks an SM in 48 registers 150
// (170 with what is brought ahead); a turn's loads in registers ahead of it 178; nothing brought ahead 158.
template <int N>
static __global__ void __launch_bounds__(256, 4) adam8_kernel(const __grid_constant__ AdamTable<N> table, const AdamStep s) {
  pdl_begin();
  __shared__ AdamFactors shared;
  adam_factors(s, shared);
  __syncthreads();
  AdamFactors f = shared;
  f.share /= f.root;
  const unsigned chunks = table.first[table.count];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long jump = (long)(kAdamTurn / kAdamBlock) * gridDim.x;      // to the warp's next block, if it is of the same tensor
  for (unsigned chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int i = tensor_of(table, chunk);
    const AdamTensor &a = table.t[i];
    const long block = (chunk - table.first[i]) * (long)(kAdamTurn / kAdamBlock) + warp, from = block * kAdamBlock;
    if (from < a.n) {
      const int n = (int)min((long)kAdamBlock, a.n - from);
      float *w = a.w + from;
      const float *g = a.g + from;
      unsigned *mc = (unsigned *)a.m + block * 64, *rc = (unsigned *)a.v + block * 64;
      const bool whole = n == kAdamBlock, vw = whole && ((uintptr_t)w & 15) == 0, vg = whole && ((uintptr_t)g & 15) == 0;
      float m[2][4], r[2][4], ww[2][4];
      unsigned mq[2], rq[2];
      const float2 scale = *reinterpret_cast<const float2 *>(a.scales + 2 * block);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int at = h * 128 + lane * 4;
        load_four(m[h], g + at, n - at, vg);
        load_four(ww[h], w + at, n - at, vw);
        mq[h] = codes_of(mc, h, lane, n);
        rq[h] = codes_of(rc, h, lane, n);
      }
      bring(a, block + jump, lane);
      float top_m = 0.f, top_r = 0.f;
      const float least = f.least * scale.y;
      const Pair share(f.share, f.share);
      const Pair scale_m2(scale.x, scale.x), scale_r2(scale.y, scale.y), beta1(s.beta1, s.beta1), beta2(s.beta2, s.beta2), rest1(s.rest1, s.rest1), rest2(s.rest2, s.rest2);
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const unsigned sizes = mq[h] & 0x7f7f7f7fu;
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const Pair gj(m[h][j], m[h][j + 1]), root = code_pair(rq[h], j, kRootShift, scale_r2);
          float x, y;
          code_pair(sizes, j, kMeanShift, scale_m2).get(x, y);
          x = __uint_as_float(__float_as_uint(x) ^ (mq[h] << (24 - 8 * j) & 0x80000000u));
          y = __uint_as_float(__float_as_uint(y) ^ (mq[h] << (16 - 8 * j) & 0x80000000u));
          add_singly(beta1 * Pair(x, y), rest1 * gj, m[h][j], m[h][j + 1]);
          add_singly(beta2 * (root * root), rest2 * (gj * gj), x, y);
          r[h][j] = __fsqrt_rn(x);
          r[h][j + 1] = __fsqrt_rn(y);
          top_m = larger_size(larger_size(top_m, m[h][j]), m[h][j + 1]);
          top_r = larger_size(larger_size(top_r, r[h][j]), r[h][j + 1]);
          // the weights' step, as adam_weight but for its bounds
          const Pair mj(m[h][j], m[h][j + 1]);
          (mj * share).get(x, y);
          x = largest_size(r[h][j], least, x);
          y = largest_size(r[h][j + 1], least, y);
          fused(Pair(x, y), Pair(f.root, f.root), Pair(s.eps, s.eps)).get(x, y);
          fused(Pair(-f.rate, -f.rate), mj * Pair(reciprocal(x), reciprocal(y)), Pair(ww[h][j], ww[h][j + 1]) * Pair(s.keep, s.keep)).get(ww[h][j], ww[h][j + 1]);
        }
        store_four(w + h * 128 + lane * 4, ww[h], n - (h * 128 + lane * 4), vw);
      }
      top_m = warp_largest(fabsf(top_m));
      top_r = warp_largest(fabsf(top_r));
      // (a NaN stays one, and makes the block's values NaN)
      float scale_m = __fmul_rn(top_m, 1.f / kMeanTop), scale_r = __fmul_rn(top_r, 1.f / kRootTop);
      if (scale_m < 0x1p-126f) scale_m = 0.f;
      if (scale_r < 0x1p-126f) scale_r = 0.f;
      const float by_m = scale_m == 0.f ? 0.f : __frcp_rn(scale_m), by_r = scale_r == 0.f ? 0.f : __frcp_rn(scale_r);
      const unsigned key = step_key(s.seed, f.step, (unsigned)(s.number + i)) + (unsigned)(from + lane * 4) * kPlaceStep;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        mq[h] = rq[h] = 0;
#pragma unroll
        for (int j = 0; j < 4; j += 2) {                       // (zeros, those behind the values among them, have the code zero whatever the noise)
          float x[2], y[2];
          (Pair(fabsf(m[h][j]), fabsf(m[h][j + 1])) * Pair(by_m, by_m)).get(x[0], x[1]);
          (Pair(r[h][j], r[h][j + 1]) * Pair(by_r, by_r)).get(y[0], y[1]);
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const unsigned bits = place_bits(key + (unsigned)(h * 128 + j + e) * kPlaceStep);
            mq[h] += (value_code(x[e], kMeanShift, mean_noise(bits)) + (m[h][j + e] < 0.f ? 128u : 0u)) << (8 * (j + e));
            rq[h] += value_code(y[e], kRootShift, root_noise(bits)) << (8 * (j + e));
          }
        }
        mc[h * 32 + lane] = mq[h];
        rc[h * 32 + lane] = rq[h];
      }
      if (lane == 0) *reinterpret_cast<float2 *>(a.scales + 2 * block) = make_float2(scale_m, scale_r);
    }
  }
  adam_count(s, f.step);
}

// What the codes stand for: m into w, v into g's place (named as the table's weights and gradients).  46 M values: 73 us, 6.4 TB/s.
template <int N>
static __global__ void __launch_bounds__(256) adam8_moments_kernel(const __grid_constant__ AdamTable<N> table) {
  pdl_begin();
  const int i = tensor_of(table, blockIdx.x), lane = threadIdx.x & 31;
  const AdamTensor &a = table.t[i];
  const long block = (blockIdx.x - table.first[i]) * (long)(kAdamTurn / kAdamBlock) + (threadIdx.x >> 5), from = block * kAdamBlock;
  if (from >= a.n) return;
  const float2 scale = *reinterpret_cast<const float2 *>(a.scales + 2 * block);
  unsigned mq[2], rq[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    mq[h] = ((const unsigned *)a.m)[block * 64 + h * 32 + lane];
    rq[h] = ((const unsigned *)a.v)[block * 64 + h * 32 + lane];
  }
  const int n = (int)min((long)kAdamBlock, a.n - from);
  float *mean = a.w + from, *square = const_cast<float *>(a.g) + from;
  const bool whole = n == kAdamBlock, vm = whole && ((uintptr_t)mean & 15) == 0, vs = whole && ((uintptr_t)square & 15) == 0;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int at = h * 128 + lane * 4;
    float m[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      const Pair root = code_pair(rq[h], j, kRootShift, Pair(scale.y, scale.y));
      (root * root).get(v[j], v[j + 1]);
      code_pair(mq[h] & 0x7f7f7f7fu, j, kMeanShift, Pair(scale.x, scale.x)).get(m[j], m[j + 1]);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) m[j] = __uint_as_float(__float_as_uint(m[j]) ^ (mq[h] << (24 - 8 * j) & 0x80000000u));
    store_four(mean + at, m, n - at, vm);
    store_four(square + at, v, n - at, vs);
  }
}

// ---- launches
enum AdamKind { kAdam32, kAdam8, kAdamMoments };
template <int N> static void adam_launch(AdamKind kind, const std::vector<AdamTensor> &all, const AdamStep &step) {
  size_t i = 0;
  do {
    AdamTable<N> table;
    AdamStep s = step;
    s.number = (int)i;
    table.count = 0;
    table.first[0] = 0;
    for (; i < all.size() && table.count < N; i++) {
      const long chunks = (all[i].n + kAdamTurn - 1) / kAdamTurn;
      THC_CHECK(chunks < (1l << 31), "tensors of more than 2^42 values");
      if (table.count && table.first[table.count] + (unsigned long)chunks >= (1ul << 31)) break;
      table.t[table.count] = all[i];
      table.first[table.count + 1] = table.first[table.count] + (unsigned)chunks;
      table.count++;
    }
    s.last = i == all.size();
    const unsigned chunks = table.first[table.count], blocks = std::max(1u, std::min(chunks, kind == kAdam8 ? (unsigned)ctx().sm_count * 4 : 1u << 31));
    if (kind == kAdam32) pdl_launch(adam_kernel<N>, blocks, 256, 0, table, s);
    else if (kind == kAdam8) pdl_launch(adam8_kernel<N>, blocks, 256, 0, table, s);
    else pdl_launch(adam8_moments_kernel<N>, blocks, 256, 0, table);
    check_launch(kind == kAdamMoments ? "AdamW_moments" : "AdamW_update");
  } while (i < all.size());
}
static void adam_launch(AdamKind kind, const std::vector<AdamTensor> &all, const AdamStep &step) {
  if (all.size() <= kFewTensors) adam_launch<kFewTensors>(kind, all, step);
  else if (all.size() <= kSomeTensors) adam_launch<kSomeTensors>(kind, all, step);
  else if (all.size() <= kMoreTensors) adam_launch<kMoreTensors>(kind, all, step);
  else adam_launch<kManyTensors>(kind, all, step);
}

// ---- checks
// Memory that a call writes may share nothing with the rest of its tensors.  Tensors of a kind often lie side by side in one storage: neighbours come together as
// they are added, so that few spans are left to sort.
class Spans {
 public:
  void add(const void *p, long values, bool written) {
    if (!values) return;
    const Span s{(uintptr_t)p, (uintptr_t)p + 4 * (uintptr_t)values, written};
    if (!spans_.empty() && spans_.back().written == written && (spans_.back().to == s.from || (!written && spans_.back().from <= s.from && s.from < spans_.back().to)))
      spans_.back().to = std::max(spans_.back().to, s.to);
    else spans_.push_back(s);
  }
  void check() {
    // Spans of one kind mostly come in order: those runs are merged, unless there are many.
    std::vector<size_t> runs{0};
    for (size_t i = 1; i < spans_.size() && runs.size() <= 16; i++)
      if (spans_[i] < spans_[i - 1]) runs.push_back(i);
    if (runs.size() > 16) std::sort(spans_.begin(), spans_.end());
    else {
      runs.push_back(spans_.size());
      for (; runs.size() > 2; ) {
        std::vector<size_t> next{0};
        for (size_t i = 2; i < runs.size(); i += 2) {
          std::inplace_merge(spans_.begin() + runs[i - 2], spans_.begin() + runs[i - 1], spans_.begin() + runs[i]);
          next.push_back(runs[i]);
        }
        if (next.back() != spans_.size()) next.push_back(spans_.size());
        runs.swap(next);
      }
    }
    uintptr_t end = 0, end_written = 0;
    for (const Span &s : spans_) {
      THC_CHECK(s.from >= (s.written ? end : end_written), "a result shares memory with another tensor of the call");
      end = std::max(end, s.to);
      if (s.written) end_written = std::max(end_written, s.to);
    }
  }

 private:
  struct Span {
    uintptr_t from, to;
    bool written;
    bool operator<(const Span &o) const { return from < o.from; }
  };
  std::vector<Span> spans_;
};
// A tensor of the call, contiguous, of n values (-1: of any number), of this device; called for every tensor, some hundreds a step.
class Flat {
 public:
  float *operator()(const THGPUTensor *t, long n, int argn, int i, const char *what) const {
    if (!t) fail("Invalid argument %d: tensors expected", argn);
    const long k = t->nDimension == 1 ? t->size[0] : nelem(t);
    if ((n >= 0 && k != n) || !((t->nDimension == 1 && t->stride[0] == 1) || is_contiguous(t)))
      fail("Invalid argument %d: contiguous %s of %ld values expected for tensor %d", argn, what, n >= 0 ? n : k, i + 1);
    if (!t->storage) return nullptr;
    const long tag = (long)(intptr_t)t->storage->allocatorContext;
    if (tag > 0 && tag != here_) fail("Invalid argument %d: tensor of device %ld while device %ld is current", argn, tag, here_);
    return data_ptr(t);
  }

 private:
  const long here_ = std::max(device_if_initialised(), 0) + 1;      // (as check_here)
};
static long values_of(const THGPUTensor *t) { return !t ? 0 : t->nDimension == 1 ? t->size[0] : nelem(t); }
static void add_codes(Spans &spans, const std::vector<AdamTensor> &all, bool codes_written, bool g_written) {
  auto blocks = [](const AdamTensor &t) { return (t.n + kAdamBlock - 1) / kAdamBlock; };
  for (const AdamTensor &t : all) spans.add(t.w, t.n, true);
  for (const AdamTensor &t : all) spans.add(t.g, t.n, g_written);
  for (const AdamTensor &t : all) spans.add(t.m, 64 * blocks(t), codes_written);
  for (const AdamTensor &t : all) spans.add(t.v, 64 * blocks(t), codes_written);
  for (const AdamTensor &t : all) spans.add(t.scales, 2 * blocks(t), codes_written);
}
static void check_rates(double lr, double beta1, double beta2, double eps, double decay, int argn) {
  THC_ARG(std::isfinite(lr) && lr >= 0, argn, "learning rate must be finite and not negative");
  THC_ARG(beta1 >= 0 && beta1 < 1, argn + 1, "beta1 must be in [0, 1)");
  THC_ARG(beta2 >= 0 && beta2 < 1, argn + 2, "beta2 must be in [0, 1)");
  THC_ARG(std::isfinite(eps) && eps >= 0x1p-126 && eps < 0x1p126, argn + 3, "epsilon must be positive and within the range of a float's normal values");
  THC_ARG(std::isfinite(decay) && decay >= 0, argn + 4, "weight decay must be finite and not negative");
}
static AdamStep adam_step(THGPUTensor *step, double lr, double beta1, double beta2, double eps, double decay, long seed) {
  AdamStep s;
  s.step = data_ptr(step);
  s.last = false;
  s.lr = (float)lr; s.beta1 = (float)beta1; s.beta2 = (float)beta2; s.rest1 = (float)(1.0 - beta1); s.rest2 = (float)(1.0 - beta2);
  s.eps = (float)eps; s.keep = (float)(1.0 - lr * decay);
  s.log1 = (float)std::log(beta1); s.log2 = (float)std::log(beta2);      // (of zero: minus infinity, and then 1 - b^t is one)
  const double left = 1.0 - beta1 * beta1 / beta2;      // (beta2 zero: minus infinity, or with beta1 zero too a NaN: no bound)
  s.most = left > 0 ? (float)std::max(2.0, (1.0 - beta1) / std::sqrt((1.0 - beta2) * left)) : INFINITY;
  s.seed = (unsigned)(unsigned long)seed;
  s.number = 0;
  return s;
}

}  // namespace thc

using namespace thc;

THC_API int THGPUNN_AdamW_update(int n, THGPUTensor **weights, THGPUTensor **grads, THGPUTensor **means, THGPUTensor **squares, THGPUTensor *step, double lr,
                                 double beta1, double beta2, double eps, double decay) {
  THC_BEGIN
  THC_ARG(n >= 0, 1, "a number of tensors expected");
  THC_ARG(n == 0 || (weights && grads && means && squares), 2, "tensors expected");
  const Flat flat;
  flat(step, 2, 6, 0, "step");
  check_rates(lr, beta1, beta2, eps, decay, 7);
  Spans spans;
  spans.add(data_ptr(step), 2, true);
  std::vector<AdamTensor> all(n);
  for (int i = 0; i < n; i++) {
    AdamTensor &t = all[i];
    t.w = flat(weights[i], -1, 2, i, "weights");
    t.n = values_of(weights[i]);
    t.g = flat(grads[i], t.n, 3, i, "gradients");
    t.m = flat(means[i], t.n, 4, i, "means");
    t.v = flat(squares[i], t.n, 5, i, "squares");
    t.scales = nullptr;
  }
  for (const AdamTensor &t : all) spans.add(t.w, t.n, true);
  for (const AdamTensor &t : all) spans.add(t.g, t.n, false);
  for (const AdamTensor &t : all) spans.add(t.m, t.n, true);
  for (const AdamTensor &t : all) spans.add(t.v, t.n, true);
  spans.check();
  adam_launch(kAdam32, all, adam_step(step, lr, beta1, beta2, eps, decay, 0));
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_AdamW8_update(int n, THGPUTensor **weights, THGPUTensor **grads, THGPUTensor **meanCodes, THGPUTensor **rootCodes, THGPUTensor **scales,
                                  THGPUTensor *step, double lr, double beta1, double beta2, double eps, double decay, long seed) {
  THC_BEGIN
  THC_ARG(n >= 0, 1, "a number of tensors expected");
  THC_ARG(n == 0 || (weights && grads && meanCodes && rootCodes && scales), 2, "tensors expected");
  const Flat flat;
  flat(step, 2, 7, 0, "step");
  check_rates(lr, beta1, beta2, eps, decay, 8);
  Spans spans;
  spans.add(data_ptr(step), 2, true);
  std::vector<AdamTensor> all(n);
  for (int i = 0; i < n; i++) {
    AdamTensor &t = all[i];
    t.w = flat(weights[i], -1, 2, i, "weights");
    t.n = values_of(weights[i]);
    const long blocks = (t.n + kAdamBlock - 1) / kAdamBlock;
    t.g = flat(grads[i], t.n, 3, i, "gradients");
    t.m = flat(meanCodes[i], 64 * blocks, 4, i, "codes of means");
    t.v = flat(rootCodes[i], 64 * blocks, 5, i, "codes of roots");
    t.scales = flat(scales[i], 2 * blocks, 6, i, "scales");
    THC_ARG(((uintptr_t)t.scales & 7) == 0, 6, "scales on a boundary of 8 bytes expected");
  }
  add_codes(spans, all, true, false);
  spans.check();
  adam_launch(kAdam8, all, adam_step(step, lr, beta1, beta2, eps, decay, seed));
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_AdamW8_moments(int n, THGPUTensor **meanCodes, THGPUTensor **rootCodes, THGPUTensor **scales, THGPUTensor **means, THGPUTensor **squares) {
  THC_BEGIN
  THC_ARG(n >= 0, 1, "a number of tensors expected");
  THC_ARG(n == 0 || (meanCodes && rootCodes && scales && means && squares), 2, "tensors expected");
  const Flat flat;
  Spans spans;
  std::vector<AdamTensor> all(n);
  for (int i = 0; i < n; i++) {
    AdamTensor &t = all[i];
    t.n = values_of(means[i]);
    const long blocks = (t.n + kAdamBlock - 1) / kAdamBlock;
    t.m = flat(meanCodes[i], 64 * blocks, 2, i, "codes of means");
    t.v = flat(rootCodes[i], 64 * blocks, 3, i, "codes of roots");
    t.scales = flat(scales[i], 2 * blocks, 4, i, "scales");
    t.w = flat(means[i], -1, 5, i, "means");
    t.g = flat(squares[i], t.n, 6, i, "squares");
    THC_ARG(((uintptr_t)t.scales & 7) == 0, 4, "scales on a boundary of 8 bytes expected");
  }
  add_codes(spans, all, false, true);
  spans.check();
  if (n) adam_launch(kAdamMoments, all, AdamStep{});
  return 0;
  THC_END(1)
}
