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
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "nn_args.h"

namespace thc {

constexpr int kAdamBlock = 256;                                // values under one scale
constexpr int kAdamChunk = 2048;                               // values of a block's turn: a warp has 256
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
constexpr int kFewTensors = 24, kManyTensors = 512;
struct AdamStep {
  float *step;               // steps taken, and the count of blocks that are done (zero between launches)
  bool last;                 // the launch that counts the step
  float lr, beta1, beta2, rest1, rest2, eps, keep;    // rest: 1 - beta, keep: 1 - lr decay
  double b1, b2;
  unsigned seed;
  int number;                // of the table's first tensor
};
// What a step's number decides: lr / (1 - b1^t) and 1 / sqrt(1 - b2^t).  1 - b^t loses a float's digits for small t: in 64 bits.
struct AdamFactors {
  float rate, root;
  unsigned step;
};
// By threads 0 and 1 into shared memory; a barrier has to follow.
static __device__ __forceinline__ void adam_factors(const AdamStep &s, AdamFactors &f) {
  if (threadIdx.x > 1) return;
  const unsigned step = (unsigned)s.step[0] + 1;
  double b = threadIdx.x ? s.b2 : s.b1, p = 1.0;
  for (unsigned t = step; t; t >>= 1, b *= b)
    if (t & 1) p *= b;
  if (threadIdx.x == 0) {
    f.rate = (float)(s.lr / (1.0 - p));
    f.step = step;
  } else f.root = (float)(1.0 / sqrt(1.0 - p));
}
// The last block of the last launch counts the step: by then every block has read its number.
static __device__ __forceinline__ void adam_count(const AdamStep &s, unsigned step) {
  if (!s.last) return;
  __syncthreads();
  if (threadIdx.x != 0) return;
  unsigned *done = reinterpret_cast<unsigned *>(s.step + 1);
  __threadfence();
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

// ---- moments in 32 bits
static __device__ __forceinline__ float reciprocal(float v) {     // within a step
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
static __device__ __forceinline__ float square_root(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
static __device__ __forceinline__ float adam_weight(float w, float m, float root, const AdamStep &s, const AdamFactors &f) {
  return fmaf(-f.rate, m * reciprocal(fmaf(root, f.root, s.eps)), w * s.keep);
}
static __device__ __forceinline__ void adam_value(float &w, float g, float &m, float &v, const AdamStep &s, const AdamFactors &f) {
  m = fmaf(s.beta1, m, s.rest1 * g);
  v = fmaf(s.beta2, v, s.rest2 * (g * g));
  w = adam_weight(w, m, square_root(v), s, f);
}
// Eight values a thread: all of a turn's loads are on their way before the first is needed, in the first turn before the step's factors are made.
template <int N>
static __global__ void __launch_bounds__(256, 4) adam_kernel(const __grid_constant__ AdamTable<N> table, const AdamStep s) {
  pdl_begin();
  __shared__ AdamFactors shared;
  AdamFactors f;
  const unsigned chunks = table.first[table.count];
  bool started = false;
  auto start = [&] {
    if (started) return;
    adam_factors(s, shared);
    __syncthreads();
    f = shared;
    started = true;
  };
  for (unsigned chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int i = tensor_of(table, chunk);
    const AdamTensor &a = table.t[i];
    const long from = (chunk - table.first[i]) * (long)kAdamChunk;
    const int n = (int)min((long)kAdamChunk, a.n - from);
    float *w = a.w + from, *m = (float *)a.m + from, *v = (float *)a.v + from;
    const float *g = a.g + from;
    if (n == kAdamChunk && (((uintptr_t)w | (uintptr_t)g | (uintptr_t)m | (uintptr_t)v) & 15) == 0) {
      float4 ww[2], gg[2], mm[2], vv[2];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int at = j * 256 + threadIdx.x;
        gg[j] = __ldcs(reinterpret_cast<const float4 *>(g) + at);
        ww[j] = reinterpret_cast<float4 *>(w)[at];
        mm[j] = reinterpret_cast<float4 *>(m)[at];
        vv[j] = reinterpret_cast<float4 *>(v)[at];
      }
      start();
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int at = j * 256 + threadIdx.x;
        adam_value(ww[j].x, gg[j].x, mm[j].x, vv[j].x, s, f);
        adam_value(ww[j].y, gg[j].y, mm[j].y, vv[j].y, s, f);
        adam_value(ww[j].z, gg[j].z, mm[j].z, vv[j].z, s, f);
        adam_value(ww[j].w, gg[j].w, mm[j].w, vv[j].w, s, f);
        reinterpret_cast<float4 *>(w)[at] = ww[j];
        reinterpret_cast<float4 *>(m)[at] = mm[j];
        reinterpret_cast<float4 *>(v)[at] = vv[j];
      }
    } else {
      float ww[8], gg[8], mm[8], vv[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int at = j * 256 + threadIdx.x;
        if (at < n) { ww[j] = w[at]; gg[j] = g[at]; mm[j] = m[at]; vv[j] = v[at]; }
      }
      start();
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int at = j * 256 + threadIdx.x;
        if (at < n) {
          adam_value(ww[j], gg[j], mm[j], vv[j], s, f);
          w[at] = ww[j]; m[at] = mm[j]; v[at] = vv[j];
        }
      }
    }
  }
  start();
  adam_count(s, f.step);
}

// ---- moments in 8 bits
static __device__ __forceinline__ float code_value(unsigned code, int shift, float scale) {
  return __fmul_rn(__fadd_rn(__uint_as_float(kCodeBits + (code << shift)), -kCodeFloor), scale);
}
// The code of x >= 0 with `noise` below 2^shift on its bits.
static __device__ __forceinline__ unsigned value_code(float x, float inverse, int shift, unsigned noise, unsigned most) {
  return min((__float_as_uint(__fadd_rn(__fmul_rn(x, inverse), kCodeFloor)) + noise - (kCodeBits - (1u << (shift - 17)))) >> shift, most);
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
// The larger of two, a NaN being the largest.
static __device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
static __device__ __forceinline__ float warp_largest(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Four values of a warp's 256: those from 4 lane on, in either half.
static __device__ __forceinline__ void load_four(float (&v)[4], const float *p, int n, bool vec) {
  if (vec) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = j < n ? p[j] : 0.f;
  }
}
static __device__ __forceinline__ void store_four(float *p, const float (&v)[4], int n, bool vec) {
  if (vec) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
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
// A warp for a block of 256 values, eight a lane.
template <int N>
static __global__ void __launch_bounds__(256, 4) adam8_kernel(const __grid_constant__ AdamTable<N> table, const AdamStep s) {
  pdl_begin();
  __shared__ AdamFactors shared;
  adam_factors(s, shared);
  __syncthreads();
  const AdamFactors f = shared;
  const unsigned chunks = table.first[table.count];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (unsigned chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int i = tensor_of(table, chunk);
    const AdamTensor &a = table.t[i];
    const long block = (chunk - table.first[i]) * (long)(kAdamChunk / kAdamBlock) + warp, from = block * kAdamBlock;
    if (from >= a.n) continue;
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
    float top_m = 0.f, top_r = 0.f;
#pragma unroll
    for (int h = 0; h < 2; h++) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float gj = m[h][j];
        const float was = code_value(mq[h] >> (8 * j) & 127u, kMeanShift, scale.x), root = code_value(rq[h] >> (8 * j) & 255u, kRootShift, scale.y);
        const float sign = __uint_as_float(__float_as_uint(was) ^ (mq[h] << (24 - 8 * j) & 0x80000000u));
        m[h][j] = __fadd_rn(__fmul_rn(s.beta1, sign), __fmul_rn(s.rest1, gj));
        r[h][j] = __fsqrt_rn(__fadd_rn(__fmul_rn(s.beta2, __fmul_rn(root, root)), __fmul_rn(s.rest2, __fmul_rn(gj, gj))));
        top_m = larger(top_m, fabsf(m[h][j]));
        top_r = larger(top_r, r[h][j]);
        ww[h][j] = adam_weight(ww[h][j], m[h][j], r[h][j], s, f);
      }
      store_four(w + h * 128 + lane * 4, ww[h], n - (h * 128 + lane * 4), vw);
    }
    top_m = warp_largest(top_m);
    top_r = warp_largest(top_r);
    // (a NaN stays one, and makes the block's values NaN)
    float scale_m = __fmul_rn(top_m, 1.f / kMeanTop), scale_r = __fmul_rn(top_r, 1.f / kRootTop);
    if (scale_m < 0x1p-126f) scale_m = 0.f;
    if (scale_r < 0x1p-126f) scale_r = 0.f;
    const float inverse_m = scale_m == 0.f ? 0.f : __fdiv_rn(1.f, scale_m), inverse_r = scale_r == 0.f ? 0.f : __fdiv_rn(1.f, scale_r);
    const unsigned key = step_key(s.seed, f.step, (unsigned)(s.number + i)) + (unsigned)(from + lane * 4) * kPlaceStep;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      mq[h] = rq[h] = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {                       // (zeros, those behind the values among them, have the code zero whatever the noise)
        const unsigned bits = place_bits(key + (unsigned)(h * 128 + j) * kPlaceStep);
        const unsigned cm = value_code(fabsf(m[h][j]), inverse_m, kMeanShift, mean_noise(bits), 127u) + (m[h][j] < 0.f ? 128u : 0u);
        mq[h] += cm << (8 * j);
        rq[h] += value_code(r[h][j], inverse_r, kRootShift, root_noise(bits), 255u) << (8 * j);
      }
      mc[h * 32 + lane] = mq[h];
      rc[h * 32 + lane] = rq[h];
    }
    if (lane == 0) *reinterpret_cast<float2 *>(a.scales + 2 * block) = make_float2(scale_m, scale_r);
  }
  adam_count(s, f.step);
}

// What the codes stand for: m into w, v into g's place (named as the table's weights and gradients).
template <int N>
static __global__ void __launch_bounds__(256) adam8_moments_kernel(const __grid_constant__ AdamTable<N> table) {
  pdl_begin();
  const unsigned chunks = table.first[table.count];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (unsigned chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int i = tensor_of(table, chunk);
    const AdamTensor &a = table.t[i];
    const long block = (chunk - table.first[i]) * (long)(kAdamChunk / kAdamBlock) + warp, from = block * kAdamBlock;
    if (from >= a.n) continue;
    const int n = (int)min((long)kAdamBlock, a.n - from);
    float *mean = a.w + from, *square = const_cast<float *>(a.g) + from;
    const unsigned *mc = (const unsigned *)a.m + block * 64, *rc = (const unsigned *)a.v + block * 64;
    const bool whole = n == kAdamBlock, vm = whole && ((uintptr_t)mean & 15) == 0, vs = whole && ((uintptr_t)square & 15) == 0;
    const float2 scale = *reinterpret_cast<const float2 *>(a.scales + 2 * block);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const unsigned mq = mc[h * 32 + lane], rq = rc[h * 32 + lane];
      const int at = h * 128 + lane * 4;
      float m[4], v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const unsigned cm = mq >> (8 * j) & 255u;
        const float value = code_value(cm & 127u, kMeanShift, scale.x), root = code_value(rq >> (8 * j) & 255u, kRootShift, scale.y);
        m[j] = cm & 128u ? -value : value;
        v[j] = __fmul_rn(root, root);
      }
      store_four(mean + at, m, n - at, vm);
      store_four(square + at, v, n - at, vs);
    }
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
      const long chunks = (all[i].n + kAdamChunk - 1) / kAdamChunk;
      THC_CHECK(chunks < (1l << 31), "tensors of more than 2^42 values");
      if (table.count && table.first[table.count] + (unsigned long)chunks >= (1ul << 31)) break;
      table.t[table.count] = all[i];
      table.first[table.count + 1] = table.first[table.count] + (unsigned)chunks;
      table.count++;
    }
    s.last = i == all.size();
    const unsigned chunks = table.first[table.count], blocks = std::max(1u, std::min(chunks, kind == kAdamMoments ? 1u << 30 : (unsigned)ctx().sm_count * 4));
    if (kind == kAdam32) pdl_launch(adam_kernel<N>, blocks, 256, 0, table, s);
    else if (kind == kAdam8) pdl_launch(adam8_kernel<N>, blocks, 256, 0, table, s);
    else pdl_launch(adam8_moments_kernel<N>, blocks, 256, 0, table);
    check_launch(kind == kAdamMoments ? "AdamW_moments" : "AdamW_update");
  } while (i < all.size());
}
static void adam_launch(AdamKind kind, const std::vector<AdamTensor> &all, const AdamStep &step) {
  if (all.size() <= kFewTensors) adam_launch<kFewTensors>(kind, all, step);
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
    if (!std::is_sorted(spans_.begin(), spans_.end())) std::sort(spans_.begin(), spans_.end());
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
static void check_flat(const THGPUTensor *t, long n, int argn, int i, const char *what) {
  if (!t || nelem(t) != n || !is_contiguous(t)) fail("Invalid argument %d: contiguous %s of %ld values expected for tensor %d", argn, what, n, i + 1);
}
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
  s.b1 = beta1; s.b2 = beta2;
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
  check_flat(step, 2, 6, 0, "step");
  check_rates(lr, beta1, beta2, eps, decay, 7);
  check_here({nullptr, nullptr, nullptr, nullptr, nullptr, step});
  Spans spans;
  spans.add(data_ptr(step), 2, true);
  std::vector<AdamTensor> all;
  all.reserve(n);
  for (int i = 0; i < n; i++) {
    THC_ARG(weights[i], 2, "tensors expected");
    const long k = nelem(weights[i]);
    check_flat(weights[i], k, 2, i, "weights");
    check_flat(grads[i], k, 3, i, "gradients");
    check_flat(means[i], k, 4, i, "means");
    check_flat(squares[i], k, 5, i, "squares");
    check_here({nullptr, weights[i], grads[i], means[i], squares[i]});
    all.push_back(AdamTensor{data_ptr(weights[i]), data_ptr(grads[i]), data_ptr(means[i]), data_ptr(squares[i]), nullptr, k});
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
  check_flat(step, 2, 7, 0, "step");
  check_rates(lr, beta1, beta2, eps, decay, 8);
  check_here({nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, step});
  Spans spans;
  spans.add(data_ptr(step), 2, true);
  std::vector<AdamTensor> all;
  all.reserve(n);
  for (int i = 0; i < n; i++) {
    THC_ARG(weights[i], 2, "tensors expected");
    const long k = nelem(weights[i]), blocks = (k + kAdamBlock - 1) / kAdamBlock;
    check_flat(weights[i], k, 2, i, "weights");
    check_flat(grads[i], k, 3, i, "gradients");
    check_flat(meanCodes[i], 64 * blocks, 4, i, "codes of means");
    check_flat(rootCodes[i], 64 * blocks, 5, i, "codes of roots");
    check_flat(scales[i], 2 * blocks, 6, i, "scales");
    check_here({nullptr, weights[i], grads[i], meanCodes[i], rootCodes[i], scales[i]});
    all.push_back(AdamTensor{data_ptr(weights[i]), data_ptr(grads[i]), data_ptr(meanCodes[i]), data_ptr(rootCodes[i]), data_ptr(scales[i]), k});
    THC_ARG(((uintptr_t)all[i].scales & 7) == 0, 6, "scales on a boundary of 8 bytes expected");
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
  Spans spans;
  std::vector<AdamTensor> all;
  all.reserve(n);
  for (int i = 0; i < n; i++) {
    THC_ARG(means[i], 5, "tensors expected");
    const long k = nelem(means[i]), blocks = (k + kAdamBlock - 1) / kAdamBlock;
    check_flat(means[i], k, 5, i, "means");
    check_flat(squares[i], k, 6, i, "squares");
    check_flat(meanCodes[i], 64 * blocks, 2, i, "codes of means");
    check_flat(rootCodes[i], 64 * blocks, 3, i, "codes of roots");
    check_flat(scales[i], 2 * blocks, 4, i, "scales");
    check_here({nullptr, meanCodes[i], rootCodes[i], scales[i], means[i], squares[i]});
    all.push_back(AdamTensor{data_ptr(means[i]), data_ptr(squares[i]), data_ptr(meanCodes[i]), data_ptr(rootCodes[i]), data_ptr(scales[i]), k});
    THC_ARG(((uintptr_t)all[i].scales & 7) == 0, 4, "scales on a boundary of 8 bytes expected");
  }
  add_codes(spans, all, false, true);
  spans.check();
  if (n) adam_launch(kAdamMoments, all, AdamStep{});
  return 0;
  THC_END(1)
}
