// Values that FP16 pairs do not hold (Stray, mm_problem.cuh), added to the results of products in FP32.
//
// Each result takes the strays of one operand against all of the other operand, and the strays of that against what the pairs hold of the
// first.  A block owns the results it changes and takes the strays in their listed order, so that sums repeat exactly.  Without
// strays, the usual case of all but the largest tensors, a launch looks at two counts and ends (about 2 us as a programmatic
// dependent); each stray of an activation costs a block about a microsecond, one of the weights a pass over a plane.
// The weight gradient's are added by UnpackGradPass (mm_planes.cuh).
#ifndef THC_MM_STRAYS_CUH
#define THC_MM_STRAYS_CUH

#include "mm_planes.cuh"

namespace thc {
namespace mm {

// Forward: src = input, out [N][K][oH][oW]; GRAD_INPUT: src = gradOutput, out [N][C][H][W].  Block (a, b) owns the images a, a + gridDim.x,
// ... of the result's planes b, b + gridDim.y, ...
template <bool GRAD_INPUT>
static __global__ void __launch_bounds__(256) window_strays_kernel(const float *src, const float *w, float *out, const LayerShape l,
                                                                   const Measured act, const Measured weight, const Ranges ranges) {
  pdl_begin();
  const bool wide = ranges.wide();
  const int na = act.strays(wide), nw = weight.strays(wide);
  if (na + nw == 0) return;
  const int Cs = GRAD_INPUT ? l.K : l.C, Hs = GRAD_INPUT ? l.oH : l.H, Ws = GRAD_INPUT ? l.oW : l.W;
  const int Co = GRAD_INPUT ? l.C : l.K, Ho = GRAD_INPUT ? l.H : l.oH, Wo = GRAD_INPUT ? l.W : l.oW;
  const int taps = l.kH * l.kW, mine = (Co - (int)blockIdx.y + (int)gridDim.y - 1) / (int)gridDim.y;   // (gridDim.y <= Co)
  for (int e = 0; e < na; e++) {
    const long at = act.list[e].at, row = at / Ws, plane = row / Hs, n = plane / Cs;
    if (n % gridDim.x != blockIdx.x) continue;
    const int x = (int)(at - row * Ws), y = (int)(row - plane * Hs), c = (int)(plane - n * Cs);
    const float v = act.list[e].v;
    for (long t = threadIdx.x; t < (long)mine * taps; t += 256) {
      const int co = (int)(blockIdx.y + t / taps * gridDim.y), tap = (int)(t % taps), i = tap / l.kW, j = tap - i * l.kW;
      int oy, ox;
      if (GRAD_INPUT) {
        oy = y * l.dH + i - l.pad; ox = x * l.dW + j - l.pad;
        if (oy < 0 || ox < 0) continue;
      } else {
        const int ty = y + l.pad - i, tx = x + l.pad - j;
        oy = ty / l.dH; ox = tx / l.dW;
        if (ty < 0 || tx < 0 || oy * l.dH != ty || ox * l.dW != tx) continue;
      }
      if (oy >= Ho || ox >= Wo) continue;
      const long k = GRAD_INPUT ? (long)c * l.C + co : (long)co * l.C + c;
      out[((n * Co + co) * Ho + oy) * (long)Wo + ox] += v * w[k * taps + tap];
    }
    __syncthreads();   // (another thread may take the same result next)
  }
  const unsigned limit = stray_limit(act.rec->max_bits) - 1u;
  for (int e = 0; e < nw; e++) {
    const long at = weight.list[e].at, k = at / taps;
    const int tap = (int)(at - k * taps), i = tap / l.kW, j = tap - i * l.kW, ko = (int)(k / l.C), ci = (int)(k - (long)ko * l.C);
    const int co = GRAD_INPUT ? ci : ko, c = GRAD_INPUT ? ko : ci;
    if (co % gridDim.y != blockIdx.y) continue;
    const float v = weight.list[e].v;
    for (long n = blockIdx.x; n < l.N; n += gridDim.x)
      for (int t = threadIdx.x; t < Ho * Wo; t += 256) {
        const int oy = t / Wo, ox = t - oy * Wo;
        int y, x;
        if (GRAD_INPUT) {
          const int ty = oy + l.pad - i, tx = ox + l.pad - j;
          y = ty / l.dH; x = tx / l.dW;
          if (ty < 0 || tx < 0 || y * l.dH != ty || x * l.dW != tx) continue;
        } else {
          y = oy * l.dH + i - l.pad; x = ox * l.dW + j - l.pad;
          if (y < 0 || x < 0) continue;
        }
        if (y >= Hs || x >= Ws) continue;
        const float s = src[((n * Cs + c) * Hs + y) * (long)Ws + x];
        if ((__float_as_uint(s) & 0x7fffffffu) - 1u >= limit) out[((n * Co + co) * Ho + oy) * (long)Wo + ox] += v * s;   // (zeros pass)
      }
    __syncthreads();
  }
}

// D(m, n) += alpha * ...: element (r, l) of a side at p[r * ld + l] (along_k) or p[l * ld + r], measured as `run` values a line.  Block (a, b)
// owns the columns of a 256-wide chunk, rows b, b + gridDim.y, ...; a thread owns a column, then a row.
struct StraySide { const float *p; long ld, run; int along_k; Measured m; };
static __global__ void __launch_bounds__(256) matrix_strays_kernel(const StraySide x, const StraySide y, long M, long N, const Epilogue epi,
                                                                   const Ranges ranges) {
  pdl_begin();
  const bool wide = ranges.wide();
  const int nx = x.m.strays(wide), ny = y.m.strays(wide);
  if (nx + ny == 0) return;
  auto place = [](const StraySide &s, int e, long &r, long &l) {
    const long at = s.m.list[e].at, line = at / s.run, c = at - line * s.run;
    r = s.along_k ? line : c;
    l = s.along_k ? c : line;
  };
  const unsigned limit = stray_limit(x.m.rec->max_bits) - 1u;
  for (long n0 = blockIdx.x * 256l; n0 < N; n0 += gridDim.x * 256l) {
    const long n = n0 + threadIdx.x;
    for (int e = 0; n < N && e < nx; e++) {
      long r, l;
      place(x, e, r, l);
      if (r % gridDim.y == blockIdx.y)
        epi.out[epi.moff(r) + n * epi.nstride] += epi.alpha * (x.m.list[e].v * y.p[y.along_k ? n * y.ld + l : l * y.ld + n]);
    }
    __syncthreads();   // rows, from here on
    for (int e = 0; e < ny; e++) {
      long c, l;
      place(y, e, c, l);
      if (c < n0 || c >= n0 + 256) continue;
      for (long m = blockIdx.y + (long)threadIdx.x * gridDim.y; m < M; m += 256l * gridDim.y) {
        const float s = x.p[x.along_k ? m * x.ld + l : l * x.ld + m];
        if ((__float_as_uint(s) & 0x7fffffffu) - 1u >= limit) epi.out[epi.moff(m) + c * epi.nstride] += epi.alpha * (y.m.list[e].v * s);
      }
    }
    __syncthreads();
  }
}

// ---- groups --------------------------------------------------------------------------------------------------------------
// Where the groups' rows start: as they are, and with each group padded to whole k tiles of 64 rows.
constexpr int kPaddedGroups = 160;
struct GroupRows {
  int n;
  int real[kPaddedGroups + 1], padded[kPaddedGroups + 1];
  // the group of a row; of several that start there the one that has rows
  static __device__ __forceinline__ int find(const int *starts, int n, int row) {
    int lo = 0, hi = n;   // starts[lo] <= row < starts[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= row) lo = mid; else hi = mid;
    }
    return lo;
  }
};
// c(r, f) += sum over k of what the pairs have left out of w[group of r](f, k) and x(r, k).  w [groups][out][in]; features are its lines (`lines`) or
// its columns.  A block owns the rows blockIdx.x, blockIdx.x + gridDim.x, ... and takes the strays in their listed order.
struct GroupStrays { const float *w; long in, out; const float *x; long ldx, run; Measured mw, mx; };
static __global__ void __launch_bounds__(256) group_row_strays_kernel(const GroupStrays g, bool lines, float *c, const Ranges ranges,
                                                                      const __grid_constant__ GroupRows rows) {
  pdl_begin();
  const bool wide = ranges.wide();
  const int nx = g.mx.strays(wide), nw = g.mw.strays(wide);
  if (nx + nw == 0) return;
  const long features = lines ? g.out : g.in;
  for (int e = 0; e < nx; e++) {
    const long at = g.mx.list[e].at, r = at / g.run, k = at - r * g.run;
    if (r % gridDim.x != blockIdx.x) continue;
    const float v = g.mx.list[e].v;
    const float *w = g.w + (long)GroupRows::find(rows.real, rows.n, (int)r) * g.out * g.in;
    for (long f = threadIdx.x; f < features; f += 256) c[r * features + f] += v * (lines ? w[f * g.in + k] : w[k * g.in + f]);
    __syncthreads();   // (another thread may take the same result next)
  }
  __syncthreads();
  const unsigned limit = stray_limit(g.mx.rec->max_bits) - 1u;
  for (int e = 0; e < nw; e++) {
    const long at = g.mw.list[e].at, line = at / g.in, i = at - line * g.in, group = line / g.out, o = line - group * g.out;
    const long f = lines ? o : i, k = lines ? i : o;
    const float v = g.mw.list[e].v;
    for (long r = blockIdx.x + (long)threadIdx.x * gridDim.x; r < rows.real[group + 1]; r += 256l * gridDim.x) {
      if (r < rows.real[group]) continue;
      const float s = g.x[r * g.ldx + k];
      if ((__float_as_uint(s) & 0x7fffffffu) - 1u >= limit) c[r * features + f] += v * s;   // (zeros pass)
    }
    __syncthreads();
  }
}
// gw[group](o, i) += scale * what the pairs have left out of the sums of gz(r, o) x(r, i) over the group's rows.  A block owns the lines blockIdx.x, ... of
// every group's matrix.
static __global__ void __launch_bounds__(256) group_sum_strays_kernel(const float *x, long ldx, long in, const float *gz, long ldg, long out, float *gw, float scale,
                                                                      const Measured mx, const Measured mg, const Ranges ranges,
                                                                      const __grid_constant__ GroupRows rows) {
  pdl_begin();
  const bool wide = ranges.wide();
  const int nx = mx.strays(wide), ng = mg.strays(wide);
  if (nx + ng == 0) return;
  for (int e = 0; e < nx; e++) {
    const long at = mx.list[e].at, r = at / in, i = at - r * in;
    const float v = scale * mx.list[e].v;
    float *c = gw + (long)GroupRows::find(rows.real, rows.n, (int)r) * out * in;
    for (long o = blockIdx.x + (long)threadIdx.x * gridDim.x; o < out; o += 256l * gridDim.x) c[o * in + i] += v * gz[r * ldg + o];
    __syncthreads();
  }
  const unsigned limit = stray_limit(mx.rec->max_bits) - 1u;
  for (int e = 0; e < ng; e++) {
    const long at = mg.list[e].at, r = at / out, o = at - r * out;
    if (o % gridDim.x != blockIdx.x) continue;
    const float v = scale * mg.list[e].v;
    float *c = gw + ((long)GroupRows::find(rows.real, rows.n, (int)r) * out + o) * in;
    for (long i = threadIdx.x; i < in; i += 256) {
      const float s = x[r * ldx + i];
      if ((__float_as_uint(s) & 0x7fffffffu) - 1u >= limit) c[i] += v * s;
    }
    __syncthreads();
  }
}
// Up to three matrices (blockIdx.y) as FP16 pairs, as split_matrix_kernel makes them: weights as they lie, rows (`grouped`) with each group padded by
// zeros to whole k tiles.
struct GroupPairJob : PairJob { int grouped; };
static __global__ void __launch_bounds__(256) split_groups_kernel(const GroupPairJob a, const GroupPairJob b, const GroupPairJob c,
                                                                  const __grid_constant__ GroupRows rows) {
  pdl_begin();
  const GroupPairJob &j = blockIdx.y == 0 ? a : blockIdx.y == 1 ? b : c;
  const SplitForm form(j);
  const int lane = threadIdx.x & 31;
  const long warps = (long)gridDim.x * 8, parts = (j.ldp + 511) / 512, lines = j.grouped ? rows.padded[rows.n] : j.lines;
  for (long w = (long)blockIdx.x * 8 + (threadIdx.x >> 5); w < lines * parts; w += warps) {
    const long l = w / parts, c0 = (w - l * parts) * 512 + lane * 4;
    long run = j.run, from = l;
    if (j.grouped) {
      const int e = GroupRows::find(rows.padded, rows.n, (int)l);
      from = l - rows.padded[e] + rows.real[e];
      if (from >= rows.real[e + 1]) run = 0;   // padding
    }
    const float *s = j.src + from * j.ld;
    float4 v[4];
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const long c = c0 + g * 128;
      if (j.vec && c + 4 <= run) v[g] = __ldg(reinterpret_cast<const float4 *>(s + c));
      else v[g] = make_float4(c < run ? s[c] : 0.f, c + 1 < run ? s[c + 1] : 0.f, c + 2 < run ? s[c + 2] : 0.f, c + 3 < run ? s[c + 3] : 0.f);
    }
    form.store(j, l, c0, v);
  }
}

}  // namespace mm
}  // namespace thc

#endif
