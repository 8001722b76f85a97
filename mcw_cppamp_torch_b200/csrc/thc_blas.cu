// BLAS front-ends on raw device pointers (column-major Fortran convention), the layer the
// reference implemented in gputorch/lib/THC/THCBlas.cpp: gemm dispatch :249-288 over four 16x16
// tile kernels :10-246 (three of which ignored the leading dimensions), gemv :291-467, axpy
// :470-483, ger :486-502.  Here gemm maps onto the shared matrix-multiply engines (tcgen05 3xTF32
// by default: the two-SM one, or a warp-level one for small and narrow products), all leading dimensions are honoured and C is not read when beta == 0.
#include "mm_launch.cuh"
#include "nn_linear.h"

namespace thc {

struct ScaleOp { float v; __device__ float operator()(const float *a) const { return a[0] * v; } };

static __global__ void scale_matrix_kernel(float *c, long m, long n, long ldc, float beta) {
  pdl_begin();
  const long t = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= m * n) return;
  const long j = t / m, i = t - j * m;
  c[i + j * ldc] = beta == 0.f ? 0.f : beta * c[i + j * ldc];
}

// out[i + j * ldc] = bias[i]
static __global__ void broadcast_rows_kernel(float *c, long m, long n, long ldc, const float *__restrict__ bias) {
  pdl_begin();
  const long t = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= m * n) return;
  const long j = t / m, i = t - j * m;
  c[i + j * ldc] = bias[i];
}
// Tensor-core path over the matrices as they lie in memory (raw-operand engine): TMA reads either layout of
// either operand, so no pass over the operands precedes the product.
// The problem of a plain product, or with a linear layer's epilogue, whose operands are K-major.
template <bool A_MN, bool B_MN, int PREC, bool FUSED> struct MatrixProblem {
  typedef mm::Problem<mm::RawOperand<A_MN, PREC>, mm::RawOperand<B_MN, PREC>, false, PREC> type;
};
template <int PREC> struct MatrixProblem<false, false, PREC, true> {
  typedef mm::FusedProblem<mm::RawOperand<false, PREC>, mm::RawOperand<false, PREC>, PREC> type;
};
template <class P> static void set_tail(P &p, const mm::LinearEpilogue *tail) {
  if constexpr (P::FUSED) p.tail = *tail;
}
template <bool A_MN, bool B_MN, bool FUSED = false>
static void gemm_raw_t(const float *a, long lda, const float *b, long ldb, long m, long n, long k, const mm::Epilogue &epi, const mm::LinearEpilogue *tail = nullptr) {
  using namespace mm;
  typename MatrixProblem<A_MN, B_MN, kTf32, FUSED>::type p;
  p.epi = epi;
  set_tail(p, tail);
  p.M = m; p.N = n; p.K = k;
  launch_raw(p, [&](auto &q, int bn2) {
    attach_raw_map<kTf32>(q.a, a, m, k, lda, TC_BM);
    attach_raw_map<kTf32>(q.b, b, n, k, ldb, bn2 / 2);
  });
}
// One side of a product: element (r, l) at p[l + r * ld] (along_k) or p[r + l * ld].
struct GemmSide { const float *p; long ld; bool along_k; long rows; };
// Orientation of the 256-row tiles and the epilogue for D(i, j) at c[i + j * ldc]: the first side takes the rows unless it has
// no more than half a tile of them and the other has more.
template <class Side>
static mm::Epilogue gemm_sides(Side &x, Side &y, float alpha, float beta, float *c, long ldc, const float *row_bias, mm::LinearEpilogue *tail = nullptr) {
  if (x.rows <= 128 && y.rows > x.rows) {
    std::swap(x, y);
    if (tail) std::swap(tail->rm, tail->rn);
    mm::Epilogue e{c, row_bias, alpha, beta, 1, ldc, 1};   // rows of the product are columns of c: out[m * ldc + n]
    return e;
  }
  mm::Epilogue e{c, nullptr, alpha, beta, LONG_MAX, 0, ldc};
  e.row_bias = row_bias;
  return e;
}
// BF16 math mode: one K-major BF16 plane per operand, BF16 products.  For results of more than half a tile's rows and more
// than 32 columns; smaller ones stay FP32-accurate.
template <bool FUSED = false>
static void gemm_half(GemmSide x, GemmSide y, long k, float alpha, float beta, float *c, long ldc, const float *row_bias, mm::LinearEpilogue *tail = nullptr) {
  using namespace mm;
  typename MatrixProblem<false, false, kBf16, FUSED>::type p;
  p.epi = gemm_sides(x, y, alpha, beta, c, ldc, row_bias, tail);
  set_tail(p, tail);
  const HalfMatrix hx = make_half_matrix(x.p, x.along_k ? x.ld : 1, x.along_k ? 1 : x.ld, x.rows, k);
  const HalfMatrix hy = make_half_matrix(y.p, y.along_k ? y.ld : 1, y.along_k ? 1 : y.ld, y.rows, k);
  p.M = x.rows; p.N = y.rows; p.K = hx.ld;
  launch_raw(p, [&](auto &q, int bn2) {
    attach_raw_map<kBf16>(q.a, hx.p, x.rows, hx.ld, hx.ld, TC_BM);
    attach_raw_map<kBf16>(q.b, hy.p, y.rows, hy.ld, hy.ld, bn2 / 2);
  });
}
// Copies the sides of products with k that have a pitch or address that TMA cannot take (a hundredth of a product's time at the sizes that come
// here) instead of feeding the products through per-thread copies.
static void pack_sides(GemmSide *const *sides, const long *k, int n) {
  mm::PackJob jobs[3] = {};
  int count = 0;
  for (int i = 0; i < n; i++) {
    GemmSide &s = *sides[i];
    if (mm::raw_matrix_ok(s.p, s.ld)) continue;
    mm::PackJob &j = jobs[count++];
    j = mm::PackJob{s.p, nullptr, s.along_k ? s.rows : k[i], s.along_k ? k[i] : s.rows, s.ld, ((s.along_k ? k[i] : s.rows) + 3) / 4 * 4};
    j.dst = (float *)ws_alloc(sizeof(float) * j.lines * j.dst_ld);
    s.p = j.dst; s.ld = j.dst_ld;
  }
  if (count) mm::launch_pack(jobs[0], jobs[1], jobs[2]);
}
template <bool FUSED = false>
static void gemm_raw(GemmSide x, GemmSide y, long k, float alpha, float beta, float *c, long ldc, const float *row_bias, mm::LinearEpilogue *tail = nullptr) {
  const mm::Epilogue epi = gemm_sides(x, y, alpha, beta, c, ldc, row_bias, tail);
  GemmSide *sides[2] = {&x, &y};
  const long ks[2] = {k, k};
  pack_sides(sides, ks, 2);
  if constexpr (FUSED) { gemm_raw_t<false, false, true>(x.p, x.ld, y.p, y.ld, x.rows, y.rows, k, epi, tail); return; }
  if (!x.along_k && y.along_k) gemm_raw_t<true, false>(x.p, x.ld, y.p, y.ld, x.rows, y.rows, k, epi);
  else if (x.along_k && y.along_k) gemm_raw_t<false, false>(x.p, x.ld, y.p, y.ld, x.rows, y.rows, k, epi);
  else if (!x.along_k) gemm_raw_t<true, true>(x.p, x.ld, y.p, y.ld, x.rows, y.rows, k, epi);
  else gemm_raw_t<false, true>(x.p, x.ld, y.p, y.ld, x.rows, y.rows, k, epi);
}
// The same over FP16 pairs: a pass measures both operands and one splits them, each as it lies in memory.
template <bool A_MN, bool B_MN, bool FUSED = false>
static void gemm_pairs_t(const mm::PairJob &a, const mm::PairJob &b, long m, long n, long k, const mm::Epilogue &epi, const mm::Ranges &ranges,
                         const mm::LinearEpilogue *tail = nullptr) {
  using namespace mm;
  typename MatrixProblem<A_MN, B_MN, kPairs, FUSED>::type p;
  p.epi = epi;
  set_tail(p, tail);
  p.M = m; p.N = n; p.K = k;
  p.range_a = ranges.rec[0]; p.range_b = ranges.rec[1]; p.ranges = ranges;
  launch_raw(p, [&](auto &q, int bn2) {
    attach_raw_map<kPairs>(q.a, a.dst, m, k, a.ldp, TC_BM, a.wide);
    attach_raw_map<kPairs>(q.b, b.dst, n, k, b.ldp, bn2 / 2, b.wide);
  });
}
// An operand as pairs.
struct PairSide : GemmSide {
  mm::Measured m;
  mm::PairJob job;
};
// Measures and splits both operands of a product with k; or of two products, with the first operand in each, whose forms are decided product by product.
// False: there is no room for the pairs, and nothing has been done.
static bool make_pairs(PairSide *const *sides, const long *k, int n) {
  using namespace mm;
  // the copies, with a little for the measures (under a hundredth of them) and the partial sums (blocks of 256 KB, up to
  // five rounds of clusters)
  double need = 96e6;
  for (int i = 0; i < n; i++) {
    const GemmSide &s = *sides[i];
    need += 4.1 * (double)(s.along_k ? s.rows : k[i]) * (double)((s.along_k ? k[i] : s.rows) + 64) * (n > 2 && i == 0 ? 2 : 1);
  }
  if (!ws_reserve((size_t)need)) return false;
  RangeJob measure[3];
  long pieces = 0;
  for (int i = 0; i < n; i++) sides[i]->m = new_measured();
  for (int i = 0; i < n; i++) {
    const GemmSide &s = *sides[i];
    const long lines = s.along_k ? s.rows : k[i], run = s.along_k ? k[i] : s.rows, ldp = (run + 63) / 64 * 64;
    measure[i] = range_job(s.p, lines, run, s.ld, sides[i]->m);
    PairJob &j = sides[i]->job;
    j = PairJob{s.p, ws_alloc(sizeof(float) * lines * ldp), lines, run, s.ld, ldp, ((uintptr_t)s.p & 15) == 0 && s.ld % 4 == 0, {}};
    j.ranges.rec[0] = sides[i]->m.rec;
    j.ranges.rec[1] = sides[i ? 0 : 1]->m.rec;
    if (n > 2 && i == 0) {
      j.wide = (float *)ws_alloc(sizeof(float) * lines * ldp);
      j.other.rec[0] = sides[0]->m.rec;
      j.other.rec[1] = sides[2]->m.rec;
    }
    pieces = std::max(pieces, lines * ((ldp + 511) / 512));
  }
  launch_ranges(measure[0], &measure[1]);
  if (n > 2) launch_ranges(measure[2], nullptr);
  const unsigned blocks = (unsigned)std::min<long>((pieces + 7) / 8, ctx().sm_count * 8l);
  pdl_launch(split_matrix_kernel, dim3(blocks, 2), 256, 0, sides[0]->job, sides[1]->job);
  check_launch("split_matrix");
  if (n > 2) {
    pdl_launch(split_matrix_kernel, dim3(blocks, 1), 256, 0, sides[2]->job, sides[2]->job);
    check_launch("split_matrix");
  }
  return true;
}
template <bool FUSED = false>
static void pairs_product(PairSide x, PairSide y, long k, float alpha, float beta, float *c, long ldc, const float *row_bias, mm::LinearEpilogue *tail = nullptr) {
  using namespace mm;
  const Epilogue epi = gemm_sides(x, y, alpha, beta, c, ldc, row_bias, tail);
  Ranges r;
  r.rec[0] = x.m.rec; r.rec[1] = y.m.rec;
  const GemmSide &xs = x, &ys = y;
  if constexpr (FUSED) {
    tail->a = x.m.rec; tail->b = y.m.rec; tail->ranges = r;
    gemm_pairs_t<false, false, true>(x.job, y.job, xs.rows, ys.rows, k, epi, r, tail);
  } else if (!xs.along_k && ys.along_k) gemm_pairs_t<true, false>(x.job, y.job, xs.rows, ys.rows, k, epi, r);
  else if (xs.along_k && ys.along_k) gemm_pairs_t<false, false>(x.job, y.job, xs.rows, ys.rows, k, epi, r);
  else if (!xs.along_k) gemm_pairs_t<true, true>(x.job, y.job, xs.rows, ys.rows, k, epi, r);
  else gemm_pairs_t<false, true>(x.job, y.job, xs.rows, ys.rows, k, epi, r);
  Epilogue sums = epi;   // (with a linear layer's epilogue: where there are strays the product has left the sums there)
  if (FUSED && tail->z) sums.out = tail->z;
  pdl_launch(matrix_strays_kernel, dim3((unsigned)std::min(ceil_div(ys.rows, 256), ctx().sm_count), 4), 256, 0, StraySide{xs.p, xs.ld, x.job.run, xs.along_k, x.m},
             StraySide{ys.p, ys.ld, y.job.run, ys.along_k, y.m}, xs.rows, ys.rows, sums, r);
  check_launch("matrix_strays");
}
// False: there is no room for the pairs, and nothing has been done.
template <bool FUSED = false>
static bool gemm_pairs(GemmSide x, GemmSide y, long k, float alpha, float beta, float *c, long ldc, const float *row_bias, mm::LinearEpilogue *tail = nullptr) {
  PairSide xp{x, {}, {}}, yp{y, {}, {}};
  PairSide *sides[2] = {&xp, &yp};
  const long ks[2] = {k, k};
  if (!make_pairs(sides, ks, 2)) return false;
  pairs_product<FUSED>(xp, yp, k, alpha, beta, c, ldc, row_bias, tail);
  return true;
}
// Whether pairs finish before TF32, the passes over the operands included.  Their copies are scratch that TF32 does without: bounded.
// Measured on both sides of the line (us, pairs / TF32): 2048^3 78.0 / 75.8, 2304^3 102.5 / 108.0, 2560^3 125 / 148, 1500 x 3001 x 2222 115 / 129, 4096 x 4096
// x 512 88 / 98, 1024 x 4096 x 4096 131 / 167.  Operands that have to stay in FP32 take up to two fifths longer than TF32 does
// (2304^3 142, 1024 x 4096 x 4096 217, 4096^3 731 / 621, 8192^3 5030 / 5004): the measuring pass, a copy, wider tiles.
static bool pairs_are_faster(long m, long n, long k) {
  if (4. * (double)k * (double)(m + n) > 16e9 || std::max(std::max(m, n), k) > 1l << 28) return false;
  const double passes = 14 + 4e-6 * (double)k * (double)(m + n) * (1 / 5.5 + 2 / 5.0);
  return mm::tc2_product_us(m, n, k, mm::kPairs, true) + passes < mm::tc2_product_us(m, n, k, mm::kTf32);
}
// Whether the warp-level engine (mm_small.cuh) finishes before the two-SM one.  The latter, as measured for the same sizes: 11 us to
// start, then the fill and fold of its long pipeline (0.026 per k up to 512) and 2.9 per GFLOP, or the operands' bytes
// at 3.3 TB/s; packing adds a launch and a pass over the operands.
static bool small_is_faster(long m, long n, long k, bool aligned) {
  const double gf = 2e-9 * (double)((m + 63) / 64 * 64) * (double)((n + 63) / 64 * 64) * (double)k, bytes = 4 * (double)k * (double)(m + n);
  double raw = 11 + std::max(0.026 * (double)std::min(k, 512l) + 2.9 * gf, bytes / 3.3e6);
  if (!aligned) raw += 5 + bytes / 2e6;
  return mm::small_product_us(m, n, k, aligned) < raw;
}

// Small and narrow products: operands as they lie, whatever their layout and alignment.
static void gemm_small(const GemmSide &x, const GemmSide &y, long k, float alpha, float beta, float *c, long ldc, const float *row_bias) {
  mm::SmallProblem p = {};
  p.a = mm::small_operand(x.p, x.ld); p.b = mm::small_operand(y.p, y.ld);
  p.M = (int)x.rows; p.N = (int)y.rows; p.K = (int)k;
  p.c = c; p.sm = 1; p.sn = ldc;
  p.alpha = alpha; p.beta = beta;
  p.bias = row_bias; p.bias_m = 1;
  mm::launch_small(p, x.along_k, y.along_k);
}

// FP32 FMA mode
static void gemm_simt(const GemmSide &x, const GemmSide &y, long k, float alpha, float beta, float *c, long ldc) {
  using namespace mm;
  Problem<Operand<LinearMap, LinearMap, 0>, Operand<LinearMap, LinearMap, 0>> p;
  auto side = [&](auto &op, const GemmSide &s) {
    op.base = s.p;
    op.rows = LinearMap{s.rows, s.along_k ? s.ld : 1};
    op.ks = LinearMap{k, s.along_k ? 1 : s.ld};
    op.H = op.W = 0; op.dH = op.dW = 1;
  };
  side(p.a, x); side(p.b, y);
  p.epi = Epilogue{c, nullptr, alpha, beta, LONG_MAX, 0, ldc};
  p.M = x.rows; p.N = y.rows; p.K = k;
  launch_simt(p);
}

void gemm(char transa, char transb, long m, long n, long k, float alpha, const float *a, long lda,
          const float *b, long ldb, float beta, float *c, long ldc, const float *row_bias) {
  const bool ta = transa == 't' || transa == 'T', tb = transb == 't' || transb == 'T';
  if (m <= 0 || n <= 0) return;
  constexpr long kPart = 1l << 30;   // the engines count rows and k in 32 bits
  if (m > kPart || n > kPart || k > kPart) {
    for (long l0 = 0; l0 < std::max(k, 1l); l0 += kPart)
      for (long j0 = 0; j0 < n; j0 += kPart)
        for (long i0 = 0; i0 < m; i0 += kPart)
          gemm(transa, transb, std::min(kPart, m - i0), std::min(kPart, n - j0), std::min(kPart, k - l0), alpha,
               a + (ta ? l0 + i0 * lda : i0 + l0 * lda), lda, b + (tb ? j0 + l0 * ldb : l0 + j0 * ldb), ldb, l0 ? 1.f : beta,
               c + i0 + j0 * ldc, ldc, l0 || !row_bias ? nullptr : row_bias + i0);
    return;
  }
  WsScope ws_scope;
  const int mode = ctx().math_mode;
  if (row_bias && (mode == 1 || k <= 0 || alpha == 0.f)) {   // engines without a bias input: D starts as the bias
    pdl_launch(broadcast_rows_kernel, ceil_div(m * n, 256), 256, 0, c, m, n, ldc, row_bias);
    check_launch("broadcast_rows");
    row_bias = nullptr;
    beta = 1.f;
  }
  if (k <= 0 || alpha == 0.f) {
    if (beta == 1.f) return;
    pdl_launch(scale_matrix_kernel, ceil_div(m * n, 256), 256, 0, c, m, n, ldc, beta);
    check_launch("scale_matrix");
    return;
  }
  // A(i,l): 'n' a[i + l*lda], 't' a[l + i*lda].  B(j,l): 'n' b[l + j*ldb], 't' b[j + l*ldb].
  const GemmSide x{a, lda, ta, m}, y{b, ldb, !tb, n};
  if (mode == 1) { gemm_simt(x, y, k, alpha, beta, c, ldc); return; }
  const bool aligned = mm::raw_matrix_ok(a, lda) && mm::raw_matrix_ok(b, ldb);
  if (mode == 2 && m > 128 && n > 32) gemm_half(x, y, k, alpha, beta, c, ldc, row_bias);
  else if (small_is_faster(m, n, k, aligned)) gemm_small(x, y, k, alpha, beta, c, ldc, row_bias);
  else if (!(mode == 0 && pairs_are_faster(m, n, k) && gemm_pairs(x, y, k, alpha, beta, c, ldc, row_bias)))
    gemm_raw(x, y, k, alpha, beta, c, ldc, row_bias);
}

// y = act(z) + residual over rows of `cols` values; y may be z.  With records of a product over pairs: only where that has left its sums.
template <int ACT>
static __global__ void __launch_bounds__(256) linear_tail_kernel(const float *z, float *y, const float *__restrict__ residual, long rows, long cols, long ldr, bool vec,
                                                                 const mm::LinearEpilogue product) {
  pdl_begin();
  if (product.a && !product.deferred()) return;
  const long stride = gridDim.x * 256l, start = blockIdx.x * 256l + threadIdx.x;
  if (vec) {
    const long per = cols / 4, n = rows * per;
    for (long i = start; i < n; i += stride) {
      float4 v = reinterpret_cast<const float4 *>(z)[i];
      v = make_float4(activation<ACT>(v.x), activation<ACT>(v.y), activation<ACT>(v.z), activation<ACT>(v.w));
      if (residual) {
        const long r = i / per;
        const float4 q = __ldg(reinterpret_cast<const float4 *>(residual + r * ldr) + (i - r * per));
        v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w;
      }
      reinterpret_cast<float4 *>(y)[i] = v;
    }
    return;
  }
  const long n = rows * cols;
  for (long i = start; i < n; i += stride) {
    float v = activation<ACT>(z[i]);
    if (residual) {
      const long r = i / cols;
      v += residual[r * ldr + (i - r * cols)];
    }
    y[i] = v;
  }
}
void linear_tail(const float *z, float *y, long rows, long out, const LinearTail &tail, const mm::LinearEpilogue &product) {
  const bool vec = out % 4 == 0 && tail.ldr % 4 == 0 && (((uintptr_t)z | (uintptr_t)y | (uintptr_t)tail.residual) & 15) == 0;
  const long n = rows * out / (vec ? 4 : 1);
  with_activation(tail.act, [&](auto a) {
    pdl_launch(linear_tail_kernel<decltype(a)::value>, (unsigned)std::min<long>((n + 255) / 256, ctx().sm_count * 16l), 256, 0, z, y, tail.residual, rows, out, tail.ldr,
               vec, product);
  });
  check_launch("linear_tail");
}
void linear_product(const float *x, long ldx, long rows, long in, long out, const float *w, const float *b, float *y, const LinearTail &tail) {
  if (rows <= 0) return;
  WsScope scope;
  const int mode = ctx().math_mode;
  if (mode == 1) {   // the FP32 engine: its result in a pass of its own
    float *z = tail.z ? tail.z : y;
    gemm('t', 'n', out, rows, in, 1.f, w, in, x, ldx, 0.f, z, out, b);
    if (tail.act != kActNone || tail.residual || z != y) linear_tail(z, y, rows, out, tail, {});
    return;
  }
  const bool aligned = mm::raw_matrix_ok(w, in) && mm::raw_matrix_ok(x, ldx);
  const GemmSide ws{w, in, true, out}, xs{x, ldx, true, rows};
  mm::LinearEpilogue e;
  e.act = tail.act; e.residual = tail.residual; e.rm = 1; e.rn = tail.ldr; e.z = tail.z;
  if (mode == 2 && out > 128 && rows > 32) {
    gemm_half<true>(ws, xs, in, 1.f, 0.f, y, out, b, &e);
  } else if (small_is_faster(out, rows, in, aligned)) {
    mm::SmallFused p = {};
    p.a = mm::small_operand(w, in); p.b = mm::small_operand(x, ldx);
    p.M = (int)out; p.N = (int)rows; p.K = (int)in;
    p.c = y; p.sm = 1; p.sn = out;
    p.alpha = 1.f;
    p.bias = b; p.bias_m = 1;
    p.act = e.act; p.residual = e.residual; p.rm = e.rm; p.rn = e.rn; p.z = e.z;
    mm::launch_small(p, true, true);
  } else if (mode == 0 && pairs_are_faster(out, rows, in) && gemm_pairs<true>(ws, xs, in, 1.f, 0.f, y, out, b, &e)) {
    linear_tail(e.z ? e.z : y, y, rows, out, tail, e);
  } else {
    gemm_raw<true>(ws, xs, in, 1.f, 0.f, y, out, b, &e);
  }
}

// gx = gz w and gw += scale * gz^T x: the products gemm() would make of them, with gz split into pairs once where both take pairs, and operands whose
// pitch TMA cannot take copied once.
void linear_gradients(const float *x, long ldx, const float *gz, long ldg, long rows, long in, long out, const float *w, float *gx, float *gw, float scale) {
  WsScope scope;
  if (gw && ctx().math_mode != 1 && few_rows_sums(Groups{&rows, 1, rows}, x, ldx, gz, ldg, in, out, gw, scale)) gw = nullptr;
  const bool gz_ok = mm::raw_matrix_ok(gz, ldg), input_ok = gz_ok && mm::raw_matrix_ok(w, in), weight_ok = gz_ok && mm::raw_matrix_ok(x, ldx);
  const bool engine = ctx().math_mode == 0 && gx && gw && !small_is_faster(in, rows, out, input_ok) && !small_is_faster(in, out, rows, weight_ok);   // for both
  if (engine && pairs_are_faster(in, rows, out) && pairs_are_faster(in, out, rows)) {
    PairSide g{{gz, ldg, true, rows}, {}, {}}, ws{{w, in, false, in}, {}, {}}, xs{{x, ldx, false, in}, {}, {}};
    PairSide *sides[3] = {&g, &ws, &xs};
    const long ks[3] = {out, out, rows};
    if (make_pairs(sides, ks, 3)) {
      pairs_product(ws, g, out, 1.f, 0.f, gx, in, nullptr);
      g.along_k = false; g.rows = out;      // the same lines, summed over
      pairs_product(xs, g, rows, scale, 1.f, gw, in, nullptr);
      return;
    }
  }
  if (engine && !(input_ok && weight_ok) && !pairs_are_faster(in, rows, out) && !pairs_are_faster(in, out, rows)) {
    GemmSide g{gz, ldg, true, rows}, ws{w, in, false, in}, xs{x, ldx, false, in};
    GemmSide *sides[3] = {&g, &ws, &xs};
    const long ks[3] = {out, out, rows};
    pack_sides(sides, ks, 3);
    gemm_raw(ws, g, out, 1.f, 0.f, gx, in, nullptr);
    g.along_k = false; g.rows = out;
    gemm_raw(xs, g, rows, scale, 1.f, gw, in, nullptr);
    return;
  }
  if (gx) gemm('n', 'n', in, rows, out, 1.f, w, in, gz, ldg, 0.f, gx, in);
  if (gw) gemm('n', 't', in, out, rows, scale, x, ldx, gz, ldg, 1.f, gw, in);
}

// y = beta*y + alpha*op(A)*x.  'n': A is m x n column-major, y has m entries: threads own rows
// (coalesced across the column).  't': y has n entries, one warp per column of A.
// block = 32 rows x 32 column slices; the slices' partial sums are folded in slice order (deterministic)
static __global__ void __launch_bounds__(1024) gemv_n_kernel(long m, long n, float alpha, const float *__restrict__ a, long lda,
                                                             const float *__restrict__ x, long incx, float beta, float *y,
                                                             long incy) {
  pdl_begin();
  __shared__ float part[32][33];
  const long i = (long)blockIdx.x * 32 + threadIdx.x;
  float acc = 0.f;
  if (i < m) {
    // eight columns on the way at once, added in their order (gradBias of three layers over 256 rows 21 -> 15 us)
    for (long j0 = threadIdx.y; j0 < n; j0 += 8 * 32) {
      float v[8], w[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const long j = j0 + 32 * k;
        v[k] = j < n ? a[i + j * lda] : 0.f;
        w[k] = j < n ? x[j * incx] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; k++)
        if (j0 + 32 * k < n) acc = fmaf(v[k], w[k], acc);
    }
  }
  part[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y == 0 && i < m) {
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < 32; s++) sum += part[s][threadIdx.x];
    y[i * incy] = (beta == 0.f ? 0.f : beta * y[i * incy]) + alpha * sum;
  }
}
static __global__ void gemv_t_kernel(long m, long n, float alpha, const float *__restrict__ a, long lda,
                                     const float *__restrict__ x, long incx, float beta, float *y, long incy) {
  pdl_begin();
  const long j = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (j >= n) return;
  const int lane = threadIdx.x & 31;
  float acc = 0.f;
  for (long i = lane; i < m; i += 32) acc = fmaf(a[i + j * lda], x[i * incx], acc);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) y[j * incy] = (beta == 0.f ? 0.f : beta * y[j * incy]) + alpha * acc;
}
static __global__ void axpy_kernel(long n, float a, const float *__restrict__ x, long incx, float *y, long incy) {
  pdl_begin();
  const long nthreads = (long)gridDim.x * blockDim.x;
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += nthreads)
    y[i * incy] = __fadd_rn(y[i * incy], __fmul_rn(a, x[i * incx]));
}
static __global__ void ger_kernel(long m, long n, float alpha, const float *__restrict__ x, long incx,
                                  const float *__restrict__ y, long incy, float *a, long lda) {
  pdl_begin();
  const long t = (long)blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= m * n) return;
  const long j = t / m, i = t - j * m;
  a[i + j * lda] += alpha * x[i * incx] * y[j * incy];
}

}  // namespace thc

using namespace thc;

THC_API void THGPUBlas_gemm(char transa, char transb, long m, long n, long k, float alpha, const float *a, long lda,
                            const float *b, long ldb, float beta, float *c, long ldc) {
  THC_BEGIN
  gemm(transa, transb, m, n, k, alpha, a, lda, b, ldb, beta, c, ldc);
  THC_END()
}

THC_API void THGPUBlas_gemv(char trans, long m, long n, float alpha, const float *a, long lda, const float *x,
                            long incx, float beta, float *y, long incy) {
  THC_BEGIN
  if (m <= 0 || n <= 0) return;
  if (trans == 't' || trans == 'T') {
    pdl_launch(gemv_t_kernel, ceil_div(n, 8), 256, 0, m, n, alpha, a, lda, x, incx, beta, y, incy);
    check_launch("gemv_t");
  } else {
    pdl_launch(gemv_n_kernel, ceil_div(m, 32), dim3(32, 32), 0, m, n, alpha, a, lda, x, incx, beta, y, incy);
    check_launch("gemv_n");
  }
  THC_END()
}

THC_API void THGPUBlas_axpy(long n, float a, const float *x, long incx, float *y, long incy) {
  THC_BEGIN
  if (n <= 0) return;
  int blocks = ceil_div(n, 256);
  const int cap = ctx().sm_count * 8;
  if (blocks > cap) blocks = cap;
  pdl_launch(axpy_kernel, blocks, 256, 0, n, a, x, incx, y, incy);
  check_launch("axpy");
  THC_END()
}

THC_API void THGPUBlas_ger(long m, long n, float alpha, const float *x, long incx, const float *y, long incy,
                           float *a, long lda) {
  THC_BEGIN
  if (m <= 0 || n <= 0) return;
  pdl_launch(ger_kernel, ceil_div(m * n, 256), 256, 0, m, n, alpha, x, incx, y, incy, a, lda);
  check_launch("ger");
  THC_END()
}

// ---- stall reporting of the tensor-core kernels ---------------------------------------------------------------
// One warp waits, with the engines' own bounded wait, on an mbarrier that nobody arrives on, and on expiry does
// what an engine CTA does: raises the stall flags and returns.  It faults nothing and waits no longer than
// `limit` SM cycles (plus one polling interval of a few tens of microseconds).
static __global__ void stall_probe_kernel(const mm::StallCtl ctl) {
  pdl_begin();
  __shared__ uint64_t bar;
  __shared__ mm::WaitCtl w;
  if (threadIdx.x == 0) {
    mm::mbar_init(mm::smem_u32(&bar), 1);
    mm::wait_ctl_init(&w, ctl);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (w.abort) return;   // a stall is already on record
  const bool ok = mm::mbar_wait(mm::smem_u32(&bar), 0, &w, mm::kWaitProbe);
  if (!ok && threadIdx.x == 0) mm::stall_raise(ctl, w.abort);
}

THC_API void THGPUSetWaitLimit(long cycles) {
  THC_BEGIN
  THC_CHECK(cycles >= 1024 && cycles <= (1l << 34), "wait limit must lie in [2^10, 2^34] SM cycles");
  ctx().stall_limit = cycles;
  THC_END()
}
THC_API long THGPUGetWaitLimit(void) { THC_BEGIN return (long)ctx().stall_limit; THC_END(-1) }

THC_API int THGPUStallProbe(long limit_cycles) {
  THC_BEGIN
  Context &c = ctx();
  if (limit_cycles < 0) {   // host only: what the host sees after a kernel has raised the flag
    *(volatile int *)c.stall_host = 1;
    return 0;
  }
  THC_CHECK(limit_cycles >= 1024 && limit_cycles <= (1l << 27), "probe limit must lie in [2^10, 2^27] SM cycles");
  mm::StallCtl ctl = stall_ctl();
  ctl.limit = limit_cycles;
  pdl_launch(stall_probe_kernel, 1, 32, 0, ctl);
  check_launch("stall_probe");
  return 0;
  THC_END(1)
}
