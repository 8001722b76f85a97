// nn.FusedLinear and nn.GroupedLinear: rows times a weight, with what follows the product done along with it.
//
//   FusedLinear    z = x w^T + b,  y = act(z) + residual          x [R][I], w [O][I], b [O], residual [R][O]
//   GroupedLinear  the same for the rows of group e with w[e], b[e], no residual: rows sorted by group, counts[e] of them each
//   backward       gz = g act'(z);  dx = gz w,  dw += scale gz^T x,  db += scale sum_rows gz  (the residual's gradient is g)
#include "nn_activation.cuh"
#include "nn_args.h"
#include "nn_linear.h"

namespace thc {

// gz = g act'(z) over [first, end) of the rows, a piece of a group (blockIdx.y), with the sums of 128 columns over them: part[blockIdx.y][cols].  gz or
// part may be null.  12 bytes a value: bound by HBM, or by latency where there are few rows.  A thread has four neighbouring columns (VEC), or one
// of each 32, and every eighth row, four rows on the way.  2048 x 4096, gelu: 25 us, 4 TB/s (100 MB, from cold caches).
struct RowPiece { int group, first, end; };
constexpr int kRowPieces = 256;
struct RowPieces {
  int count;
  long per;          // rows of a piece, where there is one group
  int groups;        // 1: pieces of `per` rows; else `at`
  long rows;
  int live;          // groups among the pieces: the i-th has [first[i], first[i + 1])
  short first[kRowPieces + 1];
  RowPiece at[kRowPieces];
  __device__ __forceinline__ RowPiece piece(int i) const {
    if (groups > 1) return at[i];
    return RowPiece{0, (int)(i * per), (int)min(rows, (i + 1) * per)};
  }
};
template <int ACT, bool VEC>
static __global__ void __launch_bounds__(256) act_grad_kernel(const float *__restrict__ g, long ldg, const float *__restrict__ z, float *gz, long cols, float *part,
                                                              const __grid_constant__ RowPieces pieces) {
  pdl_begin();
  __shared__ float sm[8][128];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const RowPiece p = pieces.piece(blockIdx.y);
  const long c0 = blockIdx.x * 128l;
  auto column = [&](int j) { return c0 + (VEC ? 4 * tx + j : tx + 32 * j); };
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
  for (long r0 = p.first + ty; r0 < p.end; r0 += 8 * U) {
    float gv[U][4], zv[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const long r = r0 + 8 * u;
      auto read = [&](const float *m, long ld, float (&v)[4]) {
        if constexpr (VEC) {
          float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < p.end && column(0) < cols) q = __ldg(reinterpret_cast<const float4 *>(m + r * ld + column(0)));
          v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; j++) v[j] = r < p.end && column(j) < cols ? __ldg(m + r * ld + column(j)) : 0.f;
        }
      };
      read(g, ldg, gv[u]);
      if constexpr (ACT != kActNone) read(z, cols, zv[u]);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const long r = r0 + 8 * u;
      if constexpr (ACT != kActNone) {
#pragma unroll
        for (int j = 0; j < 4; j++) gv[u][j] *= activation_slope<ACT>(zv[u][j]);
        if (r < p.end && gz) {
          if constexpr (VEC) {
            if (column(0) < cols) *reinterpret_cast<float4 *>(gz + r * cols + column(0)) = make_float4(gv[u][0], gv[u][1], gv[u][2], gv[u][3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
              if (column(j) < cols) gz[r * cols + column(j)] = gv[u][j];
          }
        }
      }
      if (r < p.end)
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] += gv[u][j];
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 4; j++) sm[ty][column(j) - c0] = s[j];
  __syncthreads();
  if (threadIdx.x < 128 && c0 + threadIdx.x < cols) {
    float t = sm[0][threadIdx.x];
#pragma unroll
    for (int i = 1; i < 8; i++) t += sm[i][threadIdx.x];
    part[blockIdx.y * cols + c0 + threadIdx.x] = t;
  }
}
// out[group] += scale * sum of the group's parts: eight threads a column, which take every eighth part and meet in the order of their places.  Block
// (a, b) has 32 columns of the b-th group.  192 pieces of 8 groups, 1408 columns: a block for every piece took 12 us, most of them to find nothing.
static __global__ void __launch_bounds__(256) fold_columns_kernel(const float *__restrict__ part, long cols, float *out, float scale,
                                                                  const __grid_constant__ RowPieces pieces) {
  pdl_begin();
  __shared__ float sm[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const bool one = pieces.groups == 1;
  const int first = one ? 0 : pieces.first[blockIdx.y], end = one ? pieces.count : pieces.first[blockIdx.y + 1];
  const long c = blockIdx.x * 32l + tx;
  const int group = one ? 0 : pieces.at[first].group;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int i = first + ty; i < end; i += 8) s += part[i * cols + c];
  }
  sm[ty][tx] = s;
  __syncthreads();
  if (ty || c >= cols) return;
#pragma unroll
  for (int i = 1; i < 8; i++) s += sm[i][tx];
  float *o = out + group * cols + c;
  *o = fmaf(scale, s, *o);
}
static void act_grad(const Groups &groups, const float *g, long ldg, const float *z, float *gz, long cols, int act, float *gb, float scale) {
  const bool vec = cols % 4 == 0 && ldg % 4 == 0 && (((uintptr_t)g | (uintptr_t)z | (uintptr_t)gz) & 15) == 0;
  const long tiles = (cols + 127) / 128;
  // pieces of 32 rows and more, as many as leave sixteen blocks an SM
  const long wanted = std::max(1l, ctx().sm_count * 16l / tiles), per = std::max(32l, (groups.rows + wanted - 1) / wanted);
  auto run = [&](const RowPieces &p) {
    if (!p.count) return;
    float *part = gb ? (float *)ws_alloc(sizeof(float) * p.count * cols) : nullptr;
    const dim3 grid((unsigned)tiles, (unsigned)p.count);
    with_activation(act, [&](auto a) {
      if (vec) pdl_launch(act_grad_kernel<decltype(a)::value, true>, grid, 256, 0, g, ldg, z, gz, cols, part, p);
      else pdl_launch(act_grad_kernel<decltype(a)::value, false>, grid, 256, 0, g, ldg, z, gz, cols, part, p);
    });
    check_launch("activation gradient");
    if (!gb) return;
    pdl_launch(fold_columns_kernel, dim3((unsigned)ceil_div(cols, 32), p.groups == 1 ? 1u : (unsigned)p.live), 256, 0, part, cols, gb, scale, p);
    check_launch("bias gradient");
  };
  RowPieces p;
  p.groups = groups.n; p.rows = groups.rows; p.per = per; p.count = p.live = 0;
  if (groups.n == 1) {
    p.count = (int)((groups.rows + per - 1) / per);
    run(p);
    return;
  }
  // a group's pieces stay together: one whose pieces no longer fit starts the next launch, in larger pieces if it has to
  long r = 0;
  for (int e = 0; e < groups.n; r += groups.counts[e++]) {
    const long n = groups.counts[e], step = std::max(per, (n + kRowPieces - 1) / kRowPieces);
    if (n == 0) continue;
    if (p.count + (n + step - 1) / step > kRowPieces) { run(p); p.count = p.live = 0; }
    p.first[p.live++] = (short)p.count;
    for (long i = 0; i < n; i += step) p.at[p.count++] = RowPiece{e, (int)(r + i), (int)(r + std::min(n, i + step))};
    p.first[p.live] = (short)p.count;
  }
  run(p);
}

static bool same_shape(const THGPUTensor *t, int nd, const long *size) {
  if (t->nDimension != nd) return false;
  for (int d = 0; d < nd; d++)
    if (t->size[d] != size[d]) return false;
  return true;
}
static void check_act(int act, int argn) { THC_ARG(act >= 0 && act < kActs, argn, "activation must be 0 (none), 1 (relu), 2 (gelu) or 3 (silu)"); }

// Rows, inputs and outputs are counted in 32 bits.
static void check_sizes(const THGPUTensor *input, long in, long out) {
  constexpr long kMost = 1l << 30;
  THC_ARG((nelem(input) == 0 || input->size[0] <= kMost) && in <= kMost && out <= kMost, 1, "more than 2^30 rows, inputs or outputs");
}
// What both operators check of a forward call.  `groups`: 0 for a plain layer, whose weight is a matrix.
static void check_forward(THGPUTensor *input, THGPUTensor *weight, THGPUTensor *bias, long groups, int argw) {
  const int nd = groups ? 3 : 2;
  THC_ARG(weight->nDimension == nd && is_contiguous(weight) && (!groups || weight->size[0] == groups), argw,
          groups ? "contiguous weight of one matrix a group expected" : "contiguous matrix expected");
  const long out = weight->size[nd - 2], in = weight->size[nd - 1], bs[2] = {groups, out};
  if (bias) THC_ARG(same_shape(bias, nd - 1, bs + 3 - nd) && is_contiguous(bias), argw + 1, "contiguous bias of one value a result expected");
  if (nelem(input)) THC_ARG(input->nDimension == 2 && input->size[1] == in, 1, "batch of rows of the weight's input size expected");
  check_sizes(input, in, out);
}
// Sizes the results of a forward call and holds them apart from its operands.
static void size_forward(THGPUTensor *input, THGPUTensor *residual, THGPUTensor *output, THGPUTensor *preactivation, THGPUTensor *weight, THGPUTensor *bias, long rows,
                         long out, int argo) {
  const long s[2] = {rows, out};
  size_result(output, 2, s, {input, residual, weight, bias, preactivation}, argo);
  if (preactivation) size_result(preactivation, 2, s, {input, residual, weight, bias, output}, argo + 1);
}

// What both operators check of a backward call, and the sizing of its results.
static void check_backward(THGPUTensor *input, THGPUTensor *gradOutput, THGPUTensor *gradInput, THGPUTensor *preactivation, THGPUTensor *gradPre, THGPUTensor *weight,
                           THGPUTensor *gradWeight, THGPUTensor *gradBias, int act, long groups, int first) {
  const int nd = groups ? 3 : 2;
  THC_ARG(weight->nDimension == nd && is_contiguous(weight) && (!groups || weight->size[0] == groups), first + 5,
          groups ? "contiguous weight of one matrix a group expected" : "contiguous matrix expected");
  const long out = weight->size[nd - 2], in = weight->size[nd - 1], rows = nelem(input) ? input->size[0] : 0, bs[2] = {groups, out}, s[2] = {rows, out};
  if (rows) THC_ARG(input->nDimension == 2 && input->size[1] == in, 1, "batch of rows of the weight's input size expected");
  check_sizes(input, in, out);
  THC_ARG(rows ? same_shape(gradOutput, 2, s) : nelem(gradOutput) == 0, first + 1, "gradOutput has the wrong size");
  if (gradWeight) THC_ARG(same_shape(gradWeight, nd, weight->size) && is_contiguous(gradWeight), first + 6, "contiguous gradWeight of the weight's size expected");
  if (gradBias) THC_ARG(same_shape(gradBias, nd - 1, bs + 3 - nd) && is_contiguous(gradBias), first + 7, "contiguous gradBias of one value a result expected");
  if (act != kActNone && rows) {
    THC_ARG(preactivation && same_shape(preactivation, 2, s) && is_contiguous(preactivation), first + 3, "what the forward pass kept of this input expected");
    THC_ARG(gradPre, first + 4, "room for the preactivation's gradient expected");
    size_result(gradPre, 2, s, {input, gradOutput, preactivation, weight, gradInput, gradWeight, gradBias}, first + 4);
  }
  const long gs[2] = {rows, in};
  if (gradInput) size_result(gradInput, 2, gs, {input, gradOutput, preactivation, gradPre, weight, gradWeight, gradBias}, first + 2);
  check_apart(gradWeight, {input, gradOutput, preactivation, weight, gradBias}, first + 6);
  check_apart(gradBias, {input, gradOutput, preactivation, weight}, first + 7);
}

// Sum of the counts, or a refusal.
static long check_counts(const long *counts, int groups, long rows, int argn) {
  THC_ARG(groups > 0 && counts, argn, "a count of rows for each group expected");
  long sum = 0;
  for (int e = 0; e < groups; e++) {
    THC_ARG(counts[e] >= 0 && counts[e] <= rows - sum, argn, "counts must not be negative and come to the rows of the input");
    sum += counts[e];
  }
  THC_ARG(sum == rows, argn, "counts must come to the rows of the input");
  return sum;
}

}  // namespace thc

using namespace thc;

THC_API int THGPUNN_FusedLinear_updateOutput(THGPUTensor *input, THGPUTensor *residual, THGPUTensor *output, THGPUTensor *preactivation, THGPUTensor *weight,
                                             THGPUTensor *bias, int activation) {
  THC_BEGIN
  THC_ARG(input && output && weight, 1, "tensors expected");
  check_act(activation, 7);
  check_here({input, residual, output, preactivation, weight, bias});
  check_forward(input, weight, bias, 0, 5);
  const long rows = nelem(input) ? input->size[0] : 0, out = weight->size[0], in = weight->size[1], s[2] = {rows, out};
  if (residual) THC_ARG(rows ? same_shape(residual, 2, s) : nelem(residual) == 0, 2, "residual of the output's size expected");
  size_forward(input, residual, output, preactivation, weight, bias, rows, out, 3);
  if (rows == 0) return 0;
  WsScope scope;
  DenseRows x(input);
  LinearTail tail;
  tail.act = activation;
  tail.z = preactivation ? data_ptr(preactivation) : nullptr;
  if (residual) {
    DenseRows r(residual);
    tail.residual = r.p; tail.ldr = r.ld;
    linear_product(x.p, x.ld, rows, in, out, data_ptr(weight), bias ? data_ptr(bias) : nullptr, data_ptr(output), tail);
  } else {
    linear_product(x.p, x.ld, rows, in, out, data_ptr(weight), bias ? data_ptr(bias) : nullptr, data_ptr(output), tail);
  }
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_FusedLinear_backward(THGPUTensor *input, THGPUTensor *gradOutput, THGPUTensor *gradInput, THGPUTensor *preactivation, THGPUTensor *gradPre,
                                         THGPUTensor *weight, THGPUTensor *gradWeight, THGPUTensor *gradBias, int activation, float scale) {
  THC_BEGIN
  THC_ARG(input && gradOutput && weight, 1, "tensors expected");
  check_act(activation, 9);
  check_here({input, gradOutput, gradInput, preactivation, gradPre, weight, gradWeight, gradBias});
  check_backward(input, gradOutput, gradInput, preactivation, gradPre, weight, gradWeight, gradBias, activation, 0, 1);
  const long rows = nelem(input) ? input->size[0] : 0;
  if (rows == 0) return 0;
  WsScope scope;
  DenseRows x(input), g(gradOutput);
  const bool act = activation != kActNone;
  const long out = weight->size[0], in = weight->size[1];
  const float *gz = act ? data_ptr(gradPre) : g.p;
  const long ldgz = act ? out : g.ld;
  if (act || gradBias)
    act_grad(Groups{&rows, 1, rows}, g.p, g.ld, act ? data_ptr(preactivation) : nullptr, act ? data_ptr(gradPre) : nullptr, out, activation,
             gradBias ? data_ptr(gradBias) : nullptr, scale);
  if (gradInput || gradWeight)
    linear_gradients(x.p, x.ld, gz, ldgz, rows, in, out, data_ptr(weight), gradInput ? data_ptr(gradInput) : nullptr, gradWeight ? data_ptr(gradWeight) : nullptr, scale);
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_GroupedLinear_updateOutput(THGPUTensor *input, const long *counts, int groups, THGPUTensor *output, THGPUTensor *preactivation,
                                               THGPUTensor *weight, THGPUTensor *bias, int activation) {
  THC_BEGIN
  THC_ARG(input && output && weight, 1, "tensors expected");
  check_act(activation, 8);
  const long rows = nelem(input) ? input->size[0] : 0;
  check_counts(counts, groups, rows, 2);
  check_here({input, nullptr, nullptr, output, preactivation, weight, bias});
  check_forward(input, weight, bias, groups, 6);
  const long out = weight->size[1], in = weight->size[2];
  size_forward(input, nullptr, output, preactivation, weight, bias, rows, out, 4);
  if (rows == 0) return 0;
  WsScope scope;
  DenseRows x(input);
  group_forward(Groups{counts, groups, rows}, x.p, x.ld, in, out, data_ptr(weight), bias ? data_ptr(bias) : nullptr, data_ptr(output), activation,
                preactivation ? data_ptr(preactivation) : nullptr);
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_GroupedLinear_backward(THGPUTensor *input, const long *counts, int groups, THGPUTensor *gradOutput, THGPUTensor *gradInput,
                                           THGPUTensor *preactivation, THGPUTensor *gradPre, THGPUTensor *weight, THGPUTensor *gradWeight, THGPUTensor *gradBias,
                                           int activation, float scale) {
  THC_BEGIN
  THC_ARG(input && gradOutput && weight, 1, "tensors expected");
  check_act(activation, 11);
  const long rows = nelem(input) ? input->size[0] : 0;
  check_counts(counts, groups, rows, 2);
  check_here({input, nullptr, nullptr, gradOutput, gradInput, preactivation, gradPre, weight, gradWeight, gradBias});
  check_backward(input, gradOutput, gradInput, preactivation, gradPre, weight, gradWeight, gradBias, activation, groups, 3);
  if (rows == 0) return 0;
  WsScope scope;
  DenseRows x(input), g(gradOutput);
  const bool act = activation != kActNone;
  const long out = weight->size[1], in = weight->size[2];
  const Groups gr{counts, groups, rows};
  const float *gz = act ? data_ptr(gradPre) : g.p;
  const long ldgz = act ? out : g.ld;
  if (act || gradBias)
    act_grad(gr, g.p, g.ld, act ? data_ptr(preactivation) : nullptr, act ? data_ptr(gradPre) : nullptr, out, activation, gradBias ? data_ptr(gradBias) : nullptr, scale);
  if (gradInput || gradWeight)
    group_backward(gr, x.p, x.ld, gz, ldgz, in, out, data_ptr(weight), gradInput ? data_ptr(gradInput) : nullptr, gradWeight ? data_ptr(gradWeight) : nullptr, scale);
  return 0;
  THC_END(1)
}
