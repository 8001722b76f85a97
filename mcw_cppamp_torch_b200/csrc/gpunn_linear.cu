// nn.FusedLinear and nn.GroupedLinear: rows times a weight, with what follows the product done along with it.
//
//   FusedLinear    z = x w^T + b,  y = act(z) + residual          x [R][I], w [O][I], b [O], residual [R][O]
//   GroupedLinear  the same for the rows of group e with w[e], b[e], no residual: rows sorted by group, counts[e] of them each
//   backward       gz = g act'(z);  dx = gz w,  dw += scale gz^T x,  db += scale sum_rows gz  (the residual's gradient is g)
#include <type_traits>

#include "nn_activation.cuh"
#include "nn_args.h"

namespace thc {

// y = act(z) + residual over rows of `cols` values; y may be z.
template <int ACT>
static __global__ void __launch_bounds__(256) act_rows_kernel(const float *z, float *y, const float *__restrict__ residual, long rows, long cols, long ldr) {
  pdl_begin();
  const long n = rows * cols;
  for (long i = blockIdx.x * 256l + threadIdx.x; i < n; i += gridDim.x * 256l) {
    float v = activation<ACT>(z[i]);
    if (residual) {
      const long r = i / cols;
      v += residual[r * ldr + (i - r * cols)];
    }
    y[i] = v;
  }
}

// gz = g act'(z) for a part of the rows (blockIdx.y), with the sums of 32 columns over them: part[blockIdx.y][cols].  gz or part may be null.
template <int ACT>
static __global__ void __launch_bounds__(256) act_grad_kernel(const float *__restrict__ g, long ldg, const float *__restrict__ z, float *gz, long rows, long cols,
                                                              long per, float *part) {
  pdl_begin();
  __shared__ float sm[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long end = min(rows, (blockIdx.y + 1) * per);
  for (long c0 = blockIdx.x * 32l; c0 < cols; c0 += gridDim.x * 32l) {
    const long c = c0 + tx;
    float s = 0.f;
    if (c < cols)
      for (long r = blockIdx.y * per + ty; r < end; r += 8) {
        float v = g[r * ldg + c];
        if constexpr (ACT != kActNone) {
          v *= activation_slope<ACT>(z[r * cols + c]);
          if (gz) gz[r * cols + c] = v;
        }
        s += v;
      }
    sm[ty][tx] = s;
    __syncthreads();
    if (part && ty == 0 && c < cols) {
      for (int i = 1; i < 8; i++) s += sm[i][tx];
      part[blockIdx.y * cols + c] = s;
    }
    __syncthreads();
  }
}
// out += scale * sum of the parts, in their order
static __global__ void __launch_bounds__(256) fold_columns_kernel(const float *__restrict__ part, int parts, long cols, float *out, float scale) {
  pdl_begin();
  const long c = blockIdx.x * 256l + threadIdx.x;
  if (c >= cols) return;
  float s = 0.f;
  for (int p = 0; p < parts; p++) s += part[p * cols + c];
  out[c] = fmaf(scale, s, out[c]);
}

// One product's operands and results.
struct LinearForward {
  const float *x; long ldx, rows, in, out;
  const float *w, *b;             // b may be null
  const float *residual; long ldr;   // may be null
  float *z, *y;                   // z may be null
  int act;
};
static void linear_forward(const LinearForward &l) {
  if (l.rows <= 0) return;
  float *z = l.z ? l.z : l.y;
  gemm('t', 'n', l.out, l.rows, l.in, 1.f, l.w, l.in, l.x, l.ldx, 0.f, z, l.out, l.b);
  if (l.act == kActNone && !l.residual && z == l.y) return;
  const long n = l.rows * l.out;
  with_activation(l.act, [&](auto a) {
    pdl_launch(act_rows_kernel<decltype(a)::value>, (unsigned)std::min<long>((n + 255) / 256, ctx().sm_count * 16l), 256, 0, z, l.y, l.residual, l.rows, l.out,
               l.ldr);
  });
  check_launch("linear activation");
}
struct LinearBackward {
  const float *x; long ldx, rows, in, out;
  const float *g; long ldg;
  const float *z;                 // null for no activation
  float *gz;                      // room for g act'(z); unused without an activation
  const float *w;
  float *gx, *gw, *gb;            // each may be null
  int act;
  float scale;
};
static void linear_backward(const LinearBackward &l) {
  if (l.rows <= 0) return;
  if (l.act != kActNone || l.gb) {
    const long columns = std::min<long>((l.out + 31) / 32, 1l << 20);
    const long parts = std::max(1l, std::min(std::min((l.rows + 31) / 32, (ctx().sm_count * 8l + columns - 1) / columns), 65535l)), per = (l.rows + parts - 1) / parts;
    float *part = l.gb ? (float *)ws_alloc(sizeof(float) * parts * l.out) : nullptr;
    with_activation(l.act, [&](auto a) {
      pdl_launch(act_grad_kernel<decltype(a)::value>, dim3((unsigned)columns, (unsigned)parts), 256, 0, l.g, l.ldg, l.z, l.gz, l.rows, l.out, per, part);
    });
    check_launch("linear activation gradient");
    if (l.gb) {
      pdl_launch(fold_columns_kernel, ceil_div(l.out, 256), 256, 0, part, (int)parts, l.out, l.gb, l.scale);
      check_launch("linear bias gradient");
    }
  }
  const float *gz = l.act == kActNone ? l.g : l.gz;
  const long ldgz = l.act == kActNone ? l.ldg : l.out;
  if (l.gx) gemm('n', 'n', l.in, l.rows, l.out, 1.f, l.w, l.in, gz, ldgz, 0.f, l.gx, l.in);
  if (l.gw) gemm('n', 't', l.in, l.out, l.rows, l.scale, l.x, l.ldx, gz, ldgz, 1.f, l.gw, l.in);
}

static bool same_shape(const THGPUTensor *t, int nd, const long *size) {
  if (t->nDimension != nd) return false;
  for (int d = 0; d < nd; d++)
    if (t->size[d] != size[d]) return false;
  return true;
}
static void check_act(int act, int argn) { THC_ARG(act >= 0 && act < kActs, argn, "activation must be 0 (none), 1 (relu), 2 (gelu) or 3 (silu)"); }

// What both operators check of a forward call.  `groups`: 0 for a plain layer, whose weight is a matrix.
static void check_forward(THGPUTensor *input, THGPUTensor *weight, THGPUTensor *bias, long groups, int argw) {
  const int nd = groups ? 3 : 2;
  THC_ARG(weight->nDimension == nd && is_contiguous(weight) && (!groups || weight->size[0] == groups), argw,
          groups ? "contiguous weight of one matrix a group expected" : "contiguous matrix expected");
  const long out = weight->size[nd - 2], in = weight->size[nd - 1], bs[2] = {groups, out};
  if (bias) THC_ARG(same_shape(bias, nd - 1, bs + 3 - nd) && is_contiguous(bias), argw + 1, "contiguous bias of one value a result expected");
  if (nelem(input)) THC_ARG(input->nDimension == 2 && input->size[1] == in, 1, "batch of rows of the weight's input size expected");
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
  check_act(activation, 7);
  check_here({input, residual, output, preactivation, weight, bias});
  check_forward(input, weight, bias, 0, 5);
  const long rows = nelem(input) ? input->size[0] : 0, out = weight->size[0], in = weight->size[1], s[2] = {rows, out};
  if (residual) THC_ARG(rows ? same_shape(residual, 2, s) : nelem(residual) == 0, 2, "residual of the output's size expected");
  size_forward(input, residual, output, preactivation, weight, bias, rows, out, 3);
  if (rows == 0) return 0;
  WsScope scope;
  DenseRows x(input);
  LinearForward l = {x.p, x.ld, rows, in, out, data_ptr(weight), bias ? data_ptr(bias) : nullptr, nullptr, 0, preactivation ? data_ptr(preactivation) : nullptr,
                     data_ptr(output), activation};
  if (residual) {
    DenseRows r(residual);
    l.residual = r.p; l.ldr = r.ld;
    linear_forward(l);
  } else {
    linear_forward(l);
  }
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_FusedLinear_backward(THGPUTensor *input, THGPUTensor *gradOutput, THGPUTensor *gradInput, THGPUTensor *preactivation, THGPUTensor *gradPre,
                                         THGPUTensor *weight, THGPUTensor *gradWeight, THGPUTensor *gradBias, int activation, float scale) {
  THC_BEGIN
  check_act(activation, 9);
  check_here({input, gradOutput, gradInput, preactivation, gradPre, weight, gradWeight, gradBias});
  check_backward(input, gradOutput, gradInput, preactivation, gradPre, weight, gradWeight, gradBias, activation, 0, 1);
  const long rows = nelem(input) ? input->size[0] : 0;
  if (rows == 0) return 0;
  WsScope scope;
  DenseRows x(input), g(gradOutput);
  const bool act = activation != kActNone;
  linear_backward({x.p, x.ld, rows, weight->size[1], weight->size[0], g.p, g.ld, act ? data_ptr(preactivation) : nullptr, act ? data_ptr(gradPre) : nullptr,
                   data_ptr(weight), gradInput ? data_ptr(gradInput) : nullptr, gradWeight ? data_ptr(gradWeight) : nullptr,
                   gradBias ? data_ptr(gradBias) : nullptr, activation, scale});
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_GroupedLinear_updateOutput(THGPUTensor *input, const long *counts, int groups, THGPUTensor *output, THGPUTensor *preactivation,
                                               THGPUTensor *weight, THGPUTensor *bias, int activation) {
  THC_BEGIN
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
  long r0 = 0;
  for (int e = 0; e < groups; r0 += counts[e++])
    linear_forward({x.p + r0 * x.ld, x.ld, counts[e], in, out, data_ptr(weight) + e * out * in, bias ? data_ptr(bias) + e * out : nullptr, nullptr, 0,
                    preactivation ? data_ptr(preactivation) + r0 * out : nullptr, data_ptr(output) + r0 * out, activation});
  return 0;
  THC_END(1)
}

THC_API int THGPUNN_GroupedLinear_backward(THGPUTensor *input, const long *counts, int groups, THGPUTensor *gradOutput, THGPUTensor *gradInput,
                                           THGPUTensor *preactivation, THGPUTensor *gradPre, THGPUTensor *weight, THGPUTensor *gradWeight, THGPUTensor *gradBias,
                                           int activation, float scale) {
  THC_BEGIN
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
  long r0 = 0;
  for (int e = 0; e < groups; r0 += counts[e++])
    linear_backward({x.p + r0 * x.ld, x.ld, counts[e], in, out, g.p + r0 * g.ld, g.ld, act ? data_ptr(preactivation) + r0 * out : nullptr,
                     act ? data_ptr(gradPre) + r0 * out : nullptr, data_ptr(weight) + e * out * in, gradInput ? data_ptr(gradInput) + r0 * in : nullptr,
                     gradWeight ? data_ptr(gradWeight) + e * out * in : nullptr, gradBias ? data_ptr(gradBias) + e * out : nullptr, activation, scale});
  return 0;
  THC_END(1)
}
