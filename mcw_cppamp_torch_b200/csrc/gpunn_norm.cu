// nn.LayerNorm: rows normalised to mean zero and variance one, times a weight plus a bias.
//
//   mean = sum x / D,  var = sum (x - mean)^2 / D,  inv = 1 / sqrt(var + eps),  u = (x - mean) inv,  y = u w + b
//   dx = inv (g w - mean(g w) - u mean(g w u)),  dw += scale sum_rows g u,  db += scale sum_rows g
//
// The least traffic is 8 bytes a value forward and 12 backward: everything here is bound by HBM.
// The variance is taken around the mean, not as a difference of two sums: rows whose mean is large against their spread keep their bits.
// With s1 = sum (x - m) left over from the rounding of m, mean = m + s1 / D and var = sum (x - m)^2 / D - (s1 / D)^2.
#include "nn_args.h"

namespace thc {

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
// gw += scale * sum of part[.][0], gb += scale * sum of part[.][1], in their order
static __global__ void __launch_bounds__(256) norm_fold_kernel(const float *__restrict__ part, int parts, long D, float *gw, float *gb, float scale) {
  pdl_begin();
  const long t = blockIdx.x * 256l + threadIdx.x;
  if (t >= 2 * D) return;
  float s = 0.f;
  for (int p = 0; p < parts; p++) s += part[p * 2l * D + t];
  float *o = t < D ? gw + t : gb + (t - D);
  *o = fmaf(scale, s, *o);
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
  const float *w = weight ? data_ptr(weight) : nullptr;
  if (gradInput) {
    pdl_launch(norm_rows_grad_kernel, (unsigned)std::min(rows, ctx().sm_count * 64l), 256, 0, data_ptr(x), data_ptr(g), data_ptr(gradInput), w, data_ptr(mean),
               data_ptr(invStd), rows, size);
    check_launch("LayerNorm_updateGradInput");
  }
  if (gradWeight) {
    const long columns = std::min<long>((size + 31) / 32, 1l << 20);
    const long parts = std::max(1l, std::min(std::min((rows + 31) / 32, (ctx().sm_count * 8l + columns - 1) / columns), 65535l)), per = (rows + parts - 1) / parts;
    float *part = (float *)ws_alloc(sizeof(float) * 2 * size * parts);
    pdl_launch(norm_columns_kernel, dim3((unsigned)columns, (unsigned)parts), 256, 0, data_ptr(x), data_ptr(g), data_ptr(mean), data_ptr(invStd), rows, size, per,
               part);
    check_launch("LayerNorm_accGradParameters");
    pdl_launch(norm_fold_kernel, ceil_div(2 * size, 256), 256, 0, part, (int)parts, size, data_ptr(gradWeight), data_ptr(gradBias), scale);
    check_launch("LayerNorm_accGradParameters");
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
  pdl_launch(norm_rows_kernel, (unsigned)std::min(rows, ctx().sm_count * 64l), 256, 0, data_ptr(x), data_ptr(output), weight ? data_ptr(weight) : nullptr,
             bias ? data_ptr(bias) : nullptr, mean ? data_ptr(mean) : nullptr, mean ? data_ptr(invStd) : nullptr, rows, size, (float)eps);
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
