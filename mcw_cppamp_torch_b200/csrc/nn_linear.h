// Products of nn.FusedLinear and nn.GroupedLinear: declared here, made by thc_blas.cu (plain layers) and thc_groups.cu (groups).
#ifndef THC_NN_LINEAR_H
#define THC_NN_LINEAR_H

#include <vector>

#include "thc_internal.h"

namespace thc {

// What follows a linear layer's product, for results laid out [rows][out].
struct LinearTail {
  int act = 0;                       // kActNone ...
  const float *residual = nullptr;   // row r at residual + r * ldr; may be null
  long ldr = 0;
  float *z = nullptr;                // receives the sum that the activation is taken of; may be null
};
// y = act(z) + residual with z = x w^T + b: x [rows][in] at pitch ldx, w [out][in], b may be null
void linear_product(const float *x, long ldx, long rows, long in, long out, const float *w, const float *b, float *y, const LinearTail &tail);

// gx = gz w, unless null, and gw += scale * gz^T x, unless null: gz [rows][out] at pitch ldg
void linear_gradients(const float *x, long ldx, const float *gz, long ldg, long rows, long in, long out, const float *w, float *gx, float *gw, float scale);
namespace mm { struct LinearEpilogue; }
// y = act(z) + residual in a pass of its own; with the records of a product over pairs, only where that has left its sums in z
void linear_tail(const float *z, float *y, long rows, long out, const LinearTail &tail, const mm::LinearEpilogue &product);

// Rows of group e: the counts[e] from the sum of the counts before it on.
struct Groups {
  const long *counts;
  int n;
  long rows;
};
// For the rows of each group e: y = act(z), z = x w[e]^T + b[e]
void group_forward(const Groups &g, const float *x, long ldx, long in, long out, const float *w, const float *b, float *y, int act, float *z);
// gx = gz w[e], unless null, and gw[e] += scale * gz^T x over the group's rows, unless null
void group_backward(const Groups &g, const float *x, long ldx, const float *gz, long ldg, long in, long out, const float *w, float *gx, float *gw, float scale);
// gw[e] += scale * gz^T x in FP32 where no group has more than a handful of rows; false: some has, and nothing has been done
bool few_rows_sums(const Groups &g, const float *x, long ldx, const float *gz, long ldg, long in, long out, float *gw, float scale);

}  // namespace thc

#endif
