// Arguments of the feed-forward operators: which device a tensor lives on, rows of a matrix, checks of results.
#ifndef THC_NN_ARGS_H
#define THC_NN_ARGS_H

#include <initializer_list>

#include "thc_internal.h"

namespace thc {

// The arguments from the first on (null: left out).  A storage remembers the device it was made on (0: none yet).
inline void check_here(std::initializer_list<const THGPUTensor *> args) {
  int argn = 0;
  for (const THGPUTensor *t : args) {
    argn++;
    if (!t || !t->storage) continue;
    const long tag = (long)(intptr_t)t->storage->allocatorContext, here = std::max(device_if_initialised(), 0) + 1;
    if (tag > 0 && tag != here) fail("Invalid argument %d: tensor of device %ld while device %ld is current", argn, tag, here);
  }
}
// A result may not share memory with an operand (null: left out).
inline void check_apart(const THGPUTensor *result, std::initializer_list<const THGPUTensor *> operands, int argn) {
  if (!result) return;
  for (const THGPUTensor *t : operands)
    if (t) THC_ARG(!overlap(result, t), argn, "the result shares memory with an operand");
}
// Result of `nd` sizes, apart from the operands before and after it has them.  A tensor that has them already keeps its memory and has to
// be dense.
inline void size_result(THGPUTensor *t, int nd, const long *size, std::initializer_list<const THGPUTensor *> operands, int argn) {
  check_apart(t, operands, argn);
  bool same = t->nDimension == nd;
  for (int d = 0; same && d < nd; d++) same = t->size[d] == size[d];
  if (!same) resize_nd(t, nd, size, nullptr);
  THC_ARG(is_contiguous(t), argn, "contiguous result expected");
  check_apart(t, operands, argn);
}
// A matrix whose rows are dense, at any distance of at least their length: the tensor itself, or a copy.
struct DenseRows {
  TensorRef t;
  const float *p = nullptr;
  long rows = 0, cols = 0, ld = 0;
  explicit DenseRows(THGPUTensor *m) {
    rows = m->size[0]; cols = m->size[1];
    if ((cols == 1 || m->stride[1] == 1) && (rows == 1 || m->stride[0] >= cols)) {
      THGPUTensor_retain(m);
      t.reset(m);
      ld = rows == 1 ? cols : m->stride[0];
    } else {
      t.reset(tensor_new_contiguous(m));
      ld = cols;
    }
    p = data_ptr(t);
  }
};

}  // namespace thc

#endif
