// The plain 16-bit products that dense_tc.cu makes of the gated product's gradients.
#pragma once

#include "dense.cuh"

namespace b200moe {

// D [m, n] = X W^T in the operands' type; W [n, k] is stored by column (k rows of n), X [m, k] by row or by column.
struct PlainJob {
  const void* x;
  const void* w;
  void* d;
  int32_t* status;
  int64_t m, k, x_stride, w_stride, d_stride;   // strides of stored rows, in elements
  int n;
  DenseType type;      // a 16-bit one
  bool x_by_column;
  bool early;
};
int dense_plain(const PlainJob& j, cudaStream_t st);

}  // namespace b200moe
