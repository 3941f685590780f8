// What the two kernels of the int8 product and of the gated product share (dense_rows.cu: a few rows; dense_tc.cu: many): the job
// as their launches get it, the numbers of an epilogue, and the entry points of either file.
#pragma once

#include "common.cuh"
#include "gemm_tc_common.cuh"
#include "quant_int8.cuh"

namespace b200moe {

enum DenseType { kDenseI8 = 0, kDenseBf16 = 1, kDenseF16 = 2 };

// D = X W^T for rows X [m, k] and weights W [experts][n, k], both with k dense; int8 operands with a scale for each row of
// either.  gated: D = silu(gate) * up of the products with the first and the second half of W's rows, [m, n / 2].
struct DenseJob {
  const void* x;
  const void* w;
  const float* x_scale;           // int8: [m]
  const float* w_scale;           // int8: [experts, n]
  const void* bias;               // [experts, n] in bias_f16's type, or NULL
  void* d;
  float* pre;                     // gated: the products before the activation [m, n], or NULL
  const int32_t* rows_per_expert; // NULL: one set of weights for all rows
  int32_t* status;
  int64_t m, x_stride, w_stride, d_stride;   // strides of rows in elements (w_stride: of one expert's rows)
  int n, k, experts;
  int rows_hint;                  // rows expected in use, or 0
  int max_ctas;
  DenseType type;
  b200moe_dtype x_dtype;          // int8 weights: I8, or the type of rows that the kernel quantises itself (x_scale NULL; few values)
  bool gated;
  b200moe_dtype d_dtype;          // F32, BF16, F16
  bool bias_f16;
  float clamp;                    // gated: > 0 limits gate from above and up on both sides first
  bool early;                     // launched while the kernel before it still runs
};

int dense_rows(const DenseJob& j, cudaStream_t st);      // dense_rows.cu
// Whether dense_rows takes rows of 16 or 32 bits and int8 weights, every block making the codes for itself: up to so many values
// that takes less time than a kernel of its own.
constexpr int kQuantValues = 16384;
bool dense_rows_quantises(int64_t rows, int k);
int dense_tc(const DenseJob& j, cudaStream_t st);        // dense_tc.cu

// Rows (an expert) up to which the kernel for a few rows takes a call.  By expert, layer calls, that kernel / the one for many, us:
// 8 experts of 4096 x 14336, 4 rows 246 / 257, 15 rows 365 / 265; 128 of 2048 x 768, 1 row 86.8 / 88.6, 8 rows 172 / 147; 8 of
// 2048 x 1408, 4 rows 28.4 / 36.3, 16 rows 39.8 / 36.8.
constexpr int kDenseFewRows = 16, kGroupedFewRows = 5;
inline int dense(const DenseJob& j, cudaStream_t st) {
  const int64_t rows = j.rows_hint > 0 && j.rows_hint < j.m ? j.rows_hint : j.m;
  return (rows + j.experts - 1) / j.experts <= (j.rows_per_expert != nullptr ? kGroupedFewRows : kDenseFewRows) ? dense_rows(j, st) : dense_tc(j, st);
}

namespace {
// silu(gate) * up.  The hardware's exponential and quotient: some 2^-21 of the value.
__device__ __forceinline__ float gated_product(float g, float u, float clamp) {
  if (clamp > 0.f) { g = fminf(g, clamp); u = fminf(fmaxf(u, -clamp), clamp); }
  return g * __fdividef(1.0f, 1.0f + __expf(-g)) * u;
}
__device__ __forceinline__ void store_as(void* d, b200moe_dtype t, int64_t at, float v) {
  if (t == B200MOE_F32) reinterpret_cast<float*>(d)[at] = v;
  else reinterpret_cast<uint16_t*>(d)[at] = bits16(v, t == B200MOE_F16);
}
}  // namespace
}  // namespace b200moe
