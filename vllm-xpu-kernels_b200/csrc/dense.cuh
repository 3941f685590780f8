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
// that takes less time than a kernel of its own (1 x 4096 x 4096 5.7 us, 7.2 with two kernels; 4 x 4096 x 4096 6.6 and 7.7; 1 x 4096 x
// 14336 13.2 and 13.7; 8 x 4096 x 4096 9.8 and 7.5).
constexpr int kQuantValues = 16384;
bool dense_rows_quantises(int64_t rows, int k);
int dense_tc(const DenseJob& j, cudaStream_t st);        // dense_tc.cu

// Which kernel takes a call; that for a few rows / that for many, us.  By expert: with two rows of an expert, on average, or fewer the first one; with
// up to ten where the weights of all are few, so that what a call costs besides counts.  Layer calls: 128 experts of 2048 x 768, 1 row 85 / 81,
// 4 rows 119 / 115, 10 rows 135 / 119; 8 of 4096 x 14336, 1 row 182 / 188, 3 rows 235 / 230, 10 rows 278 / 238; 8 of 2048 x 1408 (46 and 23 MB),
// 4 rows 25 / 32, 10 rows 27 / 30, 16 rows 32 / 29.  (One row an expert on average goes either way: what the first loses with many small experts, 4 us of 81,
// is less than it wins with a few large ones, 6 of 188, and the rule does not tell them apart.)
// One set: up to eight rows, and up to sixteen where the SMs have few tiles of weight rows each: then the tokens take as much of L2's
// time as the weights.  16 x 4096 x 4096 5.9 / 7.5, 16 x 4096 x 14336 14.3 / 14.0, 12 x 7168 x 2048 gated 13.4 / 13.6, 16 x 8192 x 4096 10.2 / 9.9,
// 9 x 14336 x 4096 15.8 / 13.6.
constexpr int kDenseFewRows = 16, kGroupedFewRows = 10;
constexpr int64_t kFewBytes = 64 << 20;
inline int dense(const DenseJob& j, cudaStream_t st) {
  const int64_t rows = j.rows_hint > 0 && j.rows_hint < j.m ? j.rows_hint : j.m, mean = (rows + j.experts - 1) / j.experts;
  const bool few = j.rows_per_expert != nullptr
                       ? mean <= 2 || (mean <= kGroupedFewRows && std::min<int64_t>(j.experts, rows) * j.n * j.k <= kFewBytes)
                       : mean <= 8 || (mean <= kDenseFewRows && j.n <= 64 * sm_count());
  return few ? dense_rows(j, st) : dense_tc(j, st);
}

namespace {
// silu(gate) * up.  A limit keeps a NaN: all that marks an int8 row that is not finite is its scale, and so its products.
__device__ __forceinline__ float gated_product(float g, float u, float clamp) {
  if (clamp > 0.f) { g = min_nan(g, clamp); u = clamp_nan(u, clamp); }
  return g * fast_sigmoid(g) * u;
}
__device__ __forceinline__ void store_as(void* d, b200moe_dtype t, int64_t at, float v) {
  if (t == B200MOE_F32) reinterpret_cast<float*>(d)[at] = v;
  else reinterpret_cast<uint16_t*>(d)[at] = bits16(v, t == B200MOE_F16);
}
}  // namespace
}  // namespace b200moe
