// A row's scale and codes, from a = max(amax|v|, 1e-10): scale = a / 127, q = rint(v * (127 / a)), both quotients rounded to fp32, the
// product not at all.
#pragma once

#include "common.cuh"

namespace b200moe {
namespace {

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A row that holds a NaN or an infinity gets a scale of NaN, so that every output of the product that it goes into is one.
struct Int8Scale {
  float scale, inv;
  __device__ __forceinline__ explicit Int8Scale(float amax) {
    amax = max_nan(amax, 1e-10f);
    scale = amax < INFINITY ? __fdiv_rn(amax, 127.f) : __uint_as_float(0x7fc00000u);
    inv = __fdiv_rn(127.f, amax);
  }
  // 4 * W values to W words.  Adding 1.5 * 2^23 to a product leaves the nearest whole number, ties to even, in the sum's low bits; in one
  // instruction with the multiplication, nothing else is rounded.
  template <int W, int N>
  __device__ __forceinline__ void codes(const float (&v)[N], uint32_t (&w)[W]) const {
    static_assert(4 * W <= N, "values");
#pragma unroll
    for (int i = 0; i < W; ++i) {
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(__fmaf_rn(v[4 * i + k], inv, 12582912.f));
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
};

}  // namespace
}  // namespace b200moe
