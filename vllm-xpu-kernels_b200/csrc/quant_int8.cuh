// A row's scale and codes: scale = max(amax|v|, 1e-10) / 127, q = rint(v / scale), as IEEE fp32 divisions give them.
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

__device__ __noinline__ uint32_t divided_codes(float a, float b, float c, float d, float scale) {
  if (!(scale < INFINITY)) return 0u;
  auto code = [&](float v) { return (uint32_t)(int)rintf(__fdiv_rn(v, scale)) & 0xffu; };
  return code(a) | code(b) << 8 | code(c) << 16 | code(d) << 24;
}

// Codes without a division for each value.  y = v * (1 / scale) is within 127 * 2^-22.4 of the rounded quotient (three roundings
// of 2^-24 each, of at most 127), so both round to the same whole number unless y is that close to a half: then, about once in five thousand
// values, the division is made.  Adding 1.5 * 2^23 rounds y to a whole number, ties to even, in the sum's low bits.
// A scale that is not finite (a row with a NaN or an infinity) gives codes of zero.
struct Int8Scale {
  float scale, inv;
  __device__ __forceinline__ explicit Int8Scale(float amax) {
    scale = __fdiv_rn(max_nan(amax, 1e-10f), 127.f);
    inv = __fdiv_rn(1.0f, scale);
  }
  // 4 * W values to W words
  template <int W, int N>
  __device__ __forceinline__ void codes(const float (&v)[N], uint32_t (&w)[W]) const {
    static_assert(4 * W <= N, "values");
    constexpr float kMagic = 12582912.f;
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float y = __fmul_rn(v[4 * i + k], inv), t = __fadd_rn(y, kMagic);
        far = fmaxf(far, fabsf(__fadd_rn(y, -__fadd_rn(t, -kMagic))));
        b[k] = __float_as_uint(t);
      }
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
    if (far > 0.49995f || !(scale < INFINITY)) {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = divided_codes(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], scale);
    }
  }
};

}  // namespace
}  // namespace b200moe
