// A row's scale and codes, from a = max(amax|v|, 1e-10): scale = a / 127, rounded to fp32; q = 127 v / a as the nearest whole number, ties
// to even.
//
// Rows of 16-bit values (the largest of them no less than 1e-10) get that q exactly.  Half of the row's largest value is a tie, 63.5, and common: some three of 2048 bfloat16
// values, and two roundings of a quotient leave it to chance which way they go, which the codes of a layer's second GEMM, whose rows are quantised
// again, multiply (0.9 % of the result where 16 bits cost 0.17 %).  So the product with 127 / a is not rounded, and 127 / a is rounded up:
//   * a tie k + 1/2 of 254 v = (2 k + 1) a needs a 127 among its factors.  Is 2 k + 1 = 127, the tie goes up to 64, which is even, as it does
//     with the factor a little too large.  Is it the mantissa of a, that is 254 (8 bits): 127 / a is a power of two, and exact.
//   * what is not a tie is at least 1 / 512 of v's power of two below the row's largest away from one (8 bits; 1 / 4096 with 11), and the
//     product 127 * 2^-23 of it at the most.
// Of 11 bits (float16), eight mantissas of a are multiples of 127.  Its 127 / a comes in two parts, the first of 13 bits, so that
// its product with a value is exact and the sum of both products is a tie where 127 v / a is one.
// Rows of 32-bit values: within 127 * 2^-23 of a step.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace b200moe {

// Rows up to which the int8 GEMMs and their quantiser launch early.  (More than other kernels of a layer: their blocks stay on the SMs, so none that
// waits takes the place of one that works.  Eager layer calls, 128 experts of 2048 x 768, 12000 rows 177 / 170 us, 16384 rows 198 / 190,
// 65536 rows no difference that clocks leave to be seen.)
constexpr int64_t kEarlyStayingRows = 32768;

namespace {

// The largest of a warp's values, in every lane.
__device__ __forceinline__ float warp_largest(float m) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
  return m;
}

// A row that holds a NaN or an infinity gets a scale of NaN, so that every output of the product that it goes into is one.
// T: the type of the row's values.
template <typename T>
struct Int8Scale {
  static constexpr bool kTwo = std::is_same<T, __half>::value;
  float scale, inv, rest;
  Int8Scale() = default;
  __device__ __forceinline__ explicit Int8Scale(float amax) {
    amax = max_nan(amax, 1e-10f);
    scale = amax < INFINITY ? __fdiv_rn(amax, 127.f) : __uint_as_float(0x7fc00000u);
    inv = __fdiv_ru(127.f, amax);
    if (kTwo) {
      inv = __uint_as_float(__float_as_uint(inv) & 0xfffff800u);
      rest = __fdiv_rn(__fmaf_rn(-inv, amax, 127.f), amax);
    }
  }
  // 4 * W values to W words.  Adding 1.5 * 2^23 leaves the nearest whole number, ties to even, in the sum's low bits; in one
  // instruction with the multiplication, nothing else is rounded.
  template <int W, int N>
  __device__ __forceinline__ void codes(const float (&v)[N], uint32_t (&w)[W]) const {
    static_assert(4 * W <= N, "values");
#pragma unroll
    for (int i = 0; i < W; ++i) {
      uint32_t b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float x = v[4 * i + k];
        b[k] = __float_as_uint(kTwo ? __fadd_rn(__fmaf_rn(x, inv, __fmul_rn(x, rest)), 12582912.f) : __fmaf_rn(x, inv, 12582912.f));
      }
      w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
};

// The values of 16 bytes.  (16-bit types two at a time: a conversion of a bfloat16 by itself is an instruction of a slow unit.)
__device__ __forceinline__ void unpack(const vec16& a, float (&v)[4], float) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a.w[i]);
}
__device__ __forceinline__ void unpack(const vec16& a, float (&v)[8], __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(a.w[i] << 16);
    v[2 * i + 1] = __uint_as_float(a.w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const vec16& a, float (&v)[8], __half) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a.w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
// The largest magnitude of 16 bytes and `most`, which begins as zero bits: two 16-bit values, or a float.
__device__ __forceinline__ uint32_t largest(const vec16& a, uint32_t most, float) {
  float m = __uint_as_float(most);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max_nan(m, fabsf(__uint_as_float(a.w[i])));
  return __float_as_uint(m);
}
template <typename P>
__device__ __forceinline__ uint32_t largest_pair(const vec16& a, uint32_t most) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = a.w[i] & 0x7fff7fffu;
    const P m = __hmax2_nan(*reinterpret_cast<const P*>(&most), *reinterpret_cast<const P*>(&x));
    most = *reinterpret_cast<const uint32_t*>(&m);
  }
  return most;
}
__device__ __forceinline__ uint32_t largest(const vec16& a, uint32_t most, __nv_bfloat16) { return largest_pair<__nv_bfloat162>(a, most); }
__device__ __forceinline__ uint32_t largest(const vec16& a, uint32_t most, __half) { return largest_pair<__half2>(a, most); }
__device__ __forceinline__ float largest_of(uint32_t most, float) { return __uint_as_float(most); }
template <typename T>
__device__ __forceinline__ float largest_of(uint32_t most, T) {
  const T* m = reinterpret_cast<const T*>(&most);
  return max_nan(to_f32<T>(m[0]), to_f32<T>(m[1]));
}

}  // namespace
}  // namespace b200moe
