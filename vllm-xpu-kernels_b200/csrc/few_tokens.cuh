// What the kernels of the layer for a few tokens share.
#pragma once

#include "common.cuh"

namespace b200moe {
namespace {

constexpr int kFewMaxTopk = 32, kFewMaxExperts = 1024;

// Where the scales of a 4-bit matrix are, in bytes: as they are stored, rows [E][n] one behind the other, or laid out by step, in
// words of four bytes [E][words][n] (b200moe_few_tokens_scale_words).  A step is 256 values.
struct FewScales {
  int row, bytes;        // from one row's to the next row's, and of a row (by step: of all its words)
  int step;              // of a row and step
  int next;              // from four of a row's bytes to the next four
};

struct FewMatrix {
  const void* w;
  const void* scale;
  const void* bias;      // [E, n] in the activation type, or NULL
  int format, group;     // b200moe_weight_format; int4: values per scale
  int n, k;
  FewScales scales;      // 4-bit weights
};

// Division by a number that the host knows: a quotient that is at most one too small, and put right.  (The device's own
// takes some 20 instructions, and these kernels' way to their first loads is code that runs once.)
struct FewDiv {
  uint32_t d, m;
  FewDiv() = default;
  __host__ __device__ explicit FewDiv(uint32_t d) : d(d), m(0xffffffffu / d) {}
};
__device__ __forceinline__ int operator/(uint32_t n, const FewDiv& by) {
  const uint32_t q = __umulhi(n, by.m);
  return (int)(n - q * by.d >= by.d ? q + 1 : q);
}
__device__ __forceinline__ int operator/(int n, const FewDiv& by) { return (uint32_t)n / by; }
// The same of small numbers (quotients and remainders below 2^20).
__device__ __forceinline__ int small_div(int n, int d) { return (int)__fdividef((float)n + 0.5f, (float)d); }

struct FewParams {
  const void* x;               // [tokens, hidden]
  const void* ids;             // [tokens, topk]
  const float* weights;        // [tokens, topk]
  const int32_t* expert_map;   // [id_limit], or NULL
  void* out;                   // [tokens, hidden]
  float* h;                    // [tokens * topk, inter]
  int tokens, hidden, inter, topk, experts, id_limit;
  int act;
  float alpha, limit, clamp;
  bool ids64;
  FewDiv by_topk;
  FewMatrix w13, w2;
};

// Words of four bytes that hold a row's scales of a 4-bit matrix laid out by step, in the order of k: one e8m0 byte per 32 values,
// or one 16-bit scale per group (per 128 values where groups are longer), as many as whole steps of 128 values take.
__host__ __device__ __forceinline__ int few_scale_words(int format, int group, int k) {
  const int steps = (k + 127) / 128;
  return format == B200MOE_W_MXFP4_NK || group == 64 ? steps : group == 32 ? 2 * steps : (steps + 1) / 2;
}
inline FewScales few_scales(int format, int group, int n, int k, bool by_step) {
  const int values = format == B200MOE_W_MXFP4_NK ? 32 : group, size = format == B200MOE_W_MXFP4_NK ? 1 : 2;
  if (format != B200MOE_W_MXFP4_NK && format != B200MOE_W_INT4_NK) return {};
  if (!by_step) return {k / values * size, k / values * size, 256 / values * size, 4};
  return {4, 4 * few_scale_words(format, group, k), 256 / (values < 128 ? values : 128) * size, 4 * n};
}

// The slot's expert among the local ones, -1 if it has none here.
__device__ __forceinline__ int local_expert(const FewParams& p, int slot) {
  const int64_t id = p.ids64 ? reinterpret_cast<const int64_t*>(p.ids)[slot] : (int64_t)reinterpret_cast<const int32_t*>(p.ids)[slot];
  if (id < 0 || id >= p.id_limit) return -1;
  const int e = p.expert_map ? p.expert_map[id] : (int)id;
  return e >= 0 && e < p.experts ? e : -1;
}

// Minimum and maximum that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float clamp_nan(float v, float limit) { return max_nan(min_nan(v, limit), -limit); }

// The gated activation in fp32, unrounded.
__device__ __forceinline__ float gated(int act, float alpha, float limit, float clamp, float g, float u) {
  if (clamp > 0.f) {
    g = min_nan(g, clamp);
    u = clamp_nan(u, clamp);
  }
  switch (act) {
    case B200MOE_ACT_SILU: return g / (1.0f + expf(-g)) * u;
    case B200MOE_ACT_GELU: return 0.5f * g * (1.0f + erff(g * 0.70710678118654752440f)) * u;
    case B200MOE_ACT_GELU_TANH:
      return 0.5f * g * (1.0f + tanhf(0.79788456080286535588f * (g + 0.044715f * (g * g * g)))) * u;
    case B200MOE_ACT_SWIGLUOAI:
      g = min_nan(g, limit);
      u = clamp_nan(u, limit);
      return (u + 1.0f) * (g / (1.0f + expf(-g * alpha)));
    default: return min_nan(g / (1.0f + expf(-g)), limit) * clamp_nan(u, limit);
  }
}

}  // namespace
}  // namespace b200moe
