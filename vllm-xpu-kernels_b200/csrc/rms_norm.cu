// Root-mean-square norm of rows, with the residual's addition ahead of it and an e4m3 copy of the
// rows with dynamic scales behind it: what a decoder block does between its attention and its
// Mixture-of-Experts layer, in one pass.
//
//   s = T(input + residual), stored as the new residual      (s = input without one)
//   y = s / sqrt(mean(s^2) + eps) * weight                   (fp32, mean over the row)
//   out = T(y);   per group of a row: scale = max(amax|y| / 448, 1 / (448 * 512)), q = e4m3(y / scale)
//
// The sum that is normalised is the rounded one, which the next reader of the residual sees too; y goes
// to the 8-bit rows before its rounding to T.  Scales and codes are those of per_token_group_fp8_quant on y,
// except that NaN and infinities stay visible: the scale of a group that holds one is NaN.
#include "common.cuh"

namespace b200moe {
namespace {

constexpr float kE4m3Max = 448.f, kLeastScale = 1.0f / (448.f * 512.f);

struct RmsParams {
  const void* input;
  void* residual;
  const void* weight;
  void* out;
  uint8_t* q;
  float* scales;
  int64_t rows, input_stride, residual_stride, out_stride, q_stride, s_stride_row, s_stride_group;
  int hidden, group;
  float eps;
  bool ue8m0;
};

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Smallest power of two that is at least x (x > 0, normal); NaN and infinity stay.
__device__ __forceinline__ float up_to_pow2(float x) {
  const uint32_t b = __float_as_uint(x);
  if (b >= 0x7f800000u) return x;
  return __uint_as_float((b + 0x007fffffu) & 0xff800000u);
}

__device__ __forceinline__ float scale_of(float amax, bool ue8m0) {
  const float s = max_nan(__fdiv_rn(amax, kE4m3Max), kLeastScale);
  return ue8m0 ? up_to_pow2(s) : s;
}

// Any size, stride and alignment: a block per row, one value at a time.  Every thread comes back to its own values
// only, so that `out` may be the input's memory.
template <typename T, typename W>
__global__ void __launch_bounds__(256) rms_norm_scalar_kernel(RmsParams p) {
  pdl_trigger();
  pdl_wait();
  __shared__ float red_sum[8], red_max[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.input) + r * p.input_stride;
  T* res = p.residual ? reinterpret_cast<T*>(p.residual) + r * p.residual_stride : nullptr;
  const T* s = res ? res : x;
  const W* w = reinterpret_cast<const W*>(p.weight);
  float sum = 0.f, top = 0.f;
  // A warp owns whole groups, so that what it wrote to the residual is what it reads again.
  const int group = p.q && p.group ? p.group : 32;
  for (int g0 = warp * group; g0 < p.hidden; g0 += 8 * group) {
    const int end = min(g0 + group, p.hidden);
    for (int i = g0 + lane; i < end; i += 32) {
      float v = to_f32<T>(x[i]);
      if (res) {
        const T t = from_f32<T>(v + to_f32<T>(res[i]));
        res[i] = t;
        v = to_f32<T>(t);
      }
      sum = fmaf(v, v, sum);
      top = max_nan(top, fabsf(w ? v * to_f32<W>(w[i]) : v));
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, d);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
  }
  if (lane == 0) { red_sum[warp] = sum; red_max[warp] = top; }
  __syncthreads();
  sum = 0.f;
  top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) { sum += red_sum[i]; top = max_nan(top, red_max[i]); }
  const float rs = rsqrtf(sum / (float)p.hidden + p.eps);
  float scale = 0.f, inv = 0.f;
  if (p.q && p.group == 0) {
    scale = scale_of(top * rs, p.ue8m0);
    inv = __fdiv_rn(1.0f, scale);
    if (tid == 0) p.scales[r * p.s_stride_row] = scale;
  }
  T* out = p.out ? reinterpret_cast<T*>(p.out) + r * p.out_stride : nullptr;
  uint8_t* q = p.q ? p.q + r * p.q_stride : nullptr;
  for (int g0 = warp * group; g0 < p.hidden; g0 += 8 * group) {
    const int end = min(g0 + group, p.hidden);
    if (q && p.group) {
      float m = 0.f;
      for (int i = g0 + lane; i < end; i += 32) {
        const float n = to_f32<T>(s[i]) * rs;
        m = max_nan(m, fabsf(w ? n * to_f32<W>(w[i]) : n));
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
      scale = scale_of(m, p.ue8m0);
      inv = __fdiv_rn(1.0f, scale);
      if (lane == 0) p.scales[r * p.s_stride_row + (int64_t)(g0 / group) * p.s_stride_group] = scale;
    }
    for (int i = g0 + lane; i < end; i += 32) {
      const float n = to_f32<T>(s[i]) * rs;
      const float y = w ? n * to_f32<W>(w[i]) : n;
      if (out) out[i] = from_f32<T>(y);
      if (q) q[i] = f32_to_e4m3(y * inv);
    }
  }
}

template <typename T, typename W>
int launch_rms_norm(const RmsParams& p, cudaStream_t st) {
  B200_LAUNCHED("rms_norm_scalar_kernel",
                launch_pdl(p.rows <= kEarlyLaunchRows, rms_norm_scalar_kernel<T, W>, dim3((unsigned)p.rows), dim3(256), 0, st, p));
  return B200MOE_OK;
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_add_rms_norm(const b200moe_rms_norm_args* a, b200moe_stream stream) {
  B200_CHECK_ARG(a != nullptr, "add_rms_norm: null arguments");
  B200_CHECK_ARG(a->rows >= 0 && a->rows <= 0x7fffffff && a->hidden >= 0, "add_rms_norm: negative or too large size");
  B200_CHECK_ARG(a->group_size >= 0 && (a->group_size == 0 || a->hidden % a->group_size == 0),
                 "add_rms_norm: the row length must be a multiple of group_size");
  B200_CHECK_ARG((a->q == nullptr) == (a->scales == nullptr), "add_rms_norm: 8-bit rows and scales go together");
  B200_CHECK_ARG(a->weight == nullptr || a->weight_dtype == a->dtype || a->weight_dtype == B200MOE_F32,
                 "add_rms_norm: weight must be float32 or have the input's dtype");
  if (a->rows == 0 || a->hidden == 0) return B200MOE_OK;
  B200_CHECK_ARG(a->input != nullptr, "add_rms_norm: null pointer");
  B200_CHECK_ARG(a->out != nullptr || a->q != nullptr, "add_rms_norm: nothing to write");
  RmsParams p = {a->input, a->residual, a->weight, a->out, (uint8_t*)a->q, a->scales, a->rows, a->input_stride,
                 a->residual_stride, a->out_stride, a->q_stride, a->s_stride_row, a->s_stride_group, a->hidden,
                 a->group_size == a->hidden ? 0 : a->group_size, a->eps, a->scale_ue8m0 != 0};
  const bool wide = a->weight != nullptr && a->weight_dtype == B200MOE_F32;
  B200_DISPATCH_FLOAT(a->dtype, "add_rms_norm", {
    return wide ? launch_rms_norm<scalar_t, float>(p, as_stream(stream)) : launch_rms_norm<scalar_t, scalar_t>(p, as_stream(stream));
  });
  return B200MOE_OK;
}
