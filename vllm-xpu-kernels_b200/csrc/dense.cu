// Entry points of the dense products: the int8 linear layer, the gated product and its gradients.
#include "dense.cuh"
#include "dense_tc.cuh"

namespace b200moe {
namespace {

// Gradients of the two products from the gradient of silu(g) * u, in the operands' type for the products that follow:
//   dg = d u s (1 + g (1 - s)),  du = d g s,  s = 1 / (1 + e^-g);  both = [dg | du] a row
// g and u come in 32 bits, as the forward pass had them; rounding dg and du to 16 bits is what the tensor cores ask for.  It takes the
// gradients' error from 1.7e-3 to 2.4e-3 in bfloat16 and from 2.1e-4 to 2.9e-4 in float16 (the first is the results' own 16 bits); in float16 a dg or du beyond
// 65504 is an infinity, and the rows and columns of the gradients that it goes into are not finite.
// A stream of 14 bytes for each value of d; N values a thread.
template <typename T, int N>
__global__ void __launch_bounds__(256)
gated_grad_kernel(const T* grad, const float* pre, T* both, int64_t rows, int inter, int64_t grad_stride, int64_t both_stride) {
  pdl_trigger();
  pdl_wait();
  const int per_row = inter / N;
  const int64_t total = rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / per_row;
    const int c = (int)(i - r * per_row) * N;
    const float* at = pre + r * 2 * inter + c;
    T d[N];
    float g[N], u[N];
    if (N == 8) {
      *reinterpret_cast<vec16*>(d) = ld16(grad + r * grad_stride + c);
#pragma unroll
      for (int k = 0; k < N; k += 4) {
        *reinterpret_cast<vec16*>(g + k) = ld16(at + k);
        *reinterpret_cast<vec16*>(u + k) = ld16(at + inter + k);
      }
    } else {
      d[0] = grad[r * grad_stride + c];
      g[0] = at[0];
      u[0] = at[inter];
    }
    T dg[N], du[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float s = fast_sigmoid(g[k]), x = to_f32<T>(d[k]);
      dg[k] = from_f32<T>(x * u[k] * s * (1.0f + g[k] * (1.0f - s)));
      du[k] = from_f32<T>(x * g[k] * s);
    }
    T* to = both + r * both_stride + c;
    if (N == 8) {
      st16(to, *reinterpret_cast<const vec16*>(dg));
      st16(to + inter, *reinterpret_cast<const vec16*>(du));
    } else {
      to[0] = dg[0];
      to[inter] = du[0];
    }
  }
}

// Rows of 16-byte pieces, for TMA; longer ones begin on 128 bytes, so that 128 bytes of a row are one line of L2 (both gradients of 4096 x
// 7168 x 2044 415 -> 375 us, of 1001 x 2048 x 1404 40.4 -> 36.7).
int64_t both_stride(int inter) {
  const int64_t n = 2 * (int64_t)inter, to = n <= 64 ? 8 : 64;
  return (n + to - 1) / to * to;
}

template <typename T>
int gated_grad(const b200moe_gated_linear_args* a, T* both, cudaStream_t st) {
  const int64_t stride = both_stride(a->inter);
  const bool wide = a->inter % 8 == 0 && a->grad_stride % 8 == 0 && ((uintptr_t)a->grad & 15) == 0 && ((uintptr_t)a->pre & 15) == 0;
  const int64_t threads = a->rows * (wide ? a->inter / 8 : a->inter);
  const int64_t blocks = std::min<int64_t>((threads + 255) / 256, (int64_t)sm_count() * 16);
  auto kern = wide ? gated_grad_kernel<T, 8> : gated_grad_kernel<T, 1>;
  B200_LAUNCHED("gated_grad_kernel",
                launch_pdl(a->rows <= kEarlyLaunchRows, kern, dim3((unsigned)blocks), dim3(256), 0, st, (const T*)a->grad, a->pre, both,
                           a->rows, a->inter, a->grad_stride, stride));
  return B200MOE_OK;
}

constexpr int kMaxValues = 1 << 29;      // of a gated product's rows and half of its weight rows
constexpr int kMaxFeatures = 0x7fffffff - 512;   // of an int8 product: weight rows, with those that its last tile would have, fit 32 bits
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_gated(const b200moe_gated_linear_args* a) {
  B200_CHECK_ARG(a != nullptr, "gated_linear: null argument struct");
  // (the kernels count a row's bytes and the weights' rows in 32 bits)
  B200_CHECK_ARG(a->rows >= 0 && a->rows <= 0x7fffffff && a->inter >= 0 && a->inter <= kMaxValues && a->hidden >= 0 && a->hidden <= kMaxValues,
                 "gated_linear: negative or too large size");
  B200_CHECK_ARG(a->dtype == B200MOE_BF16 || a->dtype == B200MOE_F16, "gated_linear: only float16 and bfloat16 are supported");
  B200_CHECK_ARG(a->hidden % 8 == 0 && a->x_stride % 8 == 0, "gated_linear: rows must be multiples of 16 bytes apart and long");
  B200_CHECK_ARG(aligned16(a->x) && aligned16(a->w), "gated_linear: input and weight must be 16-byte aligned");
  return B200MOE_OK;
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

// Codes of rows that are quantised on the way: longer ones begin on 128 bytes, so that 128 bytes of a row are one line of L2, not parts of two
// (4000 x 4096 x 4080 71.7 -> 59.5 us, 64 rows 11.0 -> 9.9; 30 x 3000 x 1504 7.2 -> 7.3).
static int64_t codes_pitch(int k) { return k <= 128 ? k : ((int64_t)k + 127) / 128 * 128; }

extern "C" size_t b200moe_int8_linear_workspace_bytes(int64_t rows, int k) {
  return rows <= 0 || k <= 0 ? 0 : (size_t)rows * codes_pitch(k) + (size_t)rows * 4;
}

extern "C" int b200moe_int8_linear(const b200moe_int8_linear_args* a, b200moe_stream stream) {
  B200_CHECK_ARG(a != nullptr, "int8_linear: null argument struct");
  B200_CHECK_ARG(a->rows >= 0 && a->rows <= 0x7fffffff && a->n >= 0 && a->n <= kMaxFeatures && a->k >= 0,
                 "int8_linear: negative or too large size");
  B200_CHECK_ARG(a->k <= B200MOE_INT8_MAX_K, "int8_linear: K must be at most %d, so that sums fit 32 bits", B200MOE_INT8_MAX_K);
  B200_CHECK_ARG(a->k > 0 && a->k % 16 == 0, "int8_linear: rows must be multiples of 16 values long");
  B200_CHECK_ARG(a->x_dtype == B200MOE_I8 || a->x_dtype == B200MOE_F32 || a->x_dtype == B200MOE_F16 || a->x_dtype == B200MOE_BF16,
                 "int8_linear: input must be int8, float32, float16 or bfloat16");
  B200_CHECK_ARG(a->x_dtype != B200MOE_I8 || a->x_stride % 16 == 0, "int8_linear: int8 rows must be multiples of 16 values apart");
  B200_CHECK_ARG(a->d_dtype == B200MOE_BF16 || a->d_dtype == B200MOE_F16 || a->d_dtype == B200MOE_F32,
                 "int8_linear: out must be float32, float16 or bfloat16");
  B200_CHECK_ARG(a->bias == nullptr || a->bias_dtype == B200MOE_BF16 || a->bias_dtype == B200MOE_F16,
                 "int8_linear: bias must be float16 or bfloat16");
  if (a->rows == 0 || a->n == 0) return B200MOE_OK;
  const bool codes = a->x_dtype == B200MOE_I8;
  B200_CHECK_ARG(a->x && (a->x_scale || !codes) && a->w && a->w_scale && a->d, "int8_linear: null pointer");
  B200_CHECK_ARG((aligned16(a->x) || !codes) && aligned16(a->w), "int8_linear: input and weight must be 16-byte aligned");
  DenseJob j = {};
  j.x_dtype = B200MOE_I8;
  const int size = dtype_bytes(a->x_dtype);
  if (!codes && dense_rows_quantises(a->rows, a->k) && aligned16(a->x) && a->x_stride * size % 16 == 0) {
    j.x_dtype = a->x_dtype;
  } else if (!codes) {
    if (a->workspace == nullptr || a->workspace_bytes < b200moe_int8_linear_workspace_bytes(a->rows, a->k) || !aligned16(a->workspace))
      return fail(B200MOE_E_WORKSPACE, "int8_linear: workspace missing, too small or not 16-byte aligned");
    int8_t* const q = (int8_t*)a->workspace;
    const int64_t pitch = codes_pitch(a->k);
    float* const s = (float*)(q + a->rows * pitch);
    if (int rc = b200moe_quant_int8_rows(a->x, a->x_dtype, a->x_stride, q, pitch, s, a->rows, a->k, 0, nullptr, 0, stream)) return rc;
    b200moe_int8_linear_args b = *a;
    b.x = q; b.x_scale = s; b.x_dtype = B200MOE_I8; b.x_stride = pitch;
    return b200moe_int8_linear(&b, stream);
  }
  j.x = a->x; j.w = a->w; j.x_scale = a->x_scale; j.w_scale = a->w_scale; j.bias = a->bias; j.d = a->d; j.status = a->status;
  j.m = a->rows; j.x_stride = a->x_stride; j.w_stride = a->k; j.d_stride = a->d_stride; j.n = a->n; j.k = a->k; j.experts = 1;
  j.type = kDenseI8; j.d_dtype = a->d_dtype; j.bias_f16 = a->bias_dtype == B200MOE_F16; j.early = a->rows <= kEarlyLaunchRows;
  return j.x_dtype != B200MOE_I8 ? dense_rows(j, as_stream(stream)) : dense(j, as_stream(stream));
}

extern "C" int b200moe_gated_linear(const b200moe_gated_linear_args* a, b200moe_stream stream) {
  if (int rc = check_gated(a)) return rc;
  if (a->rows == 0 || a->inter == 0) return B200MOE_OK;
  B200_CHECK_ARG(a->x && a->w && a->out && a->hidden > 0, "gated_linear: null pointer or rows without values");
  DenseJob j = {};
  j.x = a->x; j.w = a->w; j.d = a->out; j.pre = a->pre; j.status = a->status;
  j.m = a->rows; j.x_stride = a->x_stride; j.w_stride = a->hidden; j.d_stride = a->out_stride;
  j.n = 2 * a->inter; j.k = a->hidden; j.experts = 1; j.gated = true;
  j.type = a->dtype == B200MOE_BF16 ? kDenseBf16 : kDenseF16; j.d_dtype = a->dtype;
  j.early = a->rows <= kEarlyLaunchRows;
  return dense(j, as_stream(stream));
}

extern "C" size_t b200moe_gated_linear_backward_workspace_bytes(int64_t rows, int inter) {
  return rows <= 0 || inter <= 0 ? 0 : (size_t)rows * both_stride(inter) * 2;
}

extern "C" int b200moe_gated_linear_backward(const b200moe_gated_linear_args* a, b200moe_stream stream) {
  if (int rc = check_gated(a)) return rc;
  const cudaStream_t st = as_stream(stream);
  const bool early = a->rows <= kEarlyLaunchRows;
  const size_t dw_bytes = (size_t)2 * a->inter * a->hidden * 2;
  if (a->rows == 0 || a->inter == 0 || a->hidden == 0) {   // sums of nothing
    if (a->grad_w != nullptr && dw_bytes > 0) B200_CUDA_OK(cudaMemsetAsync(a->grad_w, 0, dw_bytes, st));
    if (a->grad_x != nullptr && a->rows > 0 && a->hidden > 0)
      B200_CUDA_OK(cudaMemset2DAsync(a->grad_x, (size_t)a->grad_x_stride * 2, 0, (size_t)a->hidden * 2, (size_t)a->rows, st));
    return B200MOE_OK;
  }
  if (a->grad_x == nullptr && a->grad_w == nullptr) return B200MOE_OK;
  B200_CHECK_ARG(a->grad && a->pre && (a->x || !a->grad_w) && (a->w || !a->grad_x), "gated_linear_backward: null pointer");
  if (a->workspace == nullptr || a->workspace_bytes < b200moe_gated_linear_backward_workspace_bytes(a->rows, a->inter) ||
      !aligned16(a->workspace))
    return fail(B200MOE_E_WORKSPACE, "gated_linear_backward: workspace missing, too small or not 16-byte aligned");
  const int rc = a->dtype == B200MOE_BF16 ? gated_grad<__nv_bfloat16>(a, (__nv_bfloat16*)a->workspace, st)
                                          : gated_grad<__half>(a, (__half*)a->workspace, st);
  if (rc) return rc;
  PlainJob j = {};
  j.x = a->workspace; j.status = a->status; j.x_stride = both_stride(a->inter); j.n = a->hidden;
  j.type = a->dtype == B200MOE_BF16 ? kDenseBf16 : kDenseF16; j.early = early;
  if (a->grad_x != nullptr) {      // [dg | du] W: sums over the features
    j.w = a->w; j.d = a->grad_x; j.m = a->rows; j.k = 2 * (int64_t)a->inter; j.w_stride = a->hidden; j.d_stride = a->grad_x_stride;
    if (int r = dense_plain(j, st)) return r;
  }
  if (a->grad_w != nullptr) {      // [dg | du]^T X: sums over the rows
    j.w = a->x; j.d = a->grad_w; j.m = 2 * (int64_t)a->inter; j.k = a->rows; j.w_stride = a->x_stride; j.d_stride = a->hidden;
    j.x_by_column = true;
    if (int r = dense_plain(j, st)) return r;
  }
  return B200MOE_OK;
}

namespace b200moe {

// b200moe_grouped_gemm with int8 weights.
int grouped_gemm_i8(const b200moe_gemm_args* a, cudaStream_t st) {
  const bool gated = a->epilogue == B200MOE_EPI_SILU_MUL, f32 = a->d_dtype == B200MOE_F32;
  // (no rows: nor are there scales of them)
  B200_CHECK_ARG(a->a_dtype == B200MOE_I8 && (a->a_scale != nullptr || a->m == 0) && a->w_scale != nullptr,
                 "grouped_gemm: int8 weights need int8 rows and the scales of both");
  B200_CHECK_ARG(a->k % 16 == 0 && a->k <= B200MOE_INT8_MAX_K,
                 "grouped_gemm: int8 weights need K divisible by 16 and at most %d", B200MOE_INT8_MAX_K);
  B200_CHECK_ARG(gated || a->epilogue == B200MOE_EPI_NONE, "grouped_gemm: int8 weights have the SiLU epilogue or none");
  B200_CHECK_ARG(a->d_dtype == B200MOE_BF16 || a->d_dtype == B200MOE_F16 || f32,
                 "grouped_gemm: int8 weights give float32, float16 or bfloat16");
  B200_CHECK_ARG(!f32 || a->bias == nullptr || a->mid_dtype == B200MOE_BF16 || a->mid_dtype == B200MOE_F16,
                 "grouped_gemm: a bias with float32 output has a 16-bit mid_dtype");
  B200_CHECK_ARG(a->w_experts == 0 || a->w_experts == a->num_experts,
                 "grouped_gemm: row segments that share weight sets need 16-bit or block-scaled fp8 weights");
  B200_CHECK_ARG(a->num_experts <= kMaxExperts, "grouped_gemm: more than %d experts", kMaxExperts);
  B200_CHECK_ARG(a->m <= 0x7fffffff && a->n <= kMaxFeatures, "grouped_gemm: too many rows or features");
  if (a->m == 0 || a->n == 0) return B200MOE_OK;
  B200_CHECK_ARG(a->a && a->w && a->d && a->rows_per_expert, "grouped_gemm: null pointer");
  B200_CHECK_ARG(aligned16(a->a) && aligned16(a->w), "grouped GEMM: A, W and D must be 16-byte aligned");
  if (a->impl == 2) return fail(B200MOE_E_UNSUPPORTED, "grouped_gemm: the checking kernel has no int8 weights");
  DenseJob j = {};
  j.x = a->a; j.w = a->w; j.x_scale = (const float*)a->a_scale; j.w_scale = (const float*)a->w_scale; j.bias = a->bias;
  j.d = a->d; j.rows_per_expert = a->rows_per_expert; j.status = a->status;
  j.m = a->m; j.x_stride = a->k; j.w_stride = a->k; j.n = a->n; j.k = a->k; j.experts = a->num_experts;
  j.d_stride = gated ? a->n / 2 : a->n;
  j.rows_hint = (int)(a->rows_hint > 0 && a->rows_hint < a->m ? a->rows_hint : 0);
  j.max_ctas = a->max_ctas; j.type = kDenseI8; j.x_dtype = B200MOE_I8; j.gated = gated; j.d_dtype = a->d_dtype;
  j.bias_f16 = (f32 ? a->mid_dtype : a->d_dtype) == B200MOE_F16;
  j.clamp = gated ? a->clamp_limit : 0.f;
  j.early = a->m <= kEarlyStayingRows;
  return dense(j, st);
}

}  // namespace b200moe
