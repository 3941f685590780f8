// A whole Mixture-of-Experts layer for a few tokens in two kernels:
//
//   up:    h[s] = act(W13[e] x[t] + b13[e])              for every slot s = (t, k) with a local expert e
//   down:  out[t] = sum_k w[t,k] (W2[e] h[s] + b2[e])
//
// Weights are taken as they are stored; activations stay in 16 bits or more, sums in fp32.
#include <algorithm>

#include "common.cuh"
#include "few_tokens.cuh"
#include "few_tokens_columns.cuh"
#include "few_tokens_rows.cuh"

namespace b200moe {
namespace {

// Byte i of the scales of a 4-bit matrix's row.
__device__ __forceinline__ const uint8_t* scale_at(const FewMatrix& w, int64_t e, int n, int i) {
  return reinterpret_cast<const uint8_t*>(w.scale) + e * w.n * w.scales.bytes + (int64_t)n * w.scales.row + (int64_t)(i / 4) * w.scales.next + i % 4;
}

// One weight, W_e[n, k], in fp32.
template <typename T>
__device__ __forceinline__ float weight_at(const FewMatrix& w, int64_t e, int n, int k) {
  const int64_t N = w.n, K = w.k;
  const uint8_t* b = reinterpret_cast<const uint8_t*>(w.w);
  switch (w.format) {
    case B200MOE_W_BF16_KN: return to_f32<T>(reinterpret_cast<const T*>(w.w)[(e * K + k) * N + n]);
    case B200MOE_W_FP8_BLOCK_NK:
    case B200MOE_W_FP8_BLOCK_KN: {
      const uint8_t q = w.format == B200MOE_W_FP8_BLOCK_NK ? b[(e * N + n) * K + k] : b[(e * K + k) * N + n];
      return e4m3_to_f32(q) * reinterpret_cast<const float*>(w.scale)[(e * (N / 128) + n / 128) * (K / 128) + k / 128];
    }
    case B200MOE_W_INT4_NK: {
      const uint8_t q = b[(e * N + n) * (K / 2) + k / 2];
      const int v = (int)(((k & 1) ? (q >> 4) : (q & 15)) ^ 8) - 8;
      return (float)v * to_f32<T>(*reinterpret_cast<const T*>(scale_at(w, e, n, k / (512 / w.scales.step) * 2)));
    }
    default: {
      const uint8_t q = b[(e * N + n) * (K / 2) + k / 2];
      return e2m1_to_f32((k & 1) ? (q >> 4) : (q & 15)) * e8m0_to_f32(*scale_at(w, e, n, k / 32));
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// A warp per feature of h and slot.
template <typename T>
__global__ void __launch_bounds__(256) few_up_simple_kernel(FewParams p) {
  pdl_trigger();
  pdl_wait();
  const int f = blockIdx.x * 8 + (threadIdx.x >> 5), slot = blockIdx.y, lane = threadIdx.x & 31;
  const int e = local_expert(p, slot);
  if (e < 0 || f >= p.inter) return;
  const bool pairs = p.act == B200MOE_ACT_SWIGLUOAI;   // gate and up of a feature side by side
  const int ng = pairs ? 2 * f : f, nu = pairs ? 2 * f + 1 : p.inter + f;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)(slot / p.topk) * p.hidden;
  float g = 0.f, u = 0.f;
  for (int k = lane; k < p.hidden; k += 32) {
    const float v = to_f32<T>(x[k]);
    g = fmaf(v, weight_at<T>(p.w13, e, ng, k), g);
    u = fmaf(v, weight_at<T>(p.w13, e, nu, k), u);
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (lane == 0) {
    const T* b = reinterpret_cast<const T*>(p.w13.bias);
    if (b) {
      g += to_f32<T>(b[(int64_t)e * p.w13.n + ng]);
      u += to_f32<T>(b[(int64_t)e * p.w13.n + nu]);
    }
    p.h[(int64_t)slot * p.inter + f] = gated(p.act, p.alpha, p.limit, p.clamp, g, u);
  }
}

// A warp per output feature and token.
template <typename T>
__global__ void __launch_bounds__(256) few_down_simple_kernel(FewParams p) {
  pdl_trigger();
  pdl_wait();
  const int n = blockIdx.x * 8 + (threadIdx.x >> 5), t = blockIdx.y, lane = threadIdx.x & 31;
  if (n >= p.hidden) return;
  const T* b = reinterpret_cast<const T*>(p.w2.bias);
  float sum = 0.f;
  for (int k = 0; k < p.topk; ++k) {
    const int slot = t * p.topk + k, e = local_expert(p, slot);
    if (e < 0) continue;
    const float* h = p.h + (int64_t)slot * p.inter;
    float y = 0.f;
    for (int i = lane; i < p.inter; i += 32) y = fmaf(h[i], weight_at<T>(p.w2, e, n, i), y);
    y = warp_sum(y);
    if (b) y += to_f32<T>(b[(int64_t)e * p.hidden + n]);
    sum = fmaf(p.weights[slot], y, sum);
  }
  if (lane == 0) reinterpret_cast<T*>(p.out)[(int64_t)t * p.hidden + n] = from_f32<T>(sum);
}

template <typename T>
int launch_simple(const FewParams& p, cudaStream_t st) {
  B200_LAUNCHED("few_up_simple_kernel", launch_pdl(true, few_up_simple_kernel<T>, dim3((p.inter + 7) / 8, p.tokens * p.topk), dim3(256), 0, st, p));
  B200_LAUNCHED("few_down_simple_kernel", launch_pdl(true, few_down_simple_kernel<T>, dim3((p.hidden + 7) / 8, p.tokens), dim3(256), 0, st, p));
  return B200MOE_OK;
}

// ---- on the tensor cores ------------------------------------------------------------------
constexpr int kMaxBlockSmem = 232448;

// The attribute is set once per kernel and device, and always to the most that a block may have, so that calls with
// different needs do not get into each other's way.
template <auto Kern, typename... Maps>
int launch_block_per_sm(const char* name, int grid, int threads, int smem, cudaStream_t st, const FewParams& p, const FewLaunch& l, const Maps&... maps) {
  static std::atomic<bool> done[kMaxDevices];
  const int dev = current_device();
  if (!done[dev].load(std::memory_order_acquire)) {
    B200_CUDA_OK(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBlockSmem));
    done[dev].store(true, std::memory_order_release);
  }
  B200_LAUNCHED(name, launch_pdl(true, Kern, dim3(grid), dim3(threads), smem, st, p, l, maps...));
  return B200MOE_OK;
}

// Shares of the second kernel's steps for the same rows, at most: the last of their blocks adds all of them up, some 0.2 us each and
// round of 256 sums (148 of them for 256 columns: 217 us at 16 tokens).
constexpr int kMaxSplits = 9;

// Where things are in the workspace: h, then what the blocks of the two kernels tell one another.
struct FewWorkspace {
  size_t arrived, part, bytes;
  FewWorkspace(int64_t tokens, int64_t topk, int64_t hidden, int64_t inter) {
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    arrived = up(tokens * topk * inter * sizeof(float));
    part = arrived + kFewMaxBlocks * sizeof(uint32_t);
    bytes = part + up((size_t)kMaxSplits * tokens * hidden * sizeof(float));
  }
};
// As many as make `ctas` blocks with up to `rows` rows each.
int few_splits(int64_t hidden, int ctas, int rows) {
  const int64_t n = (int64_t)ctas * rows / hidden;
  return n < 1 ? 1 : (int)std::min<int64_t>(n, std::min(ctas, kMaxSplits));
}

// The map of a matrix for loads of `box` rows (by column: columns) of a step.
template <int F>
int few_map(CUtensorMap* map, const FewMatrix& m, int experts, int box) {
  if constexpr (by_column(F)) {
    const cuuint64_t dims[3] = {(cuuint64_t)m.n, (cuuint64_t)m.k, (cuuint64_t)experts};
    const cuuint64_t strides[2] = {(cuuint64_t)m.n * 2, (cuuint64_t)m.n * m.k * 2};
    const cuuint32_t boxes[3] = {(cuuint32_t)box, (cuuint32_t)ColumnShape<F>::kK, 1};
    return encode_map(map, F == kFewBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, m.w, dims, strides, boxes,
                      box == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  } else {
    const cuuint64_t row = F == kFewFp8 ? m.k : m.k / 2;
    const cuuint64_t dims[3] = {row, (cuuint64_t)m.n, (cuuint64_t)experts};
    const cuuint64_t strides[2] = {row, row * m.n};
    const cuuint32_t boxes[3] = {128, (cuuint32_t)box, 1};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, m.w, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_128B);
  }
}
int at_least(int a, int b) { return a < b ? b : a; }

// The kernels' shared memory: what they always need, and a panel of tokens or h.
template <int F, int NT>
int launch_columns(const FewParams& p, FewLaunch l, int ctas, cudaStream_t st) {
  using S = ColumnShape<F>;
  constexpr int up_fixed = UpColumnsShape<F, NT>::kFixed, up_room = kMaxBlockSmem - up_fixed, down_room = kMaxBlockSmem - S::kRest;
  const int up_row = (p.hidden + S::kK - 1) / S::kK * S::kPanelBytes(1), down_row = (p.inter + S::kK - 1) / S::kK * S::kPanelBytes(S::kTerms);
  static_assert(up_room >= 16384 / S::kK * S::kPanelBytes(1), "a token");
  l.panel_bytes = min(p.tokens * up_row, up_room / up_row * up_row);
  l.box = S::kRows;
  // as many side by side as leave no more shares than that
  l.side = 4;
  while (l.side > 1 && (p.hidden + l.side * S::kRows - 1) / (l.side * S::kRows) * kMaxSplits * 4 < ctas * 3) l.side /= 2;
  l.columns = min(ctas, (p.hidden + l.side * S::kRows - 1) / (l.side * S::kRows));
  l.splits = min(ctas / l.columns, kMaxSplits);
  const int64_t want = (int64_t)p.tokens * p.topk * down_row;
  const int down_panel = at_least((int)(want < down_room ? want : down_room), RedShape<F, NT>::kBytes);
  l.room = down_panel / S::kPanelBytes(S::kTerms);
  l.by_columns = FewDiv(l.columns);
  l.by_splits = FewDiv(l.splits);
  l.by_down_steps = FewDiv((p.inter + S::kK - 1) / S::kK);
  // loads of 32 gates, 32 ups or 64 columns in pairs; of 64 columns of W2
  CUtensorMap up_map, down_map;
  int rc = few_map<F>(&up_map, p.w13, p.experts, p.act == B200MOE_ACT_SWIGLUOAI ? 64 : 32);
  if (rc == B200MOE_OK) rc = few_map<F>(&down_map, p.w2, p.experts, l.box);
  if (rc == B200MOE_OK)
    rc = launch_block_per_sm<few_up_columns_kernel<F, NT>>("few_up_columns_kernel", ctas, S::kThreads, up_fixed + l.panel_bytes, st, p, l, up_map);
  if (rc != B200MOE_OK) return rc;
  return launch_block_per_sm<few_down_columns_kernel<F, NT>>("few_down_columns_kernel", l.columns * l.splits, S::kThreads, S::kRest + down_panel, st, p, l,
                                                             down_map);
}
template <int F, int NT>
int launch_rows(const FewParams& p, FewLaunch l, int ctas, cudaStream_t st) {
  using S = RowShape<F>;
  constexpr int up_fixed = UpRowsShape<F, NT>::kFixed, up_room = kMaxBlockSmem - up_fixed;
  const int down_fixed = S::kRest + down_sums_bytes(p.tokens, S::kWarps), down_room = kMaxBlockSmem - down_fixed;
  const int up_row = (p.hidden + S::kK - 1) / S::kK * S::kPanelBytes, down_row = (p.inter + S::kK - 1) / S::kK * S::kPanelBytes;
  static_assert(up_room >= 16384 / S::kK * S::kPanelBytes, "a token");
  l.panel_bytes = min(p.tokens * up_row, up_room / up_row * up_row);
  l.splits = few_splits(p.hidden, ctas, kBlockRows);
  l.columns = min(ctas / l.splits, (p.hidden + 15) / 16);
  // a block's rows in as few turns as they need, and halved in each
  const int rows = (p.hidden + l.columns - 1) / l.columns, turns = (rows + kBlockRows - 1) / kBlockRows;
  l.side = 2;
  l.box = (rows + 2 * turns - 1) / (2 * turns);
  const int64_t want = (int64_t)p.tokens * p.topk * down_row;
  const int down_panel = (int)(want < down_room ? want : down_room);
  l.room = down_panel / S::kPanelBytes;
  l.most = l.panel_bytes / up_row;
  l.by_sets = FewDiv(p.inter / 16);
  l.by_steps = FewDiv((p.hidden + S::kK - 1) / S::kK);
  l.by_ctas = FewDiv(ctas);
  l.by_columns = FewDiv(l.columns);
  l.by_splits = FewDiv(l.splits);
  l.by_down_steps = FewDiv((p.inter + S::kK - 1) / S::kK);
  CUtensorMap up_map, down_map;
  int rc = few_map<F>(&up_map, p.w13, p.experts, 16);
  if (rc == B200MOE_OK) rc = few_map<F>(&down_map, p.w2, p.experts, l.box);
  if (rc == B200MOE_OK)
    rc = launch_block_per_sm<few_up_rows_kernel<F, NT>>("few_up_rows_kernel", ctas, S::kThreads, up_fixed + l.panel_bytes, st, p, l, up_map);
  if (rc != B200MOE_OK) return rc;
  return launch_block_per_sm<few_down_rows_kernel<F, NT>>("few_down_rows_kernel", l.columns * l.splits, S::kThreads, down_fixed + down_panel, st, p, l,
                                                          down_map);
}
template <int F, int NT>
int launch_mma(const FewParams& p, const FewLaunch& l, int ctas, cudaStream_t st) {
  if constexpr (by_column(F)) return launch_columns<F, NT>(p, l, ctas, st);
  else return launch_rows<F, NT>(p, l, ctas, st);
}

template <int F>
int launch_mma(const FewParams& p, const FewLaunch& l, int ctas, cudaStream_t st) {
  return p.tokens <= 8 ? launch_mma<F, 1>(p, l, ctas, st) : launch_mma<F, 2>(p, l, ctas, st);
}

// Sizes and addresses that these kernels can take; one row of tokens has to fit a block's shared memory.
bool takes_mma(const FewParams& p) {
  const bool by_columns = p.w13.format == B200MOE_W_BF16_KN;
  if (p.w13.format == B200MOE_W_FP8_BLOCK_KN) return false;
  for (const void* a : {p.x, p.w13.w, p.w13.scale, p.w2.w, p.w2.scale})
    if (((uintptr_t)a & 15) != 0) return false;
  const int whole = by_columns ? 8 : 32;
  return p.hidden % whole == 0 && p.inter % whole == 0 && p.hidden <= 16384 && p.inter <= 65536;
}

bool known_format(int f) {
  return f == B200MOE_W_BF16_KN || f == B200MOE_W_FP8_BLOCK_NK || f == B200MOE_W_FP8_BLOCK_KN || f == B200MOE_W_MXFP4_NK ||
         f == B200MOE_W_INT4_NK;
}

// What the sizes of a matrix have to be for its format.
int check_matrix(const b200moe_few_tokens_args* a, b200moe_weight_format f, const void* w, const void* scale, int group, int n, int k,
                 const char* name) {
  if (!known_format(f))
    return fail(B200MOE_E_UNSUPPORTED, "few_tokens_layer: 16-bit [E,K,N], block-scaled fp8, MXFP4 and int4 weights only");
  B200_CHECK_ARG(w != nullptr && (f == B200MOE_W_BF16_KN || scale != nullptr), "few_tokens_layer: %s or its scales are missing", name);
  if (f == B200MOE_W_FP8_BLOCK_NK || f == B200MOE_W_FP8_BLOCK_KN)
    B200_CHECK_ARG(n % 128 == 0 && k % 128 == 0, "few_tokens_layer: block-scaled %s needs sizes divisible by 128", name);
  if (f == B200MOE_W_MXFP4_NK) B200_CHECK_ARG(k % 32 == 0, "few_tokens_layer: MXFP4 %s needs rows of a multiple of 32", name);
  if (f == B200MOE_W_INT4_NK)
    B200_CHECK_ARG((group == 32 || group == 64 || group == 128 || group == 256) && k % group == 0,
                   "few_tokens_layer: int4 %s needs groups of 32, 64, 128 or 256 that divide its rows", name);
  (void)a;
  return B200MOE_OK;
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_few_tokens_scale_words(b200moe_weight_format format, int group_size, int k) {
  if (k <= 0 || (format != B200MOE_W_MXFP4_NK && format != B200MOE_W_INT4_NK)) return 0;
  return few_scale_words(format, group_size, k);
}

extern "C" size_t b200moe_few_tokens_workspace_bytes(int num_tokens, int topk, int hidden, int inter) {
  if (num_tokens <= 0 || topk <= 0 || hidden <= 0 || inter <= 0) return 0;
  return FewWorkspace(num_tokens, topk, hidden, inter).bytes;
}

namespace b200moe {
namespace {

int few_tokens_layer(const b200moe_few_tokens_args* a, b200moe_stream stream, bool scales_by_step) {
  B200_CHECK_ARG(a != nullptr, "few_tokens_layer: null arguments");
  B200_CHECK_ARG(a->dtype == B200MOE_BF16 || a->dtype == B200MOE_F16, "few_tokens_layer: hidden states must be bfloat16 or float16");
  B200_CHECK_ARG(a->num_tokens >= 0 && a->num_tokens <= B200MOE_FEW_TOKENS, "few_tokens_layer: at most %d tokens", B200MOE_FEW_TOKENS);
  B200_CHECK_ARG(a->hidden >= 1 && a->inter >= 1 && a->hidden <= (1 << 20) && a->inter <= (1 << 20),
                 "few_tokens_layer: sizes must be between 1 and 2^20");
  B200_CHECK_ARG(a->topk >= 1 && a->topk <= kFewMaxTopk, "few_tokens_layer: topk must be in [1, %d]", kFewMaxTopk);
  B200_CHECK_ARG(a->num_experts >= 1 && a->num_experts <= kFewMaxExperts, "few_tokens_layer: num_experts must be in [1, %d]", kFewMaxExperts);
  B200_CHECK_ARG(a->ids_dtype == B200MOE_I32 || a->ids_dtype == B200MOE_I64, "few_tokens_layer: topk_ids must be int32 or int64");
  B200_CHECK_ARG(a->activation >= B200MOE_ACT_SILU && a->activation <= B200MOE_ACT_SWIGLUSTEP, "few_tokens_layer: unknown activation");
  int rc = check_matrix(a, a->w13_format, a->w13, a->w13_scale, a->w13_group, 2 * a->inter, a->hidden, "w13");
  if (rc == B200MOE_OK) rc = check_matrix(a, a->w2_format, a->w2, a->w2_scale, a->w2_group, a->hidden, a->inter, "w2");
  if (rc != B200MOE_OK) return rc;
  B200_CHECK_ARG(a->w13_format == a->w2_format, "few_tokens_layer: w13 and w2 must have the same format");
  if (a->num_tokens == 0) return B200MOE_OK;
  B200_CHECK_ARG(a->x && a->topk_ids && a->topk_weights && a->out, "few_tokens_layer: null pointer");
  const size_t need = b200moe_few_tokens_workspace_bytes(a->num_tokens, a->topk, a->hidden, a->inter);
  if (a->workspace == nullptr || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15) != 0)
    return fail(B200MOE_E_WORKSPACE, "few_tokens_layer: needs %zu bytes of 16-byte aligned workspace", need);
  FewParams p = {};
  p.x = a->x; p.ids = a->topk_ids; p.ids64 = a->ids_dtype == B200MOE_I64; p.weights = a->topk_weights;
  p.expert_map = a->expert_map; p.out = a->out; p.h = (float*)a->workspace;
  p.tokens = a->num_tokens; p.hidden = a->hidden; p.inter = a->inter; p.topk = a->topk;
  p.experts = a->num_experts; p.id_limit = a->expert_map ? a->total_experts : a->num_experts;
  p.by_topk = FewDiv(a->topk);
  p.act = a->activation; p.alpha = a->act_alpha; p.limit = a->act_limit; p.clamp = a->clamp_limit;
  p.w13 = {a->w13, a->w13_scale, a->w13_bias, a->w13_format, a->w13_group, 2 * a->inter, a->hidden,
           few_scales(a->w13_format, a->w13_group, 2 * a->inter, a->hidden, scales_by_step)};
  p.w2 = {a->w2, a->w2_scale, a->w2_bias, a->w2_format, a->w2_group, a->hidden, a->inter,
          few_scales(a->w2_format, a->w2_group, a->hidden, a->inter, scales_by_step)};
  int ctas = a->max_ctas > 0 && a->max_ctas < sm_count() ? a->max_ctas : sm_count();
  if (ctas > kFewMaxBlocks) ctas = kFewMaxBlocks;
  if (takes_mma(p)) {
    FewLaunch l = {};
    l.f16 = a->dtype == B200MOE_F16;
    l.status = a->status;
    const FewWorkspace ws(p.tokens, p.topk, p.hidden, p.inter);
    l.arrived = (uint32_t*)((char*)a->workspace + ws.arrived);
    l.part = (float*)((char*)a->workspace + ws.part);
    if (p.w13.format == B200MOE_W_BF16_KN)
      return l.f16 ? launch_mma<kFewF16>(p, l, ctas, as_stream(stream)) : launch_mma<kFewBf16>(p, l, ctas, as_stream(stream));
    if (p.w13.format == B200MOE_W_FP8_BLOCK_NK) return launch_mma<kFewFp8>(p, l, ctas, as_stream(stream));
    if (p.w13.format == B200MOE_W_MXFP4_NK) return launch_mma<kFewFp4>(p, l, ctas, as_stream(stream));
    const bool fine = p.w13.group < 128 || p.w2.group < 128;
    return fine ? launch_mma<kFewInt4Fine>(p, l, ctas, as_stream(stream)) : launch_mma<kFewInt4>(p, l, ctas, as_stream(stream));
  }
  return a->dtype == B200MOE_BF16 ? launch_simple<__nv_bfloat16>(p, as_stream(stream)) : launch_simple<__half>(p, as_stream(stream));
}

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_few_tokens_layer(const b200moe_few_tokens_args* a, b200moe_stream stream) { return few_tokens_layer(a, stream, true); }

extern "C" int b200moe_few_tokens_layer_as_stored(const b200moe_few_tokens_args* a, b200moe_stream stream) {
  return few_tokens_layer(a, stream, false);
}
