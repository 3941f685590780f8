// Root-mean-square norm of rows, with the residual's addition ahead of it and an e4m3 copy of the
// rows with dynamic scales behind it: what a decoder block does between its attention and its
// Mixture-of-Experts layer, in one pass.
//
//   s = T(input + residual), stored as the new residual      (s = input without one)
//   y = s / sqrt(mean(s^2) + eps) * weight                   (fp32, mean over the row)
//   out = T(y);   per group of a row: scale = max(amax|y| / 448, 1 / (448 * 512)), q = e4m3(y * (1 / scale))
//
// The sum that is normalised is the rounded one, which the next reader of the residual sees too; y goes
// to the 8-bit rows before its rounding to T.  Scales and codes are those of per_token_group_fp8_quant on y,
// except that NaN and infinities stay visible: the scale of a group that holds one is NaN.
#include <type_traits>

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
  uint32_t least;      // bits of the least sum of squares that eps does not cover (see row_factor)
};

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

// The squares of a row are summed in fp32, which does not hold them where values are beyond some 2^63, nor to its precision where their
// sum is below 2^-80 (which counts where eps is, too).  Such a row is summed again times this power of two, and normalised so, with
// eps times its square; 1 elsewhere.  fp32 holds the squares of any float16.
__device__ __forceinline__ float row_factor(float sum, float eps) {
  if (sum == INFINITY) return 0x1p-80f;
  return sum < 0x1p-80f && eps < 0x1p-80f ? 0x1p100f : 1.f;
}
// Whether it is 1 (false also where the sum is a NaN): from `least` on, and finite.
template <typename T>
__device__ __forceinline__ bool sum_holds(float sum, uint32_t least) {
  return std::is_same_v<T, __half> || __float_as_uint(sum) - least < 0x7f800000u - least;
}

// Any size, stride and alignment: a block per row, one value at a time, four of a thread asked for together.  Every thread
// comes back to its own values only, so that `out` may be the input's memory.
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
  const int group = p.q && p.group ? p.group : 128;
  for (int g0 = warp * group; g0 < p.hidden; g0 += 8 * group) {
    const int end = min(g0 + group, p.hidden);
    for (int i0 = g0 + lane; i0 < end; i0 += 128) {
      float v[4], r[4], f[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + 32 * k;
        v[k] = i < end ? to_f32<T>(x[i]) : 0.f;
        r[k] = res && i < end ? to_f32<T>(res[i]) : 0.f;
        f[k] = w && i < end ? to_f32<W>(w[i]) : 1.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + 32 * k;
        if (i >= end) break;
        if (res) {
          const T t = from_f32<T>(v[k] + r[k]);
          res[i] = t;
          v[k] = to_f32<T>(t);
        }
        sum = fmaf(v[k], v[k], sum);
        top = max_nan(top, fabsf(v[k] * f[k]));
      }
    }
  }
  auto join = [&]() {
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
  };
  join();
  const float by = sum_holds<T>(sum, p.least) ? 1.f : row_factor(sum, p.eps);
  if (by != 1.f) {       // (the same for all threads)
    __syncthreads();
    sum = top = 0.f;
#pragma unroll 1
    for (int g0 = warp * group; g0 < p.hidden; g0 += 8 * group) {
      const int end = min(g0 + group, p.hidden);
#pragma unroll 1
      for (int i = g0 + lane; i < end; i += 32) {
        const float v = to_f32<T>(s[i]) * by;
        sum = fmaf(v, v, sum);
        top = max_nan(top, fabsf(w ? v * to_f32<W>(w[i]) : v));
      }
    }
    join();
  }
  const float rs = rsqrtf(sum / (float)p.hidden + p.eps * by * by);
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
#pragma unroll 4
      for (int i = g0 + lane; i < end; i += 32) {
        const float n = to_f32<T>(s[i]) * by * rs;
        m = max_nan(m, fabsf(w ? n * to_f32<W>(w[i]) : n));
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
      scale = scale_of(m, p.ue8m0);
      inv = __fdiv_rn(1.0f, scale);
      if (lane == 0) p.scales[r * p.s_stride_row + (int64_t)(g0 / group) * p.s_stride_group] = scale;
    }
    for (int i0 = g0 + lane; i0 < end; i0 += 128) {
      float y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + 32 * k;
        const float n = i < end ? to_f32<T>(s[i]) * by * rs : 0.f;
        y[k] = w && i < end ? n * to_f32<W>(w[i]) : n;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + 32 * k;
        if (i >= end) break;
        if (out) out[i] = from_f32<T>(y[k]);
        if (q) q[i] = f32_to_e4m3(y[k] * inv);
      }
    }
  }
}

// A thread's piece of a row: N values, moved with one access of up to 32 bytes.
template <typename T, int N> struct alignas(N * sizeof(T)) Piece { T e[N]; };
template <typename T, int N>
__device__ __forceinline__ void ld_piece(Piece<T, N>& d, const T* p) {
  if constexpr (sizeof(T) * N == 32) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&d);
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
  } else if constexpr (sizeof(T) * N == 64) {   // (fp32 weights of a 16-bit piece)
    ld_piece<T, N / 2>(reinterpret_cast<Piece<T, N / 2>*>(&d)[0], p);
    ld_piece<T, N / 2>(reinterpret_cast<Piece<T, N / 2>*>(&d)[1], p + N / 2);
  } else {
    d = *reinterpret_cast<const Piece<T, N>*>(p);
  }
}
template <typename T, int N>
__device__ __forceinline__ void st_piece(T* p, const Piece<T, N>& s) {
  if constexpr (sizeof(T) * N == 32) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&s);
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 :: "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p) : "memory");
  } else {
    *reinterpret_cast<Piece<T, N>*>(p) = s;
  }
}

enum ScaleMode { kNoScales, kRowScale, kGroupScales };

// Rows are read once and stay in registers between their sums and the result.  blockDim = (threads of a row, rows of a
// block); a thread has V pieces of N values, blockDim.x pieces apart.  A resident block takes row after row and asks for
// the next one before it waits for its sums.
// Bound by the bytes of a row, each moved once: 8192 rows of 7168 bf16 values with residual, output and e4m3 rows 86.5 us, 6.1
// TB/s (a block per row with 16-byte pieces and its values read twice 228 us).  Where only e4m3 rows are written there are fewer bytes
// for the same chain of sums, scale and codes: 8192 rows of 4096 float16 values 34 us, 2.9 TB/s.  With few rows the launch is what it
// costs: one row 2.2 us in a graph.
// Of rows that are summed again (see row_factor) the values in registers are scaled.
constexpr int kFewThreads = 448;
template <typename T, typename W, int N, int V, int kMode, int kMost>
__global__ void __launch_bounds__(kMost, kMost == 1024 ? 1 : 2) rms_norm_kernel(RmsParams p) {
  __shared__ float2 red[2][32];
  pdl_trigger();
  pdl_wait();
  const int tx = threadIdx.x, lane = tx & 31, warps = blockDim.x >> 5, warp = threadIdx.y * warps + (tx >> 5);
  const int pieces = p.hidden / N;
  const T* const input = reinterpret_cast<const T*>(p.input);
  T* const residual = reinterpret_cast<T*>(p.residual);
  const W* const w = reinterpret_cast<const W*>(p.weight);
  const int64_t step = (int64_t)gridDim.x * blockDim.y;
  Piece<T, N> x[V], b[V];
  auto ask = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int j = tx + i * blockDim.x;
      if (r < p.rows && j < pieces) {
        ld_piece<T, N>(x[i], input + r * p.input_stride + (int64_t)j * N);
        if (residual) ld_piece<T, N>(b[i], residual + r * p.residual_stride + (int64_t)j * N);
      }
    }
  };
  // Of a row's threads: a block has two rows of two warps at most.  (Numbers that the compiler knows: for one in a register the kernel is
  // given all 16 barriers, of which an SM has too few for five blocks.)
  auto row_sync = [&]() {
    if (warps == 1) __syncwarp();
    else if (threadIdx.y == 0) asm volatile("bar.sync 1, %0;" ::"r"((int)blockDim.x) : "memory");
    else asm volatile("bar.sync 2, %0;" ::"r"((int)blockDim.x) : "memory");
  };
  int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  ask(r);
  // (the rows of a block run through the same number of turns, so that its barrier is met by all)
  for (int64_t first = (int64_t)blockIdx.x * blockDim.y, turn = 0; first < p.rows; first += step, r += step, ++turn) {
    Piece<T, N> v[V];
    Piece<W, N> wv[V];
    float sum = 0.f, top = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int j = tx + i * blockDim.x;
      if (r < p.rows && j < pieces) {
        if (w) ld_piece<W, N>(wv[i], w + (int64_t)j * N);
        v[i] = x[i];
        if (residual) {
#pragma unroll
          for (int k = 0; k < N; ++k) v[i].e[k] = from_f32<T>(to_f32<T>(x[i].e[k]) + to_f32<T>(b[i].e[k]));
          st_piece<T, N>(residual + r * p.residual_stride + (int64_t)j * N, v[i]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float s = to_f32<T>(v[i].e[k]);
          sum = fmaf(s, s, sum);
          if (kMode == kRowScale) top = max_nan(top, fabsf(w ? s * to_f32<W>(wv[i].e[k]) : s));
        }
      }
    }
    ask(r + step);
    auto join = [&](auto sync) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (kMode == kRowScale) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
      }
      if (warps > 1) {   // two buffers in turn: one barrier a row
        if (lane == 0) red[turn & 1][warp] = make_float2(sum, top);
        sync();
        sum = 0.f;
        for (int i = 0; i < warps; ++i) {
          const float2 o = red[turn & 1][threadIdx.y * warps + i];
          sum += o.x;
          if (kMode == kRowScale) top = max_nan(top, o.y);
        }
      }
    };
    join([] { __syncthreads(); });
    float eps = p.eps;
    if (!sum_holds<T>(sum, p.least)) {      // (the same for all threads of a row)
      const float by = row_factor(sum, p.eps);
      row_sync();
      sum = top = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = tx + i * blockDim.x;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float s = to_f32<T>(v[i].e[k]) * by;
          v[i].e[k] = from_f32<T>(s);
          if (r < p.rows && j < pieces) {
            sum = fmaf(s, s, sum);
            if (kMode == kRowScale) top = max_nan(top, fabsf(w ? s * to_f32<W>(wv[i].e[k]) : s));
          }
        }
      }
      join(row_sync);
      eps = eps * by * by;
    }
    const float rs = rsqrtf(sum / (float)p.hidden + eps);
    float scale = 0.f, inv = 0.f;
    if (kMode == kRowScale) {
      scale = scale_of(top * rs, p.ue8m0);
      inv = __fdiv_rn(1.0f, scale);
      if (tx == 0 && r < p.rows) p.scales[r * p.s_stride_row] = scale;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int j = tx + i * blockDim.x;
      const bool mine = r < p.rows && j < pieces;
      float y[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float n = to_f32<T>(v[i].e[k]) * rs;
        y[k] = w ? n * to_f32<W>(wv[i].e[k]) : n;
      }
      if (p.out && mine) {
        Piece<T, N> o;
#pragma unroll
        for (int k = 0; k < N; ++k) o.e[k] = from_f32<T>(y[k]);
        st_piece<T, N>(reinterpret_cast<T*>(p.out) + r * p.out_stride + (int64_t)j * N, o);
      }
      if (kMode == kGroupScales) {
        const int lanes = p.group / N;   // of a group: a power of two
        float m = 0.f;
        if (mine) {
#pragma unroll
          for (int k = 0; k < N; ++k) m = max_nan(m, fabsf(y[k]));
        }
        for (int d = 1; d < lanes; d <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
        scale = scale_of(m, p.ue8m0);
        inv = __fdiv_rn(1.0f, scale);
        if (mine && (j & (lanes - 1)) == 0)
          p.scales[r * p.s_stride_row + (int64_t)(j / lanes) * p.s_stride_group] = scale;
      }
      if (kMode != kNoScales && mine) {
        uint8_t* q = p.q + r * p.q_stride + (int64_t)j * N;
        if constexpr (N == 1) {
          *q = f32_to_e4m3(y[0] * inv);
        } else {
          Piece<uint32_t, N / 4> o;
#pragma unroll
          for (int k = 0; k < N / 4; ++k)
            o.e[k] = f32x2_to_e4m3x2(y[4 * k] * inv, y[4 * k + 1] * inv) | (f32x2_to_e4m3x2(y[4 * k + 2] * inv, y[4 * k + 3] * inv) << 16);
          *reinterpret_cast<Piece<uint32_t, N / 4>*>(q) = o;
        }
      }
    }
  }
}

template <typename T, typename W, int N, int V, int kMode>
int launch_rows(const RmsParams& p, cudaStream_t st) {
  const int threads = ((p.hidden / N + V - 1) / V + 31) / 32 * 32;
  int rows = 1;   // of a block: at least 128 threads where there are rows for every SM
  while (rows * threads < 128 && p.rows > (int64_t)rows * sm_count()) rows *= 2;
  // Blocks of up to 448 threads are given 72 registers each, of which an SM has enough for two: with 64, as a block of 1024 needs, 8192 rows
  // of 7168 bf16 values take 92 us instead of 86.5, of 4096 57 instead of 50, of 512 7.9 instead of 7.0.
  const int most = rows * threads <= kFewThreads ? 2 * kFewThreads : 1024;
  const int64_t blocks = (p.rows + rows - 1) / rows, resident = (int64_t)sm_count() * (most / (rows * threads));
  const dim3 grid((unsigned)(blocks < resident ? blocks : resident));
  const auto kernel = rows * threads <= kFewThreads ? rms_norm_kernel<T, W, N, V, kMode, kFewThreads> : rms_norm_kernel<T, W, N, V, kMode, 1024>;
  B200_LAUNCHED("rms_norm_kernel", launch_pdl(p.rows <= kEarlyLaunchRows, kernel, grid, dim3(threads, rows), 0, st, p));
  return B200MOE_OK;
}
template <typename T, typename W, int N, int V>
int launch_mode(const RmsParams& p, cudaStream_t st) {
  if (p.q == nullptr) return launch_rows<T, W, N, V, kNoScales>(p, st);
  if (p.group == 0) return launch_rows<T, W, N, V, kRowScale>(p, st);
  if constexpr (N > 1) return launch_rows<T, W, N, V, kGroupScales>(p, st);
  return fail(B200MOE_E_BADARG, "add_rms_norm: no such variant");   // (not reached: see pieces_fit)
}

// Whether rows are made of pieces of n values that can be moved as such.
bool pieces_fit(const RmsParams& p, int n, int size, int weight_size) {
  auto fits = [](const void* b, int64_t stride, int bytes, int align) {
    return ((uintptr_t)b % align) == 0 && (stride * bytes) % align == 0;
  };
  const int align = n * size, lanes = p.group / n;
  return p.hidden % n == 0 && p.hidden / n <= 1024 && fits(p.input, p.input_stride, size, align) &&
         fits(p.residual, p.residual_stride, size, align) && fits(p.out, p.out_stride, size, align) &&
         fits(p.weight, 0, 1, n * weight_size < 32 ? n * weight_size : 32) && fits(p.q, p.q_stride, 1, n) &&
         (p.q == nullptr || p.group == 0 || (p.group % n == 0 && lanes <= 32 && (lanes & (lanes - 1)) == 0));
}

template <typename T, typename W>
int launch_rms_norm(const RmsParams& p, cudaStream_t st) {
  constexpr int N = 32 / sizeof(T), kSingles = 8;
  if (pieces_fit(p, N, sizeof(T), sizeof(W))) return launch_mode<T, W, N, 1>(p, st);
  if (pieces_fit(p, N / 2, sizeof(T), sizeof(W))) return launch_mode<T, W, N / 2, 1>(p, st);
  // Rows that cannot be cut into pieces: kept in registers value by value where that saves the second way through long rows, whose
  // latency counts with few of them, or where many short ones would have a block each.  us, in registers / below: 1411 bf16 values,
  // 61 rows 4.9 / 4.8, 256 rows 6.5 / 5.7, 8192 rows 81 / 51; 5001 values, 61 rows 6.0 / 9.6, 256 rows 11.7 / 12.7, 1001 rows 45 /
  // 20; 99 values, 1001 rows 4.3 / 3.8, 8192 rows 9.4 / 17.5.
  if (p.hidden <= 1024 * kSingles && (p.hidden > 2048 ? p.rows <= 256 : p.hidden < 256 && p.rows > 1024) && (p.q == nullptr || p.group == 0))
    return launch_mode<T, W, 1, kSingles>(p, st);
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
                 a->group_size == a->hidden ? 0 : a->group_size, a->eps, a->scale_ue8m0 != 0,
                 a->eps < 0x1p-80f ? 0x17800000u : 0u};
  const bool wide = a->weight != nullptr && a->weight_dtype == B200MOE_F32;
  B200_DISPATCH_FLOAT(a->dtype, "add_rms_norm", {
    return wide ? launch_rms_norm<scalar_t, float>(p, as_stream(stream)) : launch_rms_norm<scalar_t, scalar_t>(p, as_stream(stream));
  });
  return B200MOE_OK;
}
