// Rows as 8-bit integers with one scale each, as the int8 GEMM takes its activations:
//
//   v = x, or silu(gate) * up of a row [gate | up];  a = max(amax|v|, 1e-10);  scale = a / 127;  q = 127 v / a, ties to even
//
// (quant_int8.cuh on their rounding).  A row with a NaN or an infinity has a scale of NaN.
#include <algorithm>

#include "common.cuh"
#include "quant_int8.cuh"

namespace b200moe {
namespace {

struct QuantInt8Params {
  const void* in;
  int8_t* q;
  float* scales;
  const int32_t* rows_per_segment;   // or NULL: all rows
  int64_t rows, in_stride, q_stride;
  int hidden, num_segments;
};

__device__ __forceinline__ float gated_value(float g, float u) { return g * fast_sigmoid(g) * u; }   // silu(gate) * up

__device__ __forceinline__ int64_t rows_in_use(const QuantInt8Params& p) {
  if (p.rows_per_segment == nullptr) return p.rows;
  int64_t used = 0;   // (every warp for itself; plain loads: the kernel before this one may have written the counts)
  for (int e = threadIdx.x & 31; e < p.num_segments; e += 32) used += max(p.rows_per_segment[e], 0);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) used += __shfl_xor_sync(0xffffffffu, used, off);
  return used < p.rows ? used : p.rows;
}

// Largest |v| of a row over its `threads` threads (a multiple of 32); `part` holds a value per warp of the block.
__device__ __forceinline__ float row_max(float amax, int threads, float* part) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if (threads == 32) return amax;
  const int warp = threadIdx.x >> 5, warps = threads >> 5, first = warp / warps * warps;
  if ((threadIdx.x & 31) == 0) part[warp] = amax;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  amax = lane < warps ? part[first + lane] : 0.f;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  return amax;
}

// Rows whose 16-byte pieces are aligned, P of them a thread (gated: of gates and of ups), which stay in registers between the maximum
// and the codes: every byte is read once.  Blocks stay: 8192 rows of 7168 bfloat16 values 30.1 us, 5.9 TB/s (31.3 with a block a row), gated
// 72.3 (77.3); 4096 rows of 14336 float32 values 45.3, 6.5 TB/s (44.9), gated 99.9 (108.1).
template <typename T, bool kGated, int P>
__global__ void __launch_bounds__(512, kGated || P == 8 ? 1 : 2)
quant_int8_rows_kernel(const QuantInt8Params p, int threads) {
  constexpr int N = 16 / sizeof(T);
  constexpr bool kKeep = kGated && P * N <= 32;      // gated values stay; of longer rows they are made again
  __shared__ float part[2][32];
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x / threads, t = threadIdx.x - sub * threads, per_block = blockDim.x / threads;
  const int64_t rows = rows_in_use(p), step = (int64_t)gridDim.x * per_block;
  const int nvec = p.hidden / N;
  vec16 a[P], b[kGated ? P : 1];
  auto load = [&](int64_t row, vec16 (&to)[P]) {
    const T* in = reinterpret_cast<const T*>(p.in) + row * p.in_stride;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int c = t + i * threads;
      if (row < rows && c < nvec) {
        to[i] = ld16(in + (int64_t)c * N);
        if (kGated) b[kGated ? i : 0] = ld16(in + p.hidden + (int64_t)c * N);
      }
    }
  };
  int64_t row = (int64_t)blockIdx.x * per_block + sub;
  load(row, a);
  int parity = 0;
  for (int64_t first = row - sub; first < rows; first += step, row += step, parity ^= 1) {
    const bool live = row < rows;
    float amax = 0.f;
    float v[kKeep ? P : 1][N];
    auto values = [&](int i, float (&y)[N]) {
      unpack(a[i], y, T());
      if (!kGated) return;
      float u[N];
      unpack(b[kGated ? i : 0], u, T());
#pragma unroll
      for (int k = 0; k < N; ++k) y[k] = gated_value(y[k], u[k]);
    };
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if (live && t + i * threads < nvec) {
        if (kGated) {
          float y[N];
          values(i, y);
#pragma unroll
          for (int k = 0; k < N; ++k) {
            if (kKeep) v[kKeep ? i : 0][k] = y[k];
            amax = max_nan(amax, fabsf(y[k]));
          }
        } else {
          most = largest(a[i], most, T());
        }
      }
    }
    if (!kGated) amax = largest_of(most, T());
    // (the maxima of the row before are in the other half)
    const Int8Scale<std::conditional_t<kGated, float, T>> s(row_max(amax, threads, part[parity]));
    if (live) {
      if (t == 0) p.scales[row] = s.scale;
      int8_t* q = p.q + row * p.q_stride;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = t + i * threads;
        if (c < nvec) {
          float y[N];
          if (kKeep) {
#pragma unroll
            for (int k = 0; k < N; ++k) y[k] = v[kKeep ? i : 0][k];
          } else {
            values(i, y);
          }
          uint32_t w[N / 4];
          s.codes(y, w);
          if (N == 8) *reinterpret_cast<uint2*>(q + (int64_t)c * N) = make_uint2(w[0], w[N / 4 - 1]);
          else *reinterpret_cast<uint32_t*>(q + (int64_t)c * N) = w[0];
        }
      }
    }
    if (first + step < rows) load(row + step, a);
  }
}

// Any length and alignment, value by value; rows are read twice.
template <typename T, bool kGated>
__global__ void __launch_bounds__(1024)
quant_int8_any_kernel(const QuantInt8Params p) {
  __shared__ float part[32];
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x;
  if (row >= rows_in_use(p)) return;
  const T* in = reinterpret_cast<const T*>(p.in) + row * p.in_stride;
  auto value = [&](int c) {
    const float y = to_f32<T>(in[c]);
    return kGated ? gated_value(y, to_f32<T>(in[(int64_t)p.hidden + c])) : y;
  };
  float amax = 0.f;
  for (int c = threadIdx.x; c < p.hidden; c += blockDim.x) amax = max_nan(amax, fabsf(value(c)));
  const Int8Scale<std::conditional_t<kGated, float, T>> s(row_max(amax, blockDim.x, part));
  if (threadIdx.x == 0) p.scales[row] = s.scale;
  for (int c = threadIdx.x; c < p.hidden; c += blockDim.x) {
    const float y[4] = {value(c), 0.f, 0.f, 0.f};
    uint32_t w[1];
    s.codes(y, w);
    p.q[row * p.q_stride + c] = (int8_t)w[0];
  }
}

template <typename T, bool kGated, int P>
int launch_rows(const QuantInt8Params& p, int nvec, cudaStream_t st) {
  auto kern = quant_int8_rows_kernel<T, kGated, P>;
  // Threads of a row: one piece each for a few rows (latency), all of them for many.
  const int pieces = p.rows <= 256 ? 1 : P, threads = std::min(512, ((nvec + pieces - 1) / pieces + 31) / 32 * 32);
  const int per_block = threads >= 256 ? 1 : 256 / threads, block = threads * per_block;
  static std::atomic<int> resident[kMaxDevices][17];      // blocks an SM, by their warps
  std::atomic<int>& cached = resident[current_device()][block / 32];
  int n = cached.load(std::memory_order_relaxed);
  if (n == 0) {
    B200_CUDA_OK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, block, 0));
    cached.store(std::max(n, 1), std::memory_order_relaxed);
  }
  const int64_t blocks = std::min<int64_t>((p.rows + per_block - 1) / per_block, (int64_t)std::max(n, 1) * sm_count());
  B200_LAUNCHED("quant_int8_rows_kernel", launch_pdl(p.rows <= kEarlyStayingRows, kern, dim3((unsigned)blocks), dim3(block), 0, st, p, threads));
  return B200MOE_OK;
}

template <typename T, bool kGated>
int launch(const QuantInt8Params& p, cudaStream_t st) {
  constexpr int N = 16 / sizeof(T);
  const int nvec = p.hidden / N;
  const bool whole = nvec > 0 && p.hidden % N == 0 && p.in_stride % N == 0 && p.q_stride % N == 0 && ((uintptr_t)p.in & 15) == 0 &&
                     ((uintptr_t)p.q & (N - 1)) == 0 && nvec <= 4096;
  if (!whole) {
    const int threads = p.hidden >= 1024 ? 1024 : std::max(32, (p.hidden + 31) / 32 * 32);
    B200_LAUNCHED("quant_int8_any_kernel", launch_pdl(p.rows <= kEarlyLaunchRows, quant_int8_any_kernel<T, kGated>, dim3((unsigned)p.rows),
                                                      dim3(threads), 0, st, p));
    return B200MOE_OK;
  }
  // (Many short rows: a warp each, and no barrier.  16384 rows of 768 float32 values 11.6 us, 13.0 with two warps a row, 8192 of 2048 bfloat16
  // values 10.0 and 11.2; 300 of 768 2.1 and 1.7; gated 16384 of 768 23 and 16.)
  return nvec > 2048 || (!kGated && nvec <= 256 && p.rows > 1024) ? launch_rows<T, kGated, 8>(p, nvec, st) : launch_rows<T, kGated, 4>(p, nvec, st);
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" int b200moe_quant_int8_rows(const void* in, b200moe_dtype dtype, int64_t in_stride, int8_t* q, int64_t q_stride,
                                       float* scales, int64_t rows, int hidden, int gated, const int32_t* rows_per_segment,
                                       int num_segments, b200moe_stream stream) {
  B200_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && hidden >= 0, "quant_int8_rows: negative or too large size");
  B200_CHECK_ARG(rows_per_segment == nullptr || num_segments >= 0, "quant_int8_rows: negative number of segments");
  if (rows == 0) return B200MOE_OK;
  B200_CHECK_ARG(((in && q) || hidden == 0) && scales, "quant_int8_rows: null pointer");   // (rows without values have a scale too)
  const QuantInt8Params p = {in, q, scales, rows_per_segment, rows, in_stride, q_stride, hidden, num_segments};
  int rc = B200MOE_OK;
  B200_DISPATCH_FLOAT(dtype, "quant_int8_rows",
                      rc = gated ? launch<scalar_t, true>(p, as_stream(stream)) : launch<scalar_t, false>(p, as_stream(stream)));
  return rc;
}
