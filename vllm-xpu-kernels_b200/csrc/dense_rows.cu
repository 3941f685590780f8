// Products of a few rows with int8 weights, or with the 16-bit weights of a gated block: every weight is read once, straight into
// the registers of the matrix instruction.
//
//   int8:   D[m, n] = (sum_k x[m, k] w[n, k]) * x_scale[m] * w_scale[n] (+ bias[n])      sums in int32, exact
//   gated:  D[m, i] = silu(g) * u, g and u the products with rows i and I + i of W          sums in fp32
//
// The order of k inside a sum is free as long as both operands share it, so a lane loads 16 consecutive bytes of a weight row
// (and of a token's) and takes them for the four words that mma.sync wants of it, two instructions for 64 bytes of a row: no shared
// memory, no shuffle and no repacking stand between the load and the product.  A block owns 32 features (16 gates and their
// 16 ups) and up to 16 tokens; its eight warps share the row's bytes out among themselves, 128 at a time, and add their sums up in shared
// memory.  What bounds it is the weights' way from HBM.
#include "dense.cuh"

namespace b200moe {
namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 128;      // bytes of a row that a warp takes at a time

struct RowsParams {
  DenseJob j;
  int64_t x_pitch, w_pitch;     // bytes from row to row
  int k_bytes;                  // bytes of a row
  int f_tiles;                  // tiles of 32 weight rows (gated: 16 and 16)
  int t_tiles;                  // dense: tiles of tokens
};

template <int kType>
__device__ __forceinline__ void mma(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kType == kDenseI8) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(d[i]);
    if (kType == kDenseBf16)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                   : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                   : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3])
                   : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = __float_as_uint(f[i]);
  }
}
// Weights: read once, and constant while the kernel runs.
__device__ __forceinline__ uint4 ld_weights(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// NT: tiles of 8 tokens.
template <int kType, bool kGated, int NT>
__global__ void __launch_bounds__(32 * kWarps, 2)
dense_rows_kernel(const RowsParams p) {
  constexpr int BT = 8 * NT;
  __shared__ uint32_t sums[kWarps][2][NT][4][32];
  extern __shared__ __align__(16) uint8_t walk_mem[];
  const DenseJob& j = p.j;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const bool grouped = j.rows_per_expert != nullptr;
  pdl_trigger();
  pdl_wait();
  TileWalk walk = {};
  int total = p.f_tiles * p.t_tiles;
  if (grouped) {
    if (warp == 0) build_tile_walk<BT>(j.rows_per_expert, j.experts, p.f_tiles, walk_mem);
    __syncthreads();
    walk = tile_walk_at(walk_mem, j.experts);
    total = walk.total;
  }
  const int half = kGated ? j.n >> 1 : 16;        // from the tile's first 16 weight rows to its other 16
  const int limit = kGated ? j.n >> 1 : j.n;      // features
  const uint8_t *w = reinterpret_cast<const uint8_t*>(j.w), *x = reinterpret_cast<const uint8_t*>(j.x);
  int cursor = 0;
  for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
    TileInfo ti;
    if (grouped) {
      locate_tile<BT>(walk, tile, cursor, ti);
    } else {
      ti.e = 0;
      ti.n_tile = p.t_tiles == 1 ? tile : tile / p.t_tiles;
      ti.row0 = (tile - ti.n_tile * p.t_tiles) * BT;
      ti.valid = (int)(j.m - ti.row0 < BT ? j.m - ti.row0 : BT);
    }
    const int f0 = ti.n_tile * (kGated ? 16 : 32);
    // this lane's weight rows: g and g + 8 of both sixteens; rows past the end read the last one, and are not stored
    const uint8_t* wr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = f0 + g + 8 * (i & 1);
      const int row = kGated ? min(f, limit - 1) + (i >> 1) * half : min(f + (i >> 1) * half, limit - 1);
      wr[i] = w + ((int64_t)ti.e * j.n + row) * p.w_pitch;
    }
    const uint8_t* xr[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
      xr[i] = x + min((int64_t)ti.row0 + min(g + 8 * i, ti.valid - 1), j.m - 1) * p.x_pitch;
    uint32_t acc[2][NT][4] = {};
    uint4 a[2][4];
    auto load = [&](int at) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = at + 64 * s + 16 * q;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[s][i] = k < p.k_bytes ? ld_weights(wr[i] + k) : make_uint4(0, 0, 0, 0);
      }
    };
    int at = warp * kUnit;
    if (at < p.k_bytes) load(at);
    for (; at < p.k_bytes; at += kWarps * kUnit) {
      uint4 b[2][NT], c[2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int k = at + 64 * s + 16 * q;
#pragma unroll
        for (int i = 0; i < NT; ++i) b[s][i] = k < p.k_bytes ? *reinterpret_cast<const uint4*>(xr[i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[s][i] = a[s][i];
      }
      if (at + kWarps * kUnit < p.k_bytes) load(at + kWarps * kUnit);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            mma<kType>(acc[h][i], c[s][2 * h].x, c[s][2 * h + 1].x, c[s][2 * h].y, c[s][2 * h + 1].y, b[s][i].x, b[s][i].y);
            mma<kType>(acc[h][i], c[s][2 * h].z, c[s][2 * h + 1].z, c[s][2 * h].w, c[s][2 * h + 1].w, b[s][i].z, b[s][i].w);
          }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[warp][h][i][r][lane] = acc[h][i][r];
    __syncthreads();
    auto sum = [&](int h, int f, int t) {   // of feature f (of 16) and token t
      const int r = (f >> 3) * 2 + (t & 1), l = (f & 7) * 4 + ((t & 7) >> 1);
      if (kType == kDenseI8) {
        int v = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) v += (int)sums[i][h][t >> 3][r][l];
        return (float)v;
      }
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) v += __uint_as_float(sums[i][h][t >> 3][r][l]);
      return v;
    };
    auto value = [&](int h, int f, int t) {   // with scales and bias
      float v = sum(h, f, t);
      const int64_t at = (int64_t)ti.e * j.n + f0 + f + h * half;
      if (kType == kDenseI8) v = v * j.x_scale[ti.row0 + t] * j.w_scale[at];
      if (j.bias != nullptr) v += load_bias(j.bias, j.bias_f16, at);
      return v;
    };
    for (int i = threadIdx.x; i < (kGated ? 16 : 32) * BT; i += 32 * kWarps) {
      const int f = i & 15, h = kGated ? 0 : (i >> 4) & 1, t = i >> (kGated ? 4 : 5);
      const int64_t row = (int64_t)ti.row0 + t;
      if (t >= ti.valid || row >= j.m || f0 + f + (kGated ? 0 : h * half) >= limit) continue;
      if (kGated) {
        const float gate = value(0, f, t), up = value(1, f, t);
        if (j.pre != nullptr) {
          j.pre[row * j.n + f0 + f] = gate;
          j.pre[row * j.n + half + f0 + f] = up;
        }
        store_as(j.d, j.d_dtype, row * j.d_stride + f0 + f, gated_product(gate, up, j.clamp));
      } else {
        store_as(j.d, j.d_dtype, row * j.d_stride + f0 + f + h * half, value(h, f, t));
      }
    }
    if (tile + (int)gridDim.x < total) __syncthreads();   // the sums are read before they are written again
  }
}

template <int kType, bool kGated, int NT>
int launch(const RowsParams& p, cudaStream_t st) {
  constexpr int BT = 8 * NT;
  const DenseJob& j = p.j;
  const size_t smem = j.rows_per_expert != nullptr ? tile_walk_bytes(j.experts) : 0;
  const int64_t tiles = ((j.m + BT - 1) / BT + (j.rows_per_expert != nullptr ? std::min<int64_t>(j.m, j.experts) : 0)) * p.f_tiles;
  int64_t grid = (j.max_ctas > 0 ? std::min(j.max_ctas, sm_count()) : sm_count()) * 2;
  grid = std::max<int64_t>(1, std::min(grid, tiles));
  B200_LAUNCHED("dense_rows_kernel", launch_pdl(j.early, dense_rows_kernel<kType, kGated, NT>, dim3((unsigned)grid), dim3(32 * kWarps),
                                                smem, st, p));
  return B200MOE_OK;
}
template <int kType, bool kGated>
int launch_tokens(RowsParams& p, cudaStream_t st) {
  const int64_t rows = p.j.rows_hint > 0 && p.j.rows_hint < p.j.m ? p.j.rows_hint : p.j.m;
  const bool eight = (rows + p.j.experts - 1) / p.j.experts <= (p.j.rows_per_expert != nullptr ? 4 : 8);
  p.t_tiles = (int)((p.j.m + (eight ? 7 : 15)) / (eight ? 8 : 16));
  return eight ? launch<kType, kGated, 1>(p, st) : launch<kType, kGated, 2>(p, st);
}

}  // namespace

int dense_rows(const DenseJob& j, cudaStream_t st) {
  RowsParams p = {};
  p.j = j;
  const int size = j.type == kDenseI8 ? 1 : 2;
  p.k_bytes = j.k * size;
  p.x_pitch = j.x_stride * size;
  p.w_pitch = j.w_stride * size;
  p.f_tiles = j.gated ? (j.n / 2 + 15) / 16 : (j.n + 31) / 32;
  if (j.type == kDenseI8) return j.gated ? launch_tokens<kDenseI8, true>(p, st) : launch_tokens<kDenseI8, false>(p, st);
  if (!j.gated) return fail(B200MOE_E_UNSUPPORTED, "dense_rows: 16-bit products are gated");
  return j.type == kDenseBf16 ? launch_tokens<kDenseBf16, true>(p, st) : launch_tokens<kDenseF16, true>(p, st);
}

}  // namespace b200moe
