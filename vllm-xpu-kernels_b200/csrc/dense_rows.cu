// Products of a few rows with int8 weights, or with the 16-bit weights of a gated block: every weight is read once.
//
//   int8:   D[m, n] = (sum_k x[m, k] w[n, k]) * x_scale[m] * w_scale[n] (+ bias[n])      sums in int32, exact
//   gated:  D[m, i] = silu(g) * u, g and u the products with rows i and I + i of W          sums in fp32
//
// The order of k inside a sum is free as long as both operands share it, so a lane takes 16 consecutive bytes of a weight row
// (and of a token's) for the four words that mma.sync wants of it, two instructions for 64 bytes of a row, and no shuffle or
// repacking stands between the load and the product.  A block owns 16 weight rows (gated: 8 gates and their 8 ups) and up to 16
// tokens at a time; a team of its eight warps (all of them for few tiles or long rows, one or two for many short ones) shares the
// rows' bytes out, 128 at a time (a unit), and adds its sums up in shared memory.
//
// What bounds it is the weights' way from HBM, so what counts is bytes in flight: every lane has its own slots in shared memory, which
// cp.async fills several units ahead, across tiles, and which only this lane reads again, so that nothing but its own wait stands
// between the two.
//
// All blocks ask L2 for the same lines of the tokens at the same time, unit after unit.  Where that is few lines it is what takes longest: one
// token of 7168 x 2048 (gated, bfloat16) 18.6 us when lanes without a token of their own read the last one, sixteen tokens 13.9.  So
// lanes without a token bring nothing, and tiles of eight go through L1: 10.8 us, 5.1 TB/s.
#include "dense.cuh"

namespace b200moe {
namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 128;      // bytes of a row that a warp takes at a time

struct RowsParams {
  DenseJob j;
  int64_t x_pitch, w_pitch;     // bytes from row to row
  int k_bytes;                  // bytes of a row
  int units;                    // of a row
  int f_tiles;                  // tiles of 16 weight rows (gated: 8 and 8)
  int t_tiles;                  // one set of weights: tiles of tokens
  int team;                     // warps of a tile: 1, 2, 4 or 8
  int panel_pitch;              // bytes from row to row of a panel
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
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, bool there) {   // (zeros where there is nothing)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
// ... of a token, which the SM's other tiles read as well.  Tiles of eight have it, 8 x 2880 x 2880 3.4 us, 3.6 without, 4 x 2048 x 1408 gated 4.0
// and 4.3; tiles of sixteen have too many lines for L1, 16 x 4096 x 4096 6.5 us, 5.7 without.
__device__ __forceinline__ void copy16_token(uint32_t to, const uint8_t* from, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// The codes of up to eight rows, by the whole block: 8, 4, 2 or 1 warps a row.
__device__ __forceinline__ void quantise_rows(const RowsParams& p, uint8_t* codes, float* scales, float* part) {
  const DenseJob& j = p.j;
  const int m = (int)j.m, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int each = m == 1 ? 8 : m == 2 ? 4 : m <= 4 ? 2 : 1, row = warp / each, threads = 32 * each, t = (warp % each) * 32 + lane;
  const int size = j.x_dtype == B200MOE_F32 ? 4 : 2, per = 16 / size, pieces = j.k / per;
  const uint8_t* x = reinterpret_cast<const uint8_t*>(j.x) + (int64_t)min(row, m - 1) * j.x_stride * size;
  auto values = [&](int c, float (&v)[8]) {
    const vec16 a = ld16(x + (int64_t)c * 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (j.x_dtype == B200MOE_F32) v[i] = i < 4 ? __uint_as_float(a.w[i & 3]) : 0.f;
      else if (j.x_dtype == B200MOE_BF16) v[i] = __uint_as_float(i & 1 ? a.w[i / 2] & 0xffff0000u : a.w[i / 2] << 16);
      else v[i] = __half2float(reinterpret_cast<const __half*>(&a)[i]);
    }
  };
  float amax = 0.f;
#pragma unroll 4
  for (int c = t; c < pieces; c += threads) {
    float v[8];
    values(c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  if (lane == 0) part[warp] = amax;
  __syncthreads();
  for (int i = 0; i < each; ++i) amax = max_nan(amax, part[warp / each * each + i]);
  auto write = [&](const auto& s) {
    if (row >= m) return;
    if (t == 0) scales[row] = s.scale;
#pragma unroll 4
    for (int c = t; c < pieces; c += threads) {
      float v[8];
      values(c, v);
      uint32_t w[2];
      s.template codes<2>(v, w);
      if (per == 8) *reinterpret_cast<uint2*>(codes + row * p.panel_pitch + c * 8) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(codes + row * p.panel_pitch + c * 4) = w[0];
    }
  };
  if (j.x_dtype == B200MOE_F16) write(Int8Scale<__half>(amax));
  else write(Int8Scale<float>(amax));
  __syncthreads();
}

template <int NT>
struct alignas(128) Fixed {
  // (Once, with a second barrier: sums of two tiles left room for one block an SM, 5 rows each of 128 experts of 2048 x 1536 gated 97 us, 75 so.)
  uint32_t sums[kWarps][NT][4][32];
  float x_scales[8], part[kWarps];      // of rows that are quantised on the way
};

// NT: tiles of 8 tokens.  kAhead: units in flight.  kCodes: tokens come from a panel of the codes that the block makes of them, not
// beside the weights through the lanes' slots.
template <int kType, bool kGated, int NT, int kAhead, bool kCodes>
__global__ void __launch_bounds__(32 * kWarps, 2)
dense_rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int BT = 8 * NT;
  constexpr int kSlots = 4 + (kCodes ? 0 : 2 * NT);      // 16-byte pieces of a unit that a lane has
  extern __shared__ __align__(128) uint8_t dyn[];
  Fixed<NT>& fixed = *reinterpret_cast<Fixed<NT>*>(dyn);
  auto& sums = fixed.sums;
  const DenseJob& j = p.j;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int team = warp / p.team, in_team = warp - team * p.team, teams = kWarps / p.team;   // (p.team divides kWarps)
  const bool grouped = !kCodes && j.rows_per_expert != nullptr;
  uint8_t* const behind = dyn + sizeof(Fixed<NT>) + kWarps * kAhead * kSlots * 512;      // the panel, or the tile walk
  const uint32_t ring = ptx::smem_u32(dyn) + sizeof(Fixed<NT>) + warp * kAhead * kSlots * 512 + lane * 16;
  const uint32_t panel = ptx::smem_u32(behind) + min(g, (int)min(j.m, (int64_t)8) - 1) * p.panel_pitch + 16 * q;
  const int half = kGated ? j.n >> 1 : 8;         // from the tile's first 8 weight rows to its other 8
  const int limit = kGated ? j.n >> 1 : j.n;      // features
  const uint8_t *w = reinterpret_cast<const uint8_t*>(j.w), *x = reinterpret_cast<const uint8_t*>(j.x);
  TileWalk walk = {};
  int total = p.f_tiles * p.t_tiles;
  const int first_tile = team * gridDim.x + blockIdx.x, step = teams * gridDim.x;   // (neighbouring blocks: neighbouring tiles)
  auto locate = [&](int tile, int& cursor, TileInfo& ti) {
    if (grouped) {
      locate_tile<BT>(walk, tile, cursor, ti);
      return;
    }
    ti.e = 0;
    ti.n_tile = p.t_tiles == 1 ? tile : tile / p.t_tiles;
    ti.row0 = (tile - ti.n_tile * p.t_tiles) * BT;
    ti.valid = (int)(j.m - ti.row0 < BT ? j.m - ti.row0 : BT);
  };
  pdl_trigger();
  if (grouped) {
    pdl_wait();
    if (warp == 0) build_tile_walk<BT>(j.rows_per_expert, j.experts, p.f_tiles, behind);
    __syncthreads();
    walk = tile_walk_at(behind, j.experts);
    total = walk.total;
  }

  // where the copies are: tile, unit and addresses of this lane's rows in it
  int next_tile = first_tile, next_unit = in_team, next_cursor = 0;
  const uint8_t *wr[2], *xr[NT];
  auto at_tile = [&]() {
    if (next_tile >= total) return;
    TileInfo ti;
    locate(next_tile, next_cursor, ti);
    // Weight rows past the end are the last one, and not stored.  Tokens that a tile lacks are not brought: what lies in their slots
    // makes sums that nobody reads.  (9 x 4096 x 4096 5.2 us, 9.2 with copies of the last token in their place.)
    const int f = ti.n_tile * (kGated ? 8 : 16) + g;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = kGated ? min(f, limit - 1) + i * half : min(f + i * half, limit - 1);
      wr[i] = w + ((int64_t)ti.e * j.n + row) * p.w_pitch + 16 * q;
    }
    if (!kCodes) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int64_t row = (int64_t)ti.row0 + g + 8 * i;
        xr[i] = g + 8 * i < ti.valid && row < j.m ? x + row * p.x_pitch + 16 * q : nullptr;
      }
    }
  };
  auto copy = [&](uint32_t slot) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k = next_unit * kUnit + 64 * s;
      const bool there = k + 16 * q < p.k_bytes;
#pragma unroll
      for (int i = 0; i < 2; ++i) copy16(slot + (2 * s + i) * 512, wr[i] + k, there);
      if (!kCodes) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if (xr[i] == nullptr) continue;
          if (NT == 1) copy16_token(slot + (4 + NT * s + i) * 512, xr[i] + k, there);
          else copy16(slot + (4 + NT * s + i) * 512, xr[i] + k, there);
        }
      }
    }
    next_unit += p.team;
    if (next_unit < p.units) return;
    next_unit = in_team;
    next_tile += step;
    at_tile();
  };
  const bool mine = in_team < p.units;               // (a row of fewer units than warps)
  at_tile();
  if (!grouped) {
    // The first weights on their way to L2 while the kernel before this one ends.  (Only there: that kernel may be the one that
    // writes them, and L2 is where its writes are seen.)
    if (mine && next_tile < total && q == 0) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int k = (in_team + a * p.team) * kUnit;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (k < p.k_bytes) asm volatile("prefetch.global.L2 [%0];" ::"l"(wr[i] + k));
      }
    }
    pdl_wait();
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    if (mine && next_tile < total) copy(ring + a * kSlots * 512);
    commit();
  }
  if (kCodes) quantise_rows(p, behind, fixed.x_scales, fixed.part);

  // the outputs of this thread: one feature of the 8 (and of which 8), every some tokens
  const int tt = in_team * 32 + lane, f = tt & 7, h = kGated ? 0 : (tt >> 3) & 1;
  const int t0 = tt >> (kGated ? 3 : 4), t_step = 2 * p.team * (kGated ? 2 : 1);
  auto team_sync = [&]() {
    if (p.team == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(32 * p.team) : "memory");
  };
  int slot = 0, cursor = 0;
  for (int tile = first_tile; tile < total; tile += step) {
    TileInfo ti;
    locate(tile, cursor, ti);
    // scales and biases are on their way while the weights are
    const int feat = ti.n_tile * (kGated ? 8 : 16) + f + h * half;
    const int64_t at = (int64_t)ti.e * j.n + feat;
    float ws[2] = {1.f, 1.f}, bias[2] = {0.f, 0.f};
    if (feat < limit) {
#pragma unroll
      for (int i = 0; i < (kGated ? 2 : 1); ++i) {
        if (kType == kDenseI8) ws[i] = j.w_scale[at + i * half];
        if (j.bias != nullptr) bias[i] = load_bias(j.bias, j.bias_f16, at + i * half);
      }
    }
    float x_scale = 1.f;       // of the token that the lane's number says
    if (kType == kDenseI8 && !kCodes && lane < ti.valid && ti.row0 + (int64_t)lane < j.m) x_scale = j.x_scale[ti.row0 + (int64_t)lane];
    uint32_t acc[NT][4] = {};
    for (int unit = in_team; unit < p.units; unit += p.team) {
      const uint32_t from = ring + slot * kSlots * 512;
      wait_but<kAhead - 1>();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint4 a = ptx::lds128(from + 2 * s * 512), b = ptx::lds128(from + (2 * s + 1) * 512);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint4 t = kCodes ? ptx::lds128(panel + unit * kUnit + 64 * s) : ptx::lds128(from + (4 + NT * s + i) * 512);
          mma<kType>(acc[i], a.x, b.x, a.y, b.y, t.x, t.y);
          mma<kType>(acc[i], a.z, b.z, a.w, b.w, t.z, t.w);
        }
      }
      // (the slot has been read: the products above took its values)
      if (next_tile < total) copy(from);
      commit();
      if (++slot == kAhead) slot = 0;
    }
    team_sync();               // the sums of the tile before have been read
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[warp][i][r][lane] = acc[i][r];
    team_sync();
    for (int t = t0; t - t0 < ti.valid; t += t_step) {      // (every lane as often)
      const int64_t row = (int64_t)ti.row0 + t;
      const float xs = kType != kDenseI8 ? 1.f : kCodes ? fixed.x_scales[t & 7] : __shfl_sync(0xffffffffu, x_scale, t & (BT - 1));
      if (feat >= limit || t >= ti.valid || row >= j.m) continue;
      auto value = [&](int i) {
        const int r = 2 * (h + i) + (t & 1), l = f * 4 + ((t & 7) >> 1);
        if (kType == kDenseI8) {
          int sum = 0;
          for (int n = 0; n < p.team; ++n) sum += (int)sums[team * p.team + n][t >> 3][r][l];
          return (float)sum * xs * ws[i] + bias[i];
        }
        float v = 0.f;
        for (int n = 0; n < p.team; ++n) v += __uint_as_float(sums[team * p.team + n][t >> 3][r][l]);
        return v + bias[i];
      };
      float v = value(0);
      if (kGated) {
        const float up = value(1);
        if (j.pre != nullptr) {
          j.pre[row * j.n + feat] = v;
          j.pre[row * j.n + half + feat] = up;
        }
        v = gated_product(v, up, j.clamp);
      }
      store_as(j.d, j.d_dtype, row * j.d_stride + feat, v);
    }
  }
}

template <int kType, bool kGated, int NT, int kAhead, bool kCodes>
int launch(RowsParams& p, cudaStream_t st) {
  constexpr int BT = 8 * NT;
  const DenseJob& j = p.j;
  auto kern = dense_rows_kernel<kType, kGated, NT, kAhead, kCodes>;
  static SmemConfig configured;
  if (int rc = configured.ensure(kern)) return rc;
  const size_t smem = sizeof(Fixed<NT>) + (size_t)kWarps * kAhead * (4 + (kCodes ? 0 : 2 * NT)) * 512 +
                      (kCodes ? (size_t)j.m * p.panel_pitch : j.rows_per_expert != nullptr ? tile_walk_bytes(j.experts) : 0);
  const int64_t rows = j.rows_hint > 0 && j.rows_hint < j.m ? j.rows_hint : j.m;
  const int64_t tiles = j.rows_per_expert != nullptr ? (rows / BT + std::min<int64_t>(rows, j.experts)) * p.f_tiles
                                                     : (int64_t)p.t_tiles * p.f_tiles;
  const int64_t blocks = j.max_ctas > 0 ? std::min(j.max_ctas, 2 * sm_count()) : 2 * sm_count();
  // Warps of a team: rounds of tiles times the units of a warp, and as much as kTileCost units for what a tile costs besides.
  constexpr int kTileCost = 4;
  int64_t best = -1;
  for (int team = kWarps; team >= 1; team /= 2) {
    const int64_t teams = blocks * (kWarps / team), rounds = (tiles + teams - 1) / teams;
    const int64_t cost = rounds * ((p.units + team - 1) / team + kTileCost);
    if (best < 0 || cost < best) { best = cost; p.team = team; }
  }
  // Teams that have a tile are spread over all blocks (14336 weight rows of 4096, 8 tokens 11.6 us, 12.2 packed; 16 tokens 17.8 and 21.4), unless
  // packed they leave a block on each SM at the most and are tiles of eight, whose tokens they then share in L1 (6144 of 2048, 8 tokens 4.3 and 3.9).
  const int64_t packed = (tiles * p.team + kWarps - 1) / kWarps;
  const int64_t grid = std::max<int64_t>(1, std::min(blocks, NT == 1 && packed <= sm_count() ? packed : tiles));
  B200_LAUNCHED("dense_rows_kernel", launch_pdl(j.early, kern, dim3((unsigned)grid), dim3(32 * kWarps), smem, st, p));
  return B200MOE_OK;
}
template <int kType, bool kGated>
int launch_tokens(RowsParams& p, cudaStream_t st) {
  const DenseJob& j = p.j;
  const bool one_set = j.rows_per_expert == nullptr;
  const int64_t rows = j.rows_hint > 0 && j.rows_hint < j.m ? j.rows_hint : j.m;
  const bool eight = (rows + j.experts - 1) / j.experts <= (one_set ? 8 : 6);
  p.t_tiles = (int)((j.m + (eight ? 7 : 15)) / (eight ? 8 : 16));
  return eight ? launch<kType, kGated, 1, 4, false>(p, st) : launch<kType, kGated, 2, 3, false>(p, st);
}

}  // namespace

bool dense_rows_quantises(int64_t rows, int k) { return rows <= 8 && rows * k <= kQuantValues; }

int dense_rows(const DenseJob& j, cudaStream_t st) {
  RowsParams p = {};
  p.j = j;
  const int size = j.type == kDenseI8 ? 1 : 2;
  p.k_bytes = j.k * size;
  p.units = (p.k_bytes + kUnit - 1) / kUnit;
  p.x_pitch = j.x_stride * size;
  p.w_pitch = j.w_stride * size;
  p.panel_pitch = p.units * kUnit + 64;      // (half of the banks from row to row)
  p.f_tiles = j.gated ? (j.n / 2 + 7) / 8 : (j.n + 15) / 16;
  if (j.type == kDenseI8 && j.x_dtype != B200MOE_I8) {
    p.t_tiles = 1;
    return launch<kDenseI8, false, 1, 4, true>(p, st);
  }
  if (j.type == kDenseI8) return j.gated ? launch_tokens<kDenseI8, true>(p, st) : launch_tokens<kDenseI8, false>(p, st);
  if (!j.gated) return fail(B200MOE_E_UNSUPPORTED, "dense_rows: 16-bit products are gated");
  return j.type == kDenseBf16 ? launch_tokens<kDenseBf16, true>(p, st) : launch_tokens<kDenseF16, true>(p, st);
}

}  // namespace b200moe
