// Products of many rows on the sm_100a tensor cores: int8 operands with a scale for each row of either (one set of weights, or a
// set per expert's rows), the 16-bit gated product, and the plain 16-bit products that its gradients are.
//
//   D[m, n] = (sum_k X[m, k] W[n, k]) * x_scale[m] * w_scale[n] (+ bias[n])     kind::i8, sums in int32
//   D[m, i] = silu(g) * u,  g = X W[i]^T, u = X W[I + i]^T                      kind::i8 or kind::f16 (sums in fp32)
//   D = A B^T                                                                  kind::f16, either operand also stored by column
//
// A cluster of two CTAs shares a tile of 256 rows x up to 256 weight rows: each brings its 128 rows of X and one half of the
// weight rows (128 bytes of k at a time, 32 KB a CTA) into its shared memory by TMA, the even CTA issues tcgen05.mma with
// cta_group::2 for both, and each CTA's tensor memory receives its own rows' 128 x 256 sums, twice, so that the epilogue of a tile
// overlaps the products of the next.  Rows of X lie on the lanes: a thread of the epilogue owns one row, its
// scale is one register, and gate and up of a gated tile (128 gates and their 128 ups are the tile's 256 weight rows) meet in one thread.
//
// How wide a tile is follows from what the pairs have to do (tile_width below): 256 weight rows share the rows of X best, fewer leave
// fewer pairs idle in the last round.  Of a tile with few rows only those are brought in (what lies behind them in shared
// memory makes sums of rows that nobody stores).
//
//   warps 0 and 10: TMA producers of W and X;  warp 1: MMA issuer (even CTA), tensor memory;  warps 2-9: epilogue, every second 32
//   columns each four
//
// Every wait on an mbarrier is bounded, as in the grouped GEMMs (gemm_tc.cu).
#include <algorithm>

#include "dense.cuh"
#include "dense_tc.cuh"

namespace b200moe {
namespace {

constexpr int kEpi = 8;                           // epilogue warps
constexpr int kThreads = 96 + 32 * kEpi;
constexpr int kTile = 256;                        // rows of X of a pair's tile, and the most rows of W
constexpr int kOperand = 128 * 128;               // bytes of an operand in a stage: 128 rows of 128 bytes
constexpr int kRing = 6 * 2 * kOperand;           // bytes of all stages
constexpr int kMaxStages = 9;                     // (of tiles of 64 weight rows)

enum Form { kPlain, kScaled, kGated };

struct TcDense {
  const float* x_scale;
  const float* w_scale;
  const void* bias;
  void* d;
  float* pre;
  const int32_t* rows_per_expert;
  int32_t* status;
  int64_t m, d_stride;
  int n, experts;
  int num_kb;
  int m_tiles, n_tiles;
  int width;                // weight rows of a tile: a multiple of 32, gated of 64
  int stages, stage_bytes, w_bytes;   // w_bytes: of a CTA's weight rows in a stage
  int x_box;                // rows that a load of X brings
  uint32_t idesc;
  b200moe_dtype d_dtype;
  int bias_f16;
  int d_wide, pre_wide;     // bytes of a store: 32, 16, or 0 for value by value
  float clamp;
};

struct Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full[2];
  uint64_t acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  alignas(16) float scale[kEpi][128];    // per epilogue warp: of the weight rows that it has columns of
  alignas(16) float bias[kEpi][128];
  alignas(16) uint8_t narrow[kEpi][32 * 32];   // 32 bytes of each of a warp's rows, for stores that are not aligned
  alignas(16) uint8_t walk[tile_walk_bytes(kMaxExperts)];
};
constexpr size_t kSmem = 1024 + (size_t)kRing + sizeof(Ctrl);
static_assert(kSmem <= kMaxSmem, "shared memory");

// Tiles of one set of weights: eight tiles of rows side by side, so that pairs that run at the same time share both operands in L2.
__device__ __forceinline__ void locate_dense(const TcDense& p, int t, TileInfo& ti) {
  const int group = 8 * p.n_tiles, g = t / group, in = t - g * group, first = 8 * g;
  const int rows = min(8, p.m_tiles - first);
  ti.e = 0;
  ti.n_tile = in / rows;
  ti.m_tile = first + in - ti.n_tile * rows;
  ti.row0 = ti.m_tile * kTile;
  ti.valid = (int)(p.m - ti.row0 < kTile ? p.m - ti.row0 : kTile);
}

// A warp's 32 rows x 32 columns, a row a lane, of which the first `rows` rows and the columns below `limit` exist: in pieces of 32 or
// 16 bytes where they are aligned, else through shared memory, so that lanes that store together are neighbours in a row.
// (Odd row lengths, value by value from the row's own lane: 1001 x 2011 x 2032 48 us.)
__device__ __forceinline__ void store_32(void* d, b200moe_dtype t, int64_t row_at, int64_t stride, int rows, int col, int limit,
                                         const float (&v)[32], int wide, uint32_t narrow) {
  const int lane = threadIdx.x & 31;
  if (t == B200MOE_F32) {
    if (wide != 0) {
      float* to = reinterpret_cast<float*>(d) + row_at + lane * stride + col;
      if (lane >= rows) return;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        if (wide == 32) {
          if (col + i < limit)
            ptx::stg256(to + i, {__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3]),
                                 __float_as_uint(v[i + 4]), __float_as_uint(v[i + 5]), __float_as_uint(v[i + 6]), __float_as_uint(v[i + 7])});
        } else {
#pragma unroll
          for (int k = i; k < i + 8; k += 4)
            if (col + k < limit) *reinterpret_cast<float4*>(to + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
        }
      }
      return;
    }
    float* to = reinterpret_cast<float*>(d) + row_at + col;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      ptx::sts128(narrow + lane * 32, make_uint4(__float_as_uint(v[i]), __float_as_uint(v[i + 1]), __float_as_uint(v[i + 2]), __float_as_uint(v[i + 3])));
      ptx::sts128(narrow + lane * 32 + 16, make_uint4(__float_as_uint(v[i + 4]), __float_as_uint(v[i + 5]), __float_as_uint(v[i + 6]), __float_as_uint(v[i + 7])));
      __syncwarp();
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int r = 4 * n + (lane >> 3), c = i + (lane & 7);
        if (r < rows && col + c < limit) to[r * stride + c] = ptx::lds32f(narrow + r * 32 + (lane & 7) * 4);
      }
      __syncwarp();
    }
    return;
  }
  const int f16 = t == B200MOE_F16;
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = (uint32_t)bits16(v[2 * i], f16) | (uint32_t)bits16(v[2 * i + 1], f16) << 16;
  if (wide != 0) {
    uint16_t* to = reinterpret_cast<uint16_t*>(d) + row_at + lane * stride + col;
    if (lane >= rows) return;
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      if (wide == 32) {
        if (col + 2 * i < limit) ptx::stg256(to + 2 * i, {w[i], w[i + 1], w[i + 2], w[i + 3], w[i + 4], w[i + 5], w[i + 6], w[i + 7]});
      } else {
#pragma unroll
        for (int k = i; k < i + 8; k += 4)
          if (col + 2 * k < limit) *reinterpret_cast<uint4*>(to + 2 * k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
      }
    }
    return;
  }
  uint16_t* to = reinterpret_cast<uint16_t*>(d) + row_at + col;
#pragma unroll
  for (int i = 0; i < 16; i += 8) {
    ptx::sts128(narrow + lane * 32, make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
    ptx::sts128(narrow + lane * 32 + 16, make_uint4(w[i + 4], w[i + 5], w[i + 6], w[i + 7]));
    __syncwarp();
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const int r = 2 * n + (lane >> 4), c = 2 * i + (lane & 15);
      if (r < rows && col + c < limit) to[r * stride + c] = ptx::lds16(narrow + r * 32 + (lane & 15) * 2);
    }
    __syncwarp();
  }
}

// kXMn, kWMn: the operand is stored by column (its rows' index is the dense one): 16-bit types, two boxes of 64 rows x 64 k.
template <bool kI8, int kForm, bool kXMn, bool kWMn>
__global__ void __launch_bounds__(kThreads, 1)
dense_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const TcDense p) {
  constexpr int kPerKb = kI8 ? 128 : 64;
  constexpr bool kScales = kI8 || kForm == kScaled;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem + kRing);
  volatile int* abort_flag = &ctrl->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cta = ptx::cluster_ctarank();
  const int walker = (int)ptx::cluster_id_x(), walkers = (int)ptx::cluster_count_x();
  const bool grouped = kI8 && p.rows_per_expert != nullptr;

  if (warp == 0) {
    pdl_wait();
    if (grouped) build_tile_walk<kTile>(p.rows_per_expert, p.experts, p.n_tiles, ctrl->walk);
    if (lane == 0) {
      ptx::prefetch_tensormap(&tmap_x);
      ptx::prefetch_tensormap(&tmap_w);
    }
  } else if (warp == 1) {
    ptx::tmem_alloc_pair(&ctrl->tmem_base, 512);
    ptx::tmem_relinquish_pair();
  } else if (warp == 2 && lane == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      ptx::mbar_init(&ctrl->full[s], 1);
      ptx::mbar_init(&ctrl->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&ctrl->acc_full[a], 1);
      ptx::mbar_init(&ctrl->acc_empty[a], 2 * kEpi);   // the epilogue warps of both CTAs
    }
    ctrl->abort_flag = 0;
    ptx::fence_barrier_init();
  }
  pdl_wait();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();   // both CTAs' barriers and tensor memory exist before either signals the other
  ptx::tc_fence_after();

  const uint32_t tmem_base = ctrl->tmem_base;
  TileWalk walk = {};
  int total = p.m_tiles * p.n_tiles;
  if (grouped) {
    walk = tile_walk_at(ctrl->walk, p.experts);
    total = walk.total;
  }
  const int half = p.n >> 1;
  int cursor = 0;
  auto locate = [&](int t, TileInfo& ti) {
    if (grouped) locate_tile<kTile>(walk, t, cursor, ti);
    else locate_dense(p, t, ti);
  };

  if (warp == 0 || warp == 2 + kEpi) {
    // ------------------------------ TMA producers -----------------------------
    // W by the one, X by the other: a load costs its thread some 100 cycles, a K block of a tile with few rows hardly more
    // in the tensor cores.
    const bool is_w = warp == 0;
    if (ptx::elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      const uint32_t full0 = ptx::smem_u32(&ctrl->full[0]), empty0 = ptx::smem_u32(&ctrl->empty[0]);
      const uint32_t bar0 = ptx::map_to_cta(full0, 0);   // the even CTA's barriers count the bytes of both CTAs
      const uint32_t st0 = ptx::smem_u32(smem);
      uint32_t st = st0;
      auto first_row = [&](const TileInfo& ti) {   // of W, of this CTA
        return kForm == kGated ? (cta == 0 ? 0 : half) + ti.n_tile * (p.width >> 1) : ti.n_tile * p.width + (int)cta * (p.width >> 1);
      };
      for (int t = walker; t < total && ok; t += walkers) {
        TileInfo ti;
        locate(t, ti);
        // rows past the end are filled with zeros
        const int row = ti.row0 + (int)cta * 128;
        const int n0 = first_row(ti);
        // loads of X in either CTA: as many as the tile's rows take
        auto boxes = [&](int c) {
          const int rows = min(max(ti.valid - 128 * c, 0), 128);
          return kXMn ? 2 : (rows + p.x_box - 1) / p.x_box;
        };
        const int mine = boxes((int)cta);
        const uint32_t box_bytes = kXMn ? kOperand / 2 : p.x_box * 128;
        const uint32_t tx = 2 * p.w_bytes + (boxes(0) + boxes(1)) * box_bytes;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!ptx::paced::mbar_wait_s(empty0 + 8 * s, ph, abort_flag)) { ok = false; break; }
          if (is_w && cta == 0) ptx::mbar_expect_tx_s(full0 + 8 * s, tx);
          const uint32_t bar = bar0 + 8 * s;
          const int k0 = kb * kPerKb;
          if (!is_w) {
            if (kXMn) {
              ptx::tma_load_2d_pair(st, &tmap_x, bar, row, k0);
              ptx::tma_load_2d_pair(st + kOperand / 2, &tmap_x, bar, row + 64, k0);
            } else {
              for (int b = 0; b < mine; ++b) ptx::tma_load_2d_pair(st + b * box_bytes, &tmap_x, bar, k0, row + b * p.x_box);
            }
          } else if (kWMn) {
            ptx::tma_load_3d_pair(st + kOperand, &tmap_w, bar, n0, k0, ti.e);
            if (p.w_bytes > kOperand / 2) ptx::tma_load_3d_pair(st + kOperand + kOperand / 2, &tmap_w, bar, n0 + 64, k0, ti.e);
          } else {
            ptx::tma_load_3d_pair(st + kOperand, &tmap_w, bar, k0, n0, ti.e);
          }
          st += p.stage_bytes;
          if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1; st = st0; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------ MMA issuer (even CTA) -----------------------
    if (cta == 0 && ptx::elect_one()) {
      uint32_t s = 0, ph = 0, acc_it = 0;
      bool ok = true;
      const uint32_t full0 = ptx::smem_u32(&ctrl->full[0]), empty0 = ptx::smem_u32(&ctrl->empty[0]);
      const uint32_t acc_full0 = ptx::smem_u32(&ctrl->acc_full[0]), acc_empty0 = ptx::smem_u32(&ctrl->acc_empty[0]);
      // 16-byte units between the K steps of an operand: 32 bytes of its rows, or 16 of the k that are its rows
      constexpr int kXStep = kXMn ? 2048 / 16 : 2, kWStep = kWMn ? 2048 / 16 : 2;
      const uint64_t xdesc0 = ptx::make_smem_desc(ptx::smem_u32(smem), kXMn ? 8192u : 16u, 1024);
      const uint64_t wdesc0 = ptx::make_smem_desc(ptx::smem_u32(smem) + kOperand, kWMn ? 8192u : 16u, 1024);
      uint64_t xdesc = xdesc0, wdesc = wdesc0;
      const uint64_t stage16 = p.stage_bytes >> 4;
      for (int t = walker; t < total && ok; t += walkers) {
        const uint32_t a = acc_it & 1;
        if (!ptx::mbar_wait_s(acc_empty0 + 8 * a, ((acc_it >> 1) & 1) ^ 1, abort_flag)) break;
        ptx::tc_fence_after();
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!ptx::mbar_wait_s(full0 + 8 * s, ph, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          if (kI8) ptx::umma_i8_pair_block<kXStep, kWStep>(tmem_base + a * kTile, xdesc, wdesc, p.idesc, kb > 0 ? 1u : 0u);
          else ptx::umma_f16_pair_block<kXStep, kWStep>(tmem_base + a * kTile, xdesc, wdesc, p.idesc, kb > 0 ? 1u : 0u);
          ptx::umma_commit_pair(empty0 + 8 * s);
          xdesc += stage16;
          wdesc += stage16;
          if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1; xdesc = xdesc0; wdesc = wdesc0; }
        }
        if (ok) { ptx::umma_commit_pair(acc_full0 + 8 * a); ++acc_it; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue ----------------------------------
    const int quarter = warp & 3, side = (warp - 2) >> 2;
    const uint32_t lane_sel = (uint32_t)(quarter * 32) << 16;
    const uint32_t acc_empty0 = ptx::map_to_cta(ptx::smem_u32(&ctrl->acc_empty[0]), 0);
    const uint32_t scale0 = ptx::smem_u32(ctrl->scale[warp - 2]), bias0 = ptx::smem_u32(ctrl->bias[warp - 2]);
    const uint32_t narrow = ptx::smem_u32(ctrl->narrow[warp - 2]);
    uint32_t acc_it = 0;
    for (int t = walker; t < total; t += walkers) {
      TileInfo ti;
      locate(t, ti);
      const uint32_t a = acc_it & 1;
      const int row0 = (int)cta * 128 + quarter * 32;      // this warp's first row in the tile
      const int64_t first = (int64_t)ti.row0 + row0;
      const int rows = (int)min((int64_t)min(ti.valid - row0, 32), p.m - first);
      const int features = kForm == kGated ? p.width >> 1 : p.width, j0 = ti.n_tile * features;
      const int limit = kForm == kGated ? half : p.n;
      float xs = 1.f;
      if (kScales) {
        // the weight rows' scales and biases: every warp its own copy, so that no barrier couples the warps
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (gated: 32 gates, then their ups)
          const int c = 2 * (kForm == kGated ? i >> 1 : i) + side, f = j0 + 32 * c + lane;
          const bool there = 32 * c < features && f < limit;
          const int64_t at = (int64_t)ti.e * p.n + f + (kForm == kGated && (i & 1) ? half : 0);
          ptx::sts32f(scale0 + 128 * i + 4 * lane, there ? p.w_scale[at] : 0.f);
          ptx::sts32f(bias0 + 128 * i + 4 * lane, there && p.bias != nullptr ? load_bias(p.bias, p.bias_f16, at) : 0.f);
        }
        if (lane < rows) xs = p.x_scale[first + lane];
        __syncwarp();
      }
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&ctrl->acc_full[a], (acc_it >> 1) & 1, abort_flag))) {
        *abort_flag = 1;
        break;
      }
      ptx::tc_fence_after();
      const uint32_t acc = tmem_base + a * kTile + lane_sel;
      // sums as the product's values; `l`: the first one's place among the warp's scales
      auto scaled = [&](float (&f)[32], const uint32_t (&v)[32], int l) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          if (!kScales) {
            for (int k = 0; k < 4; ++k) f[i + k] = __uint_as_float(v[i + k]);
            continue;
          }
          const float4 ws = ptx::lds128f(scale0 + 4 * (l + i)), b = ptx::lds128f(bias0 + 4 * (l + i));
          f[i] = (float)(int)v[i] * xs * ws.x + b.x;
          f[i + 1] = (float)(int)v[i + 1] * xs * ws.y + b.y;
          f[i + 2] = (float)(int)v[i + 2] * xs * ws.z + b.z;
          f[i + 3] = (float)(int)v[i + 3] * xs * ws.w + b.w;
        }
      };
      if (rows > 0) {
#pragma unroll 1
        for (int c = side; 32 * c < features && j0 + 32 * c < limit; c += 2) {
          const int col = 32 * c, l = kForm == kGated ? 32 * (c & ~1) : 16 * (c & ~1);
          uint32_t g[32], u[kForm == kGated ? 32 : 1];
          __syncwarp();
          ptx::tmem_ld_32x32(acc + col, g);
          if (kForm == kGated) ptx::tmem_ld_32x32(acc + features + col, reinterpret_cast<uint32_t(&)[32]>(u));
          if (kForm == kGated) ptx::tmem_wait_ld(g, u);
          else ptx::tmem_wait_ld(g);
          float f[32];
          scaled(f, g, l);
          if (kForm == kGated) {
            float up[32];
            scaled(up, reinterpret_cast<uint32_t(&)[32]>(u), l + 32);
            if (p.pre != nullptr) {
              store_32(p.pre, B200MOE_F32, first * p.n, p.n, rows, j0 + col, limit, f, p.pre_wide, narrow);
              store_32(p.pre + half, B200MOE_F32, first * p.n, p.n, rows, j0 + col, limit, up, p.pre_wide, narrow);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = gated_product(f[i], up[i], p.clamp);
          }
          store_32(p.d, p.d_dtype, first * p.d_stride, p.d_stride, rows, j0 + col, limit, f, p.d_wide, narrow);
        }
      }
      __syncwarp();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(acc_empty0 + a * 8);
      ++acc_it;
    }
  }

  // Teardown: neither CTA frees tensor memory or leaves while the other may still use its shared memory, its barriers or MMAs
  // in flight (every thread of both CTAs gets here after bounded waits).
  pdl_trigger();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    if (*abort_flag != 0) __nanosleep(20000);
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
  if (tid == 0 && *abort_flag != 0) report_timeout(p.status);
}

template <bool kI8, int kForm, bool kXMn, bool kWMn>
int launch(const CUtensorMap& tx, const CUtensorMap& tw, const TcDense& p, int64_t tiles, int max_ctas, bool early, cudaStream_t st) {
  auto kern = dense_tc_kernel<kI8, kForm, kXMn, kWMn>;
  static SmemConfig configured;
  if (int rc = configured.ensure(kern)) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = kSmem; cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 1;
  static std::atomic<int> resident[kMaxDevices];
  const int dev = current_device();
  int pairs = resident[dev].load(std::memory_order_relaxed);
  if (pairs == 0) {
    cfg.gridDim = dim3(2 * (sm_count() / 2));
    if (cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg) != cudaSuccess || pairs < 1) {
      (void)cudaGetLastError();
      pairs = -1;   // this device (a partition with too few SMs per GPC, say) runs no such cluster
    }
    resident[dev].store(pairs, std::memory_order_relaxed);
  }
  if (pairs < 0) return fail(B200MOE_E_UNSUPPORTED, "dense products: this device runs no clusters of two CTAs");
  if (max_ctas > 0) pairs = std::min(pairs, std::max(1, max_ctas / 2));
  pairs = (int)std::max<int64_t>(1, std::min<int64_t>(pairs, tiles));
  cfg.gridDim = dim3(2 * pairs);
  cfg.numAttrs = early ? 2 : 1;
  B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, tx, tw, p));
  return B200MOE_OK;
}

CUtensorMapDataType map_type(DenseType t) {
  return t == kDenseI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                       : t == kDenseBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// An operand of `rows` rows of k (mn: stored by column, k rows of `rows`), `stride` elements from one stored row to the next;
// a load brings 128 bytes of `box` stored rows.
int operand_map(CUtensorMap* map, DenseType t, const void* base, int64_t rows, int64_t k, int64_t stride, bool mn, int experts, int box_rows) {
  const int size = t == kDenseI8 ? 1 : 2;
  const int64_t inner = mn ? rows : k, outer = mn ? k : rows;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)std::max(experts, 1)};
  const cuuint64_t strides[2] = {(cuuint64_t)(stride * size), (cuuint64_t)(stride * size * outer)};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows, 1};
  return encode_map(map, map_type(t), experts > 0 ? 3 : 2, base, dims, strides, box);
}
// Weight rows of a tile: what leaves the least for the pair that has most to do.  A K block of a tile costs 2 cycles a weight row in the
// tensor cores, 64 bytes a weight row and the rows of X on the way into a CTA (some 56 bytes a cycle), and, where no other tile of rows
// reads the same weights, 64 bytes a weight row from HBM (23 bytes a cycle and SM); a tile costs some 600 cycles besides.
int tile_width(const TcDense& p, int64_t features, bool gated, int64_t row_tiles, int rows, int pairs) {
  const int step = gated ? 64 : 32;
  int best = 0;
  double least = 0;
  for (int width = kTile; width >= 64; width -= step) {
    const int64_t tiles = row_tiles * ((features + (gated ? width / 2 : width) - 1) / (gated ? width / 2 : width));
    const double load = (128.0 * std::min(rows, 128) + 64.0 * width) / 56, hbm = row_tiles == 1 ? 64.0 * width / 23 : 0;
    const double cost = (double)((tiles + pairs - 1) / pairs) * (p.num_kb * std::max({2.0 * width, load, hbm}) + 600);
    if (best == 0 || cost < least) { best = width; least = cost; }
  }
  return best;
}
int store_width(const void* p, int64_t row_bytes, int64_t cols_bytes) {
  for (int w : {32, 16})
    if (((uintptr_t)p % w) == 0 && row_bytes % w == 0 && cols_bytes % w == 0) return w;
  return 0;
}
uint32_t idesc_of(DenseType t, bool x_mn, bool w_mn, int width) {
  if (t == kDenseI8) return ptx::make_idesc_i8(256, width);
  const uint32_t fmt = t == kDenseBf16 ? 1u : 0u;
  return ptx::make_idesc(fmt, fmt, x_mn ? 1u : 0u, w_mn ? 1u : 0u, 256, width);
}
// What follows from a tile's width.
void set_width(TcDense& p, DenseType t, bool x_mn, bool w_mn, int width, int features, bool gated) {
  p.width = width;
  p.n_tiles = (features + (gated ? width / 2 : width) - 1) / (gated ? width / 2 : width);
  p.w_bytes = w_mn ? (width > 128 ? kOperand : kOperand / 2) : width * 64;
  p.stage_bytes = kOperand + p.w_bytes;
  p.stages = std::min(kMaxStages, kRing / p.stage_bytes);
  p.idesc = idesc_of(t, x_mn, w_mn, width);
}

}  // namespace

int dense_tc(const DenseJob& j, cudaStream_t st) {
  TcDense p = {};
  p.x_scale = j.x_scale; p.w_scale = j.w_scale; p.bias = j.bias; p.d = j.d; p.pre = j.pre;
  p.rows_per_expert = j.rows_per_expert; p.status = j.status;
  p.m = j.m; p.d_stride = j.d_stride; p.n = j.n; p.experts = j.experts;
  const int per_kb = j.type == kDenseI8 ? 128 : 64, n_out = j.gated ? j.n / 2 : j.n;
  p.num_kb = (j.k + per_kb - 1) / per_kb;
  p.m_tiles = (int)((j.m + kTile - 1) / kTile);
  const int64_t rows = j.rows_hint > 0 && j.rows_hint < j.m ? j.rows_hint : j.m, each = (rows + j.experts - 1) / j.experts;
  const int64_t sets = j.rows_per_expert != nullptr ? std::min<int64_t>(j.experts, rows) : 1;
  int width = 0;
  {
    // (as if every set had the mean number of rows; sets that share a tile of rows with no other read their weights once)
    const int64_t tiles_each = (each + kTile - 1) / kTile;
    const int pairs = std::max(1, (j.max_ctas > 0 ? std::min(j.max_ctas, sm_count()) : sm_count()) / 2);
    width = tile_width(p, n_out * sets, j.gated, tiles_each, (int)std::min<int64_t>(each, kTile), pairs);
  }
  set_width(p, j.type, false, false, width, n_out, j.gated);
  p.x_box = each <= 96 ? 32 : 128;
  p.d_dtype = j.d_dtype; p.bias_f16 = j.bias_f16; p.clamp = j.clamp;
  const int out_size = dtype_bytes(j.d_dtype);
  p.d_wide = store_width(j.d, j.d_stride * out_size, (int64_t)n_out * out_size);
  if (j.pre != nullptr) p.pre_wide = store_width(j.pre, (int64_t)j.n * 4, (int64_t)n_out * 4);
  CUtensorMap tx, tw;
  if (int rc = operand_map(&tx, j.type, j.x, j.m, j.k, j.x_stride, false, 0, p.x_box)) return rc;
  if (int rc = operand_map(&tw, j.type, j.w, j.n, j.k, j.w_stride, false, j.experts, width / 2)) return rc;
  const int64_t tiles = (p.m_tiles + (j.rows_per_expert != nullptr ? (int64_t)j.experts : 0)) * p.n_tiles;
  if (j.type == kDenseI8) {
    const int rc = j.gated ? launch<true, kGated, false, false>(tx, tw, p, tiles, j.max_ctas, j.early, st)
                           : launch<true, kScaled, false, false>(tx, tw, p, tiles, j.max_ctas, j.early, st);
    return rc == B200MOE_E_UNSUPPORTED ? dense_rows(j, st) : rc;
  }
  const int rc = launch<false, kGated, false, false>(tx, tw, p, tiles, j.max_ctas, j.early, st);
  return rc == B200MOE_E_UNSUPPORTED ? dense_rows(j, st) : rc;
}

int dense_plain(const PlainJob& j, cudaStream_t st) {
  TcDense p = {};
  p.d = j.d; p.status = j.status; p.m = j.m; p.d_stride = j.d_stride; p.n = j.n; p.experts = 1;
  p.num_kb = (int)((j.k + 63) / 64);
  p.m_tiles = (int)((j.m + kTile - 1) / kTile);
  const int width = tile_width(p, j.n, false, p.m_tiles, (int)std::min<int64_t>(j.m, kTile), std::max(1, sm_count() / 2));
  set_width(p, j.type, j.x_by_column, true, width, j.n, false);
  p.x_box = 128;
  p.d_dtype = j.type == kDenseF16 ? B200MOE_F16 : B200MOE_BF16;
  p.d_wide = store_width(j.d, j.d_stride * 2, (int64_t)j.n * 2);
  CUtensorMap tx, tw;
  if (int rc = operand_map(&tx, j.type, j.x, j.m, j.k, j.x_stride, j.x_by_column, 0, j.x_by_column ? 64 : 128)) return rc;
  if (int rc = operand_map(&tw, j.type, j.w, j.n, j.k, j.w_stride, true, 1, 64)) return rc;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
  return j.x_by_column ? launch<false, kPlain, true, true>(tx, tw, p, tiles, 0, j.early, st)
                       : launch<false, kPlain, false, true>(tx, tw, p, tiles, 0, j.early, st);
}

}  // namespace b200moe
