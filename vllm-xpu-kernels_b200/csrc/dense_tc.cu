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
// How wide a tile is follows from what the pairs have to do (choose_tile below): 256 weight rows share the rows of X best, fewer leave
// fewer pairs idle in the last round.  Calls of up to 128 rows (an expert, on average) have tiles of 128 or 64 rows and instructions of
// 128 (`halved`): a CTA's 64 rows lie on the first 64 lanes with the first half of the tile's columns, on the others with the second, so the
// even CTA's weight rows, which are that first half, are then gates and their ups, and so are the odd one's.
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
constexpr int kMaxStages = 12;

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
  int half_rows;            // rows of X that a CTA has of a tile: 32, 64 or 128 (in tensor memory they are the first of 128)
  bool halved;              // tiles of at most 128 rows: instructions of M = 128, whose sums' second half of columns is on other lanes
  int stages, blocks;       // of the ring; K blocks of a stage
  int x_bytes, w_bytes;     // of a K block
  int stage_bytes;          // X of its blocks, then their W
  uint32_t idesc;
  b200moe_dtype d_dtype;
  int bias_f16;
  bool d_wide, pre_wide;    // stores in pieces of 16 bytes, else value by value
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
  alignas(16) uint16_t bias[kEpi][128];
  alignas(16) uint8_t stage[kEpi][32 * 64];    // ... 64 bytes of each of its rows on their way out
  alignas(16) uint8_t walk[tile_walk_bytes(kMaxExperts)];
};
constexpr size_t kSmem = 1024 + (size_t)kRing + sizeof(Ctrl);
static_assert(kSmem <= kMaxSmem, "shared memory");

__device__ __forceinline__ int tile_rows(const TcDense& p) { return 2 * p.half_rows; }

// Tiles of one set of weights: eight tiles of rows side by side, so that pairs that run at the same time share both operands in L2.
__device__ __forceinline__ void locate_dense(const TcDense& p, int t, TileInfo& ti) {
  const int group = 8 * p.n_tiles, g = t / group, in = t - g * group, first = 8 * g;
  const int rows = min(8, p.m_tiles - first);
  ti.e = 0;
  ti.n_tile = in / rows;
  ti.m_tile = first + in - ti.n_tile * rows;
  ti.row0 = ti.m_tile * tile_rows(p);
  ti.valid = (int)min((int64_t)tile_rows(p), p.m - ti.row0);
}

// A tile of the walk over experts' rows.  (locate_tile of gemm_tc_common.cuh with a shorter search: a pair's next tile is some experts on, as
// many as tiles fit an expert with one tile of rows, which most are.)
__device__ __forceinline__ void locate_grouped(const TcDense& p, const TileWalk& w, int t, int& cursor, TileInfo& ti) {
  if (t >= w.tile_start[cursor + 1]) {
    int hi = min(cursor + (t - w.tile_start[cursor]) / p.n_tiles, w.n - 1);   // no expert has fewer than n_tiles tiles
    if (w.tile_start[hi] > t) {
      int lo = cursor + 1;
      --hi;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (w.tile_start[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
    }
    cursor = hi;
  }
  const int local = t - w.tile_start[cursor], row = w.row_start[cursor], rows = w.row_start[cursor + 1] - row;
  const int height = tile_rows(p), m_tiles = rows <= height ? 1 : (rows + height - 1) / height;
  ti.e = w.expert[cursor];
  ti.n_tile = m_tiles == 1 ? local : local / m_tiles;
  ti.m_tile = local - ti.n_tile * m_tiles;
  ti.row0 = row + ti.m_tile * height;
  ti.valid = min(rows - ti.m_tile * height, height);
}

// B bytes of each of a warp's 32 rows, a row a lane, of which the first `rows` rows and `bytes` bytes exist, to `at` and every `pitch`
// bytes on.  Through shared memory, so that lanes that store together are neighbours in a row: in 16-byte pieces where they are aligned
// (wide), else value by value.  (A lane's own row in 32-byte pieces took a warp 1000 cycles for 32 columns, which is what bounded tiles of
// few K blocks: 128 rows each of 128 experts of 768 x 2048 59.4 us, 53.5 so.)
template <int B>
__device__ __forceinline__ void store_rows(uint8_t* at, int64_t pitch, int rows, int bytes, const uint32_t (&w)[B / 4], bool wide, int size,
                                           uint32_t stage) {
  constexpr int kPer = B / 16;
  const int lane = threadIdx.x & 31;
  auto place = [&](int row, int byte) { return stage + row * 64 + (byte ^ ((row & 6) << 3)); };    // (no two lanes of a phase in one bank)
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kPer; ++i) ptx::sts128(place(lane, 16 * i), make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
  __syncwarp();
  if (wide) {
    const int c = lane % kPer * 16, r0 = lane / kPer;
    uint8_t* to = at + r0 * pitch + c;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + i * (32 / kPer);
      const uint4 v = ptx::lds128(place(r, c));
      if (r < rows && c < bytes) *reinterpret_cast<uint4*>(to + (int64_t)i * (32 / kPer) * pitch) = v;
    }
  } else if (size == 4) {
    constexpr int kRows = 128 / B;     // at a time
    const int c = lane % (B / 4) * 4;
#pragma unroll 2
    for (int r = lane / (B / 4); r < 32; r += kRows)
      if (r < rows && c < bytes) *reinterpret_cast<uint32_t*>(at + r * pitch + c) = ptx::lds32(place(r, c));
  } else {
    constexpr int kRows = 64 / B;
    const int c = lane % (B / 2) * 2;
#pragma unroll 8
    for (int r = lane / (B / 2); r < 32; r += kRows)
      if (r < rows && c < bytes) *reinterpret_cast<uint16_t*>(at + r * pitch + c) = ptx::lds16(place(r, c));
  }
}
// The same for kN values of each row.
template <int kN>
__device__ __forceinline__ void store_values(uint8_t* at, int64_t pitch, b200moe_dtype t, int rows, int left, const float (&v)[kN], bool wide,
                                             uint32_t stage) {
  if (t == B200MOE_F32) {
#pragma unroll
    for (int h = 0; h < kN / 16; ++h) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[16 * h + i]);
      store_rows<64>(at + 64 * h, pitch, rows, 4 * left - 64 * h, w, wide, 4, stage);
    }
    return;
  }
  uint32_t w[kN / 2];
  if (t == B200MOE_F16) {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  store_rows<2 * kN>(at, pitch, rows, 2 * left, w, wide, 2, stage);
}

struct EpilogueTile {
  int64_t first;      // the warp's first row
  int rows;           // ... and how many it has
  int features, j0, limit;   // its columns of D are j0 .. limit - 1, at most `features`
  uint8_t* at;        // the first row of D, column j0
  float xs;           // scale of the lane's row
  float scale[4];     // of weight rows, on their way to shared memory
  uint16_t bias[4];
};
// What an epilogue warp does with sums: rows (quarter of the CTA's 128, a lane each) of every second 32 columns, gated 16 gates and 16 ups.
// (So few at a time: a call of few tiles runs this code once, and most of what it takes is the way of the instructions.)
template <bool kI8, int kForm>
struct Epilogue {
  const TcDense& p;
  const int side, quarter, cta, size_shift;
  const uint32_t lane_sel, scale0, bias0, stage;
  __device__ __forceinline__ Epilogue(const TcDense& job, Ctrl& ctrl, int cta_, int e)
      : p(job), side(e >> 2), quarter((threadIdx.x >> 5) & 3), cta(cta_), size_shift(job.d_dtype == B200MOE_F32 ? 2 : 1), lane_sel((uint32_t)(quarter * 32) << 16),
        scale0(ptx::smem_u32(ctrl.scale[e])), bias0(ptx::smem_u32(ctrl.bias[e])), stage(ptx::smem_u32(ctrl.stage[e])) {}
  // The warp's part of a tile, and the scales and biases that it will need: asked for a tile ahead (their way from HBM takes as long as
  // a tile of a few K blocks).
  __device__ __forceinline__ EpilogueTile fetch(const TileInfo& ti) const {
    const int lane = threadIdx.x & 31, half = p.n >> 1;
    EpilogueTile t;
    // (halved: the quarters are rows 0 and 32, then the same rows of the second half of the columns)
    const int in_cta = (p.halved ? quarter & 1 : quarter) * 32, row0 = cta * p.half_rows + in_cta, part = p.halved ? quarter >> 1 : 0;
    t.first = (int64_t)ti.row0 + row0;
    t.rows = in_cta < p.half_rows ? (int)min((int64_t)min(ti.valid - row0, 32), p.m - t.first) : 0;
    const int tile = kForm == kGated ? p.width >> 1 : p.width, all = kForm == kGated ? half : p.n;
    t.features = p.halved ? tile >> 1 : tile;
    t.j0 = ti.n_tile * tile + part * t.features;
    t.limit = min(all, t.j0 + t.features);
    t.at = reinterpret_cast<uint8_t*>(p.d) + ((t.first * p.d_stride + t.j0) << size_shift);
    t.xs = 1.f;
    if (kI8 && t.rows > 0) {
      // every second 32 columns, one after the other; gated 16 gates, then their ups.  (Nothing is done with what is loaded, not even for
      // columns that do not exist, so that nothing waits for it here.)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = 2 * i + side, f = min(t.j0 + (kForm == kGated ? 16 * c + (lane & 15) : 32 * c + lane), all - 1);
        const int64_t at = (int64_t)ti.e * p.n + f + (kForm == kGated && (lane & 16) ? half : 0);
        t.scale[i] = p.w_scale[at];
        t.bias[i] = 0;
        if (p.bias != nullptr) t.bias[i] = reinterpret_cast<const uint16_t*>(p.bias)[at];
      }
      t.xs = p.x_scale[min(t.first + lane, p.m - 1)];
    }
    return t;
  }
  // ... to shared memory (every warp its own copy, so that no barrier couples the warps)
  __device__ __forceinline__ void put(const EpilogueTile& t) const {
    if (!kI8 || t.rows <= 0) return;
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ptx::sts32f(scale0 + 128 * i + 4 * lane, t.scale[i]);
      if (p.bias != nullptr) ptx::sts16(bias0 + 64 * i + 2 * lane, t.bias[i]);
    }
    __syncwarp();
  }
  // sums as the product's values; `l`: the first one's place among the warp's scales
  template <int kN>
  __device__ __forceinline__ void scaled(float* f, const uint32_t (&v)[kN], float xs, int l) const {
    if (!kI8) {
#pragma unroll
      for (int i = 0; i < kN; ++i) f[i] = __uint_as_float(v[i]);
      return;
    }
#pragma unroll
    for (int i = 0; i < kN / 4; ++i) {
      const float4 ws = ptx::lds128f(scale0 + 4 * (l + 4 * i));
      f[4 * i] = (float)(int)v[4 * i] * xs * ws.x;
      f[4 * i + 1] = (float)(int)v[4 * i + 1] * xs * ws.y;
      f[4 * i + 2] = (float)(int)v[4 * i + 2] * xs * ws.z;
      f[4 * i + 3] = (float)(int)v[4 * i + 3] * xs * ws.w;
    }
    if (p.bias == nullptr) return;
#pragma unroll
    for (int i = 0; i < kN / 8; ++i) {
      const uint4 b = ptx::lds128(bias0 + 2 * (l + 8 * i));
      const uint16_t* const each = reinterpret_cast<const uint16_t*>(&b);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[8 * i + k] += load_bias(each, p.bias_f16, k);
    }
  }
  // Columns 32 c.. of the tile (not gated).
  __device__ __forceinline__ void store_two(const EpilogueTile& t, int c, const uint32_t (&a)[16], const uint32_t (&b)[16]) const {
    const int l = 32 * (c >> 1);
    float f[32];
    scaled(f, a, t.xs, l);
    scaled(f + 16, b, t.xs, l + 16);
    store_values(t.at + ((32 * c) << size_shift), p.d_stride << size_shift, p.d_dtype, t.rows, t.limit - t.j0 - 32 * c, f, p.d_wide, stage);
  }
  // Columns 16 c.. of the tile (u: of ups, gated).
  __device__ __forceinline__ void store(const EpilogueTile& t, int c, const uint32_t (&g)[16], const uint32_t (&u)[16]) const {
    const int left = t.limit - t.j0 - 16 * c, l = 32 * (c >> 1);
    float f[16], up[16];
    scaled(f, g, t.xs, l);
    scaled(up, u, t.xs, l + 16);
    if (p.pre != nullptr) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = h == 0 ? f[i] : up[i];
        store_values(reinterpret_cast<uint8_t*>(p.pre + t.first * p.n + h * (p.n >> 1) + t.j0 + 16 * c), (int64_t)p.n * 4, B200MOE_F32, t.rows,
                     left, v, p.pre_wide, stage);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = gated_product(f[i], up[i], p.clamp);
    store_values(t.at + ((16 * c) << size_shift), p.d_stride << size_shift, p.d_dtype, t.rows, left, f, p.d_wide, stage);
  }
};

// kWide: a load brings all K blocks of a stage (rows of whole blocks).
// kXMn, kWMn: the operand is stored by column (its rows' index is the dense one): 16-bit types, two boxes of 64 rows x 64 k.
template <bool kI8, int kForm, bool kXMn, bool kWMn, bool kWide>
__global__ void __launch_bounds__(kThreads, 1)
dense_tc_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const TcDense p) {
  constexpr int kPerKb = kI8 ? 128 : 64;
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
    if (grouped) {
      if (p.half_rows == 32) build_tile_walk<64>(p.rows_per_expert, p.experts, p.n_tiles, ctrl->walk);
      else if (p.half_rows == 64) build_tile_walk<128>(p.rows_per_expert, p.experts, p.n_tiles, ctrl->walk);
      else build_tile_walk<kTile>(p.rows_per_expert, p.experts, p.n_tiles, ctrl->walk);
    }
    if (lane == 0) {
      ptx::prefetch_tensormap(&tmap_x);
      ptx::prefetch_tensormap(&tmap_w);
    }
  } else if (warp == 1) {
    ptx::tmem_alloc_pair(&ctrl->tmem_base, 512);
    ptx::tmem_relinquish_pair();
  } else if (warp == 2 && lane == 0) {
    for (int s = 0; s < kMaxStages; ++s) {
      ptx::mbar_init(&ctrl->full[s], 3);     // the even CTA's producer of W, which announces the bytes, and both producers of X
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
  int cursor = 0;
  auto locate = [&](int t, TileInfo& ti) {
    if (grouped) locate_grouped(p, walk, t, cursor, ti);
    else locate_dense(p, t, ti);
  };

  if (warp == 0) {
    // ------------------------------ TMA producer of W -------------------------
    if (ptx::elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      const uint32_t full0 = ptx::smem_u32(&ctrl->full[0]), empty0 = ptx::smem_u32(&ctrl->empty[0]);
      const uint32_t bar0 = ptx::map_to_cta(full0, 0);   // the even CTA's barriers count the bytes of both CTAs
      const uint32_t st = ptx::smem_u32(smem) + p.blocks * p.x_bytes;
      for (int t = walker; t < total && ok; t += walkers) {
        TileInfo ti;
        locate(t, ti);
        // (rows past the end are filled with zeros)
        // (gated: the even CTA's are gates, the odd one's ups; halved: either has gates and their ups)
        const int n0 = kForm != kGated ? ti.n_tile * p.width + (int)cta * (p.width >> 1)
                       : ti.n_tile * (p.width >> 1) + (p.halved ? (int)cta * (p.width >> 2) : 0);
        const int up = kForm == kGated && !p.halved ? (int)cta : 0;
        const uint32_t tx = 2 * p.w_bytes + ((ti.valid > 0) + (ti.valid > p.half_rows)) * p.x_bytes;
        for (int kb = 0; kb < p.num_kb;) {
          if (!ptx::paced::mbar_wait_s(empty0 + 8 * s, ph, abort_flag)) { ok = false; break; }
          const uint32_t bar = bar0 + 8 * s;
          uint32_t to = st + s * p.stage_bytes;
          if (kWide) {   // (blocks past the end are zeros)
            if (cta == 0) ptx::mbar_expect_tx_s(full0 + 8 * s, tx * p.blocks);
            if (kForm == kGated) ptx::tma_load_5d_pair(to, &tmap_w, bar, 0, n0, up, kb, ti.e);
            else ptx::tma_load_4d_pair(to, &tmap_w, bar, 0, n0, kb, ti.e);
            kb += p.blocks;
          } else {
            const int end = min(kb + p.blocks, p.num_kb);
            if (cta == 0) ptx::mbar_expect_tx_s(full0 + 8 * s, tx * (end - kb));
            for (; kb < end; ++kb, to += p.w_bytes) {
              const int k0 = kb * kPerKb;
              if (kWMn) {
                ptx::tma_load_3d_pair(to, &tmap_w, bar, n0, k0, ti.e);
                if (p.w_bytes > kOperand / 2) ptx::tma_load_3d_pair(to + kOperand / 2, &tmap_w, bar, n0 + 64, k0, ti.e);
              } else if (kForm == kGated) {
                ptx::tma_load_4d_pair(to, &tmap_w, bar, k0, n0, up, ti.e);
              } else {
                ptx::tma_load_3d_pair(to, &tmap_w, bar, k0, n0, ti.e);
              }
            }
          }
          if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 2 + kEpi) {
    // ------------------------------ TMA producer of X -------------------------
    // (A thread of its own: a load costs some 100 cycles, a K block of a narrow tile hardly more in the tensor cores.)
    if (ptx::elect_one()) {
      uint32_t s = 0, ph = 1;
      bool ok = true;
      const uint32_t empty0 = ptx::smem_u32(&ctrl->empty[0]), bar0 = ptx::map_to_cta(ptx::smem_u32(&ctrl->full[0]), 0);
      const uint32_t st = ptx::smem_u32(smem);
      for (int t = walker; t < total && ok; t += walkers) {
        TileInfo ti;
        locate(t, ti);
        const int row = ti.row0 + (int)cta * p.half_rows;
        const bool mine = ti.valid > (int)cta * p.half_rows;    // (of a tile with few rows a CTA may have none)
        for (int kb = 0; kb < p.num_kb;) {
          if (!ptx::paced::mbar_wait_s(empty0 + 8 * s, ph, abort_flag)) { ok = false; break; }
          const uint32_t bar = bar0 + 8 * s;
          // An arrival besides the bytes, which a CTA may have none of: a producer must not fall behind by a round of the
          // stages, whose phases it tells apart by their parity alone.
          ptx::mbar_arrive_cluster(bar);
          uint32_t to = st + s * p.stage_bytes;
          if (kWide) {
            if (mine) ptx::tma_load_3d_pair(to, &tmap_x, bar, 0, row, kb);
            kb += p.blocks;
          } else {
            const int end = min(kb + p.blocks, p.num_kb);
            for (; kb < end; ++kb, to += p.x_bytes) {
              if (!mine) continue;
              if (kXMn) {
                ptx::tma_load_2d_pair(to, &tmap_x, bar, row, kb * kPerKb);
                ptx::tma_load_2d_pair(to + kOperand / 2, &tmap_x, bar, row + 64, kb * kPerKb);
              } else {
                ptx::tma_load_2d_pair(to, &tmap_x, bar, kb * kPerKb, row);
              }
            }
          }
          if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1; }
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
      const uint64_t wdesc0 = ptx::make_smem_desc(ptx::smem_u32(smem) + p.blocks * p.x_bytes, kWMn ? 8192u : 16u, 1024);
      const uint64_t x16 = p.x_bytes >> 4, w16 = p.w_bytes >> 4, stage16 = p.stage_bytes >> 4;
      uint64_t at = 0;     // of the stage, from the first one's descriptors
      for (int t = walker; t < total && ok; t += walkers) {
        const uint32_t a = acc_it & 1;
        if (!ptx::mbar_wait_s(acc_empty0 + 8 * a, ((acc_it >> 1) & 1) ^ 1, abort_flag)) break;
        ptx::tc_fence_after();
        for (int kb = 0; kb < p.num_kb;) {
          if (!ptx::mbar_wait_s(full0 + 8 * s, ph, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          const int end = min(kb + p.blocks, p.num_kb);
          for (uint64_t x = xdesc0 + at, w = wdesc0 + at; kb < end; ++kb, x += x16, w += w16)
            ptx::umma_pair_block<kI8, kXStep, kWStep>(tmem_base + a * kTile, x, w, p.idesc, kb > 0 ? 1u : 0u);
          ptx::umma_commit_pair(empty0 + 8 * s);
          at += stage16;
          if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1; at = 0; }
        }
        if (ok) { ptx::umma_commit_pair(acc_full0 + 8 * a); ++acc_it; }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ epilogue ----------------------------------
    const Epilogue<kI8, kForm> ep(p, *ctrl, (int)cta, warp - 2);
    const uint32_t acc_empty0 = ptx::map_to_cta(ptx::smem_u32(&ctrl->acc_empty[0]), 0);
    uint32_t acc_it = 0;
    auto fetch = [&](int t) {
      TileInfo ti;
      locate(t, ti);
      return ep.fetch(ti);
    };
    EpilogueTile next = walker < total ? fetch(walker) : EpilogueTile{};
    for (int t = walker; t < total; t += walkers) {
      const uint32_t a = acc_it & 1;
      const EpilogueTile et = next;
      ep.put(et);
      if (t + walkers < total) next = fetch(t + walkers);
      if (!__all_sync(0xffffffffu, ptx::mbar_wait(&ctrl->acc_full[a], (acc_it >> 1) & 1, abort_flag))) {
        *abort_flag = 1;
        break;
      }
      ptx::tc_fence_after();
      const uint32_t acc = tmem_base + a * kTile + ep.lane_sel;
      if (et.rows > 0) {
        constexpr int kParts = kForm == kGated ? 2 : 1;
        const int units = et.limit - et.j0;     // columns that exist
        uint32_t v[2][kParts][16];
        auto load = [&](int c, int b) {
          __syncwarp();
#pragma unroll
          for (int part = 0; part < kParts; ++part) ptx::tmem_ld_32x16(acc + part * et.features + 16 * c, v[b][part]);
        };
        auto store = [&](int c, int b) { ep.store(et, c, v[b][0], v[b][kParts - 1]); };
        auto wait = [&](int b) {
          if (kParts == 2) ptx::tmem_wait_ld(v[b][0], v[b][kParts - 1]);
          else ptx::tmem_wait_ld(v[b][0]);
        };
        if (kParts == 2) {             // the next columns are on their way while these are stored
          if (16 * ep.side < units) load(ep.side, 0);
#pragma unroll 1
          for (int c = ep.side; 16 * c < units; c += 4) {
            wait(0);
            if (16 * (c + 2) < units) load(c + 2, 1);
            store(c, 0);
            if (16 * (c + 2) >= units) break;
            wait(1);
            if (16 * (c + 4) < units) load(c + 4, 0);
            store(c + 2, 1);
          }
        } else {                       // twice as many at once (a tile's columns are there, whether or not they exist in D)
#pragma unroll 1
          for (int c = ep.side; 32 * c < units; c += 2) {
            load(2 * c, 0);
            load(2 * c + 1, 1);
            ptx::tmem_wait_ld(v[0][0], v[1][0]);
            ep.store_two(et, c, v[0][0], v[1][0]);
          }
        }
      }
      __syncwarp();
      ptx::tc_fence_before();
      __syncwarp();
      // (nobody waits for the last two: no arrival is on its way to a CTA that may have left)
      if (lane == 0 && t + 2 * walkers < total) ptx::mbar_arrive_cluster(acc_empty0 + a * 8);
      ++acc_it;
    }
  }
  // Teardown: neither CTA frees tensor memory or leaves while the other may still use its shared memory, its barriers or MMAs
  // in flight (every thread of both CTAs gets here after bounded waits).  Nothing that one CTA wrote is read by another any more: a
  // barrier that also waits until all rows that were stored have reached L2 took 2 to 4 us longer.
  pdl_trigger();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::cluster_sync_relaxed();
  if (warp == 1) {
    ptx::tc_fence_after();
    if (*abort_flag != 0) __nanosleep(20000);
    ptx::tmem_dealloc_pair(tmem_base, 512);
  }
  if (tid == 0 && *abort_flag != 0) report_timeout(p.status);
}

template <bool kI8, int kForm, bool kXMn, bool kWMn, bool kWide>
struct Kernel {
  static constexpr bool wide = kWide;
  static constexpr auto kern = dense_tc_kernel<kI8, kForm, kXMn, kWMn, kWide>;
  // How many pairs the device runs at once; 0 if none (a partition with too few SMs per GPC, say).
  static int pairs() {
    static std::atomic<int> cached[kMaxDevices];
    const int dev = current_device();
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n != 0) return n < 0 ? 0 : n;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = config(attr, 1, std::max(1, sm_count() / 2), 0);
    if (configured() != B200MOE_OK || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = -1;
    }
    cached[dev].store(n, std::memory_order_relaxed);
    return n < 0 ? 0 : n;
  }
  static int launch(const CUtensorMap& tx, const CUtensorMap& tw, const TcDense& p, int64_t pairs, bool early, cudaStream_t st) {
    if (int rc = configured()) return rc;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = config(attr, early ? 2 : 1, pairs, st);
    B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, tx, tw, p));
    return B200MOE_OK;
  }

 private:
  static int configured() {
    static SmemConfig done;
    return done.ensure(kern);
  }
  static cudaLaunchConfig_t config(cudaLaunchAttribute* attr, int attrs, int64_t pairs, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    if (attrs > 1) {
      attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[1].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.gridDim = dim3((unsigned)(2 * pairs)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = kSmem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = attrs;
    return cfg;
  }
};

CUtensorMapDataType map_type(DenseType t) {
  return t == kDenseI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                       : t == kDenseBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}
// An operand of `rows` rows of k, `stride` elements from one to the next (mn: stored by column, k rows of `rows`); a load brings 128 bytes
// of `box_rows` stored rows.  sets: of one after the other, or 0.
int operand_map(CUtensorMap* map, DenseType t, const void* base, int64_t rows, int64_t k, int64_t stride, bool mn, int sets, int box_rows) {
  const int size = t == kDenseI8 ? 1 : 2;
  const int64_t inner = mn ? rows : k, outer = mn ? k : rows;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)std::max(sets, 1)};
  const cuuint64_t strides[2] = {(cuuint64_t)(stride * size), (cuuint64_t)(stride * size * outer)};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows, 1};
  return encode_map(map, map_type(t), sets > 0 ? 3 : 2, base, dims, strides, box);
}
// The dimensions of an operand that is stored by row, one by one.
struct Dims {
  cuuint64_t dims[5], strides[5];     // (strides[i]: of dimension i, in bytes)
  cuuint32_t box[5];
  int n = 0;
  void add(int64_t size, int64_t stride, int64_t loaded) {
    dims[n] = (cuuint64_t)size;
    strides[n] = (cuuint64_t)stride;
    box[n++] = (cuuint32_t)loaded;
  }
  int encode(CUtensorMap* map, DenseType t, const void* base) const { return encode_map(map, map_type(t), n, base, dims, strides + 1, box); }
};
// blocks > 0: rows are whole blocks of 128 bytes, of which a load brings as many.  parts: the rows' equal parts (gates and ups), of which it
// brings `box_parts`, `box_rows` rows of each.
int row_map(CUtensorMap* map, DenseType t, const void* base, int64_t rows, int64_t k, int64_t stride, int sets, int parts, int box_rows, int box_parts,
            int blocks) {
  const int size = t == kDenseI8 ? 1 : 2, inner = 128 / size;
  const int64_t pitch = stride * size;
  Dims d;
  d.add(blocks > 0 ? inner : k, size, inner);
  d.add(rows / parts, pitch, box_rows);
  if (parts > 1) d.add(parts, rows / parts * pitch, box_parts);
  if (blocks > 0) d.add(k / inner, 128, blocks);
  if (sets > 0) d.add(sets, rows * pitch, 1);
  return d.encode(map, t, base);
}
// K blocks of a stage.  A wait, and what goes with it (the producers' arrivals, the issuer's commit to both CTAs), takes either single thread
// some 300 cycles, a block's instructions 100, where the tensor cores have 512 cycles of work with 256 weight rows and 256 rows of X, and
// 64 with 64 and 128.  1 / 2 / 3 / 4 / 6 / 8 blocks a stage, us: 64 x 7168 x 2048 gated, tiles of 64 weight rows 27.0 / 18.5 / 15.8 / 14.0 / 14.1 / 14.7,
// of 128 27.1 / 18.5 / 17.0 / 17.0, of 256 27.8 / 25.6 / 26.4 / 31.8 (few stages are left); 256 rows, tiles of 64 34.1 / 24.0 / 24.4 / 28.9 / 42.3.
int stage_blocks(const TcDense& p, int width, int block_bytes) {
  if (p.halved) return block_bytes <= 12288 ? 4 : 2;
  return width == kTile ? 1 : block_bytes <= 8192 ? 3 : 2;
}

// Weight rows of a tile: what takes the fewest cycles by this estimate.  A K block of a tile takes the issuer's time, the tensor cores' for
// its weight rows, or a cycle for each 60 of its bytes; a tile costs some 1400 to 2000 besides; and the weights pass HBM at 3440 bytes a
// cycle at the most.  With 64 / 128 / 192 / 256 weight rows, us: 2000 x 4096 x 4096 46 / 31 / 29 / 26, 1001 x 2016 x 2032 11.8 / 9.3 / 10.9 / 12.1,
// 64 x 4096 x 4096 7.1 / 7.8 / 8.7 / 10.4, 64 x 14336 x 4096 15.1 / 13.8 / 16.6 / 14.0, 16 rows each of 128 experts of 768 x 2048 64 / 41 / 37 / 36.
void choose_tile(TcDense& p, int64_t sets, int64_t row_tiles, int features, bool gated, bool w_mn, int64_t pairs, int64_t w_bytes) {
  const int step = gated ? 64 : 32;
  double least = 0;
  p.width = 0;
  for (int width = kTile; width >= 64; width -= step) {
    const int out = gated ? width / 2 : width, bytes = p.half_rows * 128 + (w_mn ? (width + 127) / 128 * 8192 : width * 64);
    const int64_t tiles = sets * row_tiles * ((features + out - 1) / out), rounds = (tiles + pairs - 1) / pairs;
    const int g = stage_blocks(p, width, bytes);
    const double block = p.halved ? std::max({280.0 / g + 100, 1.25 * width, bytes / 60.0}) : std::max({300.0 / g + 170, 2.45 * width, bytes / 60.0});
    const double cost = std::max(rounds * (p.num_kb * block + (p.halved ? 1400 : 2000)), w_bytes / 3440.0);
    // (of several rounds, a narrower tile that promises little more gave nothing: 64 rows each of 8 experts of 4096 x 28672 175 us with 224,
    // 170 with 256)
    if (p.width == 0 || cost < (rounds > 1 ? 0.94 : 1.0) * least) { p.width = width; least = cost; }
  }
}
bool stores_wide(const void* p, int64_t row_bytes, int64_t cols_bytes) { return ((uintptr_t)p | row_bytes | cols_bytes) % 16 == 0; }
uint32_t idesc_of(DenseType t, bool x_mn, bool w_mn, int rows, int width) {
  if (t == kDenseI8) return ptx::make_idesc_i8(rows, width);
  const uint32_t fmt = t == kDenseBf16 ? 1u : 0u;
  return ptx::make_idesc(fmt, fmt, x_mn ? 1u : 0u, w_mn ? 1u : 0u, rows, width);
}
// What follows from a tile's width.
void set_width(TcDense& p, DenseType t, bool x_mn, bool w_mn, int features, bool gated) {
  const int width = p.width;
  p.n_tiles = (features + (gated ? width / 2 : width) - 1) / (gated ? width / 2 : width);
  p.x_bytes = p.half_rows * 128;
  p.w_bytes = w_mn ? (width > 128 ? kOperand : kOperand / 2) : width * 64;
  p.blocks = std::min(p.num_kb, stage_blocks(p, width, p.x_bytes + p.w_bytes));
  p.stage_bytes = p.blocks * (p.x_bytes + p.w_bytes);
  p.stages = std::min(kMaxStages, kRing / p.stage_bytes);
  p.idesc = idesc_of(t, x_mn, w_mn, p.halved ? 128 : 256, width);
}

}  // namespace

int dense_tc(const DenseJob& j, cudaStream_t st) {
  TcDense p = {};
  p.x_scale = j.x_scale; p.w_scale = j.w_scale; p.bias = j.bias; p.d = j.d; p.pre = j.pre;
  p.rows_per_expert = j.rows_per_expert; p.status = j.status;
  p.m = j.m; p.d_stride = j.d_stride; p.n = j.n; p.experts = j.experts;
  const int per_kb = j.type == kDenseI8 ? 128 : 64, n_out = j.gated ? j.n / 2 : j.n;
  p.num_kb = (j.k + per_kb - 1) / per_kb;
  p.d_dtype = j.d_dtype; p.bias_f16 = j.bias_f16; p.clamp = j.clamp;
  const int out_size = dtype_bytes(j.d_dtype);
  p.d_wide = stores_wide(j.d, j.d_stride * out_size, (int64_t)n_out * out_size);
  if (j.pre != nullptr) p.pre_wide = stores_wide(j.pre, (int64_t)j.n * 4, (int64_t)n_out * 4);
  // (tiles as if every set of weights had the mean number of rows)
  const bool grouped = j.rows_per_expert != nullptr;
  const int64_t rows = j.rows_hint > 0 && j.rows_hint < j.m ? j.rows_hint : j.m, each = (rows + j.experts - 1) / j.experts;
  const int64_t sets = grouped ? std::min<int64_t>(j.experts, rows) : 1;
  // Rows of a tile: 256, 128 or 64 (routing is never even, so sets of rows get some headroom for 64).  Of 128 and fewer the tensor cores take
  // half the time, and an epilogue warp has half the columns: 128 rows each of 8 experts of 4096 x 28672 162 us, 186 with tiles of 256; of
  // 256 rows on average 294 and 284 (128 experts of 2048 x 768, a layer).  64 bring half as many rows of X as 128, of which there may be fewer still:
  // what follows them in shared memory makes sums that nobody reads.
  p.half_rows = each > 128 ? 128 : each > (grouped ? 40 : 64) ? 64 : 32;
  p.halved = p.half_rows <= 64;
  p.m_tiles = (int)((j.m + 2 * p.half_rows - 1) / (2 * p.half_rows));
  auto run = [&](auto kernel) {
    using K = decltype(kernel);
    if (K::pairs() == 0) return dense_rows(j, st);   // no clusters on this device
    const int64_t pairs = j.max_ctas > 0 ? std::min(K::pairs(), std::max(1, j.max_ctas / 2)) : K::pairs();
    choose_tile(p, sets, grouped ? (each + 2 * p.half_rows - 1) / (2 * p.half_rows) : p.m_tiles, n_out, j.gated, false, pairs,
                sets * j.n * (int64_t)j.k * (j.type == kDenseI8 ? 1 : 2));
    set_width(p, j.type, false, false, n_out, j.gated);
    CUtensorMap tx, tw;
    const int blocks = K::wide ? p.blocks : 0;
    if (int rc = row_map(&tx, j.type, j.x, j.m, j.k, j.x_stride, 0, 1, p.half_rows, 1, blocks)) return rc;
    if (int rc = j.gated ? row_map(&tw, j.type, j.w, j.n, j.k, j.w_stride, j.experts, 2, p.halved ? p.width / 4 : p.width / 2, p.halved ? 2 : 1, blocks)
                         : row_map(&tw, j.type, j.w, j.n, j.k, j.w_stride, j.experts, 1, p.width / 2, 1, blocks)) return rc;
    const int64_t tiles = (p.m_tiles + (grouped ? (int64_t)j.experts : 0)) * p.n_tiles;
    return K::launch(tx, tw, p, std::min(pairs, tiles), j.early, st);
  };
  const bool wide = j.k % per_kb == 0;
  if (j.type != kDenseI8) return wide ? run(Kernel<false, kGated, false, false, true>()) : run(Kernel<false, kGated, false, false, false>());
  if (j.gated) return wide ? run(Kernel<true, kGated, false, false, true>()) : run(Kernel<true, kGated, false, false, false>());
  return wide ? run(Kernel<true, kScaled, false, false, true>()) : run(Kernel<true, kScaled, false, false, false>());
}

int dense_plain(const PlainJob& j, cudaStream_t st) {
  TcDense p = {};
  p.d = j.d; p.status = j.status; p.m = j.m; p.d_stride = j.d_stride; p.n = j.n; p.experts = 1;
  p.num_kb = (int)((j.k + 63) / 64);
  p.half_rows = j.x_by_column || j.m > 128 ? 128 : j.m > 64 ? 64 : 32;
  p.halved = p.half_rows <= 64;
  p.m_tiles = (int)((j.m + 2 * p.half_rows - 1) / (2 * p.half_rows));
  p.d_dtype = j.type == kDenseF16 ? B200MOE_F16 : B200MOE_BF16;
  p.d_wide = stores_wide(j.d, j.d_stride * 2, (int64_t)j.n * 2);
  auto run = [&](auto kernel) {
    using K = decltype(kernel);
    if (K::pairs() == 0) return fail(B200MOE_E_UNSUPPORTED, "dense products: this device runs no clusters of two CTAs");
    choose_tile(p, 1, p.m_tiles, j.n, false, true, K::pairs(), 0);
    set_width(p, j.type, j.x_by_column, true, j.n, false);
    CUtensorMap tx, tw;
    if (int rc = operand_map(&tx, j.type, j.x, j.m, j.k, j.x_stride, j.x_by_column, 0, j.x_by_column ? 64 : p.half_rows)) return rc;
    if (int rc = operand_map(&tw, j.type, j.w, j.n, j.k, j.w_stride, true, 1, 64)) return rc;
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    return K::launch(tx, tw, p, std::min<int64_t>(K::pairs(), tiles), j.early, st);
  };
  return j.x_by_column ? run(Kernel<false, kPlain, true, true, false>()) : run(Kernel<false, kPlain, false, true, false>());
}

}  // namespace b200moe
