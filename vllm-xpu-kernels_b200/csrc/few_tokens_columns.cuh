// The layer for a few tokens where weights are 16 bits wide and stored by column ([E,K,N]).
//
//   D[features, tokens] += W[16 features, 16 k] x^T[16 k, 8 tokens]     (mma.sync, fp32 accumulation)
//
// A step of a warp is 4 KB of weights, 32 rows of k with 64 columns (or 32 gates and their ups), which one lane asks for by TMA into the
// warp's own ring.  A lane takes eight columns of eight rows; two rows side by side make the pairs of k that the instruction
// wants.  4096 x 14336 float16, two of 8 experts: one token 113 us, 6.2 TB/s; 16 tokens 500 us, 5.6 TB/s: the first kernel's loads
// come at 6.5, the second one's at 4.9, however many blocks share them (7, 8, 9 or 18 shares of its steps: the same; 64-byte pieces by
// lanes instead of TMA: 765 us).  Tokens next to bfloat16 weights are as they come, next to float16 weights scaled by a power of two per 32 values.
#pragma once

#include "few_tokens_mma.cuh"

namespace b200moe {
namespace {

template <int F> struct ColumnShape {
  static constexpr int kWarps = 8, kThreads = 32 * kWarps;
  static constexpr int kTiles = 4, kRows = 16 * kTiles;      // tiles of 16 columns of W (rows of the product) that a warp takes at once
  static constexpr int kK = 32;                              // values of k in a step
  // Of the panel: a row's values of a step and their scale.  h is there twice, as the weights' type has it and what that leaves
  // of it: with one rounding to 16 bits the results would be 1.4 times as far from the formula's as their own rounding puts
  // them.
  static constexpr int kTerms = 2;                           // of h
  __host__ __device__ static constexpr int kPanelBytes(int terms) { return terms * kK * 2 + 4; }
  static constexpr int kSlotBytes = 4096, kDepth = 3;
  // Shared memory: the rings, barriers, zeros, flags, the table; the rest is the kernels'.
  static constexpr int kBars = kWarps * kDepth * kSlotBytes, kZeros = kBars + 256, kFlags = kZeros + 64, kTable = kFlags + 64;
  static constexpr int kRest = kTable + kTableBytes;
  static_assert(kWarps * kDepth * 8 <= 256, "barriers");
};

// ---- tokens and activations as float16 -------------------------------------------------
// A panel holds rows of values in the order in which the lanes want them: per step of 32 values (and of h per term) a block
// of [row][4 lanes][8 values]: a lane multiplies k = 2 t, 2 t + 1 and every eighth after these.  Behind them, per row and step, the
// inverse of what the values have been multiplied by.
__device__ __forceinline__ uint32_t panel_at(int k8, int row, int rows, int terms) {   // k8: k / 8; a second term is a block on
  return (uint32_t)(((k8 >> 2) * terms * rows + row) * 64);
}

// Eight values as pairs.
template <int F>
__device__ __forceinline__ uint4 packed8(const float (&v)[8]) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F == kFewBf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Eighth j of a row to its place: a word to each of the four lanes.
__device__ __forceinline__ void store8(uint8_t* at, int j, const uint4& o) {
  uint32_t* const w = reinterpret_cast<uint32_t*>(at) + (j & 3);
  w[0] = o.x;
  w[4] = o.y;
  w[8] = o.z;
  w[12] = o.w;
}

// `len` eighths of a row (what is beyond `values` values is zero) into a panel, by `parts` warps of which this is `part`.  A warp
// asks for four times 256 values at once: the loads' latency is what this costs.  (Functions that run once in a while are not
// inlined: both kernels' code together has to stay in the SM's instruction cache.  With 160 KB of it every launch began
// with some 3 us of misses.)
template <int F, bool kF32>
__device__ __noinline__ void fill_row(uint8_t* panel, float* scales, const void* from, int values, int len, int row, int rows, int part, int parts,
                                      bool f16) {
  constexpr int kLanes = ColumnShape<F>::kK / 8;      // of a step (at most 32)
  constexpr int kWords = kF32 ? 2 : 1;
  const int lane = threadIdx.x & 31, stride = 32 * parts;
#pragma unroll 1
  for (int j0 = part * 32 + lane; j0 - lane < len; j0 += 4 * stride) {
    vec16 raw[4][kWords];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * stride;
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        raw[i][k] = vec16{{0, 0, 0, 0}};
        if (j < len && 8 * j < values) raw[i][k] = reinterpret_cast<const vec16*>(from)[j * kWords + k];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * stride;
      float v[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (kF32) {
          v[k] = __uint_as_float(raw[i][0].w[k]);
          v[4 + k] = __uint_as_float(raw[i][kWords - 1].w[k]);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw[i][0].w[k]));
          v[2 * k] = f16 ? f.x : __uint_as_float(raw[i][0].w[k] << 16);
          v[2 * k + 1] = f16 ? f.y : __uint_as_float(raw[i][0].w[k] & 0xffff0000u);
        }
      }
      uint32_t top = 0;        // (as bits: magnitudes in their order, NaN last)
#pragma unroll
      for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      float inv = 1.f;
      if constexpr (F != kFewBf16) {
        const float scale = step_scale(top, inv);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= scale;
      }
      if (j < len) {
        constexpr int kTerms = kF32 ? ColumnShape<F>::kTerms : 1;
        uint8_t* const at = panel + panel_at(j, row, rows, kTerms);
        const uint4 o = packed8<F>(v);
        store8(at, j, o);
        if constexpr (kTerms == 2) {
          const uint32_t w[4] = {o.x, o.y, o.z, o.w};
          float rest[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
            const float x = F == kFewBf16 ? __uint_as_float(w[k] << 16) : f.x, y = F == kFewBf16 ? __uint_as_float(w[k] & 0xffff0000u) : f.y;
            // (what is not finite leaves nothing)
            rest[2 * k] = fabsf(v[2 * k]) < INFINITY ? v[2 * k] - x : 0.f;
            rest[2 * k + 1] = fabsf(v[2 * k + 1]) < INFINITY ? v[2 * k + 1] - y : 0.f;
          }
          store8(at + rows * 64, j, packed8<F>(rest));
        }
        if ((j & (kLanes - 1)) == 0) scales[j / kLanes * rows + row] = inv;
      }
    }
  }
}
// Tokens of the set `now` into a panel.
template <int F>
__device__ __noinline__ void fill_tokens(uint8_t* panel, float* scales, const void* from, int hidden, uint32_t now, int len, bool f16,
                                          int member, int members) {
  const int rows = __popc(now), parts = warps_per_row(rows, members);
#pragma unroll 1
  for (int row = member / parts; row < rows; row += members / parts) {
    uint32_t left = now;
    for (int r = 0; r < row; ++r) left &= left - 1;
    const uint16_t* x = reinterpret_cast<const uint16_t*>(from) + (int64_t)(__ffs(left) - 1) * hidden;
    fill_row<F, false>(panel, scales, x, hidden, len, row, rows, member % parts, parts, f16);
  }
}

// ---- products ----------------------------------------------------------------------------
// Where a lane finds the values of its columns' tokens in the panel: the step's first block and the way to the next one.
// Without a token: zeros, and no way.
struct FewTokens {
  uint32_t at, block;
  uint32_t scale[2], step;   // the scales of the lane's columns of sums, and the way to the next step's
};
template <int NT>
__device__ __forceinline__ void find_tokens(FewTokens (&x)[NT], uint32_t used, uint32_t in_panel, uint32_t panel, uint32_t scales, uint32_t zeros, int rows) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool there = (used >> (8 * n + g)) & 1;
    x[n].at = there ? panel + rank_below(in_panel, 8 * n + g) * 64 + t * 16 : zeros;
    x[n].block = there ? rows * 64 : 0;
    // (columns without a token: any scale, nobody reads them)
#pragma unroll
    for (int c = 0; c < 2; ++c) x[n].scale[c] = scales + min(rank_below(in_panel, 8 * n + 2 * t + c), rows - 1) * 4;
    x[n].step = rows * 4;
  }
}

// acc += W x of the step in the slot: a lane has eight features of eight rows of k; two rows side by side make the pairs of k that
// the instruction wants (rows g and g + 8 of product i are the lane's features 2 i and 2 i + 1).  halves: 32 and 32 columns
// (gates, ups) behind one another, else 64.
template <int F, int NT, int kTerms>
__device__ __forceinline__ void multiply_columns(float (&acc)[ColumnShape<F>::kTiles][NT][4], uint32_t slot, bool halves, const FewTokens (&x)[NT], int s) {
  constexpr int kTiles = ColumnShape<F>::kTiles;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint4 v[kTerms][NT];
  float d[kTiles][NT][4] = {};
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int q = 0; q < kTerms; ++q) v[q][n] = lds16(x[n].at + (s * kTerms + q) * x[n].block);
  // rows 2 t and 2 t + 1 of eight; the next eight rows are 512 or 1024 bytes on
  const uint32_t at0 = halves ? slot + (g >> 2) * 2048 + t * 128 + (((g & 3) ^ t) << 4) : slot + t * 256 + ((g ^ (2 * t)) << 4);
  const uint32_t at1 = halves ? at0 + 64 : slot + t * 256 + 128 + ((g ^ (2 * t + 1)) << 4), next = halves ? 512 : 1024;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t r[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = lds16((i & 1 ? at1 : at0) + (2 * h + (i >> 1)) * next);
      r[i][0] = w.x; r[i][1] = w.y; r[i][2] = w.z; r[i][3] = w.w;
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const uint32_t a0 = __byte_perm(r[0][i], r[1][i], 0x5410), a1 = __byte_perm(r[0][i], r[1][i], 0x7632);
      const uint32_t a2 = __byte_perm(r[2][i], r[3][i], 0x5410), a3 = __byte_perm(r[2][i], r[3][i], 0x7632);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < kTerms; ++q) {
          const uint32_t b0 = h ? v[q][n].z : v[q][n].x, b1 = h ? v[q][n].w : v[q][n].y;
          if constexpr (F == kFewBf16) mma_bf16(acc[i][n], a0, a1, a2, a3, b0, b1);
          else mma(d[i][n], a0, a1, a2, a3, b0, b1);
        }
    }
  }
  if constexpr (F == kFewF16) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float s0 = ldsf(x[n].scale[0] + s * x[n].step), s1 = ldsf(x[n].scale[1] + s * x[n].step);
#pragma unroll
      for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][n][c] = fmaf(c & 1 ? s1 : s0, d[i][n][c], acc[i][n][c]);
    }
  }
}

// Takes the step in the ring's slot and fetches the next one into it.
template <int F, int NT, int kTerms, typename Next>
__device__ __forceinline__ void take_columns(float (&acc)[ColumnShape<F>::kTiles][NT][4], FewRing& ring, bool halves, const FewTokens (&x)[NT], int s,
                                             Next next) {
  using S = ColumnShape<F>;
  ring_wait(ring);
  multiply_columns<F, NT, kTerms>(acc, ring.slots + ring.slot * S::kSlotBytes, halves, x, s);
  __syncwarp();
  next(ring.slot);
  if (++ring.slot == S::kDepth) {
    ring.slot = 0;
    ring.parity ^= 1;
  }
}

// ---- the kernels -------------------------------------------------------------------------
// The tiles that the warps of a block take together: where they are among the pieces, and a warp's part.
struct FewPlace {
  int at, a, u;           // the first piece: of all, its expert (of the active ones), and within that
  int pieces;             // that the block's warps take together
  int shift, member;      // log2 of the warps of a group with the same ones, and which one this is
  int skip, tiles;        // the group's pieces: where they begin, how many (none: 0 or less)
};

// Sums of the warps, for their owner to add up.
template <int F, int NT> struct RedShape {
  static constexpr int kTile = NT * 4 * 32 + 1;      // (off the banks of the tile before)
  static constexpr int kWarpFloats = ColumnShape<F>::kTiles * kTile, kBytes = (ColumnShape<F>::kWarps * kWarpFloats * 4 + 127) / 128 * 128;
  // Where the sums of row `row` (of a tile's 16) and column `col` are.
  static __device__ __forceinline__ int at(int tile, int row, int col) {
    return tile * kTile + ((col >> 3) * 4 + (row >> 3) * 2 + (col & 1)) * 32 + (row & 7) * 4 + ((col & 7) >> 1);
  }
};
// Tile and row (of the instruction) of the sums of a warp's gate or up f, and of its output c.
__device__ __forceinline__ int2 sums_of(int f, bool up, bool pairs) {
  if (pairs) return make_int2(f & 3, (f >> 2) + (up ? 8 : 0));
  return make_int2((f & 7) >> 1, (f >> 3) + (up ? 4 : 0) + (f & 1 ? 8 : 0));
}
__device__ __forceinline__ int2 sums_of(int c) { return make_int2((c & 7) >> 1, (c >> 3) + (c & 1 ? 8 : 0)); }
// A warp's sums to its place.
template <int F, int NT>
__device__ __forceinline__ void store_sums(float* red, const float (&acc)[ColumnShape<F>::kTiles][NT][4]) {
  float* const to = red + (threadIdx.x >> 5) * RedShape<F, NT>::kWarpFloats + (threadIdx.x & 31);
#pragma unroll
  for (int i = 0; i < ColumnShape<F>::kTiles; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) to[i * RedShape<F, NT>::kTile + (n * 4 + c) * 32] = acc[i][n][c];
}
template <int F, int NT> struct UpColumnsShape {
  static constexpr int kFixed = ColumnShape<F>::kRest + RedShape<F, NT>::kBytes;
};

// ---- the first kernel where weights are stored by column ---------------------------------------
// h[row] = act(W13 x + b13).  The features of all active experts, in pieces of eight (a tile's rows: eight gates and their
// eight ups), are dealt out evenly to the blocks.  Within a block all warps work side by side, so that rows of k are read in
// long runs; where fewer pieces are left than warps times tiles several have the same ones, take their steps in turn and add
// their sums up in shared memory.
template <int F, int NT>
__global__ void __launch_bounds__(ColumnShape<F>::kThreads, 1) few_up_columns_kernel(const __grid_constant__ FewParams p, const __grid_constant__ FewLaunch launch, const __grid_constant__ CUtensorMap map) {
  using S = ColumnShape<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTiles = S::kTiles;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + S::kTable);
  uint8_t* const zeros = smem + S::kZeros;                                // a token's values where there is no token
  int* const gave_up = reinterpret_cast<int*>(smem + S::kFlags);
  float* const red = reinterpret_cast<float*>(smem + S::kRest);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  FewRing ring = make_ring(smem, S::kSlotBytes, S::kDepth, smem, 0, reinterpret_cast<uint64_t*>(smem + S::kBars), gave_up, launch.status);
  uint8_t* const panel = smem + UpColumnsShape<F, NT>::kFixed;
  if (tid == 0) {
    *gave_up = 0;
    ptx::prefetch_tensormap(&map);
  }
  prefetch_call(p, tid, kThreads);
  pdl_wait();
  pdl_trigger();
  const FewMatrix& m = p.w13;
  const int steps = (p.hidden + S::kK - 1) / S::kK, per_expert = p.inter / 8;
  const int most = launch.panel_bytes / (steps * S::kPanelBytes(1)); // rows that the panel holds
  const bool whole = most >= p.tokens;                            // all tokens
  const int k8 = steps * (S::kK / 8);
  auto scales_after = [&](uint8_t* at, int rows) { return reinterpret_cast<float*>(at + rows * steps * (S::kK * 2)); };
  if (warp == 0) {
    build_table<false>(table, p);
  } else {
    if (tid < 48) reinterpret_cast<uint32_t*>(zeros)[tid - 32] = 0;
    if (blockIdx.x == 0)   // (the second kernel counts from there)
      for (int i = tid - 32; i < kFewMaxBlocks; i += kThreads - 32) launch.arrived[i] = 0;
    if (whole) fill_tokens<F>(panel, scales_after(panel, p.tokens), p.x, p.hidden, (1u << p.tokens) - 1u, k8, launch.f16, warp - 1, kWarps - 1);
  }
  __syncthreads();
  // (blocks begin and end at whole 32-byte sectors, at whole tiles where there are enough)
  const uint32_t unit = per_expert % 2 ? 1 : per_expert % 4 || table.active * per_expert < 16 * gridDim.x ? 2 : 4;
  const uint32_t all = (uint32_t)(table.active * per_expert) / unit;     // (times the blocks below 2^32: takes_mma)
  const int begin = (int)(all * blockIdx.x / gridDim.x * unit), end = (int)(all * (blockIdx.x + 1) / gridDim.x * unit);
  const bool pairs = p.act == B200MOE_ACT_SWIGLUOAI;

#pragma unroll 1
  for (int from = begin; from < end;) {
    // As many experts as have their tokens in the panel at once; one with more tokens than that goes through its
    // features again with the rest of them.
    uint32_t tokens = (1u << p.tokens) - 1u;
    int to = end;
    if (!whole) {
      const int a0 = from / per_expert;
      tokens = table.tokens[a0];
      to = min(end, (a0 + 1) * per_expert);
      if (__popc(tokens) <= most) {
        for (int a = a0 + 1; to < end && __popc(tokens | table.tokens[a]) <= most; ++a) {
          tokens |= table.tokens[a];
          to = min(end, (a + 1) * per_expert);
        }
      }
    }
    auto place = [&](FewPlace& at) {
      const int left = min(per_expert - at.u, to - at.at);
      at.shift = left > 4 * kTiles ? 0 : left > 2 * kTiles ? 1 : left > kTiles ? 2 : 3;
      at.pieces = min(kWarps * kTiles, left);
      at.skip = (warp >> at.shift) * kTiles;
      at.member = warp & ((1 << at.shift) - 1);
      at.tiles = min(kTiles, at.pieces - at.skip);
    };
    auto place_after = [&](FewPlace& at) {
      at.at += at.pieces;
      at.u += at.pieces;
      if (at.u == per_expert) { at.u = 0; ++at.a; }
      if (at.at < to) place(at);
    };
    FewPlace start;
    start.at = from;
    start.a = from / per_expert;
    start.u = from - start.a * per_expert;
    place(start);

#pragma unroll 1
    for (uint32_t rest = tokens; rest;) {
      uint32_t now = rest;
      while (__popc(now) > most) now &= ~(1u << (31 - __clz(now)));
      rest &= ~now;

      // The ring begins to fill.  The step that is fetched next, and whether its rows have been found.
      FewPlace next = start;
      int s = start.member;
      bool found = false;
      int e = 0, row = 0;
      auto copy_next = [&](int slot) {
        while (next.at < to && (s >= steps || !found)) {
          if (found || next.tiles <= 0) {     // (without tiles for this group: on to the next ones)
            place_after(next);
            s = next.member;
            found = false;
            if (next.at >= to || next.tiles <= 0) continue;
          }
          found = true;
          e = table.expert[next.a];
          row = (next.u + next.skip) * 8;
        }
        if (next.at < to) {
          if (lane == 0) {
            const uint32_t to_slot = ring.slots + slot * S::kSlotBytes, bar = ring.bars + slot * 8;
            ptx::fence_proxy_async();      // (the warp has read what was there)
            ptx::mbar_expect_tx_s(bar, S::kSlotBytes);
            if (pairs) {
              ptx::tma_load_3d_hint_s(to_slot, &map, bar, 2 * row, s * S::kK, e, ring.once);
            } else {
              ptx::tma_load_3d_hint_s(to_slot, &map, bar, row, s * S::kK, e, ring.once);
              ptx::tma_load_3d_hint_s(to_slot + S::kSlotBytes / 2, &map, bar, p.inter + row, s * S::kK, e, ring.once);
            }
          }
          s += 1 << next.shift;
        }
      };
#pragma unroll 1
      for (int i = 0; i < S::kDepth; ++i) copy_next((ring.slot + i) % S::kDepth);
      const int rows = __popc(now);
      if (!whole) {
        fill_tokens<F>(panel, scales_after(panel, rows), p.x, p.hidden, now, k8, launch.f16, warp, kWarps);
        __syncthreads();
      }

#pragma unroll 1
      for (FewPlace at = start; at.at < to; place_after(at)) {
        const int tiles = at.tiles, group = 1 << at.shift, a = at.a;
        if (tiles <= 0) continue;
        const uint32_t mine = table.tokens[a] & now;
        FewTokens x[NT];
        find_tokens<NT>(x, mine, now, smem_at(panel), smem_at(scales_after(panel, rows)), smem_at(zeros), rows);
        float acc[kTiles][NT][4] = {};
#pragma unroll 1
        for (int cs = at.member; cs < steps; cs += group) take_columns<F, NT, 1>(acc, ring, !pairs, x, cs, copy_next);
        // The tile's sums: a lane has a feature, the members take the tokens in turn.
        store_sums<F, NT>(red, acc);
        // (a barrier for each group of each size)
        const int barrier = (kWarps >> at.shift) + (warp >> at.shift);
        if (group > 1) group_sync(barrier, group * 32);
        else __syncwarp();
        const int i = lane >> 3, f = (at.u + at.skip + i) * 8 + (lane & 7);
        const int2 at_gate = sums_of(lane, false, pairs), at_up = sums_of(lane, true, pairs);
        int turn = 0;
        for (uint32_t left = mine; left; left &= left - 1, ++turn) {
          if ((turn & (group - 1)) != at.member) continue;
          const int col = __ffs(left) - 1, row = table.first_row[a] + rank_below(table.tokens[a], col);
          if (i < tiles) {
            const float* from_red = red + (warp - at.member) * RedShape<F, NT>::kWarpFloats;
            float gate = 0.f, up = 0.f;
            for (int w = 0; w < group; ++w) {
              gate += from_red[w * RedShape<F, NT>::kWarpFloats + RedShape<F, NT>::at(at_gate.x, at_gate.y, col)];
              up += from_red[w * RedShape<F, NT>::kWarpFloats + RedShape<F, NT>::at(at_up.x, at_up.y, col)];
            }
            if (m.bias) {
              const int64_t at = (int64_t)table.expert[a] * m.n;
              gate += load16(m.bias, at + (pairs ? 2 * f : f), launch.f16);
              up += load16(m.bias, at + (pairs ? 2 * f + 1 : p.inter + f), launch.f16);
            }
            p.h[(int64_t)row * p.inter + f] = gated_once(p.act, p.alpha, p.limit, p.clamp, gate, up);
          }
        }
        // the sums' place is free again
        if (group > 1) group_sync(barrier, group * 32);
        else __syncwarp();
      }
      __syncthreads();   // the panel is free again
    }
    from = to;
  }
}

// ---- the second kernel -------------------------------------------------------------------
// out = sum over experts of weight * (W2 h + b2).  A block has up to four times 64 columns of W2, by warps side by side that
// share their steps' values of h, and a share of the steps over all active experts, which makes as many blocks as there are SMs.  It goes
// through its steps with as many of h's values at a time as its panel holds, each group of warps with a stretch of them.  Of the blocks
// with the same columns the last one to be done adds the partial sums up, in their order.
template <int F, int NT>
__global__ void __launch_bounds__(ColumnShape<F>::kThreads, 1) few_down_columns_kernel(const __grid_constant__ FewParams p, const __grid_constant__ FewLaunch launch, const __grid_constant__ CUtensorMap map) {
  using S = ColumnShape<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTiles = S::kTiles, kRows = S::kRows;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + S::kTable);
  uint8_t* const zeros = smem + S::kZeros;
  int* const gave_up = reinterpret_cast<int*>(smem + S::kFlags);
  int& last_one = *reinterpret_cast<int*>(smem + S::kFlags + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;
  FewRing ring = make_ring(smem, S::kSlotBytes, S::kDepth, smem, 0, reinterpret_cast<uint64_t*>(smem + S::kBars), gave_up, launch.status);
  uint8_t* const panel = smem + S::kRest;
  float* const red = reinterpret_cast<float*>(panel);                     // (after the last panel)
  if (tid == 0) {
    *gave_up = 0;
    ptx::prefetch_tensormap(&map);
  }
  // What routed the tokens was complete before the kernel ahead of this one let it start.
  if (warp == 0) build_table<true>(table, p);
  else if (tid < 48) reinterpret_cast<uint32_t*>(zeros)[tid - 32] = 0;
  __syncthreads();
  const FewMatrix& m = p.w2;
  const FewShare share(table, launch);
  const int steps = share.steps, step_begin = share.begin, step_end = share.end, row_begin = share.column * launch.side * kRows, row_end = p.hidden;
  const int side = launch.side, members = kWarps / side, member = warp / side, mine_side = warp % side, block_rows = side * kRows;
  float* const scales = reinterpret_cast<float*>(panel + launch.room * (S::kTerms * S::kK * 2));
  bool waited = false;

  auto finish = [&](float v, int token, int n) {
    const int64_t to = (int64_t)token * p.hidden + n;
    if (launch.f16) reinterpret_cast<__half*>(p.out)[to] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(v);
  };
  for (int block_r0 = row_begin; block_r0 < row_end || !waited; block_r0 += launch.columns * block_rows) {
    const int r0 = block_r0 + mine_side * kRows;
    const bool there = r0 < row_end;
    // The step that is fetched next, how many are left of this warp's stretch, and where the panel after that begins.
    int fetch_a = 0, fetch_s = 0, left = 0, panel_a = step_begin / steps, panel_s = step_begin - panel_a * steps;
    auto copy_next = [&](int slot) {
      while (left == 0 && panel_a * steps + panel_s < step_end) {
        int a1, s1;
        share.panel_end(table, launch.room, panel_a, panel_s, a1, s1);
        const int from = panel_a * steps + panel_s, all = a1 * steps + s1 - from, mine = all * member / members;
        left = all * (member + 1) / members - mine;
        fetch_a = (from + mine) / steps;
        fetch_s = from + mine - fetch_a * steps;
        panel_a = a1;
        panel_s = s1;
      }
      if (left > 0 && there) {
        if (fetch_s == steps) { fetch_s = 0; ++fetch_a; }
        if (lane == 0) {
          const uint32_t bar = ring.bars + slot * 8;
          ptx::fence_proxy_async();        // (the warp has read what was there)
          ptx::mbar_expect_tx_s(bar, S::kSlotBytes);
          ptx::tma_load_3d_hint_s(ring.slots + slot * S::kSlotBytes, &map, bar, r0, fetch_s * S::kK, table.expert[fetch_a], ring.once);
        }
        ++fetch_s;
        --left;
      }
    };
#pragma unroll 1
    for (int i = 0; i < S::kDepth; ++i) copy_next((ring.slot + i) % S::kDepth);
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
    }
    float out[kTiles][NT][4] = {};
    for (int a0 = step_begin / steps, s0 = step_begin - a0 * steps; a0 * steps + s0 < step_end;) {
      int a1, s1;
      share.panel_end(table, launch.room, a0, s0, a1, s1);
      const int last = s1 > 0 ? a1 : a1 - 1;           // the last expert with steps in the panel
      const int row0 = table.first_row[a0], rows = table.first_row[last + 1] - row0;
      {
        // (the first expert's rows have the steps from s0 on, the last one's those up to s1)
        constexpr int kPiece = S::kK / 8;
        const int parts = warps_per_row(rows, kWarps), n0 = table.first_row[a0 + 1] - row0;
#pragma unroll 1
        for (int row = warp / parts; row < rows; row += kWarps / parts) {
          const int r = row0 + row, a = table.row_expert[r], e0 = table.first_row[a], n = table.first_row[a + 1] - e0;
          const int k8_0 = (a == a0 ? s0 : 0) * kPiece, len = (a == a1 ? s1 : steps) * kPiece - k8_0;
          const int before = a == a0 ? 0 : n0 * (steps - s0) + (e0 - row0 - n0) * steps;   // rows times steps of earlier experts
          fill_row<F, true>(panel + before * (S::kTerms * S::kK * 2), scales + before, p.h + (int64_t)r * p.inter + 8 * k8_0, p.inter - 8 * k8_0, len,
                            r - e0, n, warp % parts, parts, false);
        }
        __syncthreads();
      }
      {
        const int from = a0 * steps + s0, all = a1 * steps + s1 - from;
        int pos = from + all * member / members;
        const int stop = there ? from + all * (member + 1) / members : 0;
        for (int a = pos / steps; pos < stop; ++a) {
          const int row = table.first_row[a], n_rows = table.first_row[a + 1] - row, end = min(stop, (a + 1) * steps);
          // rows of earlier experts in the panel, as above
          const int before = a == a0 ? 0 : (table.first_row[a0 + 1] - row0) * (steps - s0) + (row - table.first_row[a0 + 1]) * steps;
          const uint32_t base = smem_at(panel) + (before - (a == a0 ? s0 : 0) * n_rows) * (S::kTerms * S::kK * 2);
          const uint32_t base_scales = smem_at(scales) + (before - (a == a0 ? s0 : 0) * n_rows) * 4;
          const uint32_t mine = table.tokens[a];
          FewTokens x[NT];
          find_tokens<NT>(x, mine, mine, base, base_scales, smem_at(zeros), n_rows);
          float acc[kTiles][NT][4] = {};
#pragma unroll 1
          for (; pos < end; ++pos) take_columns<F, NT, S::kTerms>(acc, ring, false, x, pos - a * steps, copy_next);
          // (columns of tokens without this expert are left out: a weight that is not finite would get into them)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int token = 8 * n + 2 * t + c;
              if (!((mine >> token) & 1)) continue;
              const float w = table.weight[row + rank_below(mine, token)];
#pragma unroll
              for (int i = 0; i < kTiles; ++i) {
                out[i][n][c] = fmaf(w, acc[i][n][c], out[i][n][c]);
                out[i][n][c + 2] = fmaf(w, acc[i][n][c + 2], out[i][n][c + 2]);
              }
            }
        }
      }
      a0 = a1;
      s0 = s1;
      __syncthreads();   // the panel is free again
    }
    store_sums<F, NT>(red, out);
    __syncthreads();
    auto put = [&](float v, int token, int row) {
      const int64_t to = (int64_t)token * p.hidden + row;
      if (launch.splits == 1) finish(v, token, row);
      else launch.part[(int64_t)share.split * p.tokens * p.hidden + to] = v;
    };
    // consecutive threads, consecutive features of a token
    for (int j = tid; j < block_rows * p.tokens; j += kThreads) {
      const int row = j % block_rows, token = j / block_rows;
      if (block_r0 + row >= row_end) continue;
      const int2 at = sums_of(row % kRows);
      float v = m.bias && share.split == 0 ? weighted_bias(table, m, p.topk, launch.f16, token, block_r0 + row) : 0.f;
      for (int w = row / kRows; w < kWarps; w += side) v += red[w * RedShape<F, NT>::kWarpFloats + RedShape<F, NT>::at(at.x, at.y, token)];
      put(v, token, block_r0 + row);
    }
    __syncthreads();
  }
  if (launch.splits > 1) sum_splits(launch, p, last_one, share.column, row_begin, min(row_end - row_begin, block_rows), finish);
}

}  // namespace
}  // namespace b200moe
