// The layer for a few tokens where weights are stored by output feature ([E,N,K]: block-scaled fp8, MXFP4, int4), on the
// tensor cores.
//
//   D[features, tokens] += W[16 features, 16 k] x^T[16 k, 8 tokens]     (mma.sync, fp32 accumulation)
//
// A few tokens leave the layer to the bandwidth of its weights: every byte of an active expert passes once, from L2
// through a warp's own ring in shared memory (TMA) into the registers that the matrix instruction reads, with one
// conversion to float16 on the way, which holds every code of the three formats exactly.  The sum over k does not mind its order,
// so a lane's 16 bytes of a row go into the instruction as they come and the tokens are laid out to match.  Scales of weights
// multiply sums of their group in fp32.  Tokens and activations are float16 with a power of two per 64 or 128 values of a row,
// which keeps a bfloat16 as it is and rounds h to 11 bits.
//
// tcgen05 would have to get its weights converted in shared or tensor memory, a second pass for every byte, and its tile
// of 128 features leaves most SMs without work at one token.
#pragma once

#include "few_tokens.cuh"
#include "gemm_tc_common.cuh"
#include "sm100_ptx.cuh"

namespace b200moe {
namespace {

constexpr int kFewMaxBlocks = 160;      // of a kernel (one per SM)
constexpr int kFewMaxColumns = kFewMaxBlocks;
constexpr int kMaxSlots = kFewMaxTopk * B200MOE_FEW_TOKENS;   // routed slots of a call

enum FewFormat { kFewFp8, kFewFp4, kFewInt4Fine, kFewInt4, kFewBf16, kFewF16 };   // Fine: groups of 32 or 64
__host__ __device__ constexpr bool by_column(int f) { return f == kFewBf16 || f == kFewF16; }     // stored as [K, N]

// A step of a warp is 4 KB: 128 bytes of its 32 rows; of weights stored by column 32 rows of 128 bytes.  Codes are turned into
// float16 by every warp for itself, between loads from shared memory and products that depend on one another, and 16 warps
// hide that where 8 with twice the rows did not
template <int F> struct FewShape {
  static constexpr int kWarps = by_column(F) ? 8 : 12, kThreads = 32 * kWarps;
  static constexpr int kTiles = by_column(F) ? 4 : 2, kRows = 16 * kTiles;     // tiles of 16 rows that a warp takes at once
  static constexpr int kK = by_column(F) ? 32 : F == kFewFp8 ? 128 : 256;     // values of k
  static constexpr int kHalfBlocks = by_column(F) ? 1 : F == kFewFp8 ? 2 : 4;  // of the panel, per 64 bytes of a weight row
  static constexpr int kBlocks = kK / 32;                        // of the panel: a lane's eight values, two instructions
  // Of the panel: a row's values of a step and their scale.  h next to 16-bit weights is there twice, as the type has it
  // and what that leaves of it: with one rounding to 16 bits the results would be 1.4 times as far from the formula's as
  // their own rounding puts them.
  __host__ __device__ static constexpr int kPanelBytes(int terms) { return terms * kK * 2 + 4; }
  static constexpr int kTerms = by_column(F) ? 2 : 1;            // of h
  static constexpr int kScaleWords = F == kFewInt4Fine ? 4 : F == kFewFp4 ? 2 : 1;  // that hold a row's scales of a step
  static constexpr int kScales = F == kFewFp8 || by_column(F) ? 0 : F == kFewInt4 ? 2 : 8;                       // of a row and step, made fp32 (fp8: are so)
  static constexpr int kSlotBytes = 4096, kDepth = by_column(F) ? 3 : 2;
  static constexpr int kRing = kDepth * kSlotBytes;
  // behind the rings of all warps, per warp: scales of the steps in the ring as they come, and as fp32
  static constexpr int kSlotScales = by_column(F) ? 0 : kRows * 4 * kScaleWords;
  static constexpr int kRingScales = kDepth * kSlotScales + kRows * kScales * 4;
};

// ---- which experts a call uses ------------------------------------------------------
// Active experts in ascending order, their tokens as bits, and a row number for every (expert, token) that occurs: rows
// of an expert follow one another in token order.
struct FewTable {
  uint32_t bits[32];
  int before[32];
  int active, rows;
  int expert[kMaxSlots];
  uint32_t tokens[kMaxSlots];
  int first_row[kMaxSlots + 1];
  int slot_expert[kMaxSlots];      // the slot's expert, as an index of the active ones (-1: none)
  uint16_t row_expert[kMaxSlots];
  float weight[kMaxSlots];         // of a row: the sum over the slots that name its expert
  float slot_weight[kMaxSlots];
};

__device__ __forceinline__ int rank_below(uint32_t mask, int bit) { return __popc(mask & ((1u << bit) - 1u)); }

// By one warp; the others meet it at the block's next barrier.
template <bool kWeights>
__device__ __forceinline__ void build_table(FewTable& t, const FewParams& p) {
  const int slots = p.tokens * p.topk, lane = threadIdx.x & 31;
  t.bits[lane] = 0;
  for (int i = lane; i < slots; i += 32) t.tokens[i] = 0;
  __syncwarp();
#pragma unroll 1
  for (int i = lane; i < slots; i += 32) {
    const int e = local_expert(p, i);
    t.slot_expert[i] = e;
    if (kWeights) t.slot_weight[i] = p.weights[i];
    if (e >= 0) atomicOr(&t.bits[e >> 5], 1u << (e & 31));
  }
  __syncwarp();
  {
    const int n = __popc(t.bits[lane]);
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    t.before[lane] = sum - n;
    if (lane == 31) t.active = sum;
  }
  __syncwarp();
  bool again = false;      // a token that names an expert twice
#pragma unroll 1
  for (int i = lane; i < slots; i += 32) {
    const int e = t.slot_expert[i], tok = i / p.topk;
    if (e < 0) continue;
    const int a = t.before[e >> 5] + rank_below(t.bits[e >> 5], e & 31);
    t.slot_expert[i] = a;
    t.expert[a] = e;
    again |= (atomicOr(&t.tokens[a], 1u << tok) >> tok) & 1;
  }
  again = __any_sync(0xffffffffu, again);
  __syncwarp();
  int base = 0;
#pragma unroll 1
  for (int a0 = 0; a0 < t.active; a0 += 32) {
    const int a = a0 + lane, n = a < t.active ? __popc(t.tokens[a]) : 0;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    if (a < t.active) t.first_row[a] = base + sum - n;
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) { t.first_row[t.active] = base; t.rows = base; }
  __syncwarp();
  if (kWeights) {
#pragma unroll 1
    for (int i = lane; i < slots; i += 32) {
      const int a = t.slot_expert[i], tok = i / p.topk;
      if (a < 0) continue;
      float w = t.slot_weight[i];
      if (again) {    // the token's slots with this expert in their order, by the first of them
        bool other = false;
        for (int j = tok * p.topk; j < i; ++j) other |= t.slot_expert[j] == a;
        if (other) continue;
        for (int j = i + 1; j < (tok + 1) * p.topk; ++j)
          if (t.slot_expert[j] == a) w += t.slot_weight[j];
      }
      const int row = t.first_row[a] + rank_below(t.tokens[a], tok);
      t.weight[row] = w;
      t.row_expert[row] = (uint16_t)a;
    }
  }
}

// ---- loads ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// (volatile: they stay behind the waits and barriers ahead of them)
__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ float ldsf(uint32_t a) { return __uint_as_float(lds4(a)); }
__device__ __forceinline__ void sts16(uint32_t a, float x, float y, float z, float w) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
__device__ __forceinline__ void sts4(uint32_t a, float x) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(x) : "memory"); }

// Barrier of some of the block's warps.
__device__ __forceinline__ void group_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// ---- conversions and products ------------------------------------------------------------
// Four e4m3 codes of a word -> float16 pairs (0,1) (2,3).  (One instruction each; through the header's function, which takes
// and returns halves of registers, seven for the two.)
__device__ __forceinline__ void e4m3x4_to_h2(uint32_t w, uint32_t& a, uint32_t& b) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(a), "=r"(b) : "r"(w));
}
// Eight e2m1 codes of a word -> float16 pairs (0,1) (2,3) (4,5) (6,7).
__device__ __forceinline__ void e2m1x8_to_h2(uint32_t w, uint32_t (&o)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]) : "r"(w));
}
// Eight two's-complement nibbles -> float16 pairs (0,4) (1,5) (2,6) (3,7).  n ^ 8 = n + 8 is unsigned; below the exponent of
// 1024 it counts in ones, four bits higher in sixteenths of that.
__device__ __forceinline__ void s4x8_to_h2(uint32_t w, uint32_t (&o)[4]) {
  const __half2 one = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));       // 1024 + 8
  const __half2 down = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));      // 1 / 16
  const __half2 off = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));       // -(64 + 8)
  const uint32_t h = w >> 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = i ? h : w;
    const uint32_t lo = (v & 0x000f000fu) ^ 0x64086408u, hi = (v & 0x00f000f0u) ^ 0x64806480u;
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), one);
    const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), down, off);
    o[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
    o[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
  }
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a sum.
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// ---- tokens and activations as float16 -------------------------------------------------
// A panel holds rows of values in the order in which the lanes want them: per step blocks of [row][4 lanes][8 values].
// Where k sits: fp8 lanes hold 16 bytes of a row, 16 values; 4-bit formats hand a group of 32 values out to the four lanes,
// eight each; weights by column have 32 rows, of which a lane multiplies 2 t, 2 t + 1 and every eighth after these.  Behind them, per row and step, the inverse of what the values have been multiplied by.
template <int F>
__device__ __forceinline__ uint32_t panel_at(int k8, int row, int rows, int terms) {   // k8: k / 8; a second term is a block on
  const int block = (F == kFewFp8 ? (k8 >> 3) * 2 + (k8 & 1) : k8 >> 2) * terms;
  const int t = by_column(F) ? 0 : F == kFewFp8 ? (k8 >> 1) & 3 : k8 & 3;     // (by column: all four, see store8)
  return (uint32_t)(((block * rows + row) * 4 + t) * 16);
}

// The power of two by which values are multiplied on their way to float16, their largest magnitude then between 2^14 and 2^15,
// and its inverse.  Magnitudes below 2^-100 are taken for that; what is not finite stays as it is.
__device__ __forceinline__ float step_scale(uint32_t top, float& inverse) {   // top: bits of the largest magnitude
  int e = (int)(top >> 23);
  if (e == 255) e = 127 + 14;
  e = max(e, 127 - 100);
  inverse = __uint_as_float((uint32_t)(e - 14) << 23);
  return __uint_as_float((uint32_t)(254 - (e - 14)) << 23);
}

// Eight values as a lane wants them: int4 pairs are four apart.
template <int F>
__device__ __forceinline__ uint4 packed8(const float (&v)[8]) {
  constexpr bool kApart = F == kFewInt4 || F == kFewInt4Fine;
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F == kFewBf16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = kApart ? __floats2half2_rn(v[i], v[i + 4]) : __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Eighth j of a row to its place: at the panel's place for it, or by column a word to each of the four lanes.
template <int F>
__device__ __forceinline__ void store8(uint8_t* at, int j, const uint4& o) {
  if constexpr (by_column(F)) {
    uint32_t* const w = reinterpret_cast<uint32_t*>(at) + (j & 3);
    w[0] = o.x;
    w[4] = o.y;
    w[8] = o.z;
    w[12] = o.w;
  } else {
    *reinterpret_cast<uint4*>(at) = o;
  }
}

// `len` eighths of a row (what is beyond `values` values is zero) into a panel, by `parts` warps of which this is `part`.  A warp
// asks for four times 256 values at once: the loads' latency is what this costs.  (Functions that run once in a while are not
// inlined: both kernels' code together has to stay in the SM's instruction cache.  With 160 KB of it every launch began
// with some 3 us of misses.)
template <int F, bool kF32>
__device__ __noinline__ void fill_row(uint8_t* panel, float* scales, const void* from, int values, int len, int row, int rows, int part, int parts,
                                      bool f16) {
  constexpr int kLanes = FewShape<F>::kK / 8;      // of a step (at most 32)
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
        constexpr int kTerms = kF32 ? FewShape<F>::kTerms : 1;
        uint8_t* const at = panel + panel_at<F>(j, row, rows, kTerms);
        const uint4 o = packed8<F>(v);
        store8<F>(at, j, o);
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
          store8<F>(at + rows * 64, j, packed8<F>(rest));
        }
        if ((j & (kLanes - 1)) == 0) scales[j / kLanes * rows + row] = inv;
      }
    }
  }
}
// Warps of a row where `warps` of them fill a panel of `rows`.
__device__ __forceinline__ int warps_per_row(int rows, int warps) { return rows >= warps ? 1 : warps / rows; }

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

// ---- weights: a warp's ring ------------------------------------------------------------
// One lane asks for a step's weights by TMA, whose swizzle puts the 16-byte pieces of a row where the lanes' reads fall on
// different banks: rows of 128 bytes (a lane reads one of four pieces, or a word of each: a group of 32 4-bit codes is
// handed out to four lanes; rows of 64 bytes kept the copy unit from the memory's rate, fp8 at one token 91 us, 74 without
// it), by column rows of 128 or two halves of 64.  Scales are fetched as words, neighbouring rows
// by neighbouring lanes (those of 4-bit formats are laid out for that: as they come, a step's would be 2 or 4 bytes of every
// row, which kept the load units busy for longer than the weights did), and made fp32 by one lane per row.
// (With every lane fetching its own pieces, MXFP4 took a third more instructions, and every first touch of a page held up
// the warps: both kernels at one MXFP4 token 28.7 us, 16-bit weights at 16 tokens, whose rows are far apart, 765 us.)

// Where the rows of a step lie in a slot, and their scales: rows g and g + 8 of tile i.
struct FewOrder {
  int tile, half;             // bytes from one tile to the next, from row g to g + 8
  int place, place_half;      // the same for places of scales
};
__device__ __forceinline__ FewOrder row_order() { return {2048, 1024, 16, 8}; }         // 32 rows
__device__ __forceinline__ FewOrder halves_order() { return {1024, 2048, 8, 16}; }      // 16 gates, 16 ups
// Row of eight that the instruction's row g is: of the lanes that read 16 bytes at once (two rows g) one is in the first
// four, so that the swizzle takes them to different banks.
__device__ __forceinline__ int row_of(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ int g_of(int row) { return ((row & 3) << 1) | (row >> 2); }

// What a warp fetches: the rows of one expert's matrix that it takes at once.
struct FewRows {
  int e, row;                             // expert, first row (feature)
  int tiles;                              // that there are
  const uint8_t* s;                       // scales of step 0 of the row that the lane looks after
  bool there;                             // whether it is
};
// The matrix as a whole.
struct FewLayout {
  int row_bytes, group, k;
  int words, word_step;  // of a row's scales (4 bits), and bytes from one to the next
  bool f16;
  __device__ __forceinline__ FewLayout(const FewMatrix& m, int f, bool half) {
    row_bytes = by_column(f) ? 2 * m.n : f == kFewFp8 ? m.k : m.k / 2;
    k = m.k;
    group = m.group;
    words = f == kFewFp8 ? 0 : few_scale_words(m.format, m.group, m.k);
    word_step = f == kFewFp8 ? 4 : 4 * m.n;
    f16 = half;
  }
};
// Scales of step 0 of row n.  4 bits: [experts][words][n], words as in few_scale_words.
template <int F>
__device__ __forceinline__ const uint8_t* scales_of(const FewMatrix& m, const FewLayout& l, int e, int n) {
  if (F == kFewFp8) return reinterpret_cast<const uint8_t*>(m.scale) + (int64_t)(e * (m.n >> 7) + (n >> 7)) * (m.k >> 5);
  return reinterpret_cast<const uint8_t*>(m.scale) + (int64_t)(e * l.words) * (4 * m.n) + n * 4;
}

// Fetches the scales of step s.
template <int F>
__device__ __forceinline__ void copy_scales(uint32_t to, const FewRows& r, const FewLayout& l, int s) {
  using S = FewShape<F>;
  const int lane = threadIdx.x & 31;
  // (the other matrix of kFewInt4Fine may have groups of 128 and more: a word for 256 values)
  const int words = F == kFewInt4Fine ? (l.group == 32 ? 4 : l.group == 64 ? 2 : 1) : S::kScaleWords, word = s * words;
  if (!r.there) return;
#pragma unroll
  for (int i = 0; i < S::kScaleWords; ++i)
    // (a row's last step may have fewer; what they stand for is beyond the row)
    if (i < words && (F == kFewFp8 || word + i < l.words)) copy4(to + (lane * S::kScaleWords + i) * 4, r.s + (int64_t)(word + i) * l.word_step);
}

// A warp's ring, one slot after the other.
struct FewRing {
  uint32_t slots, bars;      // shared addresses: of slot 0, of its barrier
  uint32_t scales;           // of the scales of slot 0
  int slot, parity;          // that is taken next
  volatile int* gave_up;
  int32_t* status;
  uint64_t once;             // L2 policy of the weights
};
// Waits for a slot; a wait that runs out sets the status word, and the kernel goes on with what is there (later waits, one for
// every copy in flight, are short then).
static __device__ __noinline__ void ring_wait_long(uint32_t bar, int parity, volatile int* gave_up, int32_t* status) {
  const long long budget = *gave_up ? 1000000 : ptx::kWaitBudgetCycles, t0 = clock64();
  while (!ptx::mbar_try_wait_s(bar, parity)) {
    if (clock64() - t0 > budget) {
      *gave_up = 1;
      if (status) *reinterpret_cast<volatile int32_t*>(status) = 1;
      return;
    }
  }
}
__device__ __forceinline__ void ring_wait(const FewRing& r) {
  const uint32_t bar = r.bars + r.slot * 8;
  if (!ptx::mbar_try_wait_s(bar, r.parity)) ring_wait_long(bar, r.parity, r.gave_up, r.status);
}

// The scales of step s as fp32.
template <int F>
__device__ __forceinline__ void spread_scales(uint32_t to, uint32_t from, const FewLayout& l, int s) {
  using S = FewShape<F>;
  const int row = threadIdx.x & 31;
  const uint32_t at = from + row * S::kScaleWords * 4;
  auto value = [&](uint32_t h) { return l.f16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16); };
  if constexpr (F == kFewInt4) {
    const uint32_t v = lds4(at);
    sts4(to + row * 8, value(v & 0xffffu));
    sts4(to + row * 8 + 4, value(v >> 16));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {       // the halves of the step
      const uint32_t place = to + (h * S::kRows + row) * 16;
      if constexpr (F == kFewFp4) {
        // 2^(byte - 127): the byte is the exponent (0 gives zero for 2^-127, 255 infinity for NaN).  Beyond the row: zeros,
        // as whatever is there must not make a NaN of them.
        const uint32_t v = 2 * s + h < l.words ? lds4(at + 4 * h) : 0;
        sts16(place, __uint_as_float((v & 255u) << 23), __uint_as_float((v << 15) & 0x7f800000u), __uint_as_float((v << 7) & 0x7f800000u),
              __uint_as_float((v >> 1) & 0x7f800000u));
      } else if constexpr (F == kFewInt4Fine) {
        if (l.group == 32) {
          const uint32_t v = 4 * s + 2 * h < l.words ? lds4(at + 8 * h) : 0, w = 4 * s + 2 * h < l.words ? lds4(at + 8 * h + 4) : 0;
          sts16(place, value(v & 0xffffu), value(v >> 16), value(w & 0xffffu), value(w >> 16));
        } else if (l.group == 64) {
          const uint32_t v = 2 * s + h < l.words ? lds4(at + 4 * h) : 0;
          const float a = value(v & 0xffffu), b = value(v >> 16);
          sts16(place, a, a, b, b);
        } else {
          const float a = value(lds4(at) >> 16 * h & 0xffffu);
          sts16(place, a, a, a, a);
        }
      }
    }
  }
}

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

// acc += W x of the step in the slot, for the first `Tiles` tiles (what one of them has not got is something finite or not, in
// rows that nobody reads).
template <int F, int NT, int Tiles>
__device__ __forceinline__ void multiply_step(float (&acc)[FewShape<F>::kTiles][NT][4], uint32_t slot, uint32_t scales, const FewOrder& order,
                                              const FewTokens (&x)[NT], int s) {
  using S = FewShape<F>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, row = row_of(g);
  float sx[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) sx[n][c] = ldsf(x[n].scale[c] + s * x[n].step);
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {       // the row's first and second 64 bytes
    uint4 v[S::kHalfBlocks][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < S::kHalfBlocks; ++q) v[q][n] = lds16(x[n].at + (s * S::kBlocks + h * S::kHalfBlocks + q) * x[n].block);
#pragma unroll
    for (int i = 0; i < Tiles; ++i) {
      const int at_lo = i * order.place + row, at_hi = at_lo + order.place_half;     // places of the scales
      float d[NT][4], sum[NT][4] = {};   // products of a group of weights, and the half's
      auto add = [&](float a, float b) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sum[n][0] = fmaf(a, d[n][0], sum[n][0]);
          sum[n][1] = fmaf(a, d[n][1], sum[n][1]);
          sum[n][2] = fmaf(b, d[n][2], sum[n][2]);
          sum[n][3] = fmaf(b, d[n][3], sum[n][3]);
        }
      };
      if constexpr (F == kFewFp8) {
        const uint32_t at = slot + i * order.tile + row * 128 + (((4 * h + t) ^ row) << 4);
        const uint4 lo = lds16(at), hi = lds16(at + order.half);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_to_h2(wl[w], a0, a2);
          e4m3x4_to_h2(wh[w], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 b = v[w >> 1][n];
            if (w == 0) mma_first(d[n], a0, a1, a2, a3, b.x, b.y);
            else mma(d[n], a0, a1, a2, a3, w & 1 ? b.z : b.x, w & 1 ? b.w : b.y);
          }
        }
        add(ldsf(scales + at_lo * 4), ldsf(scales + at_hi * 4));
      } else {
        uint4 lo, hi;
        if constexpr (S::kScales == 8) {
          lo = lds16(scales + (h * S::kRows + at_lo) * 16);
          hi = lds16(scales + (h * S::kRows + at_hi) * 16);
        } else {
          lo.w = lds4(scales + at_lo * 8 + h * 4);
          hi.w = lds4(scales + at_hi * 8 + h * 4);
        }
        const uint32_t w = slot + i * order.tile + row * 128 + t * 4;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int at = ((4 * h + q) ^ row) << 4;
          const uint32_t wl = lds4(w + at), wh = lds4(w + at + order.half);
          uint32_t al[4], ah[4];
          if constexpr (F == kFewFp4) { e2m1x8_to_h2(wl, al); e2m1x8_to_h2(wh, ah); }
          else { s4x8_to_h2(wl, al); s4x8_to_h2(wh, ah); }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (S::kScales == 8 || q == 0) mma_first(d[n], al[0], ah[0], al[1], ah[1], v[q][n].x, v[q][n].y);
            else mma(d[n], al[0], ah[0], al[1], ah[1], v[q][n].x, v[q][n].y);
            mma(d[n], al[2], ah[2], al[3], ah[3], v[q][n].z, v[q][n].w);
          }
          if (S::kScales == 8 || q == 3) add(__uint_as_float(q == 0 ? lo.x : q == 1 ? lo.y : q == 2 ? lo.z : lo.w),
                                               __uint_as_float(q == 0 ? hi.x : q == 1 ? hi.y : q == 2 ? hi.z : hi.w));
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][n][c] = fmaf(sx[n][c & 1], sum[n][c], acc[i][n][c]);
    }
  }
}

// The same for weights by column: a lane has eight features of eight rows of k; two rows side by side make the pairs of k that
// the instruction wants (rows g and g + 8 of product i are the lane's features 2 i and 2 i + 1).  halves: 32 and 32 columns
// (gates, ups) behind one another, else 64.
template <int F, int NT, int kTerms>
__device__ __forceinline__ void multiply_columns(float (&acc)[FewShape<F>::kTiles][NT][4], uint32_t slot, bool halves, const FewTokens (&x)[NT], int s) {
  constexpr int kTiles = FewShape<F>::kTiles;
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
__device__ __forceinline__ void take_step(float (&acc)[FewShape<F>::kTiles][NT][4], FewRing& ring, int tiles, const FewOrder& order, bool halves, const FewLayout& l,
                                          const FewTokens (&x)[NT], int s, Next next) {
  using S = FewShape<F>;
  const uint32_t at = ring.slots + ring.slot * S::kSlotBytes;
  uint32_t scales = ring.scales + ring.slot * S::kSlotScales;
  copies_wait<S::kDepth - 1>();
  if (!by_column(F) && F != kFewFp8) {
    const uint32_t to = ring.scales + S::kDepth * S::kSlotScales;
    spread_scales<F>(to, scales, l, s);
    scales = to;
  }
  __syncwarp();
  ring_wait(ring);
  if constexpr (by_column(F)) multiply_columns<F, NT, kTerms>(acc, at, halves, x, s);
  else if (tiles > S::kTiles / 2) multiply_step<F, NT, S::kTiles>(acc, at, scales, order, x, s);
  else multiply_step<F, NT, S::kTiles / 2>(acc, at, scales, order, x, s);
  __syncwarp();
  next(ring.slot);
  if (++ring.slot == S::kDepth) {
    ring.slot = 0;
    ring.parity ^= 1;
  }
}
// Sets a warp's ring up.
template <int F>
__device__ __forceinline__ FewRing make_ring(uint8_t* rings, uint8_t* scales, uint64_t* bars, int* gave_up, int32_t* status) {
  using S = FewShape<F>;
  const int warp = threadIdx.x >> 5;
  FewRing r;
  r.slots = smem_at(rings) + warp * S::kRing;
  r.scales = smem_at(scales) + warp * S::kRingScales;
  r.bars = smem_at(bars + warp * S::kDepth);
  r.slot = r.parity = 0;
  r.gave_up = gave_up;
  r.status = status;
  r.once = ptx::l2_evict_first();
  if ((threadIdx.x & 31) == 0) {
    for (int i = 0; i < S::kDepth; ++i) ptx::mbar_init(bars + warp * S::kDepth + i, 1);
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  __syncwarp();
  return r;
}

__device__ __noinline__ float gated_once(int act, float alpha, float limit, float clamp, float gate, float up) {
  return gated(act, alpha, limit, clamp, gate, up);
}
__device__ __forceinline__ float load16(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(reinterpret_cast<const __half*>(p)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// ---- the kernels -------------------------------------------------------------------------
struct FewLaunch {
  int panel_bytes;       // of shared memory for the panel
  bool f16;
  int splits;            // shares of the second kernel's steps: blocks / splits have the same rows
  int side;              // warps side by side in the second kernel (1, 2, 4)
  uint32_t* arrived;     // per column of blocks of the second kernel
  float* part;           // [splits][tokens][hidden]: partial sums, with more than one split
  int box;               // rows (by column: columns) of a warp of the second kernel, which a load brings
  int32_t* status;       // for waits that run out, or NULL
};

// The tiles that the warps of a block take together: where they are among the pieces, and a warp's part.
struct FewPlace {
  int at, a, u;           // the first piece: of all, its expert (of the active ones), and within that
  int pieces;             // that the block's warps take together
  int shift, member;      // log2 of the warps of a group with the same ones, and which one this is
  int skip, tiles;        // the group's pieces: where they begin, how many (none: 0 or less)
};

constexpr int kBlockRows = 64;      // of W2 that a block of the second kernel has at once (by column: its own rule)
constexpr int kTableBytes = (sizeof(FewTable) + 127) / 128 * 128;
// Sums of the warps, for their owner to add up.
template <int F, int NT> struct RedShape {
  static constexpr int kTile = NT * 4 * 32 + 1;      // (off the banks of the tile before)
  static constexpr int kWarpFloats = FewShape<F>::kTiles * kTile, kBytes = (FewShape<F>::kWarps * kWarpFloats * 4 + 127) / 128 * 128;
  // Where the sums of row `row` (of a tile's 16) and column `col` are.
  static __device__ __forceinline__ int at(int tile, int row, int col) {
    return tile * kTile + ((col >> 3) * 4 + (row >> 3) * 2 + (col & 1)) * 32 + (row & 7) * 4 + ((col & 7) >> 1);
  }
};
// Tile and row (of the instruction) of the sums of a warp's gate or up f, and of its output c.
template <int F>
__device__ __forceinline__ int2 sums_of(int f, bool up, bool pairs) {
  if (!by_column(F)) {
    const int row = pairs ? 2 * (f & 7) + (up ? 1 : 0) : (f & 7) + (up ? 8 : 0);
    return make_int2(f >> 3, (row & 8) + g_of(row & 7));
  }
  if (pairs) return make_int2(f & 3, (f >> 2) + (up ? 8 : 0));
  return make_int2((f & 7) >> 1, (f >> 3) + (up ? 4 : 0) + (f & 1 ? 8 : 0));
}
template <int F>
__device__ __forceinline__ int2 sums_of(int c) {
  return by_column(F) ? make_int2((c & 7) >> 1, (c >> 3) + (c & 1 ? 8 : 0)) : make_int2(c >> 4, (c & 8) + g_of(c & 7));
}
// A warp's sums to its place.
template <int F, int NT>
__device__ __forceinline__ void store_sums(float* red, const float (&acc)[FewShape<F>::kTiles][NT][4]) {
  float* const to = red + (threadIdx.x >> 5) * RedShape<F, NT>::kWarpFloats + (threadIdx.x & 31);
#pragma unroll
  for (int i = 0; i < FewShape<F>::kTiles; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) to[i * RedShape<F, NT>::kTile + (n * 4 + c) * 32] = acc[i][n][c];
}
// Shared memory: the rings, barriers, zeros, flags, the table, scales in the rings, sums, the panel.
template <int F> struct FewSmem {
  using S = FewShape<F>;
  static constexpr int kBars = S::kWarps * S::kRing, kZeros = kBars + 256, kFlags = kZeros + 64, kTable = kFlags + 64;
  static constexpr int kScales = kTable + kTableBytes, kRest = (kScales + S::kWarps * S::kRingScales + 127) / 128 * 128;
  static_assert(S::kWarps * S::kDepth * 8 <= 256, "barriers");
};
template <int F, int NT> struct UpShape {
  static constexpr int kSums = RedShape<F, NT>::kBytes;
  static constexpr int kFixed = FewSmem<F>::kRest + kSums;
};
template <int F> struct DownShape {
  static constexpr int kFixed = FewSmem<F>::kRest;
};

// ---- the first kernel where weights are stored by column ---------------------------------------
// h[row] = act(W13 x + b13).  The features of all active experts, in pieces of eight (a tile's rows: eight gates and their
// eight ups), are dealt out evenly to the blocks.  Within a block all warps work side by side, so that rows of k are read in
// long runs; where fewer pieces are left than warps times tiles several have the same ones, take their steps in turn and add
// their sums up in shared memory.
template <int F, int NT>
__global__ void __launch_bounds__(FewShape<F>::kThreads, 1) few_up_columns_kernel(FewParams p, FewLaunch launch, const __grid_constant__ CUtensorMap map) {
  using S = FewShape<F>;
  using M = FewSmem<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTiles = S::kTiles, kRows = S::kRows;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + M::kTable);
  uint8_t* const zeros = smem + M::kZeros;                                // a token's values where there is no token
  int* const gave_up = reinterpret_cast<int*>(smem + M::kFlags);
  float* const red = reinterpret_cast<float*>(smem + M::kRest);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  FewRing ring = make_ring<F>(smem, smem + M::kScales, reinterpret_cast<uint64_t*>(smem + M::kBars), gave_up, launch.status);
  uint8_t* const panel = smem + UpShape<F, NT>::kFixed;
  if (tid == 0) {
    *gave_up = 0;
    ptx::prefetch_tensormap(&map);
  }
  pdl_wait();
  pdl_trigger();
  const FewMatrix& m = p.w13;
  const FewLayout layout(m, F, launch.f16);
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
      for (int i = tid - 32; i < kFewMaxColumns; i += kThreads - 32) launch.arrived[i] = 0;
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
      FewRows fetch;
      auto copy_next = [&](int slot) {
        while (next.at < to && (s >= steps || !found)) {
          if (found || next.tiles <= 0) {     // (without tiles for this group: on to the next ones)
            place_after(next);
            s = next.member;
            found = false;
            if (next.at >= to || next.tiles <= 0) continue;
          }
          found = true;
          fetch.e = table.expert[next.a];
          fetch.row = (next.u + next.skip) * 8;
        }
        if (next.at < to) {
          if (lane == 0) {
            const uint32_t to_slot = ring.slots + slot * S::kSlotBytes, bar = ring.bars + slot * 8;
            ptx::fence_proxy_async();      // (the warp has read what was there)
            ptx::mbar_expect_tx_s(bar, S::kSlotBytes);
            if (pairs) {
              ptx::tma_load_3d_hint_s(to_slot, &map, bar, 2 * fetch.row, s * S::kK, fetch.e, ring.once);
            } else {
              ptx::tma_load_3d_hint_s(to_slot, &map, bar, fetch.row, s * S::kK, fetch.e, ring.once);
              ptx::tma_load_3d_hint_s(to_slot + S::kSlotBytes / 2, &map, bar, p.inter + fetch.row, s * S::kK, fetch.e, ring.once);
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
        for (int cs = at.member; cs < steps; cs += group) take_step<F, NT, 1>(acc, ring, tiles, row_order(), !pairs, layout, x, cs, copy_next);
        // The tile's sums: a lane has a feature, the members take the tokens in turn.
        store_sums<F, NT>(red, acc);
        // (a barrier for each group of each size)
        const int barrier = (kWarps >> at.shift) + (warp >> at.shift);
        if (group > 1) group_sync(barrier, group * 32);
        else __syncwarp();
        const int i = lane >> 3, f = (at.u + at.skip + i) * 8 + (lane & 7);
        const int2 at_gate = sums_of<F>(lane, false, pairs), at_up = sums_of<F>(lane, true, pairs);
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

// ---- the first kernel where weights are stored by output feature ------------------------------
// Columns of a partial sum's entry: 36 floats, so that a store's 32 lanes (eight rows of four columns) hit 32 banks.
constexpr int kEntryColumn = 36;
template <int F, int NT> struct UpRowsShape {
  static constexpr int kSums = NT == 1 ? 24 * 1024 : 36 * 1024;
  static constexpr int kFixed = FewSmem<F>::kRest + kSums;
  static_assert(kSums >= (FewShape<F>::kWarps + 1) * kEntryColumn * 4 * 8 * NT, "a set with all its tokens");
};

// A block's features of one pass: pieces of eight (a tile's rows: eight gates and their eight ups), up to two of one expert to a
// set, which a warp takes at once.
struct FewPieces {
  int per_expert, from, to;     // pieces of an expert; first and last of the pass
  int a0, u0, sets0, per;       // where the first one is; sets of the first expert and of every other one
  __device__ __forceinline__ FewPieces(int per_expert, int from, int to) : per_expert(per_expert), from(from), to(to) {
    a0 = from / per_expert;
    u0 = from - a0 * per_expert;
    sets0 = (min(per_expert - u0, to - from) + 1) >> 1;
    per = (per_expert + 1) >> 1;
  }
  __device__ __forceinline__ int sets() const {
    const int rest = to - from - (per_expert - u0);     // behind the first expert
    if (rest <= 0) return sets0;
    const int experts = rest / per_expert;
    return sets0 + experts * per + ((rest - experts * per_expert + 1) >> 1);
  }
  // Set j: its expert (of the active ones), its first piece there, and how many it has.
  __device__ __forceinline__ void find(int j, int& a, int& u, int& tiles) const {
    a = a0;
    u = u0 + 2 * j;
    int end = per_expert;
    if (j >= sets0) {
      const int i = (j - sets0) / per;
      a = a0 + 1 + i;
      u = 2 * (j - sets0 - i * per);
    }
    end = min(end, to - (from - u0) - (a - a0) * per_expert);
    tiles = min(2, end - u);
  }
};

// h[row] = act(W13 x + b13).  The pieces of all active experts are dealt out evenly to the blocks.  A block's sets times the
// steps of a row are one list, of which each warp takes a stretch; what it adds up of a set goes into shared memory, and
// at the end of the pass all that there is of a set is added up in the warps' order: one barrier a pass instead of one a set (which cost
// 4 to 10 us of the kernel).
template <int F, int NT>
__global__ void __launch_bounds__(FewShape<F>::kThreads, 1) few_up_rows_kernel(FewParams p, FewLaunch launch, const __grid_constant__ CUtensorMap map,
                                                                               const __grid_constant__ CUtensorMap piece_map) {
  using S = FewShape<F>;
  using M = FewSmem<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTiles = S::kTiles;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + M::kTable);
  uint8_t* const zeros = smem + M::kZeros;                                // a token's values where there is no token
  int* const gave_up = reinterpret_cast<int*>(smem + M::kFlags);
  float* const sums = reinterpret_cast<float*>(smem + M::kRest);
  uint8_t* const panel = smem + UpRowsShape<F, NT>::kFixed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  FewRing ring = make_ring<F>(smem, smem + M::kScales, reinterpret_cast<uint64_t*>(smem + M::kBars), gave_up, launch.status);
  if (tid == 0) {
    *gave_up = 0;
    ptx::prefetch_tensormap(&map);
    ptx::prefetch_tensormap(&piece_map);
  }
  pdl_wait();
  pdl_trigger();
  const FewMatrix& m = p.w13;
  const FewLayout layout(m, F, launch.f16);
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
      for (int i = tid - 32; i < kFewMaxColumns; i += kThreads - 32) launch.arrived[i] = 0;
    if (whole) fill_tokens<F>(panel, scales_after(panel, p.tokens), p.x, p.hidden, (1u << p.tokens) - 1u, k8, launch.f16, warp - 1, kWarps - 1);
  }
  __syncthreads();
  const uint32_t all = (uint32_t)(table.active * per_expert);     // (times the blocks below 2^32: takes_mma)
  const int begin = (int)(all * blockIdx.x / gridDim.x), end = (int)(all * (blockIdx.x + 1) / gridDim.x);
  const bool pairs = p.act == B200MOE_ACT_SWIGLUOAI;
  const FewOrder order = pairs ? row_order() : halves_order();

#pragma unroll 1
  for (int from = begin; from < end;) {
    // As many experts as have their tokens in the panel at once and their sums in shared memory; one with more tokens than
    // the panel holds goes through its features again with the rest of them.
    int to = from, deep = 0;       // deep: the most tokens that an expert has
    uint32_t tokens = 0;
    for (int a = from / per_expert; to < end; ++a) {
      const uint32_t with = tokens | table.tokens[a];
      const int n = max(deep, min(__popc(table.tokens[a]), most));
      const int room = UpRowsShape<F, NT>::kSums / (kEntryColumn * 4 * n) - kWarps;             // sets
      if (tokens && (__popc(with) > most || room <= (to - from) / 2 + a - from / per_expert)) break;
      tokens = with;
      deep = n;
      // (an expert before this one may have left a set with one piece, and this one may)
      to = min(min(end, (a + 1) * per_expert), from + 2 * (room - (a - from / per_expert)));
      if (to < min(end, (a + 1) * per_expert)) break;
    }
    if (whole) tokens = (1u << p.tokens) - 1u;
    const FewPieces pieces(per_expert, from, to);
    const int total = pieces.sets() * steps;
    const int workers = min(kWarps, total);
    const int pos0 = total * min(warp, workers) / workers, pos1 = total * min(warp + 1, workers) / workers;
    const int j0 = pos0 / steps, s0 = pos0 - j0 * steps;

#pragma unroll 1
    for (uint32_t rest = tokens; rest;) {
      uint32_t now = rest;
      while (__popc(now) > most) now &= ~(1u << (31 - __clz(now)));
      rest &= ~now;

      // The ring begins to fill: the set and step that are fetched next, and how many after them.
      FewRows fetch;
      int fetch_j = j0, fetch_s = s0, left = pos1 - pos0;
      bool found = false;
      auto copy_next = [&](int slot) {
        if (left > 0) {
          if (fetch_s == steps) { fetch_s = 0; ++fetch_j; found = false; }
          if (!found) {
            int a;
            pieces.find(fetch_j, a, fetch.row, fetch.tiles);
            fetch.row *= 8;
            fetch.e = table.expert[a];
            // gates in the first half of the places, ups in the second; pairs as they are
            const int up = lane >= S::kRows / 2, fs = lane % (S::kRows / 2);
            fetch.there = pairs ? lane < 16 * fetch.tiles : fs < 8 * fetch.tiles;
            const int n = pairs ? 2 * fetch.row + lane : fetch.row + fs + up * p.inter;
            fetch.s = scales_of<F>(m, layout, fetch.e, fetch.there ? n : 0);
            found = true;
          }
          if (lane == 0) {
            const uint32_t at = ring.slots + slot * S::kSlotBytes, bar = ring.bars + slot * 8;
            const CUtensorMap* from_map = fetch.tiles == kTiles ? &map : &piece_map;
            ptx::fence_proxy_async();      // (the warp has read what was there)
            ptx::mbar_expect_tx_s(bar, fetch.tiles * 2048);
            ptx::tma_load_3d_hint_s(at, from_map, bar, fetch_s * 128, pairs ? 2 * fetch.row : fetch.row, fetch.e, ring.once);
            if (!pairs) ptx::tma_load_3d_hint_s(at + S::kSlotBytes / 2, from_map, bar, fetch_s * 128, p.inter + fetch.row, fetch.e, ring.once);
          }
          copy_scales<F>(ring.scales + slot * S::kSlotScales, fetch, layout, fetch_s);
          ++fetch_s;
          --left;
        }
        copies_end();
      };
#pragma unroll 1
      for (int i = 0; i < S::kDepth; ++i) copy_next((ring.slot + i) % S::kDepth);
      const int rows = __popc(now);
      if (!whole) {
        fill_tokens<F>(panel, scales_after(panel, rows), p.x, p.hidden, now, k8, launch.f16, warp, kWarps);
        __syncthreads();
      }

#pragma unroll 1
      for (int pos = pos0, j = j0, s = s0; pos < pos1; ++j, s = 0) {
        int a, u, tiles;
        pieces.find(j, a, u, tiles);
        const uint32_t mine = table.tokens[a] & now;
        FewTokens x[NT];
        find_tokens<NT>(x, mine, now, smem_at(panel), smem_at(scales_after(panel, rows)), smem_at(zeros), rows);
        float acc[kTiles][NT][4] = {};
        const int stop = min(steps, s + pos1 - pos);
        pos += stop - s;
#pragma unroll 1
        for (; s < stop; ++s) take_step<F, NT, 1>(acc, ring, tiles, order, !pairs, layout, x, s, copy_next);
        // sets and warps begin a new entry each
        float* const entry = sums + (j + warp) * (kEntryColumn * deep);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int token = 8 * n + 2 * (lane & 3) + c;
            if (!((mine >> token) & 1)) continue;
            float* const to_entry = entry + rank_below(mine, token) * kEntryColumn + (lane >> 2);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
              to_entry[i * 16] = acc[i][n][c];
              to_entry[i * 16 + 8] = acc[i][n][c + 2];
            }
          }
      }
      copies_wait<0>();
      __syncthreads();   // the sums are complete, and the panel is free again
      // A warp has a set, a lane one of its 16 features, for one token of two.
#pragma unroll 1
      for (int j = warp; j * steps < total; j += kWarps) {
        int a, u, tiles;
        pieces.find(j, a, u, tiles);
        const int f = 8 * u + (lane & 15), first = table.first_row[a];
        const uint32_t have = table.tokens[a], mine = have & now;
        // the warps that had the set's first and last step
        const int w0 = (workers * (j * steps + 1) - 1) / total, w1 = (workers * (j + 1) * steps - 1) / total;
        if ((lane & 15) >= 8 * tiles) continue;
        float bias_gate = 0.f, bias_up = 0.f;
        if (m.bias) {
          const int64_t at = (int64_t)table.expert[a] * m.n;
          bias_gate = load16(m.bias, at + (pairs ? 2 * f : f), launch.f16);
          bias_up = load16(m.bias, at + (pairs ? 2 * f + 1 : p.inter + f), launch.f16);
        }
        const int2 at_gate = sums_of<F>(lane & 15, false, pairs), at_up = sums_of<F>(lane & 15, true, pairs);
        const float* const gates = sums + (at_gate.x * 16 + at_gate.y), * const ups = sums + (at_up.x * 16 + at_up.y);
        uint32_t later = mine;
        if (lane >= 16) later &= later - 1;
        for (int rank = lane >> 4; later; rank += 2) {
          const int token = __ffs(later) - 1;
          float gate = bias_gate, up = bias_up;
          for (int w = w0; w <= w1; ++w) {
            const int at = ((j + w) * deep + rank) * kEntryColumn;
            gate += gates[at];
            up += ups[at];
          }
          p.h[(int64_t)(first + rank_below(have, token)) * p.inter + f] = gated_once(p.act, p.alpha, p.limit, p.clamp, gate, up);
          later &= later - 1;
          later &= later - 1;
        }
      }
      if (rest || to < end) __syncthreads();   // the sums' place is free again
    }
    from = to;
  }
}

// Routing weights times biases of a token's experts, for output n.
__device__ __noinline__ float weighted_bias(const FewTable& table, const FewMatrix& m, int topk, bool f16, int token, int n) {
  float v = 0.f;
  for (int k0 = 0; k0 < topk; k0 += 4) {
    float w[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int slot = token * topk + k0 + k, a = k0 + k < topk ? table.slot_expert[slot] : -1;
      w[k] = a >= 0 ? table.slot_weight[slot] : 0.f;
      b[k] = a >= 0 ? load16(m.bias, (int64_t)table.expert[a] * m.n + n, f16) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w[k] != 0.f) v = fmaf(w[k], b[k], v);
  }
  return v;
}

// out = sum over experts of weight * (W2 h + b2).  A block has some rows of W2 and a share of the steps over all active
// experts: of rows up to 64, so that few blocks need the same values of h, and of steps what makes as many blocks as there are
// SMs.  It goes through its steps with as many of h's values at a time as its panel holds, each warp with a stretch of them.
// Of the blocks with the same rows the last one to be done adds the partial sums up, in their order.  By column a block has
// up to four times 64, side by side by warps that share their steps' values of h.
template <int F, int NT>
__global__ void __launch_bounds__(FewShape<F>::kThreads, 1) few_down_kernel(FewParams p, FewLaunch launch, const __grid_constant__ CUtensorMap map) {
  using S = FewShape<F>;
  using M = FewSmem<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kTiles = S::kTiles, kRows = S::kRows;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + M::kTable);
  uint8_t* const zeros = smem + M::kZeros;
  int* const gave_up = reinterpret_cast<int*>(smem + M::kFlags);
  int& last_one = *reinterpret_cast<int*>(smem + M::kFlags + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;
  FewRing ring = make_ring<F>(smem, smem + M::kScales, reinterpret_cast<uint64_t*>(smem + M::kBars), gave_up, launch.status);
  uint8_t* const panel = smem + DownShape<F>::kFixed;
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
  const FewLayout layout(m, F, launch.f16);
  const int steps = (p.inter + S::kK - 1) / S::kK;
  const int columns = gridDim.x / launch.splits, column = blockIdx.x % columns, split = blockIdx.x / columns;
  // (by column: whole 64 of them, one block's after the other's)
  const int side = launch.side, members = kWarps / side, member = warp / side, mine_side = warp % side;
  const int warp_rows = launch.box, block_rows = side * warp_rows;
  const int row_begin = by_column(F) ? column * block_rows : (int)((uint32_t)p.hidden * column / columns);
  const int row_end = by_column(F) ? p.hidden : (int)((uint32_t)p.hidden * (column + 1) / columns);
  const uint32_t total = (uint32_t)(table.active * steps);
  const int step_begin = (int)(total * split / launch.splits), step_end = (int)(total * (split + 1) / launch.splits);
  const int room = launch.panel_bytes / S::kPanelBytes(S::kTerms);        // rows times steps that the panel holds
  float* const scales = reinterpret_cast<float*>(panel + room * (S::kTerms * S::kK * 2));
  bool waited = false;

  // How far a panel reaches that begins with step s0 of expert a0: whole experts, then as many steps of the next one as
  // there is room for (at least one).
  auto panel_end = [&](int a0, int s0, int& a1, int& s1) {
    const int ae = step_end / steps, se = step_end - ae * steps;      // all that is left, if it fits
    const int need = ae == a0 ? (table.first_row[a0 + 1] - table.first_row[a0]) * (se - s0)
                              : (table.first_row[a0 + 1] - table.first_row[a0]) * (steps - s0) + (table.first_row[ae] - table.first_row[a0 + 1]) * steps +
                                    (se > 0 ? (table.first_row[ae + 1] - table.first_row[ae]) * se : 0);
    a1 = ae;
    s1 = se;
    if (need <= room) return;
    int free = room;
    a1 = a0;
    s1 = s0;
    while (a1 * steps + s1 < step_end) {
      const int n = table.first_row[a1 + 1] - table.first_row[a1], fit = min(min(steps - s1, step_end - a1 * steps - s1), free / n);
      if (fit == 0) break;
      free -= fit * n;
      s1 += fit;
      if (s1 < steps) break;
      s1 = 0;
      ++a1;
    }
  };
  auto finish = [&](float v, int token, int n) {
    const int64_t to = (int64_t)token * p.hidden + n;
    if (launch.f16) reinterpret_cast<__half*>(p.out)[to] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(v);
  };
  for (int block_r0 = row_begin; block_r0 < row_end || !waited; block_r0 += by_column(F) ? columns * block_rows : block_rows) {
    const int r0 = block_r0 + mine_side * warp_rows, rows_here = max(0, min(warp_rows, row_end - r0)), tiles = (rows_here + 15) / 16;
    FewRows fetch;
    fetch.there = lane < rows_here;
    // The step that is fetched next, how many are left of this warp's stretch, and where the panel after that begins.
    int fetch_a = 0, fetch_s = 0, left = 0, panel_a = step_begin / steps, panel_s = step_begin - panel_a * steps;
    bool found = false;
    auto copy_next = [&](int slot) {
      while (left == 0 && panel_a * steps + panel_s < step_end) {
        int a1, s1;
        panel_end(panel_a, panel_s, a1, s1);
        const int from = panel_a * steps + panel_s, all = a1 * steps + s1 - from, mine = all * member / members;
        left = all * (member + 1) / members - mine;
        fetch_a = (from + mine) / steps;
        fetch_s = from + mine - fetch_a * steps;
        panel_a = a1;
        panel_s = s1;
        found = false;
      }
      if (left > 0 && rows_here > 0) {
        if (fetch_s == steps) { fetch_s = 0; ++fetch_a; found = false; }
        if (!found) {
          fetch.e = table.expert[fetch_a];
          if (!by_column(F)) fetch.s = scales_of<F>(m, layout, fetch.e, fetch.there ? r0 + lane : r0);
          found = true;
        }
        if (lane == 0) {
          const uint32_t bar = ring.bars + slot * 8;
          ptx::fence_proxy_async();        // (the warp has read what was there)
          ptx::mbar_expect_tx_s(bar, warp_rows * (by_column(F) ? 64 : 128));
          ptx::tma_load_3d_hint_s(ring.slots + slot * S::kSlotBytes, &map, bar, by_column(F) ? r0 : fetch_s * 128, by_column(F) ? fetch_s * S::kK : r0, fetch.e, ring.once);
        }
        if (!by_column(F)) copy_scales<F>(ring.scales + slot * S::kSlotScales, fetch, layout, fetch_s);
        ++fetch_s;
        --left;
      }
      copies_end();
    };
#pragma unroll 1
    for (int i = 0; i < S::kDepth; ++i) copy_next((ring.slot + i) % S::kDepth);
    // Biases while the ring fills, by the blocks with the first share (by column: when they are needed).
    constexpr int kMine = (B200MOE_FEW_TOKENS * kBlockRows + kThreads - 1) / kThreads;
    const int block_rows_here = min(block_rows, row_end - block_r0), my_row = tid % kBlockRows, my_token = tid / kBlockRows;
    float bias[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int token = my_token + i * (kThreads / kBlockRows);
      bias[i] = !by_column(F) && m.bias && split == 0 && token < p.tokens && my_row < block_rows_here
                    ? weighted_bias(table, m, p.topk, launch.f16, token, block_r0 + my_row) : 0.f;
    }
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
    }
    float out[kTiles][NT][4] = {};
    for (int a0 = step_begin / steps, s0 = step_begin - a0 * steps; a0 * steps + s0 < step_end;) {
      int a1, s1;
      panel_end(a0, s0, a1, s1);
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
        const int stop = rows_here > 0 ? from + all * (member + 1) / members : 0;
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
          for (; pos < end; ++pos) take_step<F, NT, S::kTerms>(acc, ring, tiles, row_order(), false, layout, x, pos - a * steps, copy_next);
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
    copies_wait<0>();
    __syncthreads();
    auto put = [&](float v, int token, int row) {
      const int64_t to = (int64_t)token * p.hidden + row;
      if (launch.splits == 1) finish(v, token, row);
      else launch.part[(int64_t)split * p.tokens * p.hidden + to] = v;
    };
    // consecutive threads, consecutive features of a token
    if constexpr (by_column(F)) {
      for (int j = tid; j < block_rows * p.tokens; j += kThreads) {
        const int row = j % block_rows, token = j / block_rows;
        if (block_r0 + row >= row_end) continue;
        const int2 at = sums_of<F>(row % kRows);
        float v = m.bias && split == 0 ? weighted_bias(table, m, p.topk, launch.f16, token, block_r0 + row) : 0.f;
        for (int w = row / kRows; w < kWarps; w += side) v += red[w * RedShape<F, NT>::kWarpFloats + RedShape<F, NT>::at(at.x, at.y, token)];
        put(v, token, block_r0 + row);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int token = my_token + i * (kThreads / kBlockRows);
        if (my_row >= block_rows_here || token >= p.tokens) continue;
        const int which = my_row >= warp_rows ? 1 : 0;
        const int2 at = sums_of<F>(my_row - which * warp_rows);
        float v = bias[i];
#pragma unroll
        for (int w = 0; w < kWarps / 2; ++w) v += red[(2 * w + which) * RedShape<F, NT>::kWarpFloats + RedShape<F, NT>::at(at.x, at.y, token)];
        put(v, token, block_r0 + my_row);
      }
    }
    __syncthreads();
  }
  if (launch.splits == 1) return;
  // (the barrier puts the block's partial sums ahead of the fence, and what the others have published ahead of the reads)
  if (tid == 0) {
    __threadfence();
    last_one = atomicAdd(&launch.arrived[column], 1u) == (uint32_t)launch.splits - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last_one) return;
  const int width = min(row_end - row_begin, by_column(F) ? block_rows : row_end);
  for (int j = tid; j < width * p.tokens; j += kThreads) {
    const int row = row_begin + j % width, token = j / width;
    float v = 0.f;
    const float* from = launch.part + (int64_t)token * p.hidden + row;
    const int64_t next = (int64_t)p.tokens * p.hidden;
#pragma unroll 4
    for (int i = 0; i < launch.splits; ++i) v += __ldcg(from + i * next);
    finish(v, token, row);
  }
}

}  // namespace
}  // namespace b200moe
