// The layer for a few tokens where weights are stored by output feature ([E,N,K]: block-scaled fp8, MXFP4, int4), on the
// tensor cores.
//
//   D[features, tokens] += W[16 features, 16 k] x^T[16 k, 8 tokens]     (mma.sync, fp32 accumulation)
//
// A few tokens leave the layer to the bandwidth of its weights: every byte of an active expert passes once, from L2
// through a warp's own ring in shared memory (cp.async) into the registers that the matrix instruction reads, with one
// conversion to float16 on the way, which holds every code of the three formats exactly.  The sum over k does not mind its order,
// so a lane's 16 bytes of a row go into the instruction as they come and the tokens are laid out to match.  Scales of weights
// multiply sums of their group in fp32.  Tokens and activations are float16 with a power of two per row, which keeps a
// bfloat16 as it is and rounds h to 11 bits.
//
// tcgen05 would have to get its weights converted in shared or tensor memory, a second pass for every byte, and its tile
// of 128 features leaves most SMs without work at one token.
#pragma once

#include <cuda_fp4.h>

#include "few_tokens.cuh"

namespace b200moe {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr int kMaxSlots = kFewMaxTopk * B200MOE_FEW_TOKENS;   // routed slots of a call

enum FewFormat { kFewFp8, kFewFp4, kFewInt4Fine, kFewInt4 };   // Fine: groups of 32 or 64

template <int F> struct FewShape {
  static constexpr int kChunks = F == kFewFp8 ? 2 : 1;          // 16-byte pieces of a row per lane and step of 128 k
  static constexpr int kStepBytes = F == kFewFp8 ? 128 : 64;    // of a row
  static constexpr int kScaleWords = F == kFewFp8 || F == kFewInt4 ? 1 : F == kFewFp4 ? 2 : 3;   // of a row and step
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
  uint16_t row_token[kMaxSlots];
  float weight[kMaxSlots];         // of a row: the sum over the slots that name its expert
};

__device__ __forceinline__ int rank_below(uint32_t mask, int bit) { return __popc(mask & ((1u << bit) - 1u)); }

template <bool kWeights>
__device__ __forceinline__ void build_table(FewTable& t, const FewParams& p) {
  const int slots = p.tokens * p.topk, tid = threadIdx.x, lane = tid & 31;
  if (tid < 32) t.bits[tid] = 0;
  for (int i = tid; i < slots; i += kThreads) t.tokens[i] = 0;
  __syncthreads();
  for (int i = tid; i < slots; i += kThreads) {
    const int e = local_expert(p, i);
    t.slot_expert[i] = e;
    if (e >= 0) atomicOr(&t.bits[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  if (tid < 32) {
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
  __syncthreads();
  for (int i = tid; i < slots; i += kThreads) {
    const int e = t.slot_expert[i];
    if (e < 0) continue;
    const int a = t.before[e >> 5] + rank_below(t.bits[e >> 5], e & 31);
    t.slot_expert[i] = a;
    t.expert[a] = e;
    atomicOr(&t.tokens[a], 1u << (i / p.topk));
  }
  __syncthreads();
  if (tid < 32) {
    int base = 0;
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
  }
  __syncthreads();
  if (kWeights) {
    for (int i = tid; i < slots; i += kThreads) {
      const int a = t.slot_expert[i], tok = i / p.topk, k0 = tok * p.topk;
      if (a < 0) continue;
      bool again = false;
      for (int j = k0; j < i; ++j) again |= t.slot_expert[j] == a;
      if (again) continue;
      float w = 0.f;
      for (int j = i; j < k0 + p.topk; ++j)
        if (t.slot_expert[j] == a) w += p.weights[j];
      const int row = t.first_row[a] + rank_below(t.tokens[a], tok);
      t.weight[row] = w;
      t.row_expert[row] = (uint16_t)a;
      t.row_token[row] = (uint16_t)tok;
    }
    __syncthreads();
  }
}

// ---- loads ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// `bytes` of the 16 or 4 come from memory, the rest are zeros.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

// ---- conversions and products ------------------------------------------------------------
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)v, __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
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
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- tokens and activations as float16 -------------------------------------------------
// A panel holds rows of values in the order in which the lanes want them: per step of 128 k four blocks, a block
// [row][4 lanes][8 values].  Where k sits: fp8 lanes hold 16 bytes of a row, 16 values; 4-bit formats hand a group of 32
// values out to the four lanes, eight each.
template <int F>
__device__ __forceinline__ uint32_t panel_at(int k8, int row, int rows) {   // k8: k / 8
  const int s = k8 >> 4;
  const int block = F == kFewFp8 ? ((k8 >> 2) & 2) | (k8 & 1) : (k8 >> 2) & 3;
  const int t = F == kFewFp8 ? (k8 >> 1) & 3 : k8 & 3;
  return (uint32_t)((((s * 4 + block) * rows + row) * 4 + t) * 16);
}

enum FewSource { kFromBf16, kFromF16, kFromF32 };
__device__ __forceinline__ void load8(float (&v)[8], const void* row, int source, int k8) {
  if (source == kFromF32) {
    const float4 a = reinterpret_cast<const float4*>(row)[2 * k8], b = reinterpret_cast<const float4*>(row)[2 * k8 + 1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const vec16 w = reinterpret_cast<const vec16*>(row)[k8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (source == kFromBf16) {
      v[2 * i] = __uint_as_float(w.w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w.w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w.w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// The power of two by which a row is multiplied on its way to float16, its largest magnitude then between 2^14 and 2^15, and
// its inverse.  Magnitudes below 2^-100 are taken for that; a row that is not finite stays as it is.
__device__ __forceinline__ float row_scale(float top, float& inverse) {
  int e = (int)(__float_as_uint(top) >> 23);   // (no sign)
  if (e == 255) e = 127 + 14;
  e = max(e, 127 - 100);
  inverse = __uint_as_float((uint32_t)(e - 14) << 23);
  return __uint_as_float((uint32_t)(254 - (e - 14)) << 23);
}

// One row's part of a panel: values [k8_0, k8_1) * 8 of a source row of `k` values (zeros beyond it), by `parts` warps of
// which this is `part`.
template <int F>
__device__ __forceinline__ void convert_row(uint8_t* panel, int row, int rows, const void* src, int source, int k, int k8_0, int k8_1,
                                            float scale, int part, int parts) {
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int j = k8_0 + part * 32 + lane; j < k8_1; j += parts * 32) {
    float v[8] = {};
    if (8 * j < k) load8(v, src, source, j);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // int4 pairs are four apart
      const float x = F == kFewInt4 || F == kFewInt4Fine ? v[i] : v[2 * i], y = F == kFewInt4 || F == kFewInt4Fine ? v[i + 4] : v[2 * i + 1];
      const __half2 h = __floats2half2_rn(x * scale, y * scale);
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(panel + panel_at<F>(j - k8_0, row, rows)) = make_uint4(o[0], o[1], o[2], o[3]);
  }
}
__device__ __forceinline__ float row_top(const void* src, int source, int k, int k8_0, int k8_1, int part, int parts) {
  const int lane = threadIdx.x & 31;
  float top = 0.f;
#pragma unroll 4
  for (int j = k8_0 + part * 32 + lane; j < k8_1; j += parts * 32) {
    if (8 * j >= k) break;
    float v[8];
    load8(v, src, source, j);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
  return top;
}
// Warps of a row where a panel has `rows` of them.
__device__ __forceinline__ int warps_per_row(int rows) { return rows == 1 ? 8 : rows == 2 ? 4 : rows <= 4 ? 2 : 1; }

// ---- weights: a warp's ring ------------------------------------------------------------
// A step is 128 k of MT tiles of 16 rows.  fp8: a lane finds its own bytes again; 4 bits: a lane fetches 16 bytes of a row
// (a group of 32) and reads a word of each of the row's four groups, whose places are swapped so that the eight rows of a
// read fall on different banks.
template <int F, int MT> struct FewRing {
  static constexpr int kData = MT * 16 * FewShape<F>::kStepBytes;
  static constexpr int kScales = MT * 16 * FewShape<F>::kScaleWords * 4;
  static constexpr int kSlot = kData + kScales;
};

// Where the rows of a tile lie, for one matrix of one expert.
struct FewRows {
  const uint8_t* w;       // the expert's weights and scales
  const uint8_t* s;
  int64_t row_bytes, scale_bytes;   // of a row (fp8: of a row of blocks)
};

template <int F>
__device__ __forceinline__ FewRows rows_of(const FewMatrix& m, int e) {
  FewRows r;
  const int64_t n = m.n, k = m.k;
  r.row_bytes = F == kFewFp8 ? k : k / 2;
  r.scale_bytes = F == kFewFp8 ? k / 128 * 4 : F == kFewFp4 ? k / 32 : k / m.group * 2;
  r.w = reinterpret_cast<const uint8_t*>(m.w) + e * n * r.row_bytes;
  r.s = reinterpret_cast<const uint8_t*>(m.scale) + e * (F == kFewFp8 ? n / 128 : n) * r.scale_bytes;
  return r;
}
// First byte of the scales of step s within a row.
template <int F>
__device__ __forceinline__ int scale_offset(const FewMatrix& m, int s) {
  return F == kFewFp8 ? 4 * s : F == kFewFp4 ? 4 * s : 128 * s / m.group * 2;
}

// Copies step s of the tiles into a slot.  row(i) gives row i of the 16 * MT, or -1 where there is none.
template <int F, int MT, typename Row>
__device__ __forceinline__ void copy_step(uint32_t slot, const FewRows& r, const FewMatrix& m, int s, Row row) {
  using S = FewShape<F>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int n = row(i * 8 + g);
#pragma unroll
    for (int c = 0; c < S::kChunks; ++c) {
      const int at = s * S::kStepBytes + (c * 4 + t) * 16;
      const bool there = n >= 0 && at < r.row_bytes;
      const uint32_t to = F == kFewFp8 ? slot + (i * 2 + c) * 512 + lane * 16 : slot + i * 512 + g * 64 + ((t ^ (g >> 1)) << 4);
      copy16(to, there ? r.w + n * r.row_bytes + at : r.w, there ? 16 : 0);
    }
  }
  const uint32_t sc = slot + FewRing<F, MT>::kData;
  const int off = scale_offset<F>(m, s);
#pragma unroll
  for (int i = 0; i < (MT + 1) / 2; ++i) {
    const int local = i * 32 + lane;
    if (local < 16 * MT) {
      const int n = row(local);
      // words that hold the step's scales (they need not begin at one), as far as the row goes
      const int64_t first = n < 0 ? 0 : (F == kFewFp8 ? n / 128 : n) * r.scale_bytes;
      const int64_t begin = (first + off) & ~(int64_t)3;
#pragma unroll
      for (int w = 0; w < S::kScaleWords; ++w) {
        const int64_t left = n < 0 ? 0 : first + r.scale_bytes - (begin + 4 * w);
        copy4(sc + (local * S::kScaleWords + w) * 4, left > 0 ? r.s + begin + 4 * w : r.s, left >= 4 ? 4 : left > 0 ? (int)left : 0);
      }
    }
  }
}

// The step's scale of each group of 32 values (fp8, int4 with long groups: one for all) of local row i, which is row n.
template <int F, int MT>
__device__ __forceinline__ void step_scales(float (&o)[4], uint32_t slot, const FewRows& r, const FewMatrix& m, int s, int i, int n, bool f16) {
  const uint32_t at = slot + FewRing<F, MT>::kData + i * FewShape<F>::kScaleWords * 4;
  if (F == kFewFp8) { o[0] = __uint_as_float(lds4(at)); return; }
  const int shift = (int)((n < 0 ? 0 : n * r.scale_bytes + scale_offset<F>(m, s)) & 3) * 8;
  if (F == kFewFp4) {
    // 2^(byte - 127): the byte is the exponent (0 gives zero for 2^-127, 255 infinity for NaN)
    const uint32_t v = __funnelshift_r(lds4(at), lds4(at + 4), shift);
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = __uint_as_float(((v >> (8 * q)) & 255u) << 23);
    return;
  }
  auto value = [&](uint32_t h) { return f16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16); };
  if (F == kFewInt4) { o[0] = value((lds4(at) >> shift) & 0xffffu); return; }
  const uint32_t w0 = lds4(at), w1 = lds4(at + 4), w2 = lds4(at + 8);
  const uint32_t lo = __funnelshift_r(w0, w1, shift), hi = __funnelshift_r(w1, w2, shift);
  const bool fine = m.group == 32;
  o[0] = value(lo & 0xffffu);
  o[1] = fine ? value(lo >> 16) : o[0];
  o[2] = value(fine ? hi & 0xffffu : lo >> 16);
  o[3] = fine ? value(hi >> 16) : o[2];
}

// acc += W x of one step.  b[j]: where this lane finds its token's values in the panel's first block of the step (0: no such
// token); block: bytes from one block to the next.
template <int F, int MT, int NT, typename Row>
__device__ __forceinline__ void multiply_step(float (&acc)[MT][NT][4], uint32_t slot, const FewRows& r, const FewMatrix& m, int s, bool f16,
                                              const uint32_t (&b)[NT], uint32_t block, Row row) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if constexpr (F == kFewFp8) {
    float d[MT][NT][4] = {};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint4 x[2][NT];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) x[j][n] = b[n] ? lds16(b[n] + (2 * c + j) * block) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 lo = lds16(slot + (4 * i + c) * 512 + lane * 16), hi = lds16(slot + (4 * i + 2 + c) * 512 + lane * 16);
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = e4m3x2_to_h2(wl[w] & 0xffffu), a2 = e4m3x2_to_h2(wl[w] >> 16);
          const uint32_t a1 = e4m3x2_to_h2(wh[w] & 0xffffu), a3 = e4m3x2_to_h2(wh[w] >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n)
            mma(d[i][n], a0, a1, a2, a3, w & 1 ? x[w >> 1][n].z : x[w >> 1][n].x, w & 1 ? x[w >> 1][n].w : x[w >> 1][n].y);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float lo[4], hi[4];
      step_scales<F, MT>(lo, slot, r, m, s, 16 * i + g, 0, f16);
      step_scales<F, MT>(hi, slot, r, m, s, 16 * i + 8 + g, 0, f16);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[i][n][0] = fmaf(lo[0], d[i][n][0], acc[i][n][0]);
        acc[i][n][1] = fmaf(lo[0], d[i][n][1], acc[i][n][1]);
        acc[i][n][2] = fmaf(hi[0], d[i][n][2], acc[i][n][2]);
        acc[i][n][3] = fmaf(hi[0], d[i][n][3], acc[i][n][3]);
      }
    }
  } else {
    constexpr bool kOneScale = F == kFewInt4;
    uint4 x[4][NT];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int n = 0; n < NT; ++n) x[q][n] = b[n] ? lds16(b[n] + q * block) : make_uint4(0, 0, 0, 0);
    const uint32_t at = slot + g * 64 + t * 4;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      float lo[4], hi[4];
      step_scales<F, MT>(lo, slot, r, m, s, 16 * i + g, row(16 * i + g), f16);
      step_scales<F, MT>(hi, slot, r, m, s, 16 * i + 8 + g, row(16 * i + 8 + g), f16);
      float d[NT][4] = {};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t al[4], ah[4];
        const uint32_t wl = lds4(at + 2 * i * 512 + ((q ^ (g >> 1)) << 4)), wh = lds4(at + (2 * i + 1) * 512 + ((q ^ (g >> 1)) << 4));
        if constexpr (F == kFewFp4) { e2m1x8_to_h2(wl, al); e2m1x8_to_h2(wh, ah); }
        else { s4x8_to_h2(wl, al); s4x8_to_h2(wh, ah); }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma(d[n], al[0], ah[0], al[1], ah[1], x[q][n].x, x[q][n].y);
          mma(d[n], al[2], ah[2], al[3], ah[3], x[q][n].z, x[q][n].w);
          if (!kOneScale || q == 3) {
            const int k = kOneScale ? 0 : q;
            acc[i][n][0] = fmaf(lo[k], d[n][0], acc[i][n][0]);
            acc[i][n][1] = fmaf(lo[k], d[n][1], acc[i][n][1]);
            acc[i][n][2] = fmaf(hi[k], d[n][2], acc[i][n][2]);
            acc[i][n][3] = fmaf(hi[k], d[n][3], acc[i][n][3]);
            d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
          }
        }
      }
    }
  }
}

__device__ __forceinline__ float load16(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(reinterpret_cast<const __half*>(p)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// ---- the kernels -------------------------------------------------------------------------
struct FewLaunch {
  int panel_bytes;       // of shared memory for the panel
  bool f16;
};

template <int F, int MT, int NT> struct UpShape {
  static constexpr int kDepth = 3;
  static constexpr int kRed = kWarps * MT * NT * 4 * 32 * 4;
  static constexpr int kFixed = (sizeof(FewTable) + 127) / 128 * 128 + 2 * kRed + 512 + kWarps * kDepth * FewRing<F, MT>::kSlot;
};

// h[row] = act(W13 x + b13).  The features of all active experts, in pieces of eight (a tile's rows: eight gates and their
// eight ups), are dealt out evenly to the blocks; the warps of a block take the steps of its tiles in turn and add their sums up
// in shared memory.
template <int F, int MT, int NT>
__global__ void __launch_bounds__(kThreads, 1) few_up_kernel(FewParams p, FewLaunch l) {
  using S = UpShape<F, MT, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem);
  float* const red = reinterpret_cast<float*>(smem + (sizeof(FewTable) + 127) / 128 * 128);
  float* const inverse = red + 2 * S::kRed / 4;       // of the panel's rows' scales
  float* const tops = inverse + 64;                    // (per warp)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_at(red) + 2 * S::kRed + 512 + warp * S::kDepth * FewRing<F, MT>::kSlot;
  uint8_t* const panel = smem + S::kFixed;
  pdl_wait();
  pdl_trigger();
  build_table<false>(table, p);
  const FewMatrix& m = p.w13;
  const int steps = (p.hidden + 127) / 128, per_expert = p.inter / 8;
  const int64_t all = (int64_t)table.active * per_expert;
  const int begin = (int)(all * blockIdx.x / gridDim.x), end = (int)(all * (blockIdx.x + 1) / gridDim.x);
  const bool pairs = p.act == B200MOE_ACT_SWIGLUOAI;
  const int most = l.panel_bytes / (steps * 256);      // rows that the panel holds

  for (int from = begin; from < end;) {
    // as many experts as have their tokens in the panel at once; one with more tokens than that goes through its
    // features again with the rest of them
    const int a0 = from / per_expert;
    uint32_t tokens = table.tokens[a0];
    int to = min(end, (a0 + 1) * per_expert);
    if (__popc(tokens) <= most) {
      for (int a = a0 + 1; to < end && __popc(tokens | table.tokens[a]) <= most; ++a) {
        tokens |= table.tokens[a];
        to = min(end, (a + 1) * per_expert);
      }
    }
    for (uint32_t rest = tokens; rest;) {
      uint32_t now = rest;
      while (__popc(now) > most) now &= ~(1u << (31 - __clz(now)));
      rest &= ~now;
      const int rows = __popc(now);

      // the ring begins to fill
      int tile = from, left = 0, s = warp;     // of the step that is copied next: its tile, the tile's pieces
      FewRows where = {};
      auto locate = [&]() {
        const int e = table.expert[tile / per_expert];
        where = rows_of<F>(m, e);
        left = min(MT, min(per_expert - tile % per_expert, to - tile));
      };
      auto feature_row = [&](int first, int count, int i) {   // row i of a tile whose first piece is `first`
        const int piece = i >> 4, f = (first + piece) * 8 + (i & 7);
        return piece >= count ? -1 : pairs ? 2 * f + ((i >> 3) & 1) : f + ((i >> 3) & 1) * p.inter;
      };
      auto settle = [&]() {
        while (s >= steps && tile < to) {
          s -= steps;
          tile += left;
          if (tile < to) locate();
        }
      };
      auto copy_next = [&](int slot) {
        if (tile < to) {
          copy_step<F, MT>(ring + slot * FewRing<F, MT>::kSlot, where, m, s, [&](int i) { return feature_row(tile % per_expert, left, i); });
          s += kWarps;
          settle();
        }
        copies_end();
      };
      locate();
      settle();
#pragma unroll
      for (int i = 0; i < S::kDepth; ++i) copy_next(i);

      // the panel
      {
        const int parts = warps_per_row(rows), row = warp / parts, part = warp % parts;
        const int source = l.f16 ? kFromF16 : kFromBf16, k8 = steps * 16;
        for (int r0 = 0; r0 < rows; r0 += kWarps / parts) {
          const int r = r0 + row;
          uint32_t left_tokens = now;
          for (int i = 0; i < r && i < 32; ++i) left_tokens &= left_tokens - 1;
          const uint8_t* x = reinterpret_cast<const uint8_t*>(p.x) + (int64_t)(r < rows ? __ffs(left_tokens) - 1 : 0) * p.hidden * 2;
          float top = r < rows ? row_top(x, source, p.hidden, 0, k8, part, parts) : 0.f;
          if (parts > 1) {
            if (lane == 0) tops[warp] = top;
            __syncthreads();
            for (int i = 0; i < parts; ++i) top = max_nan(top, tops[row * parts + i]);
          }
          if (r < rows) {
            float inv;
            const float scale = row_scale(top, inv);
            if (lane == 0 && part == 0) inverse[r] = inv;
            convert_row<F>(panel, r, rows, x, source, p.hidden, 0, k8, scale, part, parts);
          }
        }
        __syncthreads();
      }

      int slot = 0, turn = 0, cs = warp, count = 0;
      for (int first = from; first < to; first += count, ++turn) {
        const int a = first / per_expert;
        const FewRows rows_here = rows_of<F>(m, table.expert[a]);
        count = min(MT, min(per_expert - first % per_expert, to - first));
        const uint32_t mine = table.tokens[a] & now;
        const uint32_t block = rows * 64;
        uint32_t b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
          b[n] = (mine >> (8 * n + g)) & 1 ? smem_at(panel) + rank_below(now, 8 * n + g) * 64 + t * 16 : 0;
        float acc[MT][NT][4] = {};
        for (; cs < steps; cs += kWarps) {
          copies_wait<S::kDepth - 1>();
          __syncwarp();
          uint32_t bs[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) bs[n] = b[n] ? b[n] + cs * 4 * block : 0;
          multiply_step<F, MT, NT>(acc, ring + slot * FewRing<F, MT>::kSlot, rows_here, m, cs, l.f16, bs, block,
                                   [&](int i) { return feature_row(first % per_expert, count, i); });
          __syncwarp();
          copy_next(slot);
          slot = slot + 1 == S::kDepth ? 0 : slot + 1;
        }
        cs -= steps;
        float* const to_red = red + (turn & 1) * (S::kRed / 4);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) to_red[((warp * MT + i) * NT + n) * 128 + c * 32 + lane] = acc[i][n][c];
        __syncthreads();   // (two buffers: what the tile after next writes is read before the next one's barrier)
        for (int j = tid; j < MT * NT * 64; j += kThreads) {
          const int l2 = j & 31, c = (j >> 5) & 1, n = (j >> 6) % NT, i = (j >> 6) / NT;
          const int token = 8 * n + 2 * (l2 & 3) + c;
          if (i >= count || !((mine >> token) & 1)) continue;
          float gate = 0.f, up = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            gate += to_red[((w * MT + i) * NT + n) * 128 + c * 32 + l2];
            up += to_red[((w * MT + i) * NT + n) * 128 + (c + 2) * 32 + l2];
          }
          const float inv = inverse[rank_below(now, token)];
          const int f = (first % per_expert + i) * 8 + (l2 >> 2);
          gate *= inv;
          up *= inv;
          if (m.bias) {
            const int64_t at = (int64_t)table.expert[a] * m.n;
            gate += load16(m.bias, at + (pairs ? 2 * f : f), l.f16);
            up += load16(m.bias, at + (pairs ? 2 * f + 1 : p.inter + f), l.f16);
          }
          p.h[(int64_t)(table.first_row[a] + rank_below(table.tokens[a], token)) * p.inter + f] = gated(p, gate, up);
        }
      }
      copies_wait<0>();
      __syncthreads();   // panel, ring and sums are free again
    }
    from = to;
  }
}

template <int F, int MT, int NT> struct DownShape {
  static constexpr int kDepth = MT > 2 ? 2 : 3;
  static constexpr int kRed = kWarps * MT * NT * 4 * 32 * 4;
  static constexpr int kFixed = (sizeof(FewTable) + 127) / 128 * 128 + kRed + kMaxSlots * 4 + 128 + kWarps * kDepth * FewRing<F, MT>::kSlot;
};

// out = sum over experts of weight * (W2 h + b2).  A block has up to 16 * MT rows of W2 and goes through all active experts
// with them; its warps take the steps in turn.
template <int F, int MT, int NT>
__global__ void __launch_bounds__(kThreads, 1) few_down_kernel(FewParams p, FewLaunch l) {
  using S = DownShape<F, MT, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem);
  float* const red = reinterpret_cast<float*>(smem + (sizeof(FewTable) + 127) / 128 * 128);
  float* const coef = red + S::kRed / 4;               // of the panel's rows: routing weight and the inverse of the scale
  float* const tops = coef + kMaxSlots;                // (per warp)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_at(red) + S::kRed + kMaxSlots * 4 + 128 + warp * S::kDepth * FewRing<F, MT>::kSlot;
  uint8_t* const panel = smem + S::kFixed;
  // What routed the tokens was complete before the kernel ahead of this one let it start.
  build_table<true>(table, p);
  const FewMatrix& m = p.w2;
  const int steps = (p.inter + 127) / 128, total = table.active * steps;
  const int row_begin = (int)((int64_t)p.hidden * blockIdx.x / gridDim.x), row_end = (int)((int64_t)p.hidden * (blockIdx.x + 1) / gridDim.x);
  const int room = l.panel_bytes / 256;                // rows times steps that the panel holds
  bool waited = false;

  for (int r0 = row_begin; r0 < row_end || !waited; r0 += 16 * MT) {
    auto matrix_row = [&](int i) { return r0 + i < row_end ? r0 + i : -1; };
    int at = warp;                 // the step that is copied next, counted over all experts
    auto copy_next = [&](int slot) {
      if (at < total) {
        const int a = at / steps;
        copy_step<F, MT>(ring + slot * FewRing<F, MT>::kSlot, rows_of<F>(m, table.expert[a]), m, at - a * steps, matrix_row);
        at += kWarps;
      }
      copies_end();
    };
#pragma unroll
    for (int i = 0; i < S::kDepth; ++i) copy_next(i);
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
    }
    float out[MT][NT][4] = {};
    int slot = 0, pos = warp;
    for (int a0 = 0, s0 = 0; a0 < table.active;) {
      // how far the panel reaches: whole experts, then as many steps of the next one as there is room for (at least one)
      int a1 = a0, s1 = s0, free = room;
      while (a1 < table.active) {
        const int n = table.first_row[a1 + 1] - table.first_row[a1], fit = min(steps - s1, free / n);
        if (fit == 0) break;
        free -= fit * n;
        s1 += fit;
        if (s1 < steps) break;
        s1 = 0;
        ++a1;
      }
      const int last = s1 > 0 ? a1 : a1 - 1;           // the last expert with steps in the panel
      const int row0 = table.first_row[a0], rows = table.first_row[last + 1] - row0;
      {
        const int parts = warps_per_row(rows), row = warp / parts, part = warp % parts;
        for (int q0 = 0; q0 < rows; q0 += kWarps / parts) {
          const int r = row0 + q0 + row;
          const bool there = q0 + row < rows;
          const int a = there ? table.row_expert[r] : a0;
          const int k8_0 = a == a0 ? s0 * 16 : 0, k8_1 = (a == a1 ? s1 : steps) * 16;
          const float* h = p.h + (int64_t)(there ? r : 0) * p.inter;
          float top = there ? row_top(h, kFromF32, p.inter, k8_0, k8_1, part, parts) : 0.f;
          if (parts > 1) {
            if (lane == 0) tops[warp] = top;
            __syncthreads();
            for (int i = 0; i < parts; ++i) top = max_nan(top, tops[row * parts + i]);
          }
          if (there) {
            float inv;
            const float scale = row_scale(top, inv);
            if (lane == 0 && part == 0) coef[q0 + row] = table.weight[r] * inv;
            // rows of earlier experts in the panel: the first one's with the steps that it has there
            const int before = a == a0 ? 0 : (table.first_row[a0 + 1] - row0) * (steps - s0) + (table.first_row[a] - table.first_row[a0 + 1]) * steps;
            convert_row<F>(panel + (int64_t)before * 256, r - table.first_row[a], table.first_row[a + 1] - table.first_row[a], h, kFromF32, p.inter,
                           k8_0, k8_1, scale, part, parts);
          }
        }
        __syncthreads();
      }
      uint32_t base = smem_at(panel);
      for (int a = a0; a <= last; ++a) {
        const int first = a == a0 ? s0 : 0, stop = a == a1 ? s1 : steps, n_rows = table.first_row[a + 1] - table.first_row[a];
        const uint32_t mine = table.tokens[a], block = n_rows * 64;
        const FewRows where = rows_of<F>(m, table.expert[a]);
        uint32_t b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) b[n] = (mine >> (8 * n + g)) & 1 ? base + rank_below(mine, 8 * n + g) * 64 + t * 16 : 0;
        float acc[MT][NT][4] = {};
        for (; pos < a * steps + stop; pos += kWarps) {
          copies_wait<S::kDepth - 1>();
          __syncwarp();
          const int s = pos - a * steps;
          uint32_t bs[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) bs[n] = b[n] ? b[n] + (s - first) * 4 * block : 0;
          multiply_step<F, MT, NT>(acc, ring + slot * FewRing<F, MT>::kSlot, where, m, s, l.f16, bs, block, matrix_row);
          __syncwarp();
          copy_next(slot);
          slot = slot + 1 == S::kDepth ? 0 : slot + 1;
        }
        base += (stop - first) * 4 * block;
        // (columns of tokens without this expert are left out: a weight that is not finite would get into them)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int token = 8 * n + 2 * t + c;
            if (!((mine >> token) & 1)) continue;
            const float w = coef[table.first_row[a] - row0 + rank_below(mine, token)];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              out[i][n][c] = fmaf(w, acc[i][n][c], out[i][n][c]);
              out[i][n][c + 2] = fmaf(w, acc[i][n][c + 2], out[i][n][c + 2]);
            }
          }
      }
      a0 = a1;
      s0 = s1;
      __syncthreads();   // the panel is free again
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) red[((warp * MT + i) * NT + n) * 128 + c * 32 + lane] = out[i][n][c];
    copies_wait<0>();
    __syncthreads();
    for (int j = tid; j < 16 * MT * 8 * NT; j += kThreads) {
      // consecutive threads, consecutive features of a token
      const int row = j % (16 * MT), token = j / (16 * MT);
      if (r0 + row >= row_end || token >= p.tokens) continue;
      const int at_red = (((row >> 4) * NT) + (token >> 3)) * 128 + (((row >> 3) & 1) * 2 + (token & 1)) * 32 + (row & 7) * 4 + ((token & 7) >> 1);
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) v += red[w * MT * NT * 128 + at_red];
      if (m.bias) {
        for (int k = 0; k < p.topk; ++k) {
          const int a = table.slot_expert[token * p.topk + k];
          if (a >= 0) v = fmaf(p.weights[token * p.topk + k], load16(m.bias, (int64_t)table.expert[a] * m.n + r0 + row, l.f16), v);
        }
      }
      const int64_t to = (int64_t)token * p.hidden + r0 + row;
      if (l.f16) reinterpret_cast<__half*>(p.out)[to] = __float2half_rn(v);
      else reinterpret_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(v);
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace b200moe
