// The layer for a few tokens where weights are stored by output feature ([E,N,K]: block-scaled fp8, MXFP4, int4).
//
//   D[features, tokens] += W[16 features, 16 k] x^T[16 k, 8 tokens]     (mma.sync, fp32 accumulation)
//
// A step of a warp is 4 KB of weights, 128 bytes of 32 rows, which one lane asks for by TMA into the warp's own ring.  The sum over
// k does not mind its order, so what a lane reads of a row goes into the instruction as it comes, turned into float16 (which
// holds every code of the three formats exactly), and the tokens are laid out to match.  Scales of weights multiply the sums of
// their group in fp32.
//
// Bound by the weights' bytes with few tokens of large experts: 7168 x 2048 fp8, 8 of 256 experts, one token 65 us, 5.4 TB/s (its
// main loops alone 6.5); with small ones by what a call costs besides (few_tokens_mma.cuh).  MXFP4 and int4 take more instructions for a
// byte (two conversions, and the products of two bytes of fp8), but no unit bounds them: 2880 x 2880, 7 tokens, first and second kernel 52 and
// 43 % of the issue slots, 43 and 35 % of the ALU's cycles, 50 and 38 % of the shared-memory pipe's; int4 4 tokens 49 and 42, 50 and 40,
// 50 and 38.  What they wait for are one another's results: 12 warps hide that in part.
#pragma once

#include "few_tokens_mma.cuh"

namespace b200moe {
namespace {

template <int F> struct RowShape {
  // 12 warps hide one another's loads and products; with 8 the same work took a fifth longer where codes are many (int4)
  static constexpr int kWarps = 12, kThreads = 32 * kWarps;
  static constexpr int kK = F == kFewFp8 ? 128 : 256;           // values of k in a step
  static constexpr int kBlocks = kK / 32;                       // of the panel: a lane's eight values, two instructions
  // int4 codes go into the product as unsigned numbers (see u4x8_to_h2): groups of a step whose sums of x put that right
  static constexpr int kSums = F == kFewInt4 ? 2 : F == kFewInt4Fine ? 8 : 0;
  static constexpr int kFloats = 1 + kSums;                     // per row and step behind the panel: the scale, these sums
  static constexpr int kPanelBytes = kK * 2 + kFloats * 4;      // of the panel: a row's step
  static constexpr int kDepth = 2, kSlot = 4096;
  // Words of four bytes that a row's scales of a step (4 bits) are part of, at most: they may begin at any byte.
  static constexpr int kWords = F == kFewInt4Fine ? 5 : F == kFewFp4 ? 3 : F == kFewInt4 ? 2 : 1;
  // Behind the rings, per warp: scales of the steps in the ring as they come, a word of every row after the other, and as fp32.
  static constexpr int kSlotScales = kWords * 128, kSpread = F == kFewFp8 ? 0 : F == kFewInt4 ? 256 : 1024;
  static constexpr int kWarpScales = kDepth * kSlotScales + kSpread;
  // Shared memory: the rings, barriers, zeros, flags, the table, scales; the rest is the kernels'.
  static constexpr int kBars = kWarps * kDepth * kSlot, kZeros = kBars + 256, kFlags = kZeros + 64, kTable = kFlags + 64;
  static constexpr int kScales = kTable + kTableBytes, kRest = (kScales + kWarps * kWarpScales + 127) / 128 * 128;
  static_assert(kWarps * kDepth * 8 <= 256, "barriers");
};

// The largest value of a step's lanes (half a warp, or a warp: one instruction).
template <int kLanes>
__device__ __forceinline__ uint32_t max_of_step(uint32_t v) {
  if constexpr (kLanes == 32) return __reduce_max_sync(0xffffffffu, v);
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// ---- tokens and activations as float16 -------------------------------------------------
// A panel holds rows of values in the order in which the lanes want them: per step blocks of [row][4 lanes][8 values].  fp8
// lanes hold 16 bytes of a row, 16 values; of int4 16 bytes, 32 values; where groups are 32 values they are handed out to
// the four lanes, eight each.
template <int F>
__device__ __forceinline__ uint32_t row_panel_at(int k8, int row, int rows) {   // k8: k / 8
  const int block = F == kFewFp8 ? (k8 >> 3) * 2 + (k8 & 1) : F == kFewInt4 ? (k8 >> 4) * 4 + (k8 & 3) : k8 >> 2;
  const int t = F == kFewFp8 ? (k8 >> 1) & 3 : F == kFewInt4 ? (k8 >> 2) & 3 : k8 & 3;
  return (uint32_t)(((block * rows + row) * 4 + t) * 16);
}
// Eight values of a row's eighth j, as pairs in order and scaled, to their place, and with int4 what goes with them: pairs are four
// apart, every other one a sixteenth (its codes are 16 times as large), and the sums over a group are kept.
template <int F>
__device__ __forceinline__ void put_eight(uint8_t* panel, float* floats, int j, int row, int rows, uint32_t (&o)[4], uint32_t exponent, bool there) {
  constexpr int kLanes = RowShape<F>::kK / 8, kFloats = RowShape<F>::kFloats;
  float* const f = floats + (j / kLanes * kFloats) * rows + row;
  if constexpr (F == kFewInt4 || F == kFewInt4Fine) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&o[k]));
      sum += v.x + v.y;
    }
#pragma unroll
    for (int d = 1; d < (F == kFewInt4 ? 16 : 4); d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const uint32_t p0 = __byte_perm(o[0], o[2], 0x5410), p1 = __byte_perm(o[0], o[2], 0x7632);
    const uint32_t p2 = __byte_perm(o[1], o[3], 0x5410), p3 = __byte_perm(o[1], o[3], 0x7632);
    const __half2 sixteenth = __half2half2(__ushort_as_half(0x2c00));
    const __half2 h1 = __hmul2(*reinterpret_cast<const __half2*>(&p1), sixteenth), h3 = __hmul2(*reinterpret_cast<const __half2*>(&p3), sixteenth);
    o[0] = p0;
    o[1] = *reinterpret_cast<const uint32_t*>(&h1);
    o[2] = p2;
    o[3] = *reinterpret_cast<const uint32_t*>(&h3);
    constexpr int kGroup = F == kFewInt4 ? 16 : 4;
    if (there && (j & (kGroup - 1)) == 0) f[(1 + (j & (kLanes - 1)) / kGroup) * rows] = sum * -0x1p-21f;     // -8 times 2^-24
    exponent += 14;      // (see kCodeScale)
  }
  if (!there) return;
  *reinterpret_cast<uint4*>(panel + row_panel_at<F>(j, row, rows)) = make_uint4(o[0], o[1], o[2], o[3]);
  if ((j & (kLanes - 1)) == 0) f[0] = __uint_as_float(exponent << 23);
}
// int4 codes are numbers times 2^-24 in the products: 2^10 of that goes to the weights' scales and 2^14 to the tokens'.
constexpr float kCodeScale = 1024.f;

// `len` eighths of a token (what is beyond `values` values is zero) into a panel, by `parts` warps of which this is `part`.
// (Functions that run once in a while are not inlined: what is fetched cold costs some 0.3 us per KB of code.)
template <int F>
__device__ __noinline__ void fill_token(uint8_t* panel, float* floats, const void* from, int values, int len, int row, int rows, int part, int parts,
                                        bool f16) {
  constexpr int kLanes = RowShape<F>::kK / 8;      // of a step (at most 32)
  const int lane = threadIdx.x & 31, stride = 32 * parts;
#pragma unroll 1
  for (int j0 = part * 32 + lane; j0 - lane < len; j0 += 4 * stride) {
    vec16 raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * stride;
      raw[i] = vec16{{0, 0, 0, 0}};
      if (j < len && 8 * j < values) raw[i] = reinterpret_cast<const vec16*>(from)[j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * stride;
      if (j - lane >= len) break;
      float v[8];
      uint32_t top = 0;        // (as bits: magnitudes in their order, NaN last)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw[i].w[k]));
        v[2 * k] = f16 ? f.x : __uint_as_float(raw[i].w[k] << 16);
        v[2 * k + 1] = f16 ? f.y : __uint_as_float(raw[i].w[k] & 0xffff0000u);
        top = max(top, max(__float_as_uint(v[2 * k]) & 0x7fffffffu, __float_as_uint(v[2 * k + 1]) & 0x7fffffffu));
      }
      top = max_of_step<kLanes>(top);
      float inverse;
      const float scale = step_scale(top, inverse);
      uint32_t o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __half2 h = __floats2half2_rn(v[2 * k] * scale, v[2 * k + 1] * scale);
        o[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
      put_eight<F>(panel, floats, j, row, rows, o, __float_as_uint(inverse) >> 23, j < len);
    }
  }
}
// Tokens of the set `now` into a panel.
template <int F>
__device__ __noinline__ void fill_tokens_rows(uint8_t* panel, float* floats, const void* from, int hidden, uint32_t now, int len, bool f16, int warp,
                                              int warps) {
  const int rows = __popc(now), parts = warps_per_row(rows, warps);
  const int together = small_div(warps, parts), mine = small_div(warp, parts), part = warp - mine * parts;      // rows at once, and this warp's
#pragma unroll 1
  for (int row = mine < together ? mine : rows; row < rows; row += together) {
    uint32_t left = now;
    for (int r = 0; r < row; ++r) left &= left - 1;
    const uint16_t* x = reinterpret_cast<const uint16_t*>(from) + (int64_t)(__ffs(left) - 1) * hidden;
    fill_token<F>(panel, floats, x, hidden, len, row, rows, part, parts, f16);
  }
}

// h is float16 with a power of two for every eight values of a row (a rounding to 11 bits, as the products need one anyway), whose
// exponents are behind the values: half as many bytes as fp32 for all the blocks that read them.
__device__ __forceinline__ uint8_t* h_exponents(void* h, int inter, int rows) {
  return reinterpret_cast<uint8_t*>(h) + (int64_t)rows * inter * 2;
}
// By a whole warp: eight neighbouring lanes have the eight values.
__device__ __forceinline__ void store_h(float* h, int row, int f, int inter, int rows, float v, bool there) {
  uint32_t top = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  float inverse;
  const float scale = step_scale(top, inverse);
  if (!there) return;
  reinterpret_cast<__half*>(h)[(int64_t)row * inter + f] = __float2half_rn(v * scale);
  if ((f & 7) == 0) h_exponents(h, inter, rows)[((int64_t)row * inter + f) >> 3] = (uint8_t)(__float_as_uint(inverse) >> 23);
}
// `len` eighths of such a row from value `at` on (what is beyond it is zero) into a panel, by `parts` warps of which this is
// `part`: a step's values get its largest power of two.
template <int F>
__device__ __noinline__ void fill_h(uint8_t* panel, float* floats, void* h, int h_row, int at, int inter, int h_rows, int len, int row, int rows,
                                    int part, int parts) {
  constexpr int kLanes = RowShape<F>::kK / 8;      // of a step (at most 32)
  const int lane = threadIdx.x & 31, stride = 32 * parts, there = min(len, (inter - at) >> 3);
  const int64_t first = ((int64_t)h_row * inter + at) >> 3;
  const uint4* const from = reinterpret_cast<const uint4*>(h) + first;
  const uint8_t* const exponents = h_exponents(h, inter, h_rows) + first;
#pragma unroll 1
  for (int j0 = part * 32 + lane; j0 - lane < len; j0 += 4 * stride) {
    uint4 raw[4];
    int e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * stride;
      raw[i] = make_uint4(0, 0, 0, 0);
      e[i] = 0;
      if (j < there) {
        raw[i] = from[j];
        e[i] = exponents[j];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * stride;
      if (j - lane >= len) break;
      const int top = (int)max_of_step<kLanes>(e[i]);
      // (2^(e - top) as float16; below 2^-24 nothing is left)
      const int down = top - e[i];
      const __half f = __ushort_as_half(down < 15 ? (unsigned short)((15 - down) << 10) : down < 25 ? (unsigned short)(1 << (24 - down)) : (unsigned short)0);
      const __half2 f2 = __halves2half2(f, f);
      uint32_t o[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&o[k]), f2);
        o[k] = *reinterpret_cast<const uint32_t*>(&v);
      }
      put_eight<F>(panel, floats, j, row, rows, o, (uint32_t)top, j < len);
    }
  }
}

// ---- weights: a warp's ring ------------------------------------------------------------
// The swizzle of the copies puts the 16-byte pieces of a row's 128 bytes where the lanes' reads fall on different banks.  (Rows of
// 64 bytes kept the copy unit from the memory's rate, fp8 at one token 91 us, 68 without that; with every lane fetching its own
// pieces MXFP4 took a third more instructions.)  Rows 0 to 31 of a slot are rows g of tile (row / 8) % 2, those from 16 on in the
// upper half of the instruction; of eight rows, row_of(g) is the instruction's row g, so that of the lanes that read 16 bytes at
// once (two rows g) one is in the first four, which the swizzle takes to other banks.
__device__ __forceinline__ int row_of(int g) { return (g >> 1) | ((g & 1) << 2); }
__device__ __forceinline__ int g_of(int row) { return ((row & 3) << 1) | (row >> 2); }
// Where a column's sum of a slot's row is, among 32.
__device__ __forceinline__ int sum_of_row(int row) { return ((row >> 3) & 1) * 16 + (row >> 4) * 8 + g_of(row & 7); }
// Columns of sums are 36 floats apart, so that a store's 32 lanes (eight rows of four columns) hit 32 banks.
constexpr int kSumColumn = 36;

// Scales come by cp.async and are read where the caller has them at every call.  4-bit weights have 2 to 16 bytes of a row and step, at
// any byte (a row of 2880 MXFP4 values has 90), which are part of up to five words of four bytes; the words of a row are
// fetched by neighbouring lanes, so that an instruction has few lines to find (a row a lane: 7 MXFP4 tokens 87 us, so 81),
// and what a row's first word has ahead of its scales is taken off when they are read.  fp8: one per 128 values and 128 rows; a lane
// fetches that of its row.
template <int F>
struct RowScales {
  int words;                          // of a row and step
  int step;                           // bytes per step
  int advance;                        // bytes from a step's to the next one's
  int ahead;                          // of the lane's row: bytes ahead of the first step's scales in their first word
  bool f16;
  int place[RowShape<F>::kWords];     // of the lane's words in the expert's scales, without the step (-1: none)
};
// Slot rows up to `rows`; row(i): the matrix's row of slot row i, or one that is 16 times something below it.
template <int F, typename Row>
__device__ __forceinline__ RowScales<F> row_scales(const FewMatrix& m, int rows, bool f16, Row row) {
  const FewScales& s = m.scales;
  RowScales<F> l;
  const int lane = threadIdx.x & 31;
  l.step = s.step;
  l.advance = s.step / 4 * s.next + s.step % 4;
  l.words = s.step == 2 ? 1 : s.step / 4 + (s.row & 3 ? 1 : 0);      // (two bytes at an even place are part of one word)
  l.ahead = row(lane) * s.row & 3;
  l.f16 = f16;
#pragma unroll
  for (int i = 0; i < RowShape<F>::kWords; ++i) {
    const int j = 32 * i + lane, r = small_div(j, l.words);
    l.place[i] = i < l.words && r < rows ? row(r) * s.row + (j - r * l.words) * s.next : -1;
  }
  return l;
}
// The scales of a slot's rows from a step on.
struct ScalesFrom {
  const uint8_t* at;       // the step's of the expert, or of a row that is 16 times something
  int left;                // bytes of a row from there on
};
__device__ __forceinline__ ScalesFrom scales_from(const FewMatrix& m, int e, int row16, int step) {
  const FewScales& s = m.scales;
  const int first = step * s.step;
  return {reinterpret_cast<const uint8_t*>(m.scale) + ((int64_t)e * m.n * s.bytes + (int64_t)row16 * s.row + (int64_t)(first / 4) * s.next + first % 4),
          s.bytes - first};
}
// A step's words to their places in a slot; on to the next step.
template <int F>
__device__ __forceinline__ void copy_scales(uint32_t to, ScalesFrom& from, const RowScales<F>& l) {
  to += (threadIdx.x & 31) * 4;
  if (from.left >= l.step + 3) {
#pragma unroll
    for (int i = 0; i < RowShape<F>::kWords; ++i)
      if (l.place[i] >= 0) copy4(to + i * 128, reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(from.at + l.place[i]) & ~(uintptr_t)3));
  } else {      // the row's end: nothing from behind it
#pragma unroll
    for (int i = 0; i < RowShape<F>::kWords; ++i) {
      if (l.place[i] < 0) continue;
      const int j = 32 * i + (threadIdx.x & 31), word = j - small_div(j, l.words) * l.words;
      const uint8_t* const at = from.at + l.place[i];
      const int ahead = (int)(reinterpret_cast<uintptr_t>(at) & 3), bytes = max(min(from.left + ahead - 4 * word, 4), 0);
      copy4(to + i * 128, bytes > 0 ? at - ahead : reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(from.at) & ~(uintptr_t)3), bytes);
    }
  }
  from.at += l.advance;
  from.left -= l.step;
}
__device__ __forceinline__ const uint8_t* fp8_scale(const FewMatrix& m, int e, int n) {
  return reinterpret_cast<const uint8_t*>(m.scale) + (int64_t)(e * (m.n >> 7) + (n >> 7)) * (m.k >> 5);
}
// The scales of step s as fp32, four per row and half of the step (int4 with groups from 128 on: one).
template <int F>
__device__ __forceinline__ void spread_scales(uint32_t to, uint32_t from, const RowScales<F>& l, int s) {
  const int row = threadIdx.x & 31, shift = (l.ahead + (F == kFewFp4 ? 0 : s * l.step) & 3) * 8;
  const uint32_t at = from + row * l.words * 4;
  // (the word behind a row's last one has nothing of its scales)
  auto word = [&](int i) { return __funnelshift_r(lds4(at + i * 4), lds4(at + (i + 1) * 4), shift); };
  auto value = [&](uint32_t h) { return kCodeScale * (l.f16 ? __half2float(__ushort_as_half((unsigned short)h)) : __uint_as_float(h << 16)); };
  if constexpr (F == kFewInt4) {
    const uint32_t v = word(0);
    const float a = value(v & 0xffffu);
    sts4(to + row * 4, a);
    sts4(to + 128 + row * 4, l.step == 2 ? a : value(v >> 16));
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t place = to + (h * 32 + row) * 16;
      if constexpr (F == kFewFp4) {
        // 2^(byte - 127): the byte is the exponent (0 gives zero for 2^-127, 255 infinity for NaN).  Beyond the row: zeros.
        const uint32_t v = word(h);
        sts16(place, __uint_as_float((v & 255u) << 23), __uint_as_float((v << 15) & 0x7f800000u), __uint_as_float((v << 7) & 0x7f800000u),
              __uint_as_float((v >> 1) & 0x7f800000u));
      } else if (l.step == 16) {
        const uint32_t v = word(2 * h), w = word(2 * h + 1);
        sts16(place, value(v & 0xffffu), value(v >> 16), value(w & 0xffffu), value(w >> 16));
      } else if (l.step == 8) {
        const uint32_t v = word(h);
        const float a = value(v & 0xffffu), b = value(v >> 16);
        sts16(place, a, a, b, b);
      } else {      // (the matrix next to one with finer groups)
        const float a = value(word(0) >> (l.step == 2 ? 0 : 16 * h) & 0xffffu);
        sts16(place, a, a, a, a);
      }
    }
  }
}

// Where a lane finds the values of its columns' tokens in the panel: the first block and the way to the next one.  Without a
// token: zeros, and no way.  An expert's tokens have columns in their order, so that up to eight need one instruction, whichever they
// are.
struct RowTokens {
  uint32_t at, block;
  uint32_t floats[2], next;   // of the lane's columns of sums: the step's scale (its sums behind it), and the way to the next one
};
// `count` tokens; row(i): the panel's row of the expert's token i.
template <int NT, typename Row>
__device__ __forceinline__ void find_row_tokens(RowTokens (&x)[NT], int count, uint32_t panel, uint32_t floats, uint32_t zeros, int rows, Row row) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool there = 8 * n + g < count;
    x[n].at = there ? panel + row(8 * n + g) * 64 + t * 16 : zeros;
    x[n].block = there ? rows * 64 : 0;
    // (columns without a token: those of the last one, nobody reads them)
#pragma unroll
    for (int c = 0; c < 2; ++c) x[n].floats[c] = floats + row(min(8 * n + 2 * t + c, count - 1)) * 4;
    x[n].next = rows * 4;
  }
}
__device__ __forceinline__ int nth_bit(uint32_t bits, int n) {
  while (n-- > 0) bits &= bits - 1;
  return __ffs(bits) - 1;
}
template <int N> struct Int { static constexpr int value = N; };

// Eight two's-complement nibbles -> float16 pairs (0,4) (1,5) (2,6) (3,7) of (n + 8) 2^-24, every other pair times 16: n ^ 8 = n + 8 is
// unsigned, and a small whole number is a float16 below the normal ones.  (Made signed numbers one by one it is nine
// instructions instead of five.)  What the 8 adds, 8 times the sum of x, is where the sums begin.
__device__ __forceinline__ void u4x8_to_h2(uint32_t w, uint32_t (&o)[4]) {
  const uint32_t h = w >> 8;
  // (a & b) ^ c in one instruction; left to the compiler it is two
  auto masked = [](uint32_t v, uint32_t mask, uint32_t flip) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(v), "r"(mask), "r"(flip));
    return r;
  };
  o[0] = masked(w, 0x000f000fu, 0x00080008u);
  o[1] = masked(w, 0x00f000f0u, 0x00800080u);
  o[2] = masked(h, 0x000f000fu, 0x00080008u);
  o[3] = masked(h, 0x00f000f0u, 0x00800080u);
}

// acc += W x of the step in the slot (rows and columns that there are not: something finite or not that nobody reads).
template <int F, int NT>
__device__ __forceinline__ void multiply_rows(float (&acc)[2][NT][4], uint32_t slot, uint32_t scales, const RowTokens (&x)[NT], int s) {
  using S = RowShape<F>;
  const int lane = threadIdx.x & 31, row = row_of(lane >> 2), t = lane & 3;
  float sx[NT][2];
  uint32_t xa[NT], xf[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    xa[n] = x[n].at + s * (S::kBlocks * x[n].block);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      xf[n][c] = x[n].floats[c] + s * (S::kFloats * x[n].next);
      sx[n][c] = ldsf(xf[n][c]);
    }
  }
  const uint32_t rows = slot + row * 128;
  if constexpr (F == kFewFp8) {
    uint4 v[4][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q][n] = lds16(xa[n] + q * x[n].block);
    const uint32_t at[2] = {rows + ((t ^ row) << 4), rows + ((t ^ row ^ 4) << 4)};
    // (the tiles in turn: products of one depend on one another)
    float d[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 lo[2], hi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[i] = lds16(at[h] + i * 1024);
        hi[i] = lds16(at[h] + i * 1024 + 2048);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t a0, a1, a2, a3;
          e4m3x4_to_h2(w == 0 ? lo[i].x : w == 1 ? lo[i].y : w == 2 ? lo[i].z : lo[i].w, a0, a2);
          e4m3x4_to_h2(w == 0 ? hi[i].x : w == 1 ? hi[i].y : w == 2 ? hi[i].z : hi[i].w, a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 b = v[2 * h + (w >> 1)][n];
            if (h == 0 && w == 0) mma_first(d[i][n], a0, a1, a2, a3, b.x, b.y);
            else mma(d[i][n], a0, a1, a2, a3, w & 1 ? b.z : b.x, w & 1 ? b.w : b.y);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float a = ldsf(scales + (i * 8 + row) * 4), b = ldsf(scales + (i * 8 + row) * 4 + 64);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][n][c] = fmaf((c < 2 ? a : b) * sx[n][c & 1], d[i][n][c], acc[i][n][c]);
    }
  } else {
    const uint32_t piece = rows + (F == kFewInt4 ? (t ^ row) << 4 : (row << 4) + t * 4);
#pragma unroll(NT == 1 ? 2 : 1)
    for (int h = 0; h < 2; ++h) {       // the row's first and second 64 bytes
      uint4 v[4][NT];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q][n] = lds16(xa[n] + (4 * h + q) * x[n].block);
      float first[S::kSums ? S::kSums / 2 : 1][NT][2];
      if constexpr (S::kSums > 0) {
#pragma unroll
        for (int g = 0; g < S::kSums / 2; ++g)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) first[g][n][c] = ldsf(xf[n][c] + (1 + h * (S::kSums / 2) + g) * x[n].next);
      }
      const uint32_t half = piece ^ (h << 6);
      float d[2][NT][4];
      if constexpr (F == kFewInt4) {
        uint4 lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          lo[i] = lds16(half + i * 1024);
          hi[i] = lds16(half + i * 1024 + 2048);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) d[i][n][c] = first[0][n][c & 1];
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t al[4], ah[4];
            u4x8_to_h2(q == 0 ? lo[i].x : q == 1 ? lo[i].y : q == 2 ? lo[i].z : lo[i].w, al);
            u4x8_to_h2(q == 0 ? hi[i].x : q == 1 ? hi[i].y : q == 2 ? hi[i].z : hi[i].w, ah);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma(d[i][n], al[0], ah[0], al[1], ah[1], v[q][n].x, v[q][n].y);
              mma(d[i][n], al[2], ah[2], al[3], ah[3], v[q][n].z, v[q][n].w);
            }
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float a = ldsf(scales + h * 128 + (i * 8 + row) * 4), b = ldsf(scales + h * 128 + (i * 8 + row) * 4 + 64);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][n][c] = fmaf((c < 2 ? a : b) * sx[n][c & 1], d[i][n][c], acc[i][n][c]);
        }
      } else {
        float sum[2][NT][4];
        uint4 as[2], bs[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          as[i] = lds16(scales + (h * 32 + i * 8 + row) * 16);
          bs[i] = lds16(scales + (h * 32 + i * 8 + row) * 16 + 256);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w = (half ^ (q << 4)) + i * 1024;
            const uint32_t wl = lds4(w), wh = lds4(w + 2048);
            uint32_t al[4], ah[4];
            if constexpr (F == kFewFp4) { e2m1x8_to_h2(wl, al); e2m1x8_to_h2(wh, ah); }
            else { u4x8_to_h2(wl, al); u4x8_to_h2(wh, ah); }
            const float a = __uint_as_float(q == 0 ? as[i].x : q == 1 ? as[i].y : q == 2 ? as[i].z : as[i].w);
            const float b = __uint_as_float(q == 0 ? bs[i].x : q == 1 ? bs[i].y : q == 2 ? bs[i].z : bs[i].w);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if constexpr (F == kFewFp4) {
                mma_first(d[i][n], al[0], ah[0], al[1], ah[1], v[q][n].x, v[q][n].y);
              } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) d[i][n][c] = first[q][n][c & 1];
                mma(d[i][n], al[0], ah[0], al[1], ah[1], v[q][n].x, v[q][n].y);
              }
              mma(d[i][n], al[2], ah[2], al[3], ah[3], v[q][n].z, v[q][n].w);
#pragma unroll
              for (int c = 0; c < 4; ++c) sum[i][n][c] = q == 0 ? (c < 2 ? a : b) * d[i][n][c] : fmaf(c < 2 ? a : b, d[i][n][c], sum[i][n][c]);
            }
          }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][n][c] = fmaf(sx[n][c & 1], sum[i][n][c], acc[i][n][c]);
      }
    }
  }
}

// Takes the step in the ring's slot and fetches the next one into it.
template <int F, int NT, typename Next>
__device__ __forceinline__ void take_rows(float (&acc)[2][NT][4], FewRing& ring, const RowScales<F>& l, const RowTokens (&x)[NT], int s, Next next) {
  using S = RowShape<F>;
  uint32_t scales = ring.scales + ring.slot * S::kSlotScales;
  copies_wait<S::kDepth - 1>();
  ring_wait(ring);
  if (F != kFewFp8) {
    const uint32_t to = ring.scales + S::kDepth * S::kSlotScales;
    spread_scales<F>(to, scales, l, s);
    scales = to;
  }
  __syncwarp();
  multiply_rows<F, NT>(acc, ring.slots + ring.slot * S::kSlot, scales, x, s);
  __syncwarp();
  next(ring.slot);
  if (++ring.slot == S::kDepth) {
    ring.slot = 0;
    ring.parity ^= 1;
  }
}

// ---- the first kernel --------------------------------------------------------------------
template <int F, int NT> struct UpRowsShape {
  static constexpr int kSums = NT == 1 ? 24 * 1024 : 36 * 1024;
  static constexpr int kFixed = RowShape<F>::kRest + kSums;
  static_assert(kSums >= (RowShape<F>::kWarps + 1) * kSumColumn * 4 * 8 * NT, "a set with all its tokens");
};

// h[row] = act(W13 x + b13).  The features of all active experts, in sets of 16 (32 rows, 16 gates and their ups), are dealt out
// evenly to the blocks.  A block's sets times the steps of a row are one list, of which each warp takes a stretch; what it adds up
// of a set goes into shared memory, and at the end of a pass all that there is of a set is added up in the warps' order: one
// barrier a pass instead of one a set (which cost 4 to 10 us of the kernel).
template <int F, int NT>
__global__ void __launch_bounds__(RowShape<F>::kThreads, 1) few_up_rows_kernel(const __grid_constant__ FewParams p, const __grid_constant__ FewLaunch launch, const __grid_constant__ CUtensorMap map) {
  using S = RowShape<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + S::kTable);
  uint8_t* const zeros = smem + S::kZeros;                                // a token's values where there is no token
  int* const gave_up = reinterpret_cast<int*>(smem + S::kFlags);
  float* const sums = reinterpret_cast<float*>(smem + S::kRest);
  uint8_t* const panel = smem + UpRowsShape<F, NT>::kFixed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  FewRing ring = make_ring(smem, S::kSlot, S::kDepth, smem + S::kScales, S::kWarpScales, reinterpret_cast<uint64_t*>(smem + S::kBars), gave_up,
                           launch.status);
  if (tid == 0) {
    *gave_up = 0;
    ptx::prefetch_tensormap(&map);
  }
  prefetch_call(p, tid, kThreads);
  pdl_wait();
  pdl_trigger();
  const FewMatrix& m = p.w13;
  const int steps = launch.by_steps.d, per_expert = launch.by_sets.d, most = launch.most;
  // A few values are laid out while one warp finds the experts, which takes as long as a round of loads; more than that would keep
  // the weights from being asked for, and comes after it.
  const bool early = most >= p.tokens && p.tokens * p.hidden <= (kWarps - 1) * 1024;
  const RowScales<F> layout = row_scales<F>(m, 32, launch.f16, [&](int r) { return p.act == B200MOE_ACT_SWIGLUOAI || r < 16 ? r : p.inter + r - 16; });
  if (warp == 0) {
    build_table<false>(table, p);
  } else {
    if (tid < 48) reinterpret_cast<uint32_t*>(zeros)[tid - 32] = 0;
    if (blockIdx.x == 0)   // (the second kernel counts from there)
      for (int i = tid - 32; i < kFewMaxBlocks; i += kThreads - 32) launch.arrived[i] = 0;
    if (early)
      fill_tokens_rows<F>(panel, reinterpret_cast<float*>(panel + p.tokens * steps * (S::kK * 2)), p.x, p.hidden, (1u << p.tokens) - 1u,
                          steps * (S::kK / 8), launch.f16, warp - 1, kWarps - 1);
  }
  __syncthreads();
  const uint32_t all = (uint32_t)(table.active * per_expert);     // (times the blocks below 2^32: takes_mma)
  const int begin = all * blockIdx.x / launch.by_ctas, end = all * (blockIdx.x + 1) / launch.by_ctas;
  const bool pairs = p.act == B200MOE_ACT_SWIGLUOAI;

  // A pass: as many experts as have their tokens in the panel at once and their sums in shared memory; one with more tokens
  // than the panel holds goes through its features again with the rest of them.
  struct Pass {
    int from, to, deep;            // sets; the most tokens that an expert has
    uint32_t now, rest;            // tokens in the panel, and of a later pass over the same sets
    int total;                     // steps
    // A warp's first step; fewer steps than warps: one each.
    __device__ __forceinline__ int start(int warp) const { return total >= kWarps ? total * warp / kWarps : min(warp, total); }
    __device__ __forceinline__ int warp_of(int step, const FewDiv& by_total) const { return total >= kWarps ? (kWarps * (step + 1) - 1) / by_total : step; }
  };
  auto plan = [&](int from, int to, uint32_t rest) {       // from the set `from` on, or the rest of the tokens
    Pass pass;
    pass.from = from;
    pass.deep = min(__popc(rest), most);
    if (!rest) {
      const int a_first = from / launch.by_sets;
      to = from;
      for (int a = a_first; to < end; ++a) {
        const uint32_t with = rest | table.tokens[a];
        const int n = max(pass.deep, min(__popc(table.tokens[a]), most)), stop = min(end, (a + 1) * per_expert);
        const int room = small_div(UpRowsShape<F, NT>::kSums / (kSumColumn * 4), n) - kWarps;             // sets
        if (rest && (__popc(with) > most || room <= to - from)) break;
        rest = with;
        pass.deep = n;
        to = min(stop, from + room);
        if (to < stop) break;
      }
      if (early) rest = (1u << p.tokens) - 1u;
    }
    pass.to = to;
    pass.now = rest;
    while (__popc(pass.now) > most) pass.now &= ~(1u << (31 - __clz(pass.now)));
    pass.rest = rest & ~pass.now;
    pass.total = (to - from) * steps;
    return pass;
  };

  // The set and step that are fetched next, and how many after them.
  int fetch_j = 0, fetch_s = 0, fetch_s0 = 0, left = 0, e = 0, row = 0;
  const uint8_t* scale = nullptr;
  ScalesFrom scales_at = {};
  auto copy_next = [&](int slot) {
    if (left > 0) {
      if (fetch_s == steps) {
        fetch_s = fetch_s0;
        fetch_s0 = 0;
        const int a = fetch_j / launch.by_sets;
        row = 16 * (fetch_j - a * per_expert);
        ++fetch_j;
        e = table.expert[a];
        if (F == kFewFp8) scale = fp8_scale(m, e, pairs ? 2 * row + lane : row + (lane & 15) + (lane >= 16 ? p.inter : 0)) + fetch_s * 4;
        else scales_at = scales_from(m, e, pairs ? 2 * row : row, fetch_s);
      }
      const uint32_t scales = ring.scales + slot * S::kSlotScales;
      if (lane == 0) {
        const uint32_t at = ring.slots + slot * S::kSlot, bar = ring.bars + slot * 8;
        const int y0 = pairs ? 2 * row : row, y1 = pairs ? 2 * row + 16 : p.inter + row;
        ptx::fence_proxy_async();      // (the warp has read what was there)
        ptx::mbar_expect_tx_s(bar, S::kSlot);
        ptx::tma_load_3d_hint_s(at, &map, bar, fetch_s * 128, y0, e, ring.once);
        ptx::tma_load_3d_hint_s(at + S::kSlot / 2, &map, bar, fetch_s * 128, y1, e, ring.once);
      }
      if constexpr (F == kFewFp8) {
        copy4(scales + lane * 4, scale);
        scale += 4;
      } else {
        copy_scales<F>(scales, scales_at, layout);
      }
      ++fetch_s;
      --left;
    }
    copies_end();
  };
  auto start_fetch = [&](const Pass& pass) {
    const int pos = pass.start(warp), j = pos / launch.by_steps;
    left = pass.start(warp + 1) - pos;
    fetch_j = pass.from + j;
    fetch_s0 = pos - j * steps;
    fetch_s = steps;
#pragma unroll 1
    for (int i = 0; i < S::kDepth; ++i) copy_next((ring.slot + i) % S::kDepth);
  };
  auto lay_out = [&](uint32_t now) {
    fill_tokens_rows<F>(panel, reinterpret_cast<float*>(panel + __popc(now) * steps * (S::kK * 2)), p.x, p.hidden, now, steps * (S::kK / 8), launch.f16,
                        warp, kWarps);
  };
  Pass pass = plan(begin, begin, 0);
  if (begin < end) {
    start_fetch(pass);
    if (!early) {
      lay_out(pass.now);
      __syncthreads();
    }
  }
#pragma unroll 1
  while (pass.from < end) {
    const int from = pass.from, deep = pass.deep, rows = __popc(pass.now);
    const int pos0 = pass.start(warp), pos1 = pass.start(warp + 1), j0 = pos0 / launch.by_steps, s0 = pos0 - j0 * steps;
    const uint32_t now = pass.now;
    const FewDiv by_total(pass.total);
    const float* const floats = reinterpret_cast<float*>(panel + rows * steps * (S::kK * 2));
#pragma unroll 1
    for (int pos = pos0, j = j0, s = s0; pos < pos1; ++j, s = 0) {
      const uint32_t mine = table.tokens[(from + j) / launch.by_sets] & now;
      const int count = __popc(mine), stop = min(steps, s + pos1 - pos);
      pos += stop - s;
      // sets and warps begin a new entry each
      float* const entry = sums + (j + warp) * (kSumColumn * deep) + (lane >> 2);
      auto take = [&](auto width) {
        constexpr int N = decltype(width)::value;
        RowTokens x[N];
        find_row_tokens<N>(x, count, smem_at(panel), smem_at(floats), smem_at(zeros), rows, [&](int i) { return rank_below(now, nth_bit(mine, i)); });
        float acc[2][N][4] = {};
#pragma unroll 1
        for (; s < stop; ++s) take_rows<F, N>(acc, ring, layout, x, s, copy_next);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int column = 8 * n + 2 * (lane & 3) + c;
            if (column >= count) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              entry[column * kSumColumn + i * 16] = acc[i][n][c];
              entry[column * kSumColumn + i * 16 + 8] = acc[i][n][c + 2];
            }
          }
      };
      if (NT == 1 || count <= 8) take(Int<1>{});
      else take(Int<NT>{});
    }
    // Half a warp has a set, a lane one of its features.  What does not need the sums is there before the barrier, and for the
    // next set before the sums of this one.
    struct { int a, f, w0, w1; float gate, up; } set;
    const int sets = pass.to - from;
    auto look_up = [&](int j) {
      j = min(j, sets - 1);
      set.a = (from + j) / launch.by_sets;
      set.f = 16 * (from + j - set.a * per_expert) + (lane & 15);
      // the warps that had the set's first and last step
      set.w0 = pass.warp_of(j * steps, by_total);
      set.w1 = pass.warp_of((j + 1) * steps - 1, by_total);
      set.gate = set.up = 0.f;
      if (m.bias) {
        const int64_t at = (int64_t)table.expert[set.a] * m.n;
        set.gate = load16(m.bias, at + (pairs ? 2 * set.f : set.f), launch.f16);
        set.up = load16(m.bias, at + (pairs ? 2 * set.f + 1 : p.inter + set.f), launch.f16);
      }
    };
    const int gate_row = pairs ? 2 * (lane & 15) : lane & 15, up_row = pairs ? gate_row + 1 : 16 + gate_row;
    const float* const gates = sums + sum_of_row(gate_row), * const ups = sums + sum_of_row(up_row);
    if (2 * warp < sets) look_up(2 * warp + (lane >> 4));
    // the next pass's weights are on their way meanwhile
    const Pass next = pass.rest ? plan(from, pass.to, pass.rest) : plan(pass.to, pass.to, 0);
    if (next.from < end) start_fetch(next);
    __syncthreads();   // the sums are complete, and the panel is free again
#pragma unroll 1
    for (int j0 = 2 * warp; j0 < sets; j0 += 2 * kWarps) {
      const auto here = set;
      const int j = j0 + (lane >> 4);
      if (j0 + 2 * kWarps < sets) look_up(j + 2 * kWarps);
      const uint32_t have = table.tokens[here.a];
      uint32_t later = j < sets ? have & now : 0;
      for (int rank = 0; __any_sync(0xffffffffu, later != 0); ++rank) {
        const int token = __ffs(later) - 1;
        float v = 0.f;
        if (token >= 0) {
          float gate = here.gate, up = here.up;
          for (int w = here.w0; w <= here.w1; ++w) {
            const int at = ((j + w) * deep + rank) * kSumColumn;
            gate += gates[at];
            up += ups[at];
          }
          v = gated_once(p.act, p.alpha, p.limit, p.clamp, gate, up);
        }
        store_h(p.h, table.first_row[here.a] + (token >= 0 ? rank_below(have, token) : 0), here.f, p.inter, p.tokens * p.topk, v, token >= 0);
        later &= later - 1;
      }
    }
    if (next.from < end) {
      if (!early) lay_out(next.now);
      __syncthreads();   // the sums' place is free again
    }
    pass = next;
  }
  copies_wait<0>();
}

// ---- the second kernel -------------------------------------------------------------------
constexpr int kBlockRows = 64;      // of W2 that a block has at once
__host__ __device__ __forceinline__ int down_sums_bytes(int tokens, int warps) { return (warps * tokens * kSumColumn * 4 + 127) / 128 * 128; }

// out = sum over experts of weight * (W2 h + b2).  A block has some rows of W2 and a share of the steps over all active
// experts: of rows up to 64, so that few blocks need the same values of h, and of steps what makes as many blocks as there are
// SMs.  It goes through its steps with as many of h's values at a time as its panel holds, each warp with a stretch of them,
// half of the rows each.  Of the blocks with the same rows the last one to be done adds the partial sums up, in their order.
template <int F, int NT>
__global__ void __launch_bounds__(RowShape<F>::kThreads, 1) few_down_rows_kernel(const __grid_constant__ FewParams p, const __grid_constant__ FewLaunch launch, const __grid_constant__ CUtensorMap map) {
  using S = RowShape<F>;
  constexpr int kWarps = S::kWarps, kThreads = S::kThreads, kMembers = kWarps / 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  FewTable& table = *reinterpret_cast<FewTable*>(smem + S::kTable);
  uint8_t* const zeros = smem + S::kZeros;
  int* const gave_up = reinterpret_cast<int*>(smem + S::kFlags);
  int& last_one = *reinterpret_cast<int*>(smem + S::kFlags + 4);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;
  FewRing ring = make_ring(smem, S::kSlot, S::kDepth, smem + S::kScales, S::kWarpScales, reinterpret_cast<uint64_t*>(smem + S::kBars), gave_up,
                           launch.status);
  // every warp's sums, by token, and the panel
  float* const sums = reinterpret_cast<float*>(smem + S::kRest), * const my_sums = sums + warp * p.tokens * kSumColumn + (lane >> 2);
  uint8_t* const panel = smem + S::kRest + down_sums_bytes(p.tokens, kWarps);
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
  const int steps = share.steps, member = warp >> 1, warp_rows = launch.box;
  const int row_begin = (uint32_t)p.hidden * share.column / launch.by_columns, row_end = (uint32_t)p.hidden * (share.column + 1) / launch.by_columns;
  float* const floats = reinterpret_cast<float*>(panel + launch.room * (S::kK * 2));
  bool waited = false;
  auto finish = [&](float v, int token, int n) {
    const int64_t to = (int64_t)token * p.hidden + n;
    if (launch.f16) reinterpret_cast<__half*>(p.out)[to] = __float2half_rn(v);
    else reinterpret_cast<__nv_bfloat16*>(p.out)[to] = __float2bfloat16_rn(v);
  };
  for (int block_r0 = row_begin; block_r0 < row_end; block_r0 += 2 * warp_rows) {
    const int r0 = block_r0 + (warp & 1) * warp_rows, rows_here = max(0, min(warp_rows, row_end - r0));
    const RowScales<F> layout = row_scales<F>(m, rows_here, launch.f16, [&](int r) { return r0 + r; });
    // The step that is fetched next, how many are left of this warp's stretch, and where the panel after that begins.
    int fetch_a = 0, fetch_s = 0, left = 0, panel_a = share.begin / share.by_steps, panel_s = share.begin - panel_a * steps, e = 0;
    bool found = false;
    const uint8_t* scale = nullptr;
    ScalesFrom scales_at = {};
    auto copy_next = [&](int slot) {
      while (left == 0 && panel_a * steps + panel_s < share.end) {
        int a1, s1;
        share.panel_end(table, launch.room, panel_a, panel_s, a1, s1);
        const int from = panel_a * steps + panel_s, all = a1 * steps + s1 - from, mine = all * member / kMembers;
        left = all * (member + 1) / kMembers - mine;
        fetch_a = (from + mine) / share.by_steps;
        fetch_s = from + mine - fetch_a * steps;
        panel_a = a1;
        panel_s = s1;
        found = false;
      }
      if (left > 0 && rows_here > 0) {
        if (fetch_s == steps) { fetch_s = 0; ++fetch_a; found = false; }
        if (!found) {
          e = table.expert[fetch_a];
          if (F == kFewFp8) scale = fp8_scale(m, e, min(r0 + lane, p.hidden - 1)) + fetch_s * 4;
          else scales_at = scales_from(m, e, 0, fetch_s);
          found = true;
        }
        const uint32_t scales = ring.scales + slot * S::kSlotScales;
        if (lane == 0) {
          const uint32_t bar = ring.bars + slot * 8;
          ptx::fence_proxy_async();        // (the warp has read what was there)
          ptx::mbar_expect_tx_s(bar, warp_rows * 128);
          ptx::tma_load_3d_hint_s(ring.slots + slot * S::kSlot, &map, bar, fetch_s * 128, r0, e, ring.once);
        }
        if constexpr (F == kFewFp8) {
          copy4(scales + lane * 4, scale);
          scale += 4;
        } else {
          copy_scales<F>(scales, scales_at, layout);
        }
        ++fetch_s;
        --left;
      }
      copies_end();
    };
#pragma unroll 1
    for (int i = 0; i < S::kDepth; ++i) copy_next((ring.slot + i) % S::kDepth);
    const int block_rows_here = min(2 * warp_rows, row_end - block_r0), my_row = tid % kBlockRows, my_token = tid / kBlockRows;
    const bool with_bias = m.bias && share.split == 0;           // (by the blocks with the first share)
    if (with_bias)
      for (int i = tid; i < 2 * table.active; i += kThreads)     // into L2: what is needed once the products are done
        prefetch_l2(reinterpret_cast<const uint16_t*>(m.bias) + (int64_t)table.expert[i >> 1] * m.n + ((i & 1) ? block_r0 + block_rows_here - 1 : block_r0));
    if (!waited) {
      pdl_wait();
      pdl_trigger();
      waited = true;
    }
    for (int i = lane; i < p.tokens * kSumColumn; i += 32) sums[warp * p.tokens * kSumColumn + i] = 0.f;
    __syncwarp();
    for (int a0 = share.begin / share.by_steps, s0 = share.begin - a0 * steps; a0 * steps + s0 < share.end;) {
      int a1, s1;
      share.panel_end(table, launch.room, a0, s0, a1, s1);
      const int last = s1 > 0 ? a1 : a1 - 1;           // the last expert with steps in the panel
      const int row0 = table.first_row[a0], rows = table.first_row[last + 1] - row0;
      {
        // (the first expert's rows have the steps from s0 on, the last one's those up to s1)
        constexpr int kPiece = S::kK / 8;
        const int parts = warps_per_row(rows, kWarps), n0 = table.first_row[a0 + 1] - row0;
        const int together = small_div(kWarps, parts), mine = small_div(warp, parts), part = warp - mine * parts;
#pragma unroll 1
        for (int row = mine; row < rows; row += together) {
          const int r = row0 + row, a = table.row_expert[r], e0 = table.first_row[a], n = table.first_row[a + 1] - e0;
          const int k8_0 = (a == a0 ? s0 : 0) * kPiece, len = (a == a1 ? s1 : steps) * kPiece - k8_0;
          const int before = a == a0 ? 0 : n0 * (steps - s0) + (e0 - row0 - n0) * steps;   // rows times steps of earlier experts
          fill_h<F>(panel + before * (S::kK * 2), floats + before * S::kFloats, p.h, r, 8 * k8_0, p.inter, p.tokens * p.topk, len, r - e0, n,
                    part, parts);
        }
        __syncthreads();
      }
      {
        const int from = a0 * steps + s0, all = a1 * steps + s1 - from;
        int pos = from + all * member / kMembers;
        const int stop = rows_here > 0 ? from + all * (member + 1) / kMembers : 0;
        for (int a = pos / share.by_steps; pos < stop; ++a) {
          const int row = table.first_row[a], n_rows = table.first_row[a + 1] - row, end = min(stop, (a + 1) * steps);
          // rows of earlier experts in the panel, as above
          const int before = (a == a0 ? 0 : (table.first_row[a0 + 1] - row0) * (steps - s0) + (row - table.first_row[a0 + 1]) * steps) - (a == a0 ? s0 : 0) * n_rows;
          const uint32_t mine = table.tokens[a];
          auto take = [&](auto width) {
            constexpr int N = decltype(width)::value;
            RowTokens x[N];
            find_row_tokens<N>(x, n_rows, smem_at(panel) + before * (S::kK * 2), smem_at(floats) + before * (S::kFloats * 4), smem_at(zeros), n_rows,
                               [](int i) { return i; });
            float acc[2][N][4] = {};
#pragma unroll 1
            for (; pos < end; ++pos) take_rows<F, N>(acc, ring, layout, x, pos - a * steps, copy_next);
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int column = 8 * n + 2 * t + c;
                if (column >= n_rows) continue;
                const float w = table.weight[row + column];
                float* const to = my_sums + nth_bit(mine, column) * kSumColumn;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  to[i * 16] = fmaf(w, acc[i][n][c], to[i * 16]);
                  to[i * 16 + 8] = fmaf(w, acc[i][n][c + 2], to[i * 16 + 8]);
                }
              }
          };
          if (NT == 1 || n_rows <= 8) take(Int<1>{});
          else take(Int<NT>{});
        }
      }
      a0 = a1;
      s0 = s1;
      if (a0 * steps + s0 < share.end) __syncthreads();   // the panel is free again
    }
    // Biases while other warps are still at work.
    constexpr int kMine = (B200MOE_FEW_TOKENS * kBlockRows + kThreads - 1) / kThreads;
    float bias[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int token = my_token + i * (kThreads / kBlockRows);
      bias[i] = with_bias && token < p.tokens && my_row < block_rows_here ? weighted_bias(table, m, p.topk, launch.f16, token, block_r0 + my_row) : 0.f;
    }
    copies_wait<0>();
    __syncthreads();
    // consecutive threads, consecutive features of a token
    const int which = my_row >= warp_rows ? 1 : 0, my_sum = sum_of_row((my_row - which * warp_rows) & 31);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int token = my_token + i * (kThreads / kBlockRows);
      if (my_row >= block_rows_here || token >= p.tokens) continue;
      float v = bias[i];
#pragma unroll
      for (int w = 0; w < kMembers; ++w) v += sums[((2 * w + which) * p.tokens + token) * kSumColumn + my_sum];
      if (launch.splits == 1) finish(v, token, block_r0 + my_row);
      else launch.part[((int64_t)share.split * p.tokens + token) * p.hidden + block_r0 + my_row] = v;
    }
    __syncthreads();
  }
  if (launch.splits > 1) sum_splits(launch, p, last_one, share.column, row_begin, row_end - row_begin, finish);
}

}  // namespace
}  // namespace b200moe
