// What the tensor-core kernels of the layer for a few tokens have in common (few_tokens_rows.cuh: weights stored by output feature;
// few_tokens_columns.cuh: 16-bit weights stored by column).
//
// A few tokens leave the layer to the bandwidth of its weights: every byte of an active expert passes once, by TMA through a
// warp's own ring in shared memory into the registers that the matrix instruction reads.  The first kernel makes h =
// act(W13 x + b13), the second W2 h and what is made of it.
//
// tcgen05 would have to get its weights converted in shared or tensor memory, a second pass for every byte, and its tile
// of 128 features leaves most SMs without work at one token.  mma.sync is far from its limit here (0.4 instructions a cycle
// and SM: 12 to 26 % of the time in use).
//
// What a call costs beyond its bytes (7 tokens of MXFP4 2880 x 2880, four of 128 experts, 81 us for 52 us of weights): finding the
// experts 1.3 us in each kernel (with more than 32 routed slots 2.3), the first weights' way 2, tokens and h on their way to shared
// memory 2.5 each, the sums of the first kernel 2 to 3, of the second 1, the last of a column's blocks 1, and the kernels' ends, where blocks that
// shared the memory evenly finish up to 4 us apart.  Asking for W2 ahead from the first kernel's end into L2 gained nothing (the second
// kernel's loop is as long, the first one's 3 to 8 us longer), nor did both kernels on an SM at once with half the registers.
#pragma once

#include "few_tokens.cuh"
#include "gemm_tc_common.cuh"
#include "sm100_ptx.cuh"

namespace b200moe {
namespace {

constexpr int kFewMaxBlocks = 160;      // of a kernel (one per SM)
constexpr int kMaxSlots = kFewMaxTopk * B200MOE_FEW_TOKENS;   // routed slots of a call

enum FewFormat { kFewFp8, kFewFp4, kFewInt4Fine, kFewInt4, kFewBf16, kFewF16 };   // Fine: groups of 32 or 64
__host__ __device__ constexpr bool by_column(int f) { return f == kFewBf16 || f == kFewF16; }     // stored as [K, N]

struct FewLaunch {
  int panel_bytes;       // of shared memory for the first kernel's panel
  bool f16;
  int columns, splits;   // of the second kernel: blocks with different rows, and shares of the steps for each of them
  int side;              // by column: its warps side by side (1, 2, 4)
  int box;               // rows (by column: columns) of one of its warps, which a load brings
  int room;              // rows of h times steps that its panel holds
  int most;              // tokens that the first kernel's panel holds
  FewDiv by_sets, by_steps, by_ctas;                // the first kernel's: sets of an expert, steps of a row, blocks
  FewDiv by_columns, by_splits, by_down_steps;      // the second one's
  uint32_t* arrived;     // per column of its blocks
  float* part;           // [splits][tokens][hidden]: partial sums, with more than one split
  int32_t* status;       // for waits that run out, or NULL
};

// ---- which experts a call uses ------------------------------------------------------
// Active experts in an order that the ids alone decide, their tokens as bits, and a row number for every (expert, token) that occurs: rows
// of an expert follow one another in token order.
struct FewTable {
  uint32_t bits[32];
  int before[32];
  int active;
  int expert[kMaxSlots];
  uint32_t tokens[kMaxSlots];
  int first_row[kMaxSlots + 1];
  int slot_expert[kMaxSlots];      // the slot's expert, as an index of the active ones (-1: none)
  uint16_t row_expert[kMaxSlots];
  float weight[kMaxSlots];         // of a row: the sum over the slots that name its expert
  float slot_weight[kMaxSlots];
};

__device__ __forceinline__ int rank_below(uint32_t mask, int bit) { return __popc(mask & ((1u << bit) - 1u)); }

// The table of a call with up to 32 routed slots, a lane each; experts in the order of their first slots.  (One token: two
// thirds of the time of the other way.)
template <bool kWeights>
__device__ __forceinline__ void build_small_table(FewTable& t, const FewParams& p, int slots) {
  const int lane = threadIdx.x & 31;
  const int e = lane < slots ? local_expert(p, lane) : -1, tok = lane / p.by_topk;
  if (kWeights && lane < slots) t.slot_weight[lane] = p.weights[lane];
  const uint32_t peers = __match_any_sync(0xffffffffu, e);                       // slots with the same expert
  const int first = __ffs(peers) - 1;
  const uint32_t firsts = __ballot_sync(0xffffffffu, e >= 0 && first == lane);
  const int a = e >= 0 ? rank_below(firsts, first) : -1;
  if (lane < slots) t.slot_expert[lane] = a;
  if (e >= 0 && first == lane) {
    t.expert[a] = e;
    t.tokens[a] = 0;
  }
  __syncwarp();
  if (e >= 0) atomicOr(&t.tokens[a], 1u << tok);
  __syncwarp();
  const uint32_t tokens = e >= 0 ? t.tokens[a] : 0;
  const int n = first == lane ? __popc(tokens) : 0;
  int sum = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
  if (n > 0) t.first_row[a] = sum - n;
  if (lane == 31) {
    t.active = __popc(firsts);
    t.first_row[t.active] = sum;
  }
  __syncwarp();
  if (!kWeights || e < 0) return;
  // (a token that names an expert twice: its slots in their order, by the first of them)
  const uint32_t mine = __popc(peers) > 1 ? peers & (((2u << (p.topk - 1)) - 1u) << tok * p.topk) : 1u << lane;
  if (__ffs(mine) - 1 != lane) return;
  float w = 0.f;
  for (uint32_t left = mine; left; left &= left - 1) w += t.slot_weight[__ffs(left) - 1];
  const int row = t.first_row[a] + rank_below(tokens, tok);
  t.weight[row] = w;
  t.row_expert[row] = (uint16_t)a;
}

template <bool kWeights> __device__ __forceinline__ void build_large_table(FewTable& t, const FewParams& p);
// By one warp; the others meet it at the block's next barrier.
template <bool kWeights>
__device__ __forceinline__ void build_table(FewTable& t, const FewParams& p) {
  const int slots = p.tokens * p.topk;
  if (slots <= 32) build_small_table<kWeights>(t, p, slots);
  else build_large_table<kWeights>(t, p);
}
template <bool kWeights>
__device__ __forceinline__ void build_large_table(FewTable& t, const FewParams& p) {
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
    const int e = t.slot_expert[i], tok = i / p.by_topk;
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
  if (lane == 0) t.first_row[t.active] = base;
  __syncwarp();
  if (kWeights) {
#pragma unroll 1
    for (int i = lane; i < slots; i += 32) {
      const int a = t.slot_expert[i], tok = i / p.by_topk;
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

constexpr int kTableBytes = (sizeof(FewTable) + 127) / 128 * 128;

// ---- loads ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
// The same of a word's first `bytes` bytes (0: nothing is read); the others are zeros.
__device__ __forceinline__ void copy4(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
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

// What a call is given, into L2 while the kernels ahead of it finish (nothing is read yet: they may still write it).
__device__ __forceinline__ void prefetch_call(const FewParams& p, int tid, int threads) {
  const int slots = p.tokens * p.topk;
  const char* const ids = reinterpret_cast<const char*>(p.ids), * const x = reinterpret_cast<const char*>(p.x);
  for (int i = tid * 128; i < slots * (p.ids64 ? 8 : 4); i += threads * 128) prefetch_l2(ids + i);
  for (int i = tid * 128; i < slots * 4; i += threads * 128) prefetch_l2(reinterpret_cast<const char*>(p.weights) + i);
  if (p.expert_map)
    for (int i = tid * 32; i < p.id_limit; i += threads * 32) prefetch_l2(p.expert_map + i);
  for (int i = tid * 128; i < p.tokens * p.hidden * 2; i += threads * 128) prefetch_l2(x + i);
}

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

// The power of two by which values are multiplied on their way to float16, their largest magnitude then between 2^14 and 2^15,
// and its inverse.  Magnitudes below 2^-100 are taken for that; what is not finite stays as it is.
__device__ __forceinline__ float step_scale(uint32_t top, float& inverse) {   // top: bits of the largest magnitude
  int e = (int)(top >> 23);
  if (e == 255) e = 127 + 14;
  e = max(e, 127 - 100);
  inverse = __uint_as_float((uint32_t)(e - 14) << 23);
  return __uint_as_float((uint32_t)(254 - (e - 14)) << 23);
}

// Warps of a row where `warps` of them fill a panel of `rows`.
__device__ __forceinline__ int warps_per_row(int rows, int warps) { return rows >= warps ? 1 : small_div(warps, rows); }

// ---- a warp's ring --------------------------------------------------------------------
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

// Sets a warp's ring up: `depth` slots of `slot` bytes, and `scale_bytes` for scales.
__device__ __forceinline__ FewRing make_ring(uint8_t* rings, int slot, int depth, uint8_t* scales, int scale_bytes, uint64_t* bars, int* gave_up,
                                             int32_t* status) {
  const int warp = threadIdx.x >> 5;
  FewRing r;
  r.slots = smem_at(rings) + warp * depth * slot;
  r.scales = smem_at(scales) + warp * scale_bytes;
  r.bars = smem_at(bars + warp * depth);
  r.slot = r.parity = 0;
  r.gave_up = gave_up;
  r.status = status;
  r.once = ptx::l2_evict_first();
  if ((threadIdx.x & 31) == 0) {
    for (int i = 0; i < depth; ++i) ptx::mbar_init(bars + warp * depth + i, 1);
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
  }
  __syncwarp();
  return r;
}

// ---- what is left ----------------------------------------------------------------------
__device__ __noinline__ float gated_once(int act, float alpha, float limit, float clamp, float gate, float up) {
  return gated(act, alpha, limit, clamp, gate, up);
}
__device__ __forceinline__ float load16(const void* p, int64_t i, bool f16) {
  return f16 ? __half2float(reinterpret_cast<const __half*>(p)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
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

// What a block of the second kernel has to do: its column of blocks, and its share of the steps over all active experts.
struct FewShare {
  int steps;                   // of an expert
  FewDiv by_steps;
  int column, split, begin, end;
  __device__ __forceinline__ FewShare(const FewTable& t, const FewLaunch& l) {
    steps = l.by_down_steps.d;
    by_steps = l.by_down_steps;
    split = blockIdx.x / l.by_columns;
    column = blockIdx.x - split * l.columns;
    const uint32_t total = (uint32_t)(t.active * steps);
    begin = total * split / l.by_splits;
    end = total * (split + 1) / l.by_splits;
  }
  // How far a panel reaches that begins with step s0 of expert a0: whole experts, then as many steps of the next one as
  // there is room for (at least one).
  __device__ __forceinline__ void panel_end(const FewTable& t, int room, int a0, int s0, int& a1, int& s1) const {
    const int ae = end / by_steps, se = end - ae * steps;      // all that is left, if it fits
    const int need = ae == a0 ? (t.first_row[a0 + 1] - t.first_row[a0]) * (se - s0)
                              : (t.first_row[a0 + 1] - t.first_row[a0]) * (steps - s0) + (t.first_row[ae] - t.first_row[a0 + 1]) * steps +
                                    (se > 0 ? (t.first_row[ae + 1] - t.first_row[ae]) * se : 0);
    a1 = ae;
    s1 = se;
    if (need <= room) return;
    int free = room;
    a1 = a0;
    s1 = s0;
    while (a1 * steps + s1 < end) {
      const int n = t.first_row[a1 + 1] - t.first_row[a1], fit = min(min(steps - s1, end - a1 * steps - s1), small_div(free, n));
      if (fit == 0) break;
      free -= fit * n;
      s1 += fit;
      if (s1 < steps) break;
      s1 = 0;
      ++a1;
    }
  }
};

// The last of the blocks with the same rows to arrive adds the partial sums up.
template <typename Finish>
__device__ __forceinline__ void sum_splits(const FewLaunch& launch, const FewParams& p, int& last_one, int column, int row_begin, int width, Finish finish) {
  // (the barrier puts the block's partial sums ahead of the release, and what the others have released ahead of the reads)
  if (threadIdx.x == 0) {
    uint32_t before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(launch.arrived + column) : "memory");
    last_one = before == (uint32_t)launch.splits - 1;
  }
  __syncthreads();
  if (!last_one) return;
  // (four outputs of a thread at once, whose loads are in flight together)
  const int64_t next = (int64_t)p.tokens * p.hidden;
  const int all = width * p.tokens, stride = blockDim.x;
#pragma unroll 1
  for (int j0 = threadIdx.x; j0 < all; j0 += 4 * stride) {
    const float* from[4];
    float v[4] = {};
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const int j = min(j0 + o * stride, all - 1), token = small_div(j, width);
      from[o] = launch.part + (int64_t)token * p.hidden + row_begin + j - token * width;
    }
#pragma unroll 3
    for (int i = 0; i < launch.splits; ++i)
#pragma unroll
      for (int o = 0; o < 4; ++o) v[o] += __ldcg(from[o] + i * next);
#pragma unroll
    for (int o = 0; o < 4; ++o) {
      const int j = j0 + o * stride, token = small_div(j, width);
      if (j < all) finish(v[o], token, row_begin + j - token * width);
    }
  }
}

}  // namespace
}  // namespace b200moe
