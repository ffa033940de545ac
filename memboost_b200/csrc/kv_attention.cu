// Attention of one query token a sequence over the quantised paged cache (no
// counterpart in the reference): out = sum_t softmax_t(scale q . k_t) v_t.
//
// The query heads that share a key/value head are taken together, so that a
// code is read once: S^T = K Q^T with 16 tokens as the rows of an
// m16n8k16 product and up to 8 heads (or 16, two products) as its columns,
// then O^T += V^T P^T with 16 channels as the rows.  A sequence has one query
// token, so each key element meets at most `group` products: the work is
// bound by reading the codes, and the products only keep the arithmetic off
// the fp32 units.
//
// A CTA has kWarps warps that compute, 16 tokens each at a time, and one that
// fetches: units of 16 kWarps tokens go through a ring in shared memory by TMA
// (boxes of the code arrays as tall as the pages allow -- rows of one page and
// head are contiguous -- and bulk copies of the scales), also across the end
// of a sequence, while the others finish it.
//
// Both products' left operands are read as they lie, because the order of the
// inner index is free: in S^T lane (g, j) = (lane / 4, lane % 4) takes 16 bytes
// (4 bits: 4 of each group's 16) of the rows of tokens g and g + 8, in O^T 16
// channels of the four tokens of its columns; Q's registers follow the keys'
// channel order.  The boxes' swizzle, the 16-byte chunks 2 j + step and the
// tokens' order (token_of) keep these reads free of bank conflicts.  Between
// the products the probabilities change from S^T's layout to the right
// operand's by a transposing move.
//
// 8-bit keys enter S^T as they are: an m16n8k32 integer product with the
// query, scaled by a power of two to below 1, in three 8-bit parts (22 bits and
// a sign: off by at most 2^-22 of the query's largest channel, exact for
// channels above 2^-11 of it; with two parts, 14 bits, a channel far above the
// others cost them theirs, and 16 x 2048 took 2 % less time, 2 x 100001 4 %).
// The sums are exact.  8-bit values become exact fp16 integers (1024 +
// 128 + code by a byte permute, minus 1152); their scale multiplies the
// probability.
//
// 4-bit keys enter S^T as codes, too: their pairs under a mask are subnormal
// fp16 numbers, code 2^-24 (the upper ones code 2^-20), and exact.  The query is
// fp16 relative to its largest channel (up to 2^15: exact for channels above
// 2^-25 of it); a group's sum is multiplied by its scale in fp32, and the minima
// by the queries' sums over the groups in a product of their own (fp16, 22 bits
// of each sum in two parts).  4-bit values become m + s * code in fp16,
// one rounding (2^-11 of the value; beyond 65504 infinite).
//
// Scores, maxima, sums and the outputs' accumulators are fp32.
//
// Weights -- probabilities, with 8 bits times the value's scale -- are rounded
// to fp16 (2^-11), and for an fp16 output, whose own rounding is no larger,
// what that drops is multiplied too.  They are taken relative to the largest
// weight of the head so far, not the largest scale or score alone: a token
// whose values are huge but whose probability is nothing does not push the
// others out of fp16's range.  The reference m of a head's exponents is set so
// that the largest weight lies at 2^10, and again when one exceeds 2^15: weights
// down to 2^-24 of the largest are normal numbers, what is lost of a smaller one
// is below 2^-35 of it, and most steps rescale nothing.  The sum of probabilities
// has the same reference; with 8 bits they reach from 2^-111 (the largest scale)
// to 2^90 (a value of 0), which fp32 has room for.
//
// The units of all sequences and heads are dealt out evenly to the resident
// CTAs (two or three an SM), whatever the lengths: a CTA's share may begin and
// end inside a sequence, and pass sequences without tokens.  Those parts (maximum,
// sum, unnormalised output) go to the workspace, two a CTA at most, and a second
// kernel joins them in the order of the tokens, so the result does not depend on
// the CTAs' timing.  Where the table holds few tokens a sequence, a CTA takes a
// whole sequence's head instead and nothing is joined.
//
// Measured: 8 bits stream at 88 % of the copy rate (one sequence of 65536 tokens
// and 32 heads: 97 us for 86 us of bytes; 360 instructions a warp for 16 tokens
// of 128 channels and up to 8 query heads), 4 bits are bound by their instructions
// (470: 98 us for 52).  Beside that a call costs about 8 us (launch, the first
// units, the join) and each sequence's head about 4 us of a CTA.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "mb_cache.cuh"
#include "mb_tma.cuh"

namespace mb {
namespace {

constexpr int kBlock = 16;  // tokens a warp takes at a time

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5}, {%6}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(b));
}

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 x 8 matrix of 16-bit elements, a row's pair a lane, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 x) { return *reinterpret_cast<uint32_t*>(&x); }
__device__ __forceinline__ __half2 bits_h2(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }

// Two bytes 128 + code (in the low bytes of each half, 0x64 above: 1152 +
// code in fp16) to the codes.
__device__ __forceinline__ uint32_t code8_pair(uint32_t biased, uint32_t select) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, select);
  return h2_bits(__hsub2(bits_h2(h), bits_h2(0x64806480u)));
}

// (x & mask) | bits in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
  return d;
}

// Nibbles 0 and 4 (or, kHigh, 1 and 5) of w to m + s * code.
template <bool kHigh>
__device__ __forceinline__ uint32_t code4_pair(uint32_t w, __half2 s, __half2 m) {
  const uint32_t h = and_or(w, kHigh ? 0x00F000F0u : 0x000F000Fu, 0x64006400u);
  const __half2 c = kHigh ? __hfma2(bits_h2(h), bits_h2(0x2C002C00u), bits_h2(0xD400D400u))
                          : __hsub2(bits_h2(h), bits_h2(0x64006400u));  // (h - 1024) / 16
  return h2_bits(__hfma2(c, s, m));
}

struct Query {
  const void* data;
  int64_t batch_stride, head_stride;
  bool bf16, vec;
};

__device__ __forceinline__ void store_out(void* out, bool bf16, int64_t i, float y) {
  if (bf16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(y);
  else
    static_cast<__half*>(out)[i] = __float2half_rn(y);
}

// How rows of a head_dim in (64 (kQuarters - 1), 64 kQuarters] are taken.
template <int BITS, int kQuarters>
struct Layout {
  static constexpr int kWarps = 4;                         // that compute
  static constexpr int kUnit = kWarps * kBlock;            // tokens a stage
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kRow = kQuarters >= 3 ? (BITS == 8 ? 256 : 128) : kQuarters * 8 * BITS;
  static constexpr int kBoxRow = kRow < 128 ? kRow : 128;  // bytes of a row in one box
  static constexpr int kBoxes = kRow / kBoxRow;
  static constexpr int kColumn = kUnit * kBoxRow;          // a box column of a stage
  static constexpr int kCodes = kUnit * kRow;              // of keys, or of values
  static constexpr int kSwizzle = kBoxRow == 128 ? 0x70 : kBoxRow == 64 ? 0x30 : 0x10;
  // bytes of a token's scales, and what a stage keeps for them at most
  __host__ __device__ static constexpr uint32_t scale_bytes(uint32_t dim) {
    return BITS == 8 ? 4 : dim / kGroup4 * 4;
  }
  static constexpr int kScales = kUnit * (BITS == 8 ? 4 : 2 * kQuarters * 4);
  // a stage: the keys' codes, the values', the keys' scales, the values'
  static constexpr int kStage = (2 * (kCodes + kScales) + 1023) / 1024 * 1024;
  static constexpr int kStages = kQuarters > 2 ? 2 : BITS == 8 ? 3 : 5;
  // CTAs an SM: what registers and shared memory leave room for
  __host__ __device__ static constexpr int ctas(int tiles) {
    return kQuarters > 2 || tiles == 2 ? 2 : 3;
  }

  // S^T: steps of 4 lanes x 4 words, or groups of 4 lanes x a word; O^T: passes of 8
  // lanes x 16 channels
  static constexpr int kSteps = kRow / 64;                           // 8 bits
  static constexpr int kGroups = kRow / 16;                          // 4 bits: of 32 channels
  static constexpr int kProducts = 2 * (BITS == 8 ? kSteps : kGroups);  // of S^T, and a part
  static constexpr int kPieces = BITS == 8 ? 2 * kSteps : kGroups;   // a lane's, of 8 channels
  // 8 bits: parts of the query (of three, the lower ones) that registers have no
  // room for and shared memory holds, each lane its own
  __host__ __device__ static constexpr int parts_in_smem(int tiles) {
    return BITS == 4 ? 0 : tiles == 2 ? 2 : kQuarters > 2 ? 1 : 0;
  }
  static constexpr int kPasses = (kQuarters + 1) / 2;

  // The warps' outputs of 8 heads before they are joined: [warp][8][kJoinRow],
  // channel ch at ch + 4 (ch / 32) (free of bank conflicts).
  static constexpr int kJoinRow = 64 * kQuarters + 8 * kQuarters + 1;
  static constexpr int kJoin = kWarps * 8 * kJoinRow * 4;
  static constexpr int kRing = kStages * kStage;
  __host__ __device__ static constexpr int smem(int tiles) {
    return 1024 + kRing + kJoin + kWarps * 32 * 8 * parts_in_smem(tiles) * kProducts * tiles;
  }

  // Place in a stage's keys (or values) of a byte of a row.
  __device__ __forceinline__ static uint32_t at(uint32_t row, uint32_t byte) {
    const uint32_t o = row * kBoxRow + byte % kBoxRow;
    return byte / kBoxRow * kColumn + (o ^ ((o >> 3) & kSwizzle));
  }
  // 8 bits: first byte of lane j's part of a key's row in a step.
  __device__ __forceinline__ static uint32_t key_byte(int step, int j) {
    if constexpr (kSteps == 1) return 16 * j;
    return 128 * (step / 2) + 16 * (2 * j + step % 2);
  }
  // First channel of lane j's piece of 8.
  __device__ __forceinline__ static uint32_t piece_channel(int piece, int j) {
    if constexpr (BITS == 8) return key_byte(piece / 2, j) + 8 * (piece % 2);
    return 32 * piece + 8 * j;
  }
};

// Token (of 16) at row g of S^T and column k = g of O^T's inner index: pairs
// change places in every other pair of pairs, which spreads a warp's reads of
// the values over the banks.
__device__ __forceinline__ int token_of(int k) { return k ^ ((k >> 1) & 1); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -0x1.fffffep127f;  // a maximum of nothing
// Exponents of the largest weight: when it is set, and above which it is set again.
constexpr int kAim = 10, kMost = 15;
// 8 bits: a probability above which it is set again, and the least exponent that a
// value's scale counts as when it is (one of 0 has no weight, but belongs to the sum).
constexpr float kMostP = 0x1p90f;
constexpr int kLeastScale = -70;

// Integer products begin at the bits of 1.5 2^23: sums of up to 2^22 (256 channels
// of 128 times 128) then are the bits of 1.5 2^23 plus the sum, which a subtraction
// makes an fp32 number (converting goes through the unit that exp2 needs).
constexpr int kSumBits = 0x4B400000;
__device__ __forceinline__ float whole_sum(int x) { return __int_as_float(x) - kRoundMagic; }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
// Four 8 x 16-byte matrices, a row a lane's address: lane (g, j) has bytes 4 j .. of
// row g of each.
__device__ __forceinline__ void ldmatrix4(uint32_t (&v)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(at));
}
__device__ __forceinline__ void sts64(uint32_t at, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(x), "r"(y));
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}

__device__ __forceinline__ void prefetch_l1(const void* p) {
  asm volatile("prefetch.global.L1 [%0];" ::"l"(p));
}

// Bulk copy of n bytes (a multiple of 16, both sides 16-byte aligned).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t n, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(n), "r"(smem_u32(bar))
      : "memory");
}

// mbar_wait of a whole warp: lanes may see the time run out apart, and what
// follows needs all of them.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

struct Lengths {
  const int32_t* data;
  int64_t most;  // tokens the table can name
  uint32_t batch, unit, idle;
  __device__ __forceinline__ int of(uint32_t b) const {
    return (int)max64(0, min64(data[b], most));
  }
  // Units of `unit` tokens, and before them `idle` without tokens: what
  // beginning and ending a sequence's head costs.
  __device__ __forceinline__ uint32_t units(int len) const {
    return idle + ((uint32_t)len + unit - 1) / unit;
  }
};

// Dealing the tokens' units alone leaves CTAs with many short sequences behind.
// 16 sequences of 1 .. 2048 tokens, a head a group: 40 us with two idle units, 43
// with four; 48 of 1 .. 8192, eight heads a group: 89 with two, 81 with four.
inline uint32_t idle_units(uint32_t group) { return 2 + std::min(group, 16u) / 4; }

// The units in order: sequences, in them rows (a key/value head's block of
// query heads), in them tokens.  before(b): the units of a row of the
// sequences before b.
struct Deal {
  unsigned long long before;  // of sequence b
  uint32_t b, n;              // that sequence, its units
  unsigned long long total;   // of a row of all sequences
};

// The sequence that holds unit `u(total)` of all rows, found by the whole CTA
// of kThreads.
template <int kThreads, typename U>
__device__ __forceinline__ Deal find_unit(const Lengths& lengths, uint32_t rows, U&& u) {
  constexpr int kParts = kThreads / 32;
  __shared__ unsigned long long sums[kParts], found_before, total;
  __shared__ uint32_t found_b, found_n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned long long mine = 0;
  for (uint32_t b = threadIdx.x; b < lengths.batch; b += kThreads)
    mine += lengths.units(lengths.of(b));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if (lane == 0) sums[warp] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long t = 0;
    for (int w = 0; w < kParts; ++w) t += sums[w];
    total = t;
    found_b = lengths.batch;
  }
  __syncthreads();
  const unsigned long long at = u(total);
  unsigned long long done = 0;
  for (uint32_t b0 = 0; b0 < lengths.batch; b0 += kThreads) {
    const uint32_t b = b0 + threadIdx.x;
    const uint32_t n = b < lengths.batch ? lengths.units(lengths.of(b)) : 0;
    unsigned long long upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += x;
    }
    __syncthreads();  // sums of the last round are read
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    unsigned long long all = 0;
    for (int w = 0; w < kParts; ++w) {
      if (w == warp) upto += all;
      all += sums[w];
    }
    const unsigned long long before = done + upto - n;
    if (n > 0 && at >= before * rows && at < (before + n) * rows) {
      found_b = b;
      found_n = n;
      found_before = before;
    }
    done += all;
  }
  __syncthreads();
  return Deal{found_before, found_b, found_n, total};
}

// A run of a CTA's units inside one row of one sequence.
struct Segment {
  uint32_t b, row, c0, c1;  // sequence, row, units c0 .. c1 - 1
  uint32_t n;               // units of the sequence
  uint32_t idle;
  int len;
  // those with tokens
  __device__ __forceinline__ uint32_t first() const { return max(c0, idle) - idle; }
  __device__ __forceinline__ uint32_t last() const { return max(c1, idle) - idle; }
};

// A CTA's segments in turn.
struct Segments {
  const Lengths* lengths;
  uint32_t rows;
  unsigned long long left;  // units
  Segment s;

  __device__ __forceinline__ void begin(const Lengths* all, uint32_t rows_, const Deal& d,
                                        unsigned long long u0, unsigned long long u1) {
    lengths = all;
    rows = rows_;
    s.idle = all->idle;
    left = u1 - u0;
    if (left == 0) return;
    const unsigned long long in = u0 - d.before * rows;
    s.b = d.b;
    s.n = d.n;
    s.row = (uint32_t)(in / d.n);
    s.c0 = (uint32_t)(in - (unsigned long long)s.row * d.n);
    s.len = lengths->of(s.b);
    s.c1 = (uint32_t)min((unsigned long long)s.n, s.c0 + left);
  }
  __device__ __forceinline__ bool more() const { return left > 0; }
  __device__ __forceinline__ void next() {
    left -= s.c1 - s.c0;
    if (left == 0) return;
    if (++s.row == rows) {
      s.row = 0;
      ++s.b;
      s.len = lengths->of(s.b);
      s.n = lengths->units(s.len);
    }
    s.c0 = 0;
    s.c1 = (uint32_t)min((unsigned long long)s.n, left);
  }
};

// No more CTAs share the units than there are, so that none between two others
// has nothing; first unit of CTA i's share.
__device__ __forceinline__ unsigned long long shares_used(unsigned long long units,
                                                          uint32_t shares) {
  return units < shares ? units : shares;
}
__device__ __forceinline__ unsigned long long share_begin(unsigned long long i,
                                                          unsigned long long units,
                                                          unsigned long long used) {
  return i * units / used;
}

struct Heads {
  uint32_t all, group, blocks;  // of q; of a key/value head; blocks of a group
};

// shares: CTAs the units are dealt to (then gridDim.x = shares and `parts` has
// two places a CTA: [8 kTiles heads][head_dim] outputs, behind all of them
// (maximum, sum) pairs), or 0: CTA i takes row i % rows of sequence i / rows.
template <int BITS, int kQuarters, int kTiles>
__global__ void
__launch_bounds__(Layout<BITS, kQuarters>::kThreads, (Layout<BITS, kQuarters>::ctas(kTiles)))
    cache_attention_kernel(const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map, CacheView c,
                           uint32_t box_rows, Query q, Heads heads,
                           const int32_t* __restrict__ table, int64_t table_stride,
                           const __grid_constant__ Lengths lengths, float scale, uint32_t shares,
                           float* __restrict__ parts, void* __restrict__ out) {
  using L = Layout<BITS, kQuarters>;
  constexpr int kHeads = 8 * kTiles;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                             ~(uintptr_t)1023);
  float* join = reinterpret_cast<float*>(ring + L::kRing);
  __shared__ float sm[L::kWarps][8], sl[L::kWarps][8];
  __shared__ uint64_t full[L::kStages], empty[L::kStages];
  __shared__ int tokens[L::kStages][L::kWarps];  // of a warp's 16 that there are
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const uint32_t rows = c.heads * heads.blocks;
  const uint32_t token_scales = L::scale_bytes(c.dim);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], L::kWarps);
    }
    fence_mbar_init();
  }
  // in this order: the joining kernel reads the lengths before it waits
  grid_dependency_wait();
  grid_launch_dependents();
  Segments run;
  if (shares > 0) {
    unsigned long long u0 = 0, u1 = 0;
    const Deal d = find_unit<L::kThreads>(
        lengths, rows, [&](unsigned long long total) {
          const unsigned long long units = total * rows, n = shares_used(units, shares);
          if (blockIdx.x < n) {
            u0 = share_begin(blockIdx.x, units, n);
            u1 = share_begin(blockIdx.x + 1, units, n);
          }
          return u0;
        });
    run.begin(&lengths, rows, d, u0, u1);
  } else {
    const uint32_t b = blockIdx.x / rows;
    const Deal d{0, b, lengths.units(lengths.of(b)), 0};
    const unsigned long long u0 = (unsigned long long)(blockIdx.x - b * rows) * d.n;
    run.begin(&lengths, rows, d, u0, u0 + d.n);
  }
  __syncthreads();

  if (warp == L::kWarps) {
    // ---- the warp that fetches: lane x the x-th box of a unit
    const uint32_t boxes = L::kUnit / box_rows, mine = lane * box_rows;
    const bool holds = lane < (int)boxes;
    int stage = 0, issued = 0;
    uint32_t phase = 1;
    bool ok = true;
    // the page of this lane's box of a unit, read a unit ahead
    const auto page_of = [&](const Segment& s, uint32_t u) -> int32_t {
      const uint32_t t = u * L::kUnit + mine;
      return holds && t < (uint32_t)s.len
                 ? table[(int64_t)s.b * table_stride + t / c.page_size]
                 : -1;
    };
    const auto first_page = [&]() -> int32_t {
      return run.more() && run.s.first() < run.s.last() ? page_of(run.s, run.s.first()) : -1;
    };
    int32_t next_page = first_page();
    while (run.more() && ok) {
      const Segment s = run.s;
      const uint32_t kvh = s.row / heads.blocks;
      run.next();
      if (run.more()) {  // the next row's query, which the other warps want at its begin
        const uint32_t next = run.s.row / heads.blocks, lines = (2 * c.dim + 127) / 128;
        const uint32_t from = (run.s.row - next * heads.blocks) * kHeads;
        for (uint32_t x = lane; x < kHeads * lines; x += 32)
          if (from + x / lines < heads.group)
            prefetch_l1(static_cast<const uint8_t*>(q.data) +
                        2 * ((int64_t)run.s.b * q.batch_stride +
                             (int64_t)(next * heads.group + from + x / lines) * q.head_stride) +
                        128 * (x % lines));
      }
      // nothing to fetch (idle units, a sequence without tokens): the page read
      // ahead is that of the segment behind it
      if (s.first() >= s.last()) next_page = first_page();
      for (uint32_t u = s.first(); u < s.last(); ++u) {
        const uint32_t t = u * L::kUnit + mine;
        const uint32_t p = t / c.page_size;
        const int32_t page = next_page;
        next_page = u + 1 < s.last() ? page_of(s, u + 1) : first_page();
        const bool there = page >= 0 && page < c.pages;
        if (!warp_wait(&empty[stage], phase)) {
          ok = false;
          break;
        }
        const uint32_t lanes = __ballot_sync(0xffffffffu, there);
        if (holds)
          for (uint32_t x = 0; x < box_rows / kBlock; ++x)
            tokens[stage][lane * (box_rows / kBlock) + x] =
                there ? min(kBlock, max(0, s.len - (int)(t + x * kBlock))) : 0;
        __syncwarp();
        if (lane == 0)
          mbar_arrive_expect_tx(&full[stage],
                                __popc(lanes) * 2 * box_rows * (L::kRow + token_scales));
        __syncwarp();
        if (there) {
          const int64_t row =
              ((int64_t)page * c.heads + kvh) * c.page_size + (t - p * c.page_size);
          uint8_t* at = ring + stage * L::kStage + mine * L::kBoxRow;
          uint8_t* sc = ring + stage * L::kStage + 2 * L::kCodes + mine * token_scales;
#pragma unroll
          for (int x = 0; x < L::kBoxes; ++x) {
            tma_load_2d(at + x * L::kColumn, &k_map, &full[stage], x * L::kBoxRow, (int)row);
            tma_load_2d(at + L::kCodes + x * L::kColumn, &v_map, &full[stage], x * L::kBoxRow,
                        (int)row);
          }
          const int64_t first = row * token_scales;
          bulk_load(sc, c.scales[0] + first, box_rows * token_scales, &full[stage]);
          bulk_load(sc + L::kScales, c.scales[1] + first, box_rows * token_scales, &full[stage]);
        }
        ++issued;
        if (++stage == L::kStages) stage = 0, phase ^= 1u;
      }
    }
    // a reader that gave up leaves: not before the copies are in
    for (int x = max(0, issued - L::kStages); x < issued; ++x)
      mbar_wait(&full[x % L::kStages], (uint32_t)((x / L::kStages) & 1));
    return;
  }

  // ---- the warps that compute
  // Tokens (of the warp's 16): token_of(g) and 8 further at S^T's rows,
  // token_of(2 j), token_of(2 j + 1) and 8 further at O^T's columns.  Eight rows
  // further on is a fixed distance: the swizzle repeats.
  const int row0 = token_of(g), column[2] = {token_of(2 * j), token_of(2 * j + 1)};
  const uint32_t ring0 = smem_u32(ring);
  constexpr uint32_t kEight = 8 * L::kBoxRow;
  uint32_t key_at[2], value_at[2];  // in a stage: steps 0 and 1 (2 and 3: a box column on)
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    // 4 bits: lane 8 i + r names row r of the i-th of four 8 x 16-byte matrices
    key_at[x] = ring0 + (BITS == 8
                             ? L::at(16 * warp + row0, L::key_byte(L::kSteps > 1 ? x : 0, j))
                             : L::at(16 * warp + token_of(lane & 7) + (lane & 8), lane & 16));
    // past the row (64-channel rows have 4 lanes' pieces): any, not stored
    const uint32_t byte = (kQuarters == 1 ? g & 3 : g) * 2 * BITS;
    value_at[x] = ring0 + L::kCodes + L::at(16 * warp + column[x], byte);
  }
  const int last_group = (int)c.dim / kGroup4 - 1;
  const uint32_t eight_scales = 8 * token_scales;
  const uint32_t key_scale = ring0 + 2 * L::kCodes + (16 * warp + row0) * token_scales;
  const uint32_t value_scale[2] = {
      ring0 + 2 * L::kCodes + L::kScales + (16 * warp + column[0]) * token_scales,
      ring0 + 2 * L::kCodes + L::kScales + (16 * warp + column[1]) * token_scales};
  uint32_t stage_at = 0;  // bytes
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  constexpr int kHeld = L::parts_in_smem(kTiles);
  // of part x (1 middle, 2 lower), tile n and product i
  const auto held_at = [&](int x, int n, int i) {
    return ring0 + L::kRing + L::kJoin +
           8 * (((warp * kHeld + 2 - x) * kTiles + n) * L::kProducts + i) * 32 + 8 * lane;
  };
  const bool fine = !q.bf16;  // an fp16 output: what fp16 drops of the probabilities too
  for (uint32_t place = 0; run.more(); run.next(), place = 1) {
    const Segment& seg = run.s;
    const uint32_t kvh = seg.row / heads.blocks, h0 = (seg.row - kvh * heads.blocks) * kHeads;

    // Q in the order of the keys' registers, below 1 by a power of two a head
    // 8 bits: qf[0] the upper part, qf[1] the middle, qf[2] the lower
    uint32_t qf[BITS == 8 ? 3 - kHeld : 1][kTiles][L::kProducts][2];
    // 4 bits: the query's sum over group j (and j + 4) in two parts, 22 bits
    [[maybe_unused]] uint32_t qs[kTiles][(L::kGroups + 3) / 4];
    float factor[kTiles][2];  // of heads 2 j, 2 j + 1: scale log2(e) and that power
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const uint32_t h = h0 + 8 * n + g;
      const bool live = h < heads.group;
      const int64_t at = (int64_t)seg.b * q.batch_stride +
                         (int64_t)(kvh * heads.group + (live ? h : 0)) * q.head_stride;
      float x[L::kPieces][8] = {};
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < L::kPieces; ++s) {
        const uint32_t ch = L::piece_channel(s, j);
        if (live && ch < c.dim) {
          if (q.bf16)
            load8(static_cast<const __nv_bfloat16*>(q.data) + at + ch, q.vec, x[s]);
          else
            load8(static_cast<const __half*>(q.data) + at + ch, q.vec, x[s]);
        }
        top = max(top, abs_bits_max(x[s]));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // down = 2^-p with 2^(p - 1) <= max < 2^p (subnormal for the largest two
      // exponents), up = 2^(p - 8); a query below 2^-118 is taken relative to
      // that; NaN where it is not finite
      const uint32_t ex = min(max(top >> 23, 8u), 254u);
      const float down = __uint_as_float(ex <= 252 ? (253 - ex) << 23 : 0x00800000u >> (ex - 252));
      const float up = __uint_as_float(top >= 0x7F800000u ? 0x7FC00000u : (ex - 7) << 23);
      if constexpr (BITS == 8) {
#pragma unroll
        for (int s = 0; s < L::kSteps; ++s) {
          // q 2^22 = 65536 upper + 256 middle + lower, all signed bytes: those of
          // v = q 2^22 + 128 (256 + 1), the lower two less 128
          uint32_t part[3][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = __float_as_uint(fmaf(x[2 * s + i / 2][4 * (i & 1) + e] * down, 0x1p22f,
                                          kRoundMagic)) -
                     (uint32_t)kSumBits + 0x8080u;
            const uint32_t a = __byte_perm(v[0], v[1], 0x5140), b = __byte_perm(v[2], v[3], 0x5140);
            part[0][i] = __byte_perm(__byte_perm(v[0], v[1], 0x0062),
                                     __byte_perm(v[2], v[3], 0x0062), 0x5410);
            part[1][i] = __byte_perm(a, b, 0x7632) ^ 0x80808080u;
            part[2][i] = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int y = 0; y < 3; ++y) {
              if (y < 3 - kHeld) {
                qf[y < 3 - kHeld ? y : 0][n][2 * s + i][0] = part[y][2 * i];
                qf[y < 3 - kHeld ? y : 0][n][2 * s + i][1] = part[y][2 * i + 1];
              } else {
                sts64(held_at(y, n, 2 * s + i), part[y][2 * i], part[y][2 * i + 1]);
              }
            }
        }
      } else {
#pragma unroll
        for (int s = 0; s < L::kGroups; ++s) {
          // channels as the codes' pairs have them, to below 2^15 (2^11: codes times 16)
          float sum = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[s][i] *= down;
            sum += x[s][i];
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t(&f)[2] = qf[0][n][2 * s + i];
            f[0] = h2_bits(__floats2half2_rn(x[s][2 * i] * 0x1p15f, x[s][2 * i + 4] * 0x1p15f));
            f[1] = h2_bits(__floats2half2_rn(x[s][2 * i + 1] * 0x1p11f, x[s][2 * i + 5] * 0x1p11f));
          }
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (s % 4 == 0) qs[n][s / 4] = 0u;
          if (j == s % 4) {
            const __half high = __float2half_rn(sum * 0x1p9f);
            qs[n][s / 4] = h2_bits(__halves2half2(
                high, __float2half_rn(fmaf(sum, 0x1p9f, -__half2float(high)))));
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        // (finite, so that a sum of 0 stays 0; NaN stays NaN)
        const float y = __shfl_sync(0xffffffffu, up, 4 * (2 * j + r)) *
                        (BITS == 8 ? 0x1p-14f : 1.0f) * (scale * kLog2e) *
                        (BITS == 8 ? 1.0f : 0x1p17f);
        factor[n][r] = isinf(y) ? copysignf(-kLowest, y) : y;
      }
    }

    // o[n][p][i]: channels 16 (g + 8 p) + 2 i, + 1 of heads 2 j, 2 j + 1
    float o[kTiles][L::kPasses][8][4] = {};
    float m[kTiles][2], l[kTiles][2] = {};
#pragma unroll
    for (int n = 0; n < kTiles; ++n) m[n][0] = m[n][1] = kLowest;

#pragma unroll 1
    for (uint32_t u = seg.first(); u < seg.last(); ++u) {
      if (!ok || !warp_wait(&full[stage], phase)) {  // ran out: NaN from here on
        ok = false;
        break;
      }
      const int seen = tokens[stage][warp];
      const bool whole = seen == kBlock;

      if (seen > 0) {
        // the values of a pass: those of the first are on the way during S^T
        constexpr int kWords = BITS / 2;
        uint32_t vw[4][kWords];
        uint32_t gr[4];
        const auto load_values = [&](int p) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if constexpr (BITS == 8) {
              const uint4 v =
                  lds128(value_at[r & 1] + stage_at + p * L::kColumn + (r >> 1) * kEight);
              vw[r][0] = v.x; vw[r][1] = v.y; vw[r][2] = v.z; vw[r][3] = v.w;
            } else {
              // the second pass is the row's other half: chunks 4 .. 7
              const uint2 v = lds64((value_at[r & 1] ^ (p * 64)) + stage_at + (r >> 1) * kEight);
              vw[r][0] = v.x; vw[r][1] = v.y;
              gr[r] = lds32(value_scale[r & 1] + stage_at + 4 * min((g + 8 * p) / 2, last_group) +
                            (r >> 1) * eight_scales);
            }
          }
        };
        if constexpr (BITS == 4) load_values(0);

        // ---- S^T = K Q^T
        float s[kTiles][4] = {};
        if constexpr (BITS == 8) {
          int sums[3][kTiles][4];  // with the upper, middle and lower part
#pragma unroll
          for (int y = 0; y < 3; ++y)
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) sums[y][n][e] = kSumBits;
#pragma unroll
          for (int st = 0; st < L::kSteps; ++st) {
            uint4 kw[2];
#pragma unroll
            for (int r = 0; r < 2; ++r)
              kw[r] = lds128(key_at[st % 2] + stage_at + st / 2 * L::kColumn + r * kEight);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t a0 = i ? kw[0].z : kw[0].x, a1 = i ? kw[1].z : kw[1].x;
                const uint32_t a2 = i ? kw[0].w : kw[0].y, a3 = i ? kw[1].w : kw[1].y;
#pragma unroll
                for (int y = 0; y < 3; ++y) {
                  uint2 f;
                  if (y < 3 - kHeld)
                    f = make_uint2(qf[y < 3 - kHeld ? y : 0][n][2 * st + i][0],
                                   qf[y < 3 - kHeld ? y : 0][n][2 * st + i][1]);
                  else
                    f = lds64(held_at(y, n, 2 * st + i));
                  mma_s8(sums[y][n], a0, a1, a2, a3, f.x, f.y);
                }
              }
            }
          }
          const float ks[2] = {__uint_as_float(lds32(key_scale + stage_at)),
                               __uint_as_float(lds32(key_scale + stage_at + 32))};
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[n][e] = fmaf(whole_sum(sums[0][n][e]), 65536.0f,
                             fmaf(whole_sum(sums[1][n][e]), 256.0f, whole_sum(sums[2][n][e]))) *
                        ks[e >> 1];
        } else {
          // sum of q k = sum over the groups of s (sum of q code) + m (sum of q): the
          // second is a product of its own, over groups, with both parts of a sum
          uint64_t both[kTiles][2];  // heads 2 j, 2 j + 1 of a token
          {
            float low[kTiles][4] = {};
#pragma unroll
            for (int i = 0; i < L::kGroups; i += 4) {
              uint32_t gm[2];
#pragma unroll
              for (int r = 0; r < 2; ++r)
                // past head_dim the query is 0 (any group's minimum will do)
                gm[r] = h2_bits(__high2half2(
                    bits_h2(lds32(key_scale + stage_at + r * eight_scales +
                                  4 * min(i + j, last_group)))));
#pragma unroll
              for (int n = 0; n < kTiles; ++n) mma_f16_k8(low[n], gm[0], gm[1], qs[n][i / 4]);
            }
            const uint64_t to = f2_pack(0x1p-18f, 0x1p-18f);  // 2^6 less the codes' 2^24
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                both[n][r] = f2_mul(f2_pack(low[n][2 * r], low[n][2 * r + 1]), to);
          }
#pragma unroll
          for (int i = 0; i < L::kGroups; i += 2) {
            uint32_t kw[4];
            ldmatrix4(kw, (key_at[0] ^ (16 * i)) + stage_at);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint64_t gs[2];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float x = __low2float(
                    bits_h2(lds32(key_scale + stage_at + r * eight_scales +
                                  4 * min(i + h, last_group))));
                gs[r] = f2_pack(x, x);
              }
              const uint32_t w0 = kw[2 * h], w1 = kw[2 * h + 1];
              float sum[kTiles][4] = {};
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const uint32_t a0 = w0 >> (8 * x) & 0x000F000Fu, a1 = w1 >> (8 * x) & 0x000F000Fu;
                const uint32_t a2 = w0 >> (8 * x) & 0x00F000F0u, a3 = w1 >> (8 * x) & 0x00F000F0u;
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                  const uint32_t(&f)[2] = qf[0][n][2 * (i + h) + x];
                  mma_f16(sum[n], a0, a1, a2, a3, f[0], f[1]);
                }
              }
#pragma unroll
              for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                  both[n][r] = f2_fma(gs[r], f2_pack(sum[n][2 * r], sum[n][2 * r + 1]),
                                      both[n][r]);
            }
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) f2_unpack(both[n][r], s[n][2 * r], s[n][2 * r + 1]);
        }

        // ---- scores in powers of two; weights, and what they are relative to
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[n][e] *= factor[n][e & 1];
          }
        if (!whole) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (row0 + 8 * (e >> 1) >= seen) s[n][e] = -INFINITY;
        }
        float vs[2] = {1.0f, 1.0f};
        if constexpr (BITS == 8) {
          vs[0] = __uint_as_float(lds32(key_scale + stage_at + L::kScales));
          vs[1] = __uint_as_float(lds32(key_scale + stage_at + L::kScales + 32));
          if (!whole) {  // what lies behind the sequence's end is not used
            if (row0 >= seen) vs[0] = 0.0f;
            if (row0 + 8 >= seen) vs[1] = 0.0f;
          }
        }
        float p[kTiles][4], w[kTiles][4];
        const auto weigh = [&](int n, int e) {
          p[n][e] = exp2_fast(s[n][e] - m[n][e & 1]);
          w[n][e] = BITS == 8 ? p[n][e] * vs[e >> 1] : p[n][e];
        };
        float most = 0.0f, most_p = 0.0f;  // (a NaN is in neither)
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            weigh(n, e);
            most = fmaxf(most, w[n][e]);
            if constexpr (BITS == 8) most_p = fmaxf(most_p, p[n][e]);
          }
        if (__any_sync(0xffffffffu, most > (float)(1 << kMost) || most_p > kMostP)) {
          // how far below a score its weight's reference lies
          float below[2] = {(float)kAim, (float)kAim};
          if constexpr (BITS == 8) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const uint32_t x = __float_as_uint(vs[t]) & 0x7FFFFFFFu;
              // (a scale that is not finite has no say)
              const int e = x < 0x7F800000u ? (int)(x >> 23) - 127 : kLeastScale;
              below[t] -= (float)max(e, kLeastScale);
            }
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            float f[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float top = fmaxf(s[n][r] - below[0], s[n][r + 2] - below[1]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              top = fmaxf(top, m[n][r]);
              f[r] = exp2_fast(m[n][r] - top);
              l[n][r] *= f[r];
              m[n][r] = top;
              weigh(n, r);
              weigh(n, r + 2);
            }
#pragma unroll
            for (int t = 0; t < L::kPasses; ++t)
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][t][i][e] *= f[e & 1];
          }
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) l[n][e & 1] += p[n][e];
        uint32_t pt[kTiles][2], low[kTiles][2] = {};
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const __half2 high = __floats2half2_rn(w[n][2 * r], w[n][2 * r + 1]);
            pt[n][r] = transpose8x8(h2_bits(high));
            if (fine) {
              const float2 back = __half22float2(high);
              low[n][r] = transpose8x8(
                  h2_bits(__floats2half2_rn(w[n][2 * r] - back.x, w[n][2 * r + 1] - back.y)));
            }
          }
        }

        // ---- O^T += V^T P^T
#pragma unroll
        for (int p = 0; p < L::kPasses; ++p) {
          if (BITS == 8 || p > 0) load_values(p);
          if constexpr (BITS == 4) {
            if (!whole) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (column[r & 1] + 8 * (r >> 1) >= seen) gr[r] = 0u;
            }
          }
          if constexpr (BITS == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t w0 = vw[0][i] ^ 0x80808080u, w1 = vw[1][i] ^ 0x80808080u;
              const uint32_t w2 = vw[2][i] ^ 0x80808080u, w3 = vw[3][i] ^ 0x80808080u;
#pragma unroll
              for (int h = 0; h < 2; ++h) {  // channels 4 i + 2 h, + 1
                const uint32_t x = __byte_perm(w0, w1, h ? 0x7362 : 0x5140);
                const uint32_t y = __byte_perm(w2, w3, h ? 0x7362 : 0x5140);
                const uint32_t a0 = code8_pair(x, 0x4140), a1 = code8_pair(x, 0x4342);
                const uint32_t a2 = code8_pair(y, 0x4140), a3 = code8_pair(y, 0x4342);
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                  mma_f16(o[n][p][2 * i + h], a0, a1, a2, a3, pt[n][0], pt[n][1]);
                  if (fine) mma_f16(o[n][p][2 * i + h], a0, a1, a2, a3, low[n][0], low[n][1]);
                }
              }
            }
          } else {
            const __half2 s01 = bits_h2(__byte_perm(gr[0], gr[1], 0x5410));
            const __half2 m01 = bits_h2(__byte_perm(gr[0], gr[1], 0x7632));
            const __half2 s23 = bits_h2(__byte_perm(gr[2], gr[3], 0x5410));
            const __half2 m23 = bits_h2(__byte_perm(gr[2], gr[3], 0x7632));
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int h = 0; h < 4; ++h) {  // channels 8 i + 2 h, + 1
                const uint32_t sel = h < 2 ? 0x5410 : 0x7632;
                const uint32_t x = __byte_perm(vw[0][i], vw[1][i], sel) >> (8 * (h & 1));
                const uint32_t y = __byte_perm(vw[2][i], vw[3][i], sel) >> (8 * (h & 1));
                const uint32_t a0 = code4_pair<false>(x, s01, m01);
                const uint32_t a1 = code4_pair<true>(x, s01, m01);
                const uint32_t a2 = code4_pair<false>(y, s23, m23);
                const uint32_t a3 = code4_pair<true>(y, s23, m23);
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                  mma_f16(o[n][p][4 * i + h], a0, a1, a2, a3, pt[n][0], pt[n][1]);
                  if (fine) mma_f16(o[n][p][4 * i + h], a0, a1, a2, a3, low[n][0], low[n][1]);
                }
              }
          }
        }
      }

      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      stage_at += L::kStage;
      if (++stage == L::kStages) stage = 0, stage_at = 0, phase ^= 1u;
    }

    // ---- the warps' parts joined, 8 heads at a time
    const bool part = seg.c1 - seg.c0 != seg.n;
    const uint32_t slot = 2 * blockIdx.x + place;
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const uint32_t first = h0 + 8 * n;
      const uint32_t here = first < heads.group ? min(8u, heads.group - first) : 0u;
      if (here == 0) break;
      // the outputs joined before are read
      asm volatile("bar.sync 1, %0;" ::"n"(32 * L::kWarps) : "memory");
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float sum = ok ? l[n][r] : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const uint32_t h = 2 * j + r;
        if (g == 0) sm[warp][h] = m[n][r], sl[warp][h] = sum;
        if (h < here) {
          float* to = join + (warp * 8 + j + 4 * r) * L::kJoinRow;
#pragma unroll
          for (int p = 0; p < L::kPasses; ++p) {
            const uint32_t ch = 16 * (g + 8 * p);
            if (ch < 64 * kQuarters)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                to[ch + ch / 32 * 4 + 2 * i] = o[n][p][i][r];
                to[ch + ch / 32 * 4 + 2 * i + 1] = o[n][p][i][r + 2];
              }
          }
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(32 * L::kWarps) : "memory");
      // a warp a head; with fewer heads several, taking turns at 32 channels
      const uint32_t turns = max(1u, (uint32_t)L::kWarps / here);
      for (uint32_t x = warp; x < here * turns; x += L::kWarps) {
        const uint32_t h = x % here;
        const float* from = join + ((h >> 1) + 4 * (h & 1)) * L::kJoinRow;
        float top = kLowest, sum = 0.0f, f[L::kWarps];
#pragma unroll
        for (int w = 0; w < L::kWarps; ++w) f[w] = sm[w][h];
#pragma unroll
        for (int w = 0; w < L::kWarps; ++w) top = fmaxf(top, f[w]);
#pragma unroll
        for (int w = 0; w < L::kWarps; ++w) {
          f[w] = exp2_fast(f[w] - top);
          sum = fmaf(sl[w][h], f[w], sum);
        }
        const uint32_t at = slot * kHeads + 8 * n + h;
        const uint64_t head = (uint64_t)seg.b * heads.all + kvh * heads.group + first + h;
        const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (uint32_t ch = x / here * 32 + lane; ch < c.dim; ch += turns * 32) {
          float y = 0.0f;
#pragma unroll
          for (int w = 0; w < L::kWarps; ++w)
            y = fmaf(from[w * 8 * L::kJoinRow + ch + ch / 32 * 4], f[w], y);
          if (part)
            parts[(uint64_t)at * c.dim + ch] = y;
          else
            store_out(out, q.bf16, head * c.dim + ch, y * by);
        }
        if (part && x < here && lane == 0)
          reinterpret_cast<float2*>(parts + (uint64_t)2 * shares * kHeads * c.dim)[at] =
              make_float2(top, sum);
      }
    }
  }
}

// What the join kernels work on: the parts of a row of a sequence, those of
// CTAs i0 .. i1.
constexpr int kJoinWarps = 8;
struct Join {
  const float* parts;
  uint32_t shares, part_heads, kv_heads;
  Heads heads;
  uint32_t dim;
  Lengths lengths;
  bool bf16;
  void* out;
};
struct Row {
  uint32_t i0, i1, second, kvh, h0, b;
  // a CTA's first part, or its second where it begins before this row
  __device__ __forceinline__ uint32_t slot(uint32_t i, uint32_t part_heads) const {
    return (2 * i + (i == i0 ? second : 0u)) * part_heads;
  }
};
// Of this CTA's row (blockIdx.x); i0 == i1: one CTA took it and wrote its output.
__device__ __forceinline__ Row find_row(const Join& a) {
  __shared__ unsigned long long counts[2][kJoinWarps];
  const uint32_t rows = a.kv_heads * a.heads.blocks;
  Row r;
  r.b = blockIdx.x / rows;
  const uint32_t row = blockIdx.x - r.b * rows;
  r.kvh = row / a.heads.blocks;
  r.h0 = (row - r.kvh * a.heads.blocks) * a.part_heads;
  // units of a row before this sequence, and of all
  unsigned long long before = 0, total = 0;
  for (uint32_t i = threadIdx.x; i < a.lengths.batch; i += 32 * kJoinWarps) {
    const uint32_t x = a.lengths.units(a.lengths.of(i));
    total += x;
    if (i < r.b) before += x;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, d);
    total += __shfl_xor_sync(0xffffffffu, total, d);
  }
  const uint32_t warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) counts[0][warp] = before, counts[1][warp] = total;
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) before += counts[0][w], total += counts[1][w];
  const uint32_t n = a.lengths.units(a.lengths.of(r.b));
  const unsigned long long units = total * rows, used = shares_used(units, a.shares);
  const unsigned long long s0 = before * rows + (unsigned long long)row * n, s1 = s0 + n - 1;
  r.i0 = (uint32_t)(((s0 + 1) * used - 1) / units);
  r.i1 = (uint32_t)(((s1 + 1) * used - 1) / units);
  r.second = share_begin(r.i0, units, used) < s0 ? 1u : 0u;
  return r;
}

// Few parts a row: a CTA a row, a thread four channels of a head at a time.
__global__ void __launch_bounds__(32 * kJoinWarps)
    cache_attention_join_rows_kernel(const __grid_constant__ Join a) {
  const Row r = find_row(a);
  grid_dependency_wait();  // by CTAs without work too: their end is the call's
  if (r.i0 == r.i1) return;
  const uint32_t here = min(a.part_heads, a.heads.group - r.h0);
  const float2* ml =
      reinterpret_cast<const float2*>(a.parts + (uint64_t)2 * a.shares * a.part_heads * a.dim);
  for (uint32_t x = threadIdx.x; x < here * a.dim / 4; x += 32 * kJoinWarps) {
    const uint32_t h = 4 * x / a.dim, ch = 4 * x - h * a.dim;
    float top = kLowest, sum = 0.0f;
#pragma unroll 4
    for (uint32_t i = r.i0; i <= r.i1; ++i)
      top = fmaxf(top, ml[r.slot(i, a.part_heads) + h].x);
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (uint32_t i = r.i0; i <= r.i1; ++i) {
      const uint32_t at = r.slot(i, a.part_heads) + h;
      const float2 m = ml[at];
      const float4 v = *reinterpret_cast<const float4*>(a.parts + (uint64_t)at * a.dim + ch);
      const float f = exp2_fast(m.x - top);
      sum = fmaf(m.y, f, sum);
      y.x = fmaf(v.x, f, y.x);
      y.y = fmaf(v.y, f, y.y);
      y.z = fmaf(v.z, f, y.z);
      y.w = fmaf(v.w, f, y.w);
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t at =
        ((uint64_t)r.b * a.heads.all + r.kvh * a.heads.group + r.h0 + h) * a.dim + ch;
    store_out(a.out, a.bf16, at, y.x * by);
    store_out(a.out, a.bf16, at + 1, y.y * by);
    store_out(a.out, a.bf16, at + 2, y.z * by);
    store_out(a.out, a.bf16, at + 3, y.w * by);
  }
}

// Many: a CTA a head of a row, each of its warps every eighth part; then the
// warps' sums in order.
__global__ void __launch_bounds__(32 * kJoinWarps)
    cache_attention_join_heads_kernel(const __grid_constant__ Join a) {
  __shared__ float tops[kJoinWarps], sums[kJoinWarps];
  __shared__ __align__(16) float so[kJoinWarps][256];
  const Row r = find_row(a);
  const uint32_t h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  if (r.i0 == r.i1 || r.h0 + h >= a.heads.group) return;
  const float2* ml =
      reinterpret_cast<const float2*>(a.parts + (uint64_t)2 * a.shares * a.part_heads * a.dim);
  float top = kLowest;
  for (uint32_t i = r.i0 + threadIdx.x; i <= r.i1; i += 32 * kJoinWarps)
    top = fmaxf(top, ml[r.slot(i, a.part_heads) + h].x);
  top = warp_max(top);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, tops[w]);
  float sum = 0.0f;
  float4 y[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
  constexpr int kAtOnce = 8;  // parts a warp has on the way
  for (uint32_t i = r.i0 + warp; i <= r.i1; i += kAtOnce * kJoinWarps) {
    float2 m[kAtOnce];
    float4 v[kAtOnce][2];
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      const uint32_t from = i + e * kJoinWarps;
      const uint32_t at = r.slot(min(from, r.i1), a.part_heads) + h;
      m[e] = ml[at];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        v[e][x] = 4 * (lane + 32 * x) < a.dim
                      ? *reinterpret_cast<const float4*>(a.parts + (uint64_t)at * a.dim +
                                                         4 * (lane + 32 * x))
                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int e = 0; e < kAtOnce; ++e) {
      if (i + e * kJoinWarps > r.i1) break;
      const float f = exp2_fast(m[e].x - top);
      sum = fmaf(m[e].y, f, sum);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        y[x].x = fmaf(v[e][x].x, f, y[x].x);
        y[x].y = fmaf(v[e][x].y, f, y[x].y);
        y[x].z = fmaf(v[e][x].z, f, y[x].z);
        y[x].w = fmaf(v[e][x].w, f, y[x].w);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x)
    *reinterpret_cast<float4*>(&so[warp][4 * (lane + 32 * x)]) = y[x];
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  const uint32_t ch = threadIdx.x;
  if (ch >= a.dim) return;
  float all = 0.0f, z = 0.0f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) all += sums[w], z += so[w][ch];
  const uint64_t head = (uint64_t)r.b * a.heads.all + r.kvh * a.heads.group + r.h0 + h;
  store_out(a.out, a.bf16, head * a.dim + ch, all == 0.0f ? 0.0f : z / all);
}

// Two column tiles (16 heads) where their registers fit (head_dim up to 128),
// else head blocks of 8 that read the codes again.
inline uint32_t head_tiles(uint32_t group, uint32_t dim) { return group > 8 && dim <= 128 ? 2 : 1; }

// Sequences of tables this narrow are taken whole, a CTA a row: nothing to join.
// A row costs its CTA about 1 us for 64 tokens, dealing and joining 4 us; with
// many rows the CTAs have enough to do either way.  Whole and dealt out, 32 rows:
// 256 tokens 7.0 and 8.4 us, 352 8.7 and 9.1, 512 10.4 and 9.1; 128 rows of 512:
// 10.6 and 12.8; 512 rows of 512: 19.3 and 23.4.
constexpr int64_t kWholeTokens = 320, kWholeTokensOfMany = 512, kManyRows = 64;
constexpr int64_t kMostShares = 3 * 148;  // Layout::ctas an SM at most
inline bool whole(int64_t most, int64_t rows) {
  return most <= (rows > kManyRows ? kWholeTokensOfMany : kWholeTokens);
}

// Rows of codes as TMA reads them: [all rows, bytes].
bool rows_map(CUtensorMap* map, const void* codes, const CacheView& c, int bits, uint32_t box_row,
              uint32_t box_rows) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  std::memset(map, 0, sizeof(*map));
  const cuuint64_t bytes = (cuuint64_t)c.dim * bits / 8;
  const cuuint64_t dims[2] = {bytes, (cuuint64_t)(c.pages * c.heads * c.page_size)};
  const cuuint64_t strides[1] = {bytes};
  const cuuint32_t box[2] = {box_row, box_rows};
  const cuuint32_t ones[2] = {1, 1};
  const CUtensorMapSwizzle swizzle = box_row == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : box_row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                     : CU_TENSOR_MAP_SWIZZLE_32B;
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_NONE,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Call {
  CacheView c;
  Query q;
  Heads heads;
  const int32_t* table;
  int64_t table_stride;
  Lengths lengths;
  float scale;
  float* parts;  // null: sequences are taken whole
  void* out;
  cudaStream_t stream;
};

template <int BITS, int kQuarters, int kTiles>
mb_status launch(const Call& a) {
  using L = Layout<BITS, kQuarters>;
  // boxes as tall as units and pages allow
  uint32_t box_rows = L::kUnit;
  while (a.c.page_size % box_rows != 0) box_rows /= 2;
  CUtensorMap k_map, v_map;
  if (!rows_map(&k_map, a.c.codes[0], a.c, BITS, L::kBoxRow, box_rows) ||
      !rows_map(&v_map, a.c.codes[1], a.c, BITS, L::kBoxRow, box_rows))
    return set_error(MB_ERR_CUDA, "cuTensorMapEncodeTiled rejected the cache");
  auto* kernel = cache_attention_kernel<BITS, kQuarters, kTiles>;
  static std::atomic<uint64_t> attr_done{0};
  MB_CUDA_TRY(set_smem_limit_once(kernel, L::smem(kTiles), attr_done));
  const uint32_t rows = a.c.heads * a.heads.blocks;
  Lengths lengths = a.lengths;
  lengths.unit = L::kUnit;
  lengths.idle = idle_units(a.heads.group);
  const uint32_t shares = a.parts == nullptr ? 0 : 148 * L::ctas(kTiles);
  const unsigned grid = shares > 0 ? shares : a.lengths.batch * rows;
  MB_CUDA_TRY(launch_dependent(kernel, grid, L::kThreads, L::smem(kTiles), a.stream, k_map, v_map,
                               a.c, box_rows, a.q, a.heads, a.table, a.table_stride, lengths, a.scale,
                               shares, a.parts, a.out));
  if (shares > 0) {
    dim3 joins(a.lengths.batch * rows);
    const Join join{a.parts, shares,  (uint32_t)(8 * kTiles), a.c.heads, a.heads,
                    a.c.dim, lengths, a.q.bf16,               a.out};
    // Parts a row of eight and more: 1 x 100000 tokens of one key/value head 26 us
    // with the heads' kernel, 114 with the rows'; 48 x 8192 of eight 103 and 80.
    const bool by_heads = shares >= 8 * joins.x;
    if (by_heads) joins.y = std::min<uint32_t>(8 * kTiles, a.heads.group);
    MB_CUDA_TRY(launch_dependent(
        by_heads ? cache_attention_join_heads_kernel : cache_attention_join_rows_kernel, joins,
        32 * kJoinWarps, 0, a.stream, join));
  }
  return MB_OK;
}

template <int BITS>
mb_status dispatch(const Call& a, uint32_t tiles) {
  if (a.c.dim <= 64) return tiles == 2 ? launch<BITS, 1, 2>(a) : launch<BITS, 1, 1>(a);
  if (a.c.dim <= 128) return tiles == 2 ? launch<BITS, 2, 2>(a) : launch<BITS, 2, 1>(a);
  if (a.c.dim <= 192) return launch<BITS, 3, 1>(a);
  return launch<BITS, 4, 1>(a);
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" size_t mb_cache_attention_workspace_size(const mb_kv_cache* cache, int64_t batch,
                                                    int64_t heads, int64_t table_width) {
  if (cache == nullptr || cache->kv_heads <= 0 || cache->page_size <= 0 || batch <= 0 ||
      heads < cache->kv_heads || table_width <= 0)
    return 0;
  const int64_t group = heads / cache->kv_heads;
  const uint32_t tiles = head_tiles((uint32_t)group, (uint32_t)cache->head_dim);
  const int64_t rows = batch * cache->kv_heads * ceil_div(group, 8 * tiles);
  if (whole(table_width * cache->page_size, rows)) return 0;
  return (size_t)(2 * kMostShares * 8 * tiles) * (size_t)(cache->head_dim + 2) * sizeof(float);
}

extern "C" mb_status mb_cache_attention(const mb_kv_cache* cache, const void* q,
                                        int64_t q_batch_stride, int64_t q_head_stride,
                                        mb_dtype type, int64_t batch, int64_t heads,
                                        const int32_t* page_table, int64_t table_stride,
                                        int64_t table_width, const int32_t* lengths, float scale,
                                        void* out, void* workspace, size_t workspace_bytes,
                                        mb_stream_t stream_) {
  clear_error();
  if (const mb_status st = check_cache(cache); st != MB_OK) return st;
  MB_REQUIRE(q && lengths && out && (page_table || table_width == 0),
             "cache_attention pointers must not be null");
  MB_REQUIRE(type == MB_FP16 || type == MB_BF16, "q must be fp16 or bf16");
  MB_REQUIRE(batch > 0 && batch <= 65535, "batch must be 1 to 65535");
  MB_REQUIRE(heads > 0 && heads % cache->kv_heads == 0 && heads <= 65535,
             "heads must be a multiple of kv_heads up to 65535");
  MB_REQUIRE(table_width >= 0, "table_width must not be negative");
  MB_REQUIRE(table_width <= ((int64_t(1) << 31) - 1024) / cache->page_size,
             "table_width too large: positions must fit 31 bits");
  MB_REQUIRE(std::isfinite(scale), "scale must be finite");
  MB_REQUIRE(aligned(q, 2) && aligned(out, 2) && aligned(page_table, 4) && aligned(lengths, 4),
             "misaligned q, out, page_table or lengths");
  const CacheView c = cache_view(cache);
  MB_REQUIRE(c.pages * c.heads * c.page_size < (int64_t(1) << 31),
             "cache too large: pages * kv_heads * page_size must fit 31 bits");
  const int64_t most = table_width * c.page_size;
  const uint32_t group = (uint32_t)(heads / c.heads), tiles = head_tiles(group, c.dim);
  const Heads hs{(uint32_t)heads, group, (uint32_t)ceil_div(group, 8 * tiles)};
  MB_REQUIRE(batch * c.heads * hs.blocks < (int64_t(1) << 31), "too many sequences and heads");
  const size_t need = mb_cache_attention_workspace_size(cache, batch, heads, table_width);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return set_error(MB_ERR_WORKSPACE,
                     "cache_attention workspace missing, misaligned or too small");
  const Call call{c,
                  Query{q, q_batch_stride, q_head_stride, type == MB_BF16,
                        aligned(q, 16) && (batch == 1 || q_batch_stride % 8 == 0) &&
                            (heads == 1 || q_head_stride % 8 == 0)},
                  hs,
                  page_table,
                  table_stride,
                  Lengths{lengths, most, (uint32_t)batch, 0, 0},  // units: launch
                  scale,
                  need > 0 ? static_cast<float*>(workspace) : nullptr,
                  out,
                  reinterpret_cast<cudaStream_t>(stream_)};
  return cache->bits == 8 ? dispatch<8>(call, tiles) : dispatch<4>(call, tiles);
}
