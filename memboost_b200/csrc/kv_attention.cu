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
// Codes and scales reach a warp through a ring of its own in shared memory,
// 16 tokens a stage, filled by TMA: a 16-row box of each code array (rows of
// one page and head are contiguous) and a bulk copy of each scale array, all
// issued by one lane and awaited on one mbarrier.  With a stage of 4.2 KB
// (8 bits, head_dim 128), three stages and 16 warps an SM has up to 200 KB on
// the way; held in registers instead, two thirds of a stage a warp were.
//
// Both products' left operands are read as they lie, because the order of the
// inner index is free: in S^T lane (g, j) = (lane / 4, lane % 4) takes 16 bytes
// of the rows of tokens g and g + 8, in O^T 16 channels of the four tokens of
// its columns; Q's registers follow the keys' channel order.  The boxes' swizzle,
// the 16-byte chunks 2 j + step and the tokens' order (token_of) keep these
// reads free of bank conflicts.  Between the products the probabilities
// change from S^T's layout to the right operand's by a transposing move.
//
// 8-bit codes become exact fp16 integers (1024 + 128 + code by a byte
// permute, minus 1152); the key's scale multiplies the score and the value's
// the probability, relative to a power of two at or above every scale so far,
// so that the product stays in fp16's range.  4-bit codes become
// m + s * code in fp16, one rounding, as cache_read returns them.  The query
// is scaled by a power of two to below 1 (a bf16 value then fits fp16);
// probabilities are rounded to fp16 (2^-11); scores, maxima, sums and the
// accumulators are fp32.
//
// The running maximum is raised only when a score exceeds it by 8 (in powers
// of two): probabilities then stay below 256 and most steps rescale nothing.
//
// Long sequences are split over CTAs in chunks of `chunk` tokens; each leaves
// its maximum, sum and unnormalised output in the workspace, and a second
// kernel joins them in the chunks' order, so the result does not depend on
// the CTAs' timing.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "mb_cache.cuh"
#include "mb_tma.cuh"

namespace mb {
namespace {

constexpr int kWarps = 4;
constexpr int kBlock = 16;  // tokens a warp takes at a time

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
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

// Nibbles 0 and 4 (or, `high`, 1 and 5) of w to m + s * code.
template <bool kHigh>
__device__ __forceinline__ uint32_t code4_pair(uint32_t w, __half2 s, __half2 m) {
  const uint32_t h = (w & (kHigh ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
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

// How rows of a head_dim in (64 (kQuarters - 1), 64 kQuarters] lie in a stage.
template <int BITS, int kQuarters>
struct Layout {
  static constexpr int kRow = kQuarters >= 3 ? (BITS == 8 ? 256 : 128) : kQuarters * 8 * BITS;
  static constexpr int kBoxRow = kRow < 128 ? kRow : 128;  // bytes of a row in one box
  static constexpr int kBoxes = kRow / kBoxRow;
  static constexpr int kBox = kBlock * kBoxRow;
  static constexpr int kCodes = kBlock * kRow;             // of keys, or of values
  static constexpr int kSwizzle = kBoxRow == 128 ? 0x70 : kBoxRow == 64 ? 0x30 : 0x10;
  // bytes of 16 tokens' scales, and what a stage keeps for them
  __host__ __device__ static constexpr uint32_t scale_bytes(uint32_t dim) {
    return kBlock * (BITS == 8 ? 4 : dim / kGroup4 * 4);
  }
  static constexpr int kScales = kBlock * (BITS == 8 ? 4 : 2 * kQuarters * 4);
  static constexpr int kStage = 2 * (kCodes + kScales);

  // S^T: steps of 4 lanes x kKeyWords words; O^T: passes of 8 lanes x 16 channels
  static constexpr int kKeyWords = BITS == 4 && kQuarters == 1 ? 2 : 4;
  static constexpr int kSteps = kRow / (16 * kKeyWords);
  static constexpr int kProducts = kSteps * kKeyWords * (BITS == 8 ? 1 : 2);  // of S^T
  static constexpr int kPasses = (kQuarters + 1) / 2;

  // Place in a stage's keys (or values) of a byte of a row.
  __device__ __forceinline__ static uint32_t at(uint32_t row, uint32_t byte) {
    const uint32_t o = row * kBoxRow + byte % kBoxRow;
    return byte / kBoxRow * kBox + (o ^ ((o >> 3) & kSwizzle));
  }
  // First byte of lane j's part of a key's row in a step.
  __device__ __forceinline__ static uint32_t key_byte(int step, int j) {
    if constexpr (kKeyWords == 2) return 8 * j;
    if constexpr (kSteps == 1) return 16 * j;
    return 128 * (step / 2) + 16 * (2 * j + step % 2);
  }
};

// Token (of 16) at row g of S^T and column k = g of O^T's inner index: pairs
// change places in every other pair of pairs, which spreads a warp's reads of
// the values over the banks.
__device__ __forceinline__ int token_of(int k) { return k ^ ((k >> 1) & 1); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;  // how far a score may exceed the maximum in use

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bulk copy of n bytes (a multiple of 16, both sides 16-byte aligned).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t n, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(n), "r"(smem_u32(bar))
      : "memory");
}

// A warp's walk over its blocks' places in the pages.
struct Walk {
  uint32_t page, place;  // of the next block
  __device__ __forceinline__ void start(uint32_t t, uint32_t page_size) {
    page = t / page_size;
    place = t - page * page_size;
  }
  __device__ __forceinline__ void advance(uint32_t pages, uint32_t rest, uint32_t page_size) {
    page += pages;
    place += rest;
    if (place >= page_size) place -= page_size, ++page;
  }
};

struct Lengths {
  const int32_t* data;
  int64_t most;  // tokens the table can name
  __device__ __forceinline__ int64_t of(int64_t b) const {
    return max64(0, min64(data[b], most));
  }
};

// Grid: (chunks, kv heads x head blocks, batch).  parts: per (sequence, head,
// chunk) head_dim outputs, then all (maximum, sum) pairs; null with one chunk.
template <int BITS, int kQuarters, int kTiles, int kStages>
__global__ void __launch_bounds__(32 * kWarps)
    cache_attention_kernel(const __grid_constant__ CUtensorMap k_map,
                           const __grid_constant__ CUtensorMap v_map, CacheView c, Query q,
                           uint32_t heads, uint32_t head_blocks, const int32_t* __restrict__ table,
                           int64_t table_stride, Lengths lengths, float scale, uint32_t chunk,
                           float* __restrict__ parts, void* __restrict__ out) {
  using L = Layout<BITS, kQuarters>;
  constexpr int kHeads = 8 * kTiles;
  extern __shared__ uint8_t raw[];
  uint8_t* shared = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                               ~(uintptr_t)1023);
  __shared__ float sm[kWarps][kHeads], sl[kWarps][kHeads];
  __shared__ uint64_t bars[kWarps][kStages];
  const uint32_t group = heads / c.heads;
  const uint32_t kvh = blockIdx.y / head_blocks, h0 = (blockIdx.y % head_blocks) * kHeads;
  const int64_t b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int64_t len = lengths.of(b);
  const int64_t t0 = (int64_t)blockIdx.x * chunk;
  if (t0 >= len && blockIdx.x > 0) return;  // the join reads no such part
  const int here = (int)min64(chunk, len - t0);
  const int blocks = (here + kBlock - 1) / kBlock;
  const int32_t* pages = table + b * table_stride;

  uint8_t* codes = shared + warp * kStages * 2 * L::kCodes;  // per stage: keys, values
  uint8_t* scales = shared + kWarps * kStages * 2 * L::kCodes + warp * kStages * 2 * L::kScales;
  uint64_t* bar = bars[warp];
  const uint32_t scale_bytes = L::scale_bytes(c.dim);
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    fence_mbar_init();
  }
  __syncwarp();

  // The next block to fetch: its number, and its page, read one fetch ahead.
  constexpr uint32_t kStride = kWarps * kBlock;
  const uint32_t stride_pages = kStride / c.page_size, stride_rest = kStride % c.page_size;
  Walk walk;
  walk.start((uint32_t)t0 + warp * kBlock, c.page_size);
  int fetch = warp;
  int32_t page = fetch < blocks ? pages[walk.page] : 0;
  // Fetches the next block whose page exists into a stage; the number of its
  // tokens that the sequence has, or 0 if there is none.
  const auto fetch_into = [&](int s) -> int {
    while (fetch < blocks) {
      const int32_t p = page;
      const uint32_t place = walk.place;
      const int seen = min(kBlock, here - fetch * kBlock);
      fetch += kWarps;
      walk.advance(stride_pages, stride_rest, c.page_size);
      if (fetch < blocks) page = pages[walk.page];
      if (p < 0 || p >= c.pages) continue;
      if (lane == 0) {
        const int64_t row = ((int64_t)p * c.heads + kvh) * c.page_size + place;
        uint8_t* at = codes + s * 2 * L::kCodes;
        uint8_t* sc = scales + s * 2 * L::kScales;
        mbar_arrive_expect_tx(&bar[s], 2 * (L::kCodes + scale_bytes));
#pragma unroll
        for (int x = 0; x < L::kBoxes; ++x) {
          tma_load_2d(at + x * L::kBox, &k_map, &bar[s], x * L::kBoxRow, (int)row);
          tma_load_2d(at + L::kCodes + x * L::kBox, &v_map, &bar[s], x * L::kBoxRow, (int)row);
        }
        const int64_t first = row * (scale_bytes / kBlock);
        bulk_load(sc, c.scales[0] + first, scale_bytes, &bar[s]);
        bulk_load(sc + L::kScales, c.scales[1] + first, scale_bytes, &bar[s]);
      }
      return seen;
    }
    return 0;
  };
  int seen[kStages];  // of the stages in order, the next to use first
#pragma unroll
  for (int s = 0; s < kStages; ++s) seen[s] = fetch_into(s);

  // Q in the order of the keys' registers, below 1 by a power of two a head
  uint32_t qf[kTiles][L::kProducts][2];
  float factor[kTiles][2];  // of heads 2 j, 2 j + 1: scale log2(e) and that power
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const uint32_t h = h0 + 8 * n + g;
    const bool live = h < group;
    const int64_t at = b * q.batch_stride + (int64_t)(kvh * group + (live ? h : 0)) * q.head_stride;
    constexpr int kPer = L::kKeyWords * 32 / BITS;  // channels of a lane in a step
    float x[L::kSteps][kPer];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) {
      const uint32_t ch = L::key_byte(s, j) * 8 / BITS;
#pragma unroll
      for (int e = 0; e < kPer / 8; ++e) {
        float y[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (live && ch + 8 * e < c.dim) {
          if (q.bf16)
            load8(static_cast<const __nv_bfloat16*>(q.data) + at + ch + 8 * e, q.vec, 8, y);
          else
            load8(static_cast<const __half*>(q.data) + at + ch + 8 * e, q.vec, 8, y);
        }
        top = max(top, abs_bits_max(y));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[s][8 * e + i] = y[i];
      }
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^-p with 2^(p - 1) <= max < 2^p; 1 for zeros, and where the query is not finite
    const uint32_t ex = top >> 23;
    const bool plain = ex == 0 || ex == 255;
    const float down = plain ? 1.0f : __uint_as_float((253u - min(ex, 252u)) << 23);
    const float up = plain ? 1.0f : __uint_as_float((1u + min(ex, 252u)) << 23);
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s)
#pragma unroll
      for (int i = 0; i < L::kProducts / L::kSteps; ++i) {
        // channels of the products' registers: code8_pair and code4_pair
        const int c0 = BITS == 8 ? 4 * i : 8 * (i / 2) + 2 * (i & 1);
        const int d = BITS == 8 ? 1 : 4, e = BITS == 8 ? 2 : 1;
        uint32_t(&f)[2] = qf[n][s * (L::kProducts / L::kSteps) + i];
        f[0] = h2_bits(__floats2half2_rn(x[s][c0] * down, x[s][c0 + d] * down));
        f[1] = h2_bits(__floats2half2_rn(x[s][c0 + e] * down, x[s][c0 + e + d] * down));
      }
#pragma unroll
    for (int r = 0; r < 2; ++r)
      factor[n][r] = __shfl_sync(0xffffffffu, up, 4 * (2 * j + r)) * (scale * kLog2e);
  }

  // o[n][p][i]: channels 16 (g + 8 p) + 2 i, + 1 of heads 2 j, 2 j + 1
  float o[kTiles][L::kPasses][8][4] = {};
  float m[kTiles][2], l[kTiles][2] = {};
#pragma unroll
  for (int n = 0; n < kTiles; ++n) m[n][0] = m[n][1] = -INFINITY;
  uint32_t v_exp = 1;  // exponent of the power of two the value scales are taken by
  const int row0 = token_of(g);        // and row0 + 8: the tokens of S^T's rows
  const int column0 = token_of(2 * j), column1 = token_of(2 * j + 1);  // of O^T, and + 8

  int stage = 0;
  uint32_t phase = 0;
#pragma unroll 1
  while (seen[0] > 0) {
    if (!mbar_wait(&bar[stage], phase)) {  // ran out: NaN, once the other copies are in
#pragma unroll
      for (int x = 1; x < kStages; ++x)
        if (seen[x] > 0)
          mbar_wait(&bar[(stage + x) % kStages], phase ^ (stage + x >= kStages ? 1u : 0u));
#pragma unroll
      for (int n = 0; n < kTiles; ++n) l[n][0] = l[n][1] = __uint_as_float(0x7FC00000u);
      break;
    }
    const uint8_t* keys = codes + stage * 2 * L::kCodes;
    const uint8_t* values = keys + L::kCodes;
    const uint32_t* ksc = reinterpret_cast<const uint32_t*>(scales + stage * 2 * L::kScales);
    const uint32_t* vsc = ksc + L::kScales / 4;
    const bool whole = seen[0] == kBlock;

    // ---- S^T = K Q^T
    float s[kTiles][4] = {};
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st) {
      uint32_t w[2][4];
      __half2 gs[2], gm[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t byte = L::key_byte(st, j);
        const uint8_t* p = keys + L::at(row0 + 8 * r, byte);
        if constexpr (L::kKeyWords == 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(p);
          w[r][0] = u.x; w[r][1] = u.y; w[r][2] = u.z; w[r][3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(p);
          w[r][0] = u.x; w[r][1] = u.y;
        }
        if constexpr (BITS == 4) {
          const uint32_t of = byte / 16;  // the group; past head_dim the codes are 0
          const __half2 sm2 =
              bits_h2(of * kGroup4 < c.dim ? ksc[(row0 + 8 * r) * (c.dim / kGroup4) + of] : 0u);
          gs[r] = __low2half2(sm2);
          gm[r] = __high2half2(sm2);
        }
      }
#pragma unroll
      for (int i = 0; i < L::kProducts / L::kSteps; ++i) {
        uint32_t a[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (BITS == 8) {
            const uint32_t x = w[r][i] ^ 0x80808080u;
            a[r][0] = code8_pair(x, 0x4140);
            a[r][1] = code8_pair(x, 0x4342);
          } else {
            const uint32_t x = w[r][i / 2] >> (8 * (i & 1));
            a[r][0] = code4_pair<false>(x, gs[r], gm[r]);
            a[r][1] = code4_pair<true>(x, gs[r], gm[r]);
          }
        }
        const int at = st * (L::kProducts / L::kSteps) + i;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          mma_f16(s[n], a[0][0], a[1][0], a[0][1], a[1][1], qf[n][at][0], qf[n][at][1]);
      }
    }

    // ---- scores in powers of two; the maximum in use
    if constexpr (BITS == 8) {
      const float ks[2] = {__uint_as_float(ksc[row0]), __uint_as_float(ksc[row0 + 8])};
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= ks[e >> 1];
    }
    bool raise = false;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= factor[n][e & 1];
        if (!whole && row0 + 8 * (e >> 1) >= seen[0]) s[n][e] = -INFINITY;
        raise |= s[n][e] > m[n][e & 1] + kRaise;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < kTiles; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = fmaxf(s[n][r], s[n][r + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(top, m[n][r]);
          const float keep = top == m[n][r] ? 1.0f : exp2f(m[n][r] - top);
          m[n][r] = top;
          l[n][r] *= keep;
#pragma unroll
          for (int p = 0; p < L::kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[n][p][i][r] *= keep;
              o[n][p][i][r + 2] *= keep;
            }
        }
    }
    float vs[2] = {1.0f, 1.0f};
    if constexpr (BITS == 8) {
      // scales relative to 2^(v_exp - 127), above every scale so far
      uint32_t e0 = vsc[row0], e1 = vsc[row0 + 8];
      if (!whole) {  // what lies behind the sequence's end is not used
        if (row0 >= seen[0]) e0 = 0u;
        if (row0 + 8 >= seen[0]) e1 = 0u;
      }
      const uint32_t e = max(e0, e1);
      if (__any_sync(0xffffffffu, e < 0x7F800000u && (e >> 23) >= v_exp)) {
        const uint32_t now =
            max(v_exp, 1u + __reduce_max_sync(0xffffffffu, e < 0x7F800000u ? e >> 23 : 0u));
        const uint32_t drop = now - v_exp;  // by 2^-drop
        const float down = drop < 127u ? __uint_as_float((127u - drop) << 23) : 0.0f;
        v_exp = now;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int p = 0; p < L::kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[n][p][i][r] *= down;
      }
      const float by = __uint_as_float((254u - v_exp) << 23);
      vs[0] = __uint_as_float(e0) * by;
      vs[1] = __uint_as_float(e1) * by;
    }
    uint32_t pt[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float top = m[n][e & 1];
        p[e] = exp2_fast(s[n][e] - (top == -INFINITY ? 0.0f : top));
        l[n][e & 1] += p[e];
        if constexpr (BITS == 8) p[e] *= vs[e >> 1];
      }
      pt[n][0] = transpose8x8(h2_bits(__floats2half2_rn(p[0], p[1])));
      pt[n][1] = transpose8x8(h2_bits(__floats2half2_rn(p[2], p[3])));
    }

    // ---- O^T += V^T P^T
#pragma unroll
    for (int p = 0; p < L::kPasses; ++p) {
      // past the row (64-channel rows have 4 lanes' pieces): any, not stored
      const uint32_t byte = ((kQuarters == 1 ? g & 3 : g) + 8 * p) * 2 * BITS;
      constexpr int kWords = BITS / 2;
      uint32_t w[4][kWords];
      uint32_t gr[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int t = (r & 1 ? column1 : column0) + 8 * (r >> 1);
        const uint8_t* at = values + L::at(t, byte);
        if constexpr (BITS == 8) {
          const uint4 u = *reinterpret_cast<const uint4*>(at);
          w[r][0] = u.x; w[r][1] = u.y; w[r][2] = u.z; w[r][3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(at);
          w[r][0] = u.x; w[r][1] = u.y;
          const uint32_t of = byte / 16;
          gr[r] = of * kGroup4 < c.dim ? vsc[t * (c.dim / kGroup4) + of] : 0u;
          if (!whole && t >= seen[0]) gr[r] = 0u;
        }
      }
      if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w0 = w[0][i] ^ 0x80808080u, w1 = w[1][i] ^ 0x80808080u;
          const uint32_t w2 = w[2][i] ^ 0x80808080u, w3 = w[3][i] ^ 0x80808080u;
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // channels 4 i + 2 h, + 1
            const uint32_t x = __byte_perm(w0, w1, h ? 0x7362 : 0x5140);
            const uint32_t y = __byte_perm(w2, w3, h ? 0x7362 : 0x5140);
            const uint32_t a0 = code8_pair(x, 0x4140), a1 = code8_pair(x, 0x4342);
            const uint32_t a2 = code8_pair(y, 0x4140), a3 = code8_pair(y, 0x4342);
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
              mma_f16(o[n][p][2 * i + h], a0, a1, a2, a3, pt[n][0], pt[n][1]);
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
            const uint32_t x = __byte_perm(w[0][i], w[1][i], sel) >> (8 * (h & 1));
            const uint32_t y = __byte_perm(w[2][i], w[3][i], sel) >> (8 * (h & 1));
            const uint32_t a0 = code4_pair<false>(x, s01, m01), a1 = code4_pair<true>(x, s01, m01);
            const uint32_t a2 = code4_pair<false>(y, s23, m23), a3 = code4_pair<true>(y, s23, m23);
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
              mma_f16(o[n][p][4 * i + h], a0, a1, a2, a3, pt[n][0], pt[n][1]);
          }
      }
    }

    // ---- the stage is read: the next block into it
    __syncwarp();
    const int more = fetch_into(stage);
#pragma unroll
    for (int x = 0; x + 1 < kStages; ++x) seen[x] = seen[x + 1];
    seen[kStages - 1] = more;
    if (++stage == kStages) stage = 0, phase ^= 1u;
  }

  // the warps' parts, in the rings' memory
  __syncthreads();
  float* so = reinterpret_cast<float*>(shared);  // [kWarps][kHeads][dim]
  const float up = BITS == 8 ? __uint_as_float(v_exp << 23) : 1.0f;
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[n][r] += __shfl_xor_sync(0xffffffffu, l[n][r], d);
      const int h = 8 * n + 2 * j + r;
      if (g == 0) sm[warp][h] = m[n][r], sl[warp][h] = l[n][r];
#pragma unroll
      for (int p = 0; p < L::kPasses; ++p) {
        const uint32_t ch = 16 * (g + 8 * p);
        if (ch < c.dim)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float2*>(&so[(warp * kHeads + h) * c.dim + ch + 2 * i]) =
                make_float2(o[n][p][i][r] * up, o[n][p][i][r + 2] * up);
      }
    }
  }
  __syncthreads();
  const int64_t rows = (int64_t)gridDim.z * heads * gridDim.x;  // parts
  for (uint32_t i = threadIdx.x; i < kHeads * c.dim; i += 32 * kWarps) {
    const uint32_t h = i / c.dim, ch = i - h * c.dim;
    if (h0 + h >= group) break;
    float top = -INFINITY, sum = 0.0f, y = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w][h]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = sm[w][h] == -INFINITY ? 0.0f : exp2f(sm[w][h] - top);
      sum = fmaf(sl[w][h], f, sum);
      y = fmaf(so[(w * kHeads + h) * c.dim + ch], f, y);
    }
    const int64_t head = b * heads + kvh * group + h0 + h;
    if (parts == nullptr) {
      store_out(out, q.bf16, head * c.dim + ch, sum == 0.0f ? 0.0f : y / sum);
    } else {
      const int64_t part = head * gridDim.x + blockIdx.x;
      parts[part * c.dim + ch] = y;
      if (ch == 0)
        reinterpret_cast<float2*>(parts + rows * c.dim)[part] = make_float2(top, sum);
    }
  }
}

// A CTA a (sequence, head): the chunks' parts in order.
__global__ void __launch_bounds__(256)
    cache_attention_join_kernel(const float* __restrict__ parts, uint32_t chunks, uint32_t chunk,
                                uint32_t heads, uint32_t dim, Lengths lengths, bool bf16,
                                void* __restrict__ out) {
  const int64_t head = (int64_t)blockIdx.y * heads + blockIdx.x;
  const int64_t len = lengths.of(blockIdx.y);
  const int n = max((int)((len + chunk - 1) / chunk), 1);
  const float2* ml = reinterpret_cast<const float2*>(
                         parts + (int64_t)gridDim.y * heads * chunks * dim) + head * chunks;
  const float* o = parts + head * chunks * dim;
  float top = -INFINITY;
  for (int i = 0; i < n; ++i) top = fmaxf(top, ml[i].x);
  for (uint32_t ch = threadIdx.x; ch < dim; ch += 256) {
    float sum = 0.0f, y = 0.0f;
    for (int i = 0; i < n; ++i) {
      const float2 a = ml[i];
      const float f = a.x == -INFINITY ? 0.0f : exp2f(a.x - top);
      sum = fmaf(a.y, f, sum);
      y = fmaf(o[(int64_t)i * dim + ch], f, y);
    }
    store_out(out, bf16, head * dim + ch, sum == 0.0f ? 0.0f : y / sum);
  }
}

// Two column tiles (16 heads) where their registers fit (head_dim up to 128),
// else head blocks of 8 that read the codes again.
inline uint32_t head_tiles(uint32_t group, uint32_t dim) { return group > 8 && dim <= 128 ? 2 : 1; }

struct Split {
  uint32_t head_blocks, chunk, chunks;
};

// Chunks: enough CTAs for a few rounds of the GPU's resident ones, none
// shorter than 256 tokens.
inline Split split_for(const CacheView& c, int64_t batch, int64_t heads, int64_t most) {
  Split s;
  const uint32_t group = (uint32_t)(heads / c.heads);
  s.head_blocks = (uint32_t)ceil_div(group, 8 * head_tiles(group, c.dim));
  const int64_t rows = batch * c.heads * s.head_blocks;
  const int64_t want = max64(1, ceil_div(148 * 4 * 2, rows));
  const int64_t chunk = max64(256, ceil_div(ceil_div(most, want), 64) * 64);
  s.chunks = (uint32_t)max64(1, ceil_div(most, chunk));
  s.chunk = (uint32_t)chunk;
  return s;
}

// Rows of codes as TMA reads them: [all rows, bytes], boxes of 16 rows.
bool rows_map(CUtensorMap* map, const void* codes, const CacheView& c, int bits, uint32_t box_row) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  std::memset(map, 0, sizeof(*map));
  const cuuint64_t bytes = (cuuint64_t)c.dim * bits / 8;
  const cuuint64_t dims[2] = {bytes, (cuuint64_t)(c.pages * c.heads * c.page_size)};
  const cuuint64_t strides[1] = {bytes};
  const cuuint32_t box[2] = {box_row, (cuuint32_t)kBlock};
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
  uint32_t heads;
  Split split;
  dim3 grid;
  const int32_t* table;
  int64_t table_stride;
  Lengths lengths;
  float scale;
  float* parts;
  void* out;
  cudaStream_t stream;
};

template <int BITS, int kQuarters, int kTiles>
mb_status launch(const Call& a) {
  using L = Layout<BITS, kQuarters>;
  constexpr int kStages = 3;
  CUtensorMap k_map, v_map;
  if (!rows_map(&k_map, a.c.codes[0], a.c, BITS, L::kBoxRow) ||
      !rows_map(&v_map, a.c.codes[1], a.c, BITS, L::kBoxRow))
    return set_error(MB_ERR_CUDA, "cuTensorMapEncodeTiled rejected the cache");
  const size_t ring = (size_t)kWarps * kStages * L::kStage;
  const size_t join = (size_t)kWarps * 8 * kTiles * a.c.dim * sizeof(float);
  const size_t smem = (ring > join ? ring : join) + 1024;
  auto* kernel = cache_attention_kernel<BITS, kQuarters, kTiles, kStages>;
  static std::atomic<uint64_t> attr_done{0};
  MB_CUDA_TRY(set_smem_limit_once(kernel, 160 * 1024, attr_done));
  kernel<<<a.grid, 32 * kWarps, smem, a.stream>>>(
      k_map, v_map, a.c, a.q, a.heads, a.split.head_blocks, a.table, a.table_stride, a.lengths,
      a.scale, a.split.chunk, a.parts, a.out);
  MB_LAUNCH_CHECK("cache_attention_kernel");
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
  const CacheView c = cache_view(cache);
  const Split s = split_for(c, batch, heads, table_width * c.page_size);
  if (s.chunks == 1) return 0;
  return (size_t)(batch * heads) * s.chunks * (c.dim + 2) * sizeof(float);
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
  MB_REQUIRE(table_width <= ((int64_t(1) << 31) - 1) / cache->page_size,
             "table_width too large: positions must fit 31 bits");
  MB_REQUIRE(std::isfinite(scale), "scale must be finite");
  MB_REQUIRE(aligned(q, 2) && aligned(out, 2) && aligned(page_table, 4) && aligned(lengths, 4),
             "misaligned q, out, page_table or lengths");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const CacheView c = cache_view(cache);
  const int64_t most = table_width * c.page_size;
  const uint32_t group = (uint32_t)(heads / c.heads), tiles = head_tiles(group, c.dim);
  const Split s = split_for(c, batch, heads, most);
  const size_t need = mb_cache_attention_workspace_size(cache, batch, heads, table_width);
  float* parts = nullptr;
  if (need > 0) {
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 8))
      return set_error(MB_ERR_WORKSPACE,
                       "cache_attention workspace missing, misaligned or too small");
    parts = static_cast<float*>(workspace);
  }
  const Query qs{q, q_batch_stride, q_head_stride, type == MB_BF16,
                 aligned(q, 16) && (batch == 1 || q_batch_stride % 8 == 0) &&
                     (heads == 1 || q_head_stride % 8 == 0)};
  const dim3 grid(s.chunks, (unsigned)(c.heads * s.head_blocks), (unsigned)batch);
  MB_REQUIRE(grid.y <= 65535u, "too many head blocks");
  MB_REQUIRE(c.pages * c.heads * c.page_size < (int64_t(1) << 31),
             "cache too large: pages * kv_heads * page_size must fit 31 bits");
  const Lengths all{lengths, most};
  const Call call{c,     qs,  (uint32_t)heads, s,     grid, page_table, table_stride,
                  all,   scale, parts,         out,   stream};
  const mb_status st = cache->bits == 8 ? dispatch<8>(call, tiles) : dispatch<4>(call, tiles);
  if (st != MB_OK) return st;
  if (parts != nullptr) {
    cache_attention_join_kernel<<<dim3((unsigned)heads, (unsigned)batch), 256, 0, stream>>>(
        parts, s.chunks, s.chunk, (uint32_t)heads, c.dim, all, type == MB_BF16, out);
    MB_LAUNCH_CHECK("cache_attention_join_kernel");
  }
  return MB_OK;
}
