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
// No shared memory on the way in: both products' left operands come straight
// from global memory, because the order of the inner index is free.  In
// S^T the lane (g, j) = (lane / 4, lane % 4) holds 16 consecutive channels of
// tokens g and g + 8 (channel 64 s + 16 j + .. in step s), and Q's registers
// follow the same order; in O^T it holds 16 consecutive channels
// (16 g + .., and 128 further for head_dim > 128) of tokens 2 j, 2 j + 1,
// 2 j + 8, 2 j + 9.  Each load is 16 (8 bits) or 8 bytes (4 bits) of a row,
// neighbours within a row.  Between the products the probabilities change
// from S^T's layout to the right operand's by a transposing move.
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

#include "mb_cache.cuh"

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

__device__ __forceinline__ float query_at(const Query& q, int64_t i) {
  return q.bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(q.data)[i])
                : __half2float(static_cast<const __half*>(q.data)[i]);
}

__device__ __forceinline__ void store_out(void* out, bool bf16, int64_t i, float y) {
  if (bf16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(y);
  else
    static_cast<__half*>(out)[i] = __float2half_rn(y);
}

// One lane's part of 16 tokens' keys and values.  kSteps: 64-channel steps.
template <int BITS, int kSteps>
struct Tokens {
  static constexpr int kWords = BITS == 8 ? 4 : 2;        // of 16 channels
  static constexpr int kPasses = (kSteps + 1) / 2;        // 128-channel passes over V
  uint32_t k[2][kSteps][kWords];                          // tokens g, g + 8
  uint32_t v[4][kPasses][kWords];                         // tokens 2j, 2j + 1, 2j + 8, 2j + 9
  float k_scale[2], v_scale[2];                           // 8 bits: tokens g, g + 8
  uint32_t k_group[BITS == 4 ? 2 : 1][BITS == 4 ? kSteps : 1];   // 4 bits: (s, m)
  uint32_t v_group[BITS == 4 ? 4 : 1][BITS == 4 ? kPasses : 1];

  __device__ __forceinline__ static void load_words(uint32_t (&w)[kWords], const uint8_t* p) {
    if constexpr (BITS == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    }
  }

  // Tokens row .. row + 15; those from `seen` on get scales (4 bits: scale
  // and minimum) of 0: what a place behind the sequence's end holds is not
  // used.  The codes there lie in the same page.
  __device__ __forceinline__ void load_keys(const CacheView& c, int64_t row, int seen, int g,
                                            int j) {
    const uint32_t bytes = c.dim * BITS / 8;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t at = row + g + 8 * r;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint32_t piece = 4 * s + j;
        if (piece * 16 < c.dim)
          load_words(k[r][s], c.codes[0] + at * bytes + piece * (2 * BITS));
        if constexpr (BITS == 4) {
          k_group[r][s] = 0;
          if (piece * 16 < c.dim && g + 8 * r < seen)
            k_group[r][s] =
                reinterpret_cast<const uint32_t*>(c.scales[0])[at * (c.dim / kGroup4) + piece / 2];
        }
      }
      if constexpr (BITS == 8)
        k_scale[r] = g + 8 * r < seen ? reinterpret_cast<const float*>(c.scales[0])[at] : 0.0f;
    }
  }

  __device__ __forceinline__ void load_values(const CacheView& c, int64_t row, int seen, int g,
                                              int j) {
    const uint32_t bytes = c.dim * BITS / 8;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 2 * j + (r & 1) + 8 * (r >> 1);
      const int64_t at = row + t;
#pragma unroll
      for (int p = 0; p < kPasses; ++p) {
        const uint32_t piece = g + 8 * p;
        if (piece * 16 < c.dim)
          load_words(v[r][p], c.codes[1] + at * bytes + piece * (2 * BITS));
        if constexpr (BITS == 4) {
          v_group[r][p] = 0;
          if (piece * 16 < c.dim && t < seen)
            v_group[r][p] =
                reinterpret_cast<const uint32_t*>(c.scales[1])[at * (c.dim / kGroup4) + piece / 2];
        }
      }
    }
    if constexpr (BITS == 8) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        v_scale[r] =
            g + 8 * r < seen ? reinterpret_cast<const float*>(c.scales[1])[row + g + 8 * r] : 0.0f;
    }
  }

  // Nothing to see: values that contribute nothing, whatever the codes.
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      k_scale[r] = v_scale[r] = 0.0f;
      if constexpr (BITS == 4)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) k_group[r][s] = 0;
    }
    if constexpr (BITS == 4)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int p = 0; p < kPasses; ++p) v_group[r][p] = 0;
  }

  // S^T += K Q^T
  template <int kTiles>
  __device__ __forceinline__ void scores(float (&s)[kTiles][4],
                                         const uint32_t (&q)[kTiles][kSteps][4][2]) const {
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if constexpr (BITS == 8) {
            const uint32_t w = k[r][st][i] ^ 0x80808080u;
            a[r][0] = code8_pair(w, 0x4140);
            a[r][1] = code8_pair(w, 0x4342);
          } else {
            const __half2 gm = bits_h2(k_group[r][st]);
            const uint32_t w = k[r][st][i / 2] >> (8 * (i & 1));
            a[r][0] = code4_pair<false>(w, __low2half2(gm), __high2half2(gm));
            a[r][1] = code4_pair<true>(w, __low2half2(gm), __high2half2(gm));
          }
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
          mma_f16(s[n], a[0][0], a[1][0], a[0][1], a[1][1], q[n][st][i][0], q[n][st][i][1]);
      }
    }
  }

  // O^T += V^T P^T; o[n][p][m]: channels 16 (g + 8 p) + 2 m, + 1 of heads 2 j, 2 j + 1
  template <int kTiles>
  __device__ __forceinline__ void outputs(float (&o)[kTiles][kPasses][8][4],
                                          const uint32_t (&pt)[kTiles][2]) const {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (BITS == 8) {
          const uint32_t w0 = v[0][p][i] ^ 0x80808080u, w1 = v[1][p][i] ^ 0x80808080u;
          const uint32_t w2 = v[2][p][i] ^ 0x80808080u, w3 = v[3][p][i] ^ 0x80808080u;
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
        } else {
          const uint32_t g01[2] = {v_group[0][p], v_group[1][p]};
          const uint32_t g23[2] = {v_group[2][p], v_group[3][p]};
          const __half2 s01 = bits_h2(__byte_perm(g01[0], g01[1], 0x5410));
          const __half2 m01 = bits_h2(__byte_perm(g01[0], g01[1], 0x7632));
          const __half2 s23 = bits_h2(__byte_perm(g23[0], g23[1], 0x5410));
          const __half2 m23 = bits_h2(__byte_perm(g23[0], g23[1], 0x7632));
#pragma unroll
          for (int h = 0; h < 4; ++h) {  // channels 8 i + 2 h, + 1
            const uint32_t sel = h < 2 ? 0x5410 : 0x7632;
            const uint32_t x = __byte_perm(v[0][p][i], v[1][p][i], sel) >> (8 * (h & 1));
            const uint32_t y = __byte_perm(v[2][p][i], v[3][p][i], sel) >> (8 * (h & 1));
            const uint32_t a0 = code4_pair<false>(x, s01, m01), a1 = code4_pair<true>(x, s01, m01);
            const uint32_t a2 = code4_pair<false>(y, s23, m23), a3 = code4_pair<true>(y, s23, m23);
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
              mma_f16(o[n][p][4 * i + h], a0, a1, a2, a3, pt[n][0], pt[n][1]);
          }
        }
      }
    }
  }
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;  // how far a score may exceed the maximum in use

// Grid: (chunks, kv heads x head blocks, batch).  parts: per (sequence, head,
// chunk) head_dim outputs, then all (maximum, sum) pairs; null with one chunk.
template <int BITS, int kSteps, int kTiles>
__global__ void __launch_bounds__(32 * kWarps)
    cache_attention_kernel(CacheView c, Query q, uint32_t heads, uint32_t head_blocks,
                           const int32_t* __restrict__ table, int64_t table_stride,
                           int64_t most, const int32_t* __restrict__ lengths, float scale,
                           uint32_t chunk, float* __restrict__ parts, void* __restrict__ out) {
  constexpr int kHeads = 8 * kTiles;
  using Piece = Tokens<BITS, kSteps>;
  __shared__ float sm[kWarps][kHeads], sl[kWarps][kHeads];
  extern __shared__ float so[];  // [kWarps][kHeads][dim]
  const uint32_t group = heads / c.heads;
  const uint32_t kvh = blockIdx.y / head_blocks, h0 = (blockIdx.y % head_blocks) * kHeads;
  const int64_t b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
  const int64_t len = max64(0, min64(lengths[b], most));
  const int64_t t0 = (int64_t)blockIdx.x * chunk;
  if (t0 >= len && blockIdx.x > 0) return;  // the join reads no such part
  const int here = (int)min64(chunk, len - t0);
  const int blocks = (here + kBlock - 1) / kBlock;
  const int32_t* pages = table + b * table_stride;

  // first row of a block, or -1 if its page lies outside the cache
  const auto row_of = [&](int block) -> int64_t {
    const uint32_t t = (uint32_t)t0 + (uint32_t)block * kBlock;
    const uint32_t p = t / c.page_size;
    const int64_t page = pages[p];
    if (page < 0 || page >= c.pages) return -1;
    return (page * c.heads + kvh) * c.page_size + (t - p * c.page_size);
  };

  Piece tok = {};
  int64_t row = -1;
  int seen = 0;
  if (warp < blocks) {
    row = row_of(warp);
    seen = row < 0 ? 0 : min(kBlock, here - warp * kBlock);
    if (row >= 0) {
      tok.load_keys(c, row, seen, g, j);
      tok.load_values(c, row, seen, g, j);
    }
  }

  // Q in the order of the keys' registers, below 1 by a power of two a head
  uint32_t qf[kTiles][kSteps][4][2];
  float factor[kTiles][2];  // of heads 2 j, 2 j + 1: scale log2(e) and that power
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const uint32_t h = h0 + 8 * n + g;
    const bool live = h < group;
    const int64_t at = b * q.batch_stride + (int64_t)(kvh * group + (live ? h : 0)) * q.head_stride;
    float x[kSteps][16];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const uint32_t ch = 64 * s + 16 * j;
      const bool in = live && ch < c.dim;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float y[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (in) {
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
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // channels of the products' registers: code8_pair and code4_pair
        const int c0 = BITS == 8 ? 4 * i : 8 * (i / 2) + 2 * (i & 1);
        const int d = BITS == 8 ? 1 : 4, e = BITS == 8 ? 2 : 1;
        qf[n][s][i][0] =
            h2_bits(__floats2half2_rn(x[s][c0] * down, x[s][c0 + d] * down));
        qf[n][s][i][1] =
            h2_bits(__floats2half2_rn(x[s][c0 + e] * down, x[s][c0 + e + d] * down));
      }
#pragma unroll
    for (int r = 0; r < 2; ++r)
      factor[n][r] = __shfl_sync(0xffffffffu, up, 4 * (2 * j + r)) * (scale * kLog2e);
  }

  float o[kTiles][Piece::kPasses][8][4] = {};
  float m[kTiles][2], l[kTiles][2] = {};
#pragma unroll
  for (int n = 0; n < kTiles; ++n) m[n][0] = m[n][1] = -INFINITY;
  uint32_t v_exp = 1;  // exponent of the power of two the value scales are taken by

#pragma unroll 1
  for (int block = warp; block < blocks; block += kWarps) {
    const int next = block + kWarps;
    const int64_t next_row = next < blocks ? row_of(next) : -1;
    const int next_seen = next_row < 0 ? 0 : min(kBlock, here - next * kBlock);

    float s[kTiles][4] = {};
    tok.template scores<kTiles>(s, qf);
    const float ks[2] = {tok.k_scale[0], tok.k_scale[1]};
    if (next_row >= 0) tok.load_keys(c, next_row, next_seen, g, j);

    // scores in powers of two; the maximum in use
    bool raise = false;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y = s[n][e] * factor[n][e & 1];
        if constexpr (BITS == 8) y *= ks[e >> 1];
        s[n][e] = g + 8 * (e >> 1) < seen ? y : -INFINITY;
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
          for (int p = 0; p < Piece::kPasses; ++p)
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
      const uint32_t e = max(__float_as_uint(tok.v_scale[0]), __float_as_uint(tok.v_scale[1]));
      if (__any_sync(0xffffffffu, e < 0x7F800000u && (e >> 23) >= v_exp)) {
        const uint32_t now = max(v_exp, 1u + __reduce_max_sync(0xffffffffu,
                                                  e < 0x7F800000u ? e >> 23 : 0u));
        const uint32_t drop = now - v_exp;  // by 2^-drop
        const float down = drop < 127u ? __uint_as_float((127u - drop) << 23) : 0.0f;
        v_exp = now;
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int p = 0; p < Piece::kPasses; ++p)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[n][p][i][r] *= down;
      }
      const float by = __uint_as_float((254u - v_exp) << 23);
      vs[0] = tok.v_scale[0] * by;
      vs[1] = tok.v_scale[1] * by;
    }
    uint32_t pt[kTiles][2];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float top = m[n][e & 1];
        p[e] = exp2f(s[n][e] - (top == -INFINITY ? 0.0f : top));
        l[n][e & 1] += p[e];
        p[e] *= vs[e >> 1];
      }
      pt[n][0] = transpose8x8(h2_bits(__floats2half2_rn(p[0], p[1])));
      pt[n][1] = transpose8x8(h2_bits(__floats2half2_rn(p[2], p[3])));
    }
    tok.template outputs<kTiles>(o, pt);
    if (next_row >= 0)
      tok.load_values(c, next_row, next_seen, g, j);
    else
      tok.clear();
    seen = next_seen;
  }

  // the warps' parts, in shared memory
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
      for (int p = 0; p < Piece::kPasses; ++p) {
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
                                uint32_t heads, uint32_t dim, int64_t most,
                                const int32_t* __restrict__ lengths, bool bf16,
                                void* __restrict__ out) {
  const int64_t head = (int64_t)blockIdx.y * heads + blockIdx.x;
  const int64_t len = max64(0, min64(lengths[blockIdx.y], most));
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
  const size_t smem = (size_t)kWarps * 8 * tiles * c.dim * sizeof(float);
  const auto go = [&](auto kernel) {
    kernel<<<grid, 32 * kWarps, smem, stream>>>(c, qs, (uint32_t)heads, s.head_blocks, page_table,
                                                table_stride, most, lengths, scale, s.chunk, parts,
                                                out);
  };
  const auto steps = [&](auto bits) {
    constexpr int B = decltype(bits)::value;
    if (c.dim <= 64)
      tiles == 2 ? go(cache_attention_kernel<B, 1, 2>) : go(cache_attention_kernel<B, 1, 1>);
    else if (c.dim <= 128)
      tiles == 2 ? go(cache_attention_kernel<B, 2, 2>) : go(cache_attention_kernel<B, 2, 1>);
    else if (c.dim <= 192)
      go(cache_attention_kernel<B, 3, 1>);
    else
      go(cache_attention_kernel<B, 4, 1>);
  };
  if (cache->bits == 8)
    steps(std::integral_constant<int, 8>{});
  else
    steps(std::integral_constant<int, 4>{});
  MB_LAUNCH_CHECK("cache_attention_kernel");
  if (parts != nullptr) {
    cache_attention_join_kernel<<<dim3((unsigned)heads, (unsigned)batch), 256, 0, stream>>>(
        parts, s.chunks, s.chunk, (uint32_t)heads, c.dim, most, lengths, type == MB_BF16, out);
    MB_LAUNCH_CHECK("cache_attention_join_kernel");
  }
  return MB_OK;
}
