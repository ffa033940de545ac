// Keys and values quantised to 8 or 4 bits as they are written into a paged
// cache, and read back (no counterpart in the reference).
//
// A row (one token's head of k or v) is taken by the 2 .. 32 lanes that hold
// its channels, eight a lane: a 16-byte load, the maximum (8 bits: of the
// row) or minimum and maximum (4 bits: of 32 channels, four lanes) by
// shuffles, and one 8- or 4-byte store.  Bound by memory: 2 bytes in and 1 or
// 0.63 out a value.
#include <algorithm>

#include "mb_cache.cuh"

namespace mb {
namespace {

// Up to so many tokens, a row looks through the later tokens' slots itself
// for its own; above, a table says which token a slot belongs to.
constexpr int64_t kScanTokens = 512;

__host__ __device__ inline uint32_t claim_hash(uint32_t slot, uint32_t mask) {
  return (slot * 2654435761u >> 7) & mask;
}

inline uint32_t claim_entries(int64_t tokens) {
  uint32_t n = 1024;
  while (n < 2 * tokens) n *= 2;
  return n;
}

// Entry: slot + 1 in the upper half, the largest token with that slot in the
// lower.  The table has at least two entries a token, so a free one is found
// within its length.
__global__ void __launch_bounds__(256)
    cache_claim_kernel(const int64_t* __restrict__ slots, uint32_t tokens, int64_t n_slots,
                       unsigned long long* __restrict__ table, uint32_t mask) {
  const uint32_t t = blockIdx.x * 256u + threadIdx.x;
  if (t >= tokens) return;
  const int64_t slot = slots[t];
  if (slot < 0 || slot >= n_slots) return;
  const unsigned long long mine = ((unsigned long long)(slot + 1) << 32) | t;
  for (uint32_t i = 0, at = claim_hash((uint32_t)slot, mask); i <= mask; ++i, at = (at + 1) & mask) {
    const unsigned long long old = atomicCAS(&table[at], 0ull, mine);
    if (old == 0ull) return;
    if (old >> 32 == mine >> 32) {
      atomicMax(&table[at], mine);
      return;
    }
  }
}

__device__ __forceinline__ bool claimed(const unsigned long long* __restrict__ table,
                                        uint32_t mask, uint32_t slot, uint32_t t) {
  for (uint32_t i = 0, at = claim_hash(slot, mask); i <= mask; ++i, at = (at + 1) & mask) {
    const unsigned long long e = table[at];
    if (e >> 32 == (unsigned long long)slot + 1) return (uint32_t)e == t;
  }
  return false;
}

struct KvSource {
  const void* data[2];
  int64_t token_stride[2], head_stride[2];
  bool vec[2];
};

// `width` lanes a row (a power of two, at least dim / 8).
template <typename X, int BITS>
__global__ void __launch_bounds__(256)
    cache_write_kernel(CacheView c, KvSource src, const int64_t* __restrict__ slots,
                       uint32_t tokens, uint32_t width, const unsigned long long* __restrict__ table,
                       uint32_t mask) {
  const uint32_t per = 256u / width;
  const uint32_t lane = threadIdx.x & (width - 1);
  const uint64_t r = (uint64_t)blockIdx.x * per + threadIdx.x / width;
  const uint32_t rows_per_token = 2 * c.heads;
  const uint64_t t64 = r / rows_per_token;
  const bool live = t64 < tokens;
  const uint32_t t = live ? (uint32_t)t64 : 0u;
  const uint32_t in = (uint32_t)(r - t64 * rows_per_token);
  const uint32_t which = in >= c.heads, head = in - (which ? c.heads : 0u);
  const int64_t slot = slots[t];
  bool mine = live && slot >= 0 && slot < cache_slots(c);
  const bool holds = lane * 8 < c.dim;
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (mine && holds)
    load8(static_cast<const X*>(which ? src.data[1] : src.data[0]) +
              t * (which ? src.token_stride[1] : src.token_stride[0]) +
              head * (which ? src.head_stride[1] : src.head_stride[0]) + 8 * lane,
          which ? src.vec[1] : src.vec[0], 8, v);
  // the last token with this slot is the one that is kept
  if (table != nullptr) {
    if (mine) mine = claimed(table, mask, (uint32_t)slot, t);
  } else {
    bool later = false;
    if (mine)
      for (uint32_t o = t + 1 + lane; o < tokens; o += width) later |= slots[o] == slot;
    for (uint32_t o = width / 2; o > 0; o >>= 1)
      later |= __shfl_xor_sync(0xffffffffu, (int)later, o) != 0;
    mine = mine && !later;
  }
  const int64_t row = mine ? cache_row(c, (uint32_t)slot, head) : 0;
  uint8_t* codes = which ? c.codes[1] : c.codes[0];
  uint8_t* scales = which ? c.scales[1] : c.scales[0];
  if constexpr (BITS == 8) {
    uint32_t m = abs_bits_max(v);
    for (uint32_t o = width / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!mine || !holds) return;
    const RowScale s = row_scale(m);
    *reinterpret_cast<uint2*>(codes + row * c.dim + 8 * lane) = codes8(v, s);
    if (lane == 0) reinterpret_cast<float*>(scales)[row] = s.scale;
  } else {
    // fminf and fmaxf pass over a NaN: carry it by a sum of its own
    float lo = v[0], hi = v[0], bad = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo = fminf(lo, v[i]);
      hi = fmaxf(hi, v[i]);
      bad += v[i] * 0.0f;
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      bad += __shfl_xor_sync(0xffffffffu, bad, o);
    }
    if (!mine || !holds) return;
    const GroupScale g = group_scale(lo + bad, hi + bad);
    *reinterpret_cast<uint32_t*>(codes + row * (c.dim / 2) + 4 * lane) = codes4(v, g);
    if (lane % 4 == 0)
      reinterpret_cast<__half2*>(scales)[row * (c.dim / kGroup4) + lane / 4] =
          __halves2half2(g.scale, g.low);
  }
}

template <typename Y, int BITS>
__global__ void __launch_bounds__(256)
    cache_read_kernel(CacheView c, const int64_t* __restrict__ slots, uint32_t tokens,
                      uint32_t width, Y* __restrict__ k_out, Y* __restrict__ v_out) {
  const uint32_t per = 256u / width;
  const uint32_t lane = threadIdx.x & (width - 1);
  const uint64_t r = (uint64_t)blockIdx.x * per + threadIdx.x / width;
  const uint32_t rows_per_token = 2 * c.heads;
  const uint64_t t = r / rows_per_token;
  if (t >= tokens || lane * 8 >= c.dim) return;
  const uint32_t in = (uint32_t)(r - t * rows_per_token);
  const uint32_t which = in >= c.heads, head = in - (which ? c.heads : 0u);
  const int64_t slot = slots[t];
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (slot >= 0 && slot < cache_slots(c)) {
    const int64_t row = cache_row(c, (uint32_t)slot, head);
    const uint8_t* codes = which ? c.codes[1] : c.codes[0];
    const uint8_t* scales = which ? c.scales[1] : c.scales[0];
    if constexpr (BITS == 8) {
      const uint2 q = *reinterpret_cast<const uint2*>(codes + row * c.dim + 8 * lane);
      const float s = reinterpret_cast<const float*>(scales)[row];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = __fmul_rn((float)(int)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3))), s);
    } else {
      const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + row * (c.dim / 2) + 4 * lane);
      const __half2 g =
          reinterpret_cast<const __half2*>(scales)[row * (c.dim / kGroup4) + lane / 4];
      const float s = __low2float(g), m = __high2float(g);
      // s * code is exact in fp32: 11 + 4 bits
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(s, (float)((q >> (4 * i)) & 15u), m);
    }
  }
  store8((which ? v_out : k_out) + (t * c.heads + head) * c.dim + 8 * lane, true, 8, v);
}

inline uint32_t row_width(uint32_t dim) {
  uint32_t w = 4;
  while (w * 8 < dim) w *= 2;
  return w;
}

template <typename X>
void launch_write(const CacheView& c, int bits, const KvSource& src, const int64_t* slots,
                  uint32_t tokens, const unsigned long long* table, uint32_t mask,
                  cudaStream_t stream) {
  const uint32_t width = row_width(c.dim);
  const unsigned grid = (unsigned)ceil_div((int64_t)tokens * 2 * c.heads, 256 / width);
  if (bits == 8)
    cache_write_kernel<X, 8><<<grid, 256, 0, stream>>>(c, src, slots, tokens, width, table, mask);
  else
    cache_write_kernel<X, 4><<<grid, 256, 0, stream>>>(c, src, slots, tokens, width, table, mask);
}

template <typename Y>
void launch_read(const CacheView& c, int bits, const int64_t* slots, uint32_t tokens, void* k,
                 void* v, cudaStream_t stream) {
  const uint32_t width = row_width(c.dim);
  const unsigned grid = (unsigned)ceil_div((int64_t)tokens * 2 * c.heads, 256 / width);
  if (bits == 8)
    cache_read_kernel<Y, 8><<<grid, 256, 0, stream>>>(c, slots, tokens, width,
                                                      static_cast<Y*>(k), static_cast<Y*>(v));
  else
    cache_read_kernel<Y, 4><<<grid, 256, 0, stream>>>(c, slots, tokens, width,
                                                      static_cast<Y*>(k), static_cast<Y*>(v));
}

mb_status check_tokens(const mb_kv_cache* c, int64_t tokens) {
  MB_REQUIRE(tokens > 0, "tokens must be positive");
  MB_REQUIRE(tokens < (int64_t(1) << 30) &&
                 tokens * 2 * c->kv_heads / (256 / row_width((uint32_t)c->head_dim)) <
                     (int64_t(1) << 31) - 1,
             "too many tokens");
  return MB_OK;
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" size_t mb_cache_write_workspace_size(int64_t tokens) {
  if (tokens <= kScanTokens || tokens >= (int64_t(1) << 30)) return 0;
  return (size_t)claim_entries(tokens) * 8;
}

extern "C" mb_status mb_cache_write(const mb_kv_cache* cache, const void* k,
                                    int64_t k_token_stride, int64_t k_head_stride, const void* v,
                                    int64_t v_token_stride, int64_t v_head_stride, mb_dtype type,
                                    int64_t tokens, const int64_t* slots, void* workspace,
                                    size_t workspace_bytes, mb_stream_t stream_) {
  clear_error();
  if (const mb_status st = check_cache(cache); st != MB_OK) return st;
  MB_REQUIRE(k && v && slots, "cache_write pointers must not be null");
  MB_REQUIRE(type == MB_FP16 || type == MB_BF16, "k and v must be fp16 or bf16");
  MB_REQUIRE(aligned(k, 2) && aligned(v, 2) && aligned(slots, 8), "misaligned k, v or slots");
  if (const mb_status st = check_tokens(cache, tokens); st != MB_OK) return st;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const CacheView c = cache_view(cache);
  const auto vec = [&](const void* p, int64_t ts, int64_t hs) {
    return aligned(p, 16) && (tokens == 1 || ts % 8 == 0) && (c.heads == 1 || hs % 8 == 0);
  };
  const KvSource src{{k, v},
                     {k_token_stride, v_token_stride},
                     {k_head_stride, v_head_stride},
                     {vec(k, k_token_stride, k_head_stride),
                      vec(v, v_token_stride, v_head_stride)}};
  unsigned long long* table = nullptr;
  uint32_t mask = 0;
  if (tokens > kScanTokens) {
    const size_t need = mb_cache_write_workspace_size(tokens);
    if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 8))
      return set_error(MB_ERR_WORKSPACE, "cache_write workspace missing, misaligned or too small");
    table = static_cast<unsigned long long*>(workspace);
    mask = claim_entries(tokens) - 1;
    MB_CUDA_TRY(cudaMemsetAsync(table, 0, need, stream));
    cache_claim_kernel<<<(unsigned)ceil_div(tokens, 256), 256, 0, stream>>>(
        slots, (uint32_t)tokens, cache_slots(c), table, mask);
    MB_LAUNCH_CHECK("cache_claim_kernel");
  }
  if (type == MB_FP16)
    launch_write<__half>(c, cache->bits, src, slots, (uint32_t)tokens, table, mask, stream);
  else
    launch_write<__nv_bfloat16>(c, cache->bits, src, slots, (uint32_t)tokens, table, mask, stream);
  MB_LAUNCH_CHECK("cache_write_kernel");
  return MB_OK;
}

extern "C" mb_status mb_cache_read(const mb_kv_cache* cache, const int64_t* slots, int64_t tokens,
                                   void* k_out, void* v_out, mb_dtype out_type,
                                   mb_stream_t stream_) {
  clear_error();
  if (const mb_status st = check_cache(cache); st != MB_OK) return st;
  MB_REQUIRE(slots && k_out && v_out, "cache_read pointers must not be null");
  MB_REQUIRE(dtype_known(out_type), "unknown type of the outputs");
  MB_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16) && aligned(slots, 8),
             "outputs must be 16-byte aligned");
  if (const mb_status st = check_tokens(cache, tokens); st != MB_OK) return st;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const CacheView c = cache_view(cache);
  if (out_type == MB_FP16)
    launch_read<__half>(c, cache->bits, slots, (uint32_t)tokens, k_out, v_out, stream);
  else if (out_type == MB_BF16)
    launch_read<__nv_bfloat16>(c, cache->bits, slots, (uint32_t)tokens, k_out, v_out, stream);
  else
    launch_read<float>(c, cache->bits, slots, (uint32_t)tokens, k_out, v_out, stream);
  MB_LAUNCH_CHECK("cache_read_kernel");
  return MB_OK;
}
