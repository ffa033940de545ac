// Attention of one query token a sequence over the quantised paged cache (no
// counterpart in the reference): out = sum_t softmax_t(scale q . k_t) v_t.
//
// A CTA a (sequence, head); its warps take tokens in turn, a lane holding
// every 32nd channel, with the running maximum and sum of the softmax, and
// join at the end.
#include <cmath>

#include "mb_cache.cuh"

namespace mb {
namespace {

constexpr int kWarps = 8;

template <int BITS>
__device__ __forceinline__ float cache_value(const CacheView& c, int which, int64_t row,
                                             uint32_t ch) {
  if constexpr (BITS == 8) {
    return (float)(int)(int8_t)c.codes[which][row * c.dim + ch] *
           reinterpret_cast<const float*>(c.scales[which])[row];
  } else {
    const uint32_t q = (c.codes[which][row * (c.dim / 2) + ch / 2] >> (4 * (ch & 1))) & 15u;
    const __half2 g = reinterpret_cast<const __half2*>(
        c.scales[which])[row * (c.dim / kGroup4) + ch / kGroup4];
    return fmaf(__low2float(g), (float)q, __high2float(g));
  }
}

template <typename X, int BITS>
__global__ void __launch_bounds__(32 * kWarps)
    cache_attention_kernel(CacheView c, const X* __restrict__ q, int64_t q_batch_stride,
                           int64_t q_head_stride, uint32_t heads,
                           const int32_t* __restrict__ table, int64_t table_stride,
                           int64_t table_width, const int32_t* __restrict__ lengths, float scale,
                           X* __restrict__ out) {
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][256];
  const int64_t b = blockIdx.y;
  const uint32_t h = blockIdx.x, kvh = h / (heads / c.heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float qv[8], o[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t ch = lane + 32 * i;
    qv[i] = ch < c.dim ? to_float<X>(q[b * q_batch_stride + h * q_head_stride + ch]) * scale : 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const int64_t len = min64(lengths[b], table_width * c.page_size);
  for (int64_t t = warp; t < len; t += kWarps) {
    const int64_t page = table[b * table_stride + t / c.page_size];
    if (page < 0 || page >= c.pages) continue;
    const int64_t row = (page * c.heads + kvh) * c.page_size + t % c.page_size;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < c.dim) s = fmaf(qv[i], cache_value<BITS>(c, 0, row, lane + 32 * i), s);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float top = fmaxf(m, s);
    const float keep = m == top ? 1.0f : expf(m - top), p = expf(s - top);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < c.dim)
        o[i] = fmaf(p, cache_value<BITS>(c, 1, row, lane + 32 * i), o[i] * keep);
  }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < kWarps; ++w)
    if (sl[w] != 0.0f) top = fmaxf(top, sm[w]);
  for (int w = 0; w < kWarps; ++w)
    if (sl[w] != 0.0f) sum += sl[w] * expf(sm[w] - top);
  for (uint32_t ch = threadIdx.x; ch < c.dim; ch += 32 * kWarps) {
    float y = 0.0f;
    for (int w = 0; w < kWarps; ++w)
      if (sl[w] != 0.0f) y += so[w][ch] * expf(sm[w] - top);
    out[(b * heads + h) * c.dim + ch] = from_float<X>(sum != 0.0f ? y / sum : 0.0f);
  }
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" size_t mb_cache_attention_workspace_size(const mb_kv_cache* cache, int64_t batch,
                                                    int64_t heads, int64_t table_width) {
  (void)cache, (void)batch, (void)heads, (void)table_width;
  return 0;
}

extern "C" mb_status mb_cache_attention(const mb_kv_cache* cache, const void* q,
                                        int64_t q_batch_stride, int64_t q_head_stride,
                                        mb_dtype type, int64_t batch, int64_t heads,
                                        const int32_t* page_table, int64_t table_stride,
                                        int64_t table_width, const int32_t* lengths, float scale,
                                        void* out, void* workspace, size_t workspace_bytes,
                                        mb_stream_t stream_) {
  (void)workspace, (void)workspace_bytes;
  clear_error();
  if (const mb_status st = check_cache(cache); st != MB_OK) return st;
  MB_REQUIRE(q && lengths && out && (page_table || table_width == 0),
             "cache_attention pointers must not be null");
  MB_REQUIRE(type == MB_FP16 || type == MB_BF16, "q must be fp16 or bf16");
  MB_REQUIRE(batch > 0 && batch <= 65535, "batch must be 1 to 65535");
  MB_REQUIRE(heads > 0 && heads % cache->kv_heads == 0 && heads <= 65535,
             "heads must be a multiple of kv_heads up to 65535");
  MB_REQUIRE(table_width >= 0, "table_width must not be negative");
  MB_REQUIRE(std::isfinite(scale), "scale must be finite");
  MB_REQUIRE(aligned(q, 2) && aligned(out, 2) && aligned(page_table, 4) && aligned(lengths, 4),
             "misaligned q, out, page_table or lengths");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const CacheView c = cache_view(cache);
  const dim3 grid((unsigned)heads, (unsigned)batch);
  const auto go = [&](auto* typed, auto kernel) {
    using X = std::remove_pointer_t<decltype(typed)>;
    kernel<<<grid, 32 * kWarps, 0, stream>>>(c, static_cast<const X*>(q), q_batch_stride,
                                             q_head_stride, (uint32_t)heads, page_table,
                                             table_stride, table_width, lengths, scale, typed);
  };
  if (type == MB_FP16) {
    auto* o = static_cast<__half*>(out);
    cache->bits == 8 ? go(o, cache_attention_kernel<__half, 8>)
                     : go(o, cache_attention_kernel<__half, 4>);
  } else {
    auto* o = static_cast<__nv_bfloat16*>(out);
    cache->bits == 8 ? go(o, cache_attention_kernel<__nv_bfloat16, 8>)
                     : go(o, cache_attention_kernel<__nv_bfloat16, 4>);
  }
  MB_LAUNCH_CHECK("cache_attention_kernel");
  return MB_OK;
}
