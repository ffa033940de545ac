// Keys and values quantised to 8 or 4 bits as they are written into a paged
// cache, and read back (no counterpart in the reference).
//
// A CTA takes a few tokens: first the row of each in the cache (and, writing,
// whether a later token has the same slot), then the tokens' heads.  A head's
// row is taken by the 2 .. 32 lanes that hold its channels, eight a lane: a
// 16-byte load, the maximum (8 bits: of the row) or minimum and maximum (4
// bits: of 32 channels, four lanes) by shuffles, and one 8- or 4-byte store.
// Bound by memory: 2 bytes in and 1 or 0.63 out a value; at usual sizes by the
// chain of loads (slot, row, codes), by the slots that each writing CTA looks
// through, and by the launches: 2048 tokens of 8 heads of 128 channels written and
// 8000 read (4 bits) in 20.9 us as two calls in turn, where their bytes take 1.7 and
// 6.7 (under ncu, with cold caches, 11.7 and 12.9).
#include <algorithm>

#include "mb_cache.cuh"
#include "mb_tma.cuh"

namespace mb {
namespace {

// Which token of a slot is kept: up to kOwnTokens tokens, each writing CTA looks
// through the later tokens' slots itself; up to kScanTokens a kernel before
// does so for 32 tokens a CTA; above, where that reads too much, a table says
// which token a slot belongs to (two launches more).  The kernels leave each
// token's first row in the workspace.
// 2048 tokens (8000 read, 4 bits): 20.2 us themselves, 23.6 with the kernel; 8192
// tokens (8 bits): 46 and 42.6.
constexpr int64_t kOwnTokens = 2048, kScanTokens = 16384;
constexpr uint32_t kThreads = 256;
constexpr uint32_t kMostTokens = 4;  // of a CTA
constexpr uint32_t kTurns = 4;       // of a CTA over its tokens' lanes

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
__global__ void __launch_bounds__(kThreads)
    cache_claim_kernel(const int64_t* __restrict__ slots, uint32_t tokens, int64_t n_slots,
                       unsigned long long* __restrict__ table, uint32_t mask) {
  const uint32_t t = blockIdx.x * kThreads + threadIdx.x;
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
  bool vec;
};

// How the work is cut: `tokens` a CTA; a token has 2 heads rows of 2^shift
// lanes (at least dim / 8); a CTA's lanes are dealt to gridDim.y CTAs.
struct Cut {
  uint32_t tokens, shift, heads;  // lanes a row: 2^shift
  uint32_t inverse;               // 2^32 / (2 heads), up: divides what is below 2^16
};
struct Place {
  uint32_t token, which, head, lane;
};
__device__ __forceinline__ Place place_of(uint32_t x, const Cut& cut) {
  Place p;
  const uint32_t row = x >> cut.shift;
  p.lane = x - (row << cut.shift);
  p.token = __umulhi(row, cut.inverse);
  const uint32_t in = row - p.token * 2 * cut.heads;
  p.which = in >= cut.heads;
  p.head = in - (p.which ? cut.heads : 0u);
  return p;
}

// A slot in 32 bits (those of a cache fit), others as one that no cache has.
constexpr uint32_t kNoKey = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t key_of(int64_t slot) {
  return (uint64_t)slot >> 32 == 0 ? (uint32_t)slot : kNoKey;
}

// First row (head 0) of a slot, -1 outside the cache.
__device__ __forceinline__ int64_t first_row(const CacheView& c, int64_t slot) {
  return slot >= 0 && slot < cache_slots(c) ? cache_row(c, (uint32_t)slot, 0) : -1;
}

// Every token's first row, -1 where it is not written.  table: from
// cache_claim_kernel, or null: later tokens are looked through, most of them
// only against a bit that says whether one of the CTA's slots has their hash.
constexpr uint32_t kScanOwn = 32, kScanBits = 2048;
__global__ void __launch_bounds__(kThreads)
    cache_rows_kernel(CacheView c, const int64_t* __restrict__ slots, uint32_t tokens,
                      const unsigned long long* __restrict__ table, uint32_t mask,
                      int64_t* __restrict__ rows) {
  grid_dependency_wait();
  grid_launch_dependents();  // the writing kernel begins with the values
  if (table != nullptr) {
    const uint32_t t = blockIdx.x * kThreads + threadIdx.x;
    if (t >= tokens) return;
    const int64_t slot = slots[t], row = first_row(c, slot);
    rows[t] = row >= 0 && claimed(table, mask, (uint32_t)slot, t) ? row : -1;
    return;
  }
  __shared__ uint32_t bits[kScanBits / 32], own[kScanOwn];
  __shared__ int64_t first[kScanOwn];
  const uint32_t t0 = blockIdx.x * kScanOwn, here = min(kScanOwn, tokens - t0);
  if (threadIdx.x < kScanBits / 32) bits[threadIdx.x] = 0;
  __syncthreads();
  if (threadIdx.x < here) {
    const int64_t slot = slots[t0 + threadIdx.x];
    const uint32_t key = key_of(slot);
    own[threadIdx.x] = key;
    first[threadIdx.x] = first_row(c, slot);
    if (key != kNoKey) atomicOr(&bits[key % kScanBits / 32], 1u << key % 32);
  }
  __syncthreads();
#pragma unroll 8
  for (uint32_t o = t0 + 1 + threadIdx.x; o < tokens; o += kThreads) {
    const uint32_t key = key_of(slots[o]);
    if (key == kNoKey || (bits[key % kScanBits / 32] >> key % 32 & 1u) == 0) continue;
    for (uint32_t k = 0; k < here; ++k)
      if (key == own[k] && o > t0 + k) first[k] = -1;
  }
  __syncthreads();
  if (threadIdx.x < here) rows[t0 + threadIdx.x] = first[threadIdx.x];
}

// kVec: 16-byte loads.
template <typename X, int BITS, bool kVec>
__global__ void __launch_bounds__(kThreads)
    cache_write_kernel(CacheView c, KvSource src, const int64_t* __restrict__ slots,
                       uint32_t tokens, Cut cut, const int64_t* __restrict__ first_rows) {
  __shared__ int64_t rows[kMostTokens];
  __shared__ uint32_t mine[kMostTokens];
  const uint32_t t0 = blockIdx.x * cut.tokens, here = min(cut.tokens, tokens - t0);
  const uint32_t lanes = (here * 2 * cut.heads) << cut.shift;
  if (first_rows == nullptr) grid_dependency_wait();
  // the values are on the way while the slots are looked at
  Raw8<X> raw[kTurns];
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) {
    const uint32_t x = (blockIdx.y + i * gridDim.y) * kThreads + threadIdx.x;
    const Place p = place_of(x, cut);
    if (x < lanes && 8 * p.lane < c.dim)
      raw[i].load(static_cast<const X*>(p.which ? src.data[1] : src.data[0]) +
                      (t0 + p.token) * (p.which ? src.token_stride[1] : src.token_stride[0]) +
                      p.head * (p.which ? src.head_stride[1] : src.head_stride[0]) + 8 * p.lane,
                  kVec, 8);
  }
  if (first_rows != nullptr) {
    grid_dependency_wait();
    if (threadIdx.x < here) rows[threadIdx.x] = first_rows[t0 + threadIdx.x];
    __syncthreads();
  } else {  // the last token with a slot is the one that is kept
    if (threadIdx.x < here) {
      const int64_t slot = slots[t0 + threadIdx.x];
      rows[threadIdx.x] = first_row(c, slot);
      mine[threadIdx.x] = key_of(slot);
    }
    __syncthreads();
    uint32_t own[kMostTokens];
#pragma unroll
    for (uint32_t k = 0; k < kMostTokens; ++k) own[k] = k < here ? mine[k] : kNoKey;
#pragma unroll 4
    for (uint32_t o = t0 + 1 + threadIdx.x; o < tokens; o += kThreads) {
      const uint32_t key = key_of(slots[o]);
      if (key == kNoKey) continue;
#pragma unroll
      for (uint32_t k = 0; k < kMostTokens; ++k)
        if (key == own[k] && o > t0 + k) rows[k] = -1;
    }
    __syncthreads();
  }
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) {
    const uint32_t x = (blockIdx.y + i * gridDim.y) * kThreads + threadIdx.x;
    if (x - threadIdx.x >= lanes) break;  // the whole CTA
    const Place p = place_of(x, cut);
    const int64_t first = x < lanes ? rows[p.token] : -1;
    const bool holds = first >= 0 && 8 * p.lane < c.dim;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (holds) raw[i].floats(v);
    const int64_t row = first + (int64_t)p.head * c.page_size;
    uint8_t* codes = p.which ? c.codes[1] : c.codes[0];
    uint8_t* scales = p.which ? c.scales[1] : c.scales[0];
    if constexpr (BITS == 8) {
      uint32_t m = abs_bits_max(v);
      for (uint32_t o = 1u << cut.shift >> 1; o > 0; o >>= 1)
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (!holds) continue;
      const RowScale s = row_scale(m);
      *reinterpret_cast<uint2*>(codes + row * c.dim + 8 * p.lane) = codes8(v, s);
      if (p.lane == 0) reinterpret_cast<float*>(scales)[row] = s.scale;
    } else {
      // fminf and fmaxf pass over a NaN: carry it by a sum of its own
      float lo = v[0], hi = v[0], bad = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
        bad = fmaf(v[i], 0.0f, bad);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad += __shfl_xor_sync(0xffffffffu, bad, o);
      }
      if (!holds) continue;
      const GroupScale g = group_scale(lo + bad, hi + bad);
      *reinterpret_cast<uint32_t*>(codes + row * (c.dim / 2) + 4 * p.lane) = codes4(v, g);
      if (p.lane % 4 == 0)
        reinterpret_cast<__half2*>(scales)[row * (c.dim / kGroup4) + p.lane / 4] =
            __halves2half2(g.scale, g.low);
    }
  }
}

template <typename Y, int BITS>
__global__ void __launch_bounds__(kThreads)
    cache_read_kernel(CacheView c, const int64_t* __restrict__ slots, uint32_t tokens, Cut cut,
                      Y* __restrict__ k_out, Y* __restrict__ v_out) {
  __shared__ int64_t rows[kMostTokens];
  const uint32_t t0 = blockIdx.x * cut.tokens, here = min(cut.tokens, tokens - t0);
  grid_dependency_wait();
  if (threadIdx.x < here) rows[threadIdx.x] = first_row(c, slots[t0 + threadIdx.x]);
  __syncthreads();
  const uint32_t lanes = (here * 2 * cut.heads) << cut.shift;
  // eight codes and their scale (4 bits: and minimum) of each turn, then the values
  uint2 q[kTurns];
  uint32_t scale[kTurns];
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) {
    const uint32_t x = (blockIdx.y + i * gridDim.y) * kThreads + threadIdx.x;
    const Place p = place_of(x, cut);
    q[i] = make_uint2(0u, 0u);
    scale[i] = 0u;
    if (x >= lanes || 8 * p.lane >= c.dim || rows[p.token] < 0) continue;
    const int64_t row = rows[p.token] + (int64_t)p.head * c.page_size;
    const uint8_t* codes = p.which ? c.codes[1] : c.codes[0];
    const uint32_t* scales =
        reinterpret_cast<const uint32_t*>(p.which ? c.scales[1] : c.scales[0]);
    if constexpr (BITS == 8) {
      q[i] = *reinterpret_cast<const uint2*>(codes + row * c.dim + 8 * p.lane);
      scale[i] = scales[row];
    } else {
      q[i].x = *reinterpret_cast<const uint32_t*>(codes + row * (c.dim / 2) + 4 * p.lane);
      scale[i] = scales[row * (c.dim / kGroup4) + p.lane / 4];
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kTurns; ++i) {
    const uint32_t x = (blockIdx.y + i * gridDim.y) * kThreads + threadIdx.x;
    const Place p = place_of(x, cut);
    if (x >= lanes || 8 * p.lane >= c.dim) continue;
    float v[8];
    if constexpr (BITS == 8) {
      const float s = __uint_as_float(scale[i]);
      // 2^23 + 128 + code from the code's byte, less 2^23 + 128
      const uint32_t w[2] = {q[i].x ^ 0x80808080u, q[i].y ^ 0x80808080u};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = __fmul_rn(
            __uint_as_float(__byte_perm(w[e / 4], 0x4B000000u, 0x7440 + (e & 3))) - 8388736.0f, s);
    } else {
      const __half2 g = *reinterpret_cast<const __half2*>(&scale[i]);
      const float s = __low2float(g), m = __high2float(g);
      // s * code is exact in fp32: 11 + 4 bits; the code from 2^23 + code
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = fmaf(s, __uint_as_float(((q[i].x >> (4 * e)) & 15u) | 0x4B000000u) - 8388608.0f, m);
    }
    store8((p.which ? v_out : k_out) + ((int64_t)(t0 + p.token) * c.heads + p.head) * c.dim +
               8 * p.lane,
           v);
  }
}

inline uint32_t row_shift(uint32_t dim) {
  uint32_t w = 2;
  while (8u << w < dim) ++w;
  return w;
}

// As many tokens a CTA as fill its turns; fewer, and a token's heads over
// several CTAs, where there are not enough for the GPU or a token has more.
struct Launch {
  Cut cut;
  dim3 grid;
};
inline Launch launch_for(const CacheView& c, uint32_t tokens) {
  Launch l;
  l.cut.shift = row_shift(c.dim);
  l.cut.heads = c.heads;
  l.cut.inverse = (uint32_t)((((uint64_t)1 << 32) + 2 * c.heads - 1) / (2 * c.heads));
  const uint32_t lanes = 2 * c.heads << l.cut.shift;  // of a token
  uint32_t n = std::max(1u, kTurns * kThreads / lanes);
  n = std::min(n, std::max(1u, tokens / (4 * 148)));
  l.cut.tokens = std::min(n, kMostTokens);
  l.grid.x = (unsigned)ceil_div(tokens, l.cut.tokens);
  const uint32_t turns = (uint32_t)ceil_div((int64_t)l.cut.tokens * lanes, kThreads);
  l.grid.y = std::max((turns + kTurns - 1) / kTurns,
                      std::min(turns, std::max(1u, 4 * 148 / l.grid.x)));
  return l;
}

template <typename X>
mb_status launch_write(const CacheView& c, int bits, const KvSource& src, const int64_t* slots,
                       uint32_t tokens, const int64_t* rows, cudaStream_t stream) {
  const Launch l = launch_for(c, tokens);
  const auto go = [&](auto kernel) {
    return launch_dependent(kernel, l.grid, kThreads, 0, stream, c, src, slots, tokens, l.cut,
                            rows);
  };
  if (bits == 8)
    MB_CUDA_TRY(src.vec ? go(cache_write_kernel<X, 8, true>) : go(cache_write_kernel<X, 8, false>));
  else
    MB_CUDA_TRY(src.vec ? go(cache_write_kernel<X, 4, true>) : go(cache_write_kernel<X, 4, false>));
  return MB_OK;
}

template <typename Y>
void launch_read(const CacheView& c, int bits, const int64_t* slots, uint32_t tokens, void* k,
                 void* v, cudaStream_t stream) {
  const Launch l = launch_for(c, tokens);
  if (bits == 8)
    launch_dependent(cache_read_kernel<Y, 8>, l.grid, kThreads, 0, stream, c, slots, tokens, l.cut,
                     static_cast<Y*>(k), static_cast<Y*>(v));
  else
    launch_dependent(cache_read_kernel<Y, 4>, l.grid, kThreads, 0, stream, c, slots, tokens, l.cut,
                     static_cast<Y*>(k), static_cast<Y*>(v));
}

mb_status check_tokens(int64_t tokens) {
  MB_REQUIRE(tokens > 0, "tokens must be positive");
  MB_REQUIRE(tokens < (int64_t(1) << 30), "too many tokens");
  return MB_OK;
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" size_t mb_cache_write_workspace_size(int64_t tokens) {
  if (tokens <= kOwnTokens || tokens >= (int64_t(1) << 30)) return 0;
  return (size_t)tokens * 8 + (tokens > kScanTokens ? (size_t)claim_entries(tokens) * 8 : 0);
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
  if (const mb_status st = check_tokens(tokens); st != MB_OK) return st;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const CacheView c = cache_view(cache);
  const auto vec = [&](const void* p, int64_t ts, int64_t hs) {
    return aligned(p, 16) && (tokens == 1 || ts % 8 == 0) && (c.heads == 1 || hs % 8 == 0);
  };
  const KvSource src{{k, v},
                     {k_token_stride, v_token_stride},
                     {k_head_stride, v_head_stride},
                     vec(k, k_token_stride, k_head_stride) &&
                         vec(v, v_token_stride, v_head_stride)};
  int64_t* rows = nullptr;
  if (tokens > kOwnTokens) {
    if (workspace == nullptr || workspace_bytes < mb_cache_write_workspace_size(tokens) ||
        !aligned(workspace, 8))
      return set_error(MB_ERR_WORKSPACE, "cache_write workspace missing, misaligned or too small");
    rows = static_cast<int64_t*>(workspace);
    unsigned long long* table = nullptr;
    uint32_t mask = 0;
    unsigned grid = (unsigned)ceil_div(tokens, kScanOwn);
    if (tokens > kScanTokens) {
      table = reinterpret_cast<unsigned long long*>(rows + tokens);
      mask = claim_entries(tokens) - 1;
      MB_CUDA_TRY(cudaMemsetAsync(table, 0, ((size_t)mask + 1) * 8, stream));
      grid = (unsigned)ceil_div(tokens, kThreads);
      cache_claim_kernel<<<grid, kThreads, 0, stream>>>(slots, (uint32_t)tokens, cache_slots(c),
                                                        table, mask);
      MB_LAUNCH_CHECK("cache_claim_kernel");
    }
    MB_CUDA_TRY(launch_dependent(cache_rows_kernel, grid, kThreads, 0, stream, c, slots,
                                 (uint32_t)tokens, table, mask, rows));
  }
  return type == MB_FP16 ? launch_write<__half>(c, cache->bits, src, slots, (uint32_t)tokens, rows,
                                                stream)
                         : launch_write<__nv_bfloat16>(c, cache->bits, src, slots,
                                                       (uint32_t)tokens, rows, stream);
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
  if (const mb_status st = check_tokens(tokens); st != MB_OK) return st;
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
