// out = (a_scales b_scales^T) o (A B^T) + bias for 8-bit codes A (tokens) and
// B (weights, an output channel a row), on the tcgen05 tensor cores: the sums
// are whole numbers, exact in int32 (127^2 K < 2^31), scaled once at the end.
//
// The weights are the 128-row operand (accumulator row = TMEM lane = output
// channel), the tokens the columns, so the same kernel serves one token and
// thousands: a tile is 128 channels by kN tokens.  Both operands are read by
// TMA in 128-byte steps of K with the 128-byte swizzle ("K-major"); rows and
// columns past the matrices read 0.  A warp issues the loads, a warp the
// products, and the four warps then drain the accumulator: a thread owns a
// channel, so its scale and bias are registers and a warp writes 32
// consecutive channels of a token.
//
// Few tiles (few tokens): K is split over the CTAs of a cluster, which add
// their int32 parts through distributed shared memory -- whole numbers, so
// the result does not depend on the split.
//
// One token is bound by what comes one after another: 4096 x 4096 takes 8.2 us, 2
// of them the quantising launch, the others set-up, the weights (131 KB for each
// of 128 CTAs, 1.5 to 1.8 us at the 75 to 90 GB/s that one SM takes in), the join
// over the cluster and the drain.  11008 x 4096 at 48 tokens takes 15.6 us, bound by
// that intake: 790 KB for each of the 86 SMs that have a tile.  Thousands of
// tokens are bound by the tensor cores and, back to back, by the card's power: 8192
// x 11008 x 4096 takes 277 us in a replayed graph, 2.7e15 operations a second, 322 us
// a call, 2.3e15 (the pipe is busy for 71 % of a launch alone).
#include <algorithm>
#include <cstring>

#include "mb_codes.cuh"
#include "mb_tma.cuh"

namespace mb {
namespace {

constexpr int kChannels = 128;            // tile rows: output channels
constexpr int kStepK = 128;               // bytes of K a stage
constexpr int kWeightBytes = kChannels * kStepK;
constexpr int kThreads = 192;             // warps 0-3 drain, 4 loads, 5 multiplies

// Shared memory of a tile of kN tokens: a ring of stages (128 bytes of K of
// both operands), whose memory the int32 parts of a split reuse (128
// channels by kN tokens and padding).
template <int kN>
struct Shape {
  static constexpr int kStage = kWeightBytes + kN * kStepK;
  static constexpr uint32_t kTmem = kN < 32 ? 32 : kN;
  static constexpr int smem(int stages) { return stages * kStage + 1024; }
  static constexpr int kLeast = ((kN + 4) * kChannels * 4 + kStage - 1) / kStage;  // stages
};
constexpr int kMaxStages = 12;
constexpr uint32_t kMostParts = 8;  // of K: a portable cluster
// A CTA's shared memory, less what is declared statically.  CTAs of a cluster wait
// for one another, and each for its TMEM columns: two clusters that share two
// SMs, each with the columns on one that the other waits for on the second, would
// never end.  So a CTA of a cluster takes so much shared memory that no second one
// for whose columns there is no room comes beside it: a pair's, with all 512, all
// of it, the others, with 256 at most, half of it at least (all would leave too few
// places for clusters of eight: 8 x 2048 x 2048 10.9 us instead of 7.0).  Lone CTAs
// wait for no other.
constexpr int kMostSmem = 227 * 1024 - 2048;
constexpr int kSms = 148;

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// Shared-memory descriptor of a K-major operand written by TMA with the
// 128-byte swizzle: rows of 128 bytes, 8-row atoms of 1024 bytes.
__device__ __forceinline__ uint64_t umma_desc_k_sw128(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)1 << 16;                         // (unused with this swizzle)
  d |= (uint64_t)((1024u >> 4) & 0x3FFFu) << 32;  // between 8-row groups
  d |= (uint64_t)1 << 46;                         // descriptor version (sm_100)
  d |= (uint64_t)2 << 61;                         // 128-byte swizzle
  return d;
}

// Instruction descriptor, kind::i8: int32 accumulate, signed 8-bit operands,
// both K-major, M = 128.
__host__ __device__ constexpr uint32_t int8_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kChannels >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory address of the same place in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t cluster_address(uint32_t saddr, uint32_t rank) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(saddr), "r"(rank));
  return d;
}
__device__ __forceinline__ uint32_t load_cluster(uint32_t saddr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(saddr) : "memory");
  return v;
}
__device__ __forceinline__ int4 load_cluster4(uint32_t saddr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(saddr)
               : "memory");
  return v;
}

struct Epilogue {
  const float* a_scales;
  const float* b_scales;
  const void* bias;
  void* out;
  int64_t out_stride;
  int bias_type;
};

__device__ __forceinline__ float bias_at(const Epilogue& e, int64_t n) {
  if (e.bias == nullptr) return 0.0f;
  return e.bias_type == MB_FP16   ? __half2float(static_cast<const __half*>(e.bias)[n])
         : e.bias_type == MB_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(e.bias)[n])
                                  : static_cast<const float*>(e.bias)[n];
}

// The sum times the token's scale is at most 2^31 times it: past this scale it
// may be infinite, below the smallest normal scale lose bits, where the result
// is an ordinary number.
__device__ __forceinline__ bool extreme(float sa) {
  return sa > 0x1p96f || (sa > 0.0f && sa < 0x1p-126f);
}
__device__ __forceinline__ float scaled(int sum, float sa, float sb, float bias) {
  return fmaf(__fmul_rn((float)sum, sa), sb, bias);
}
// In 64 bits where the token's scale is extreme: of a tile that has such a token
// (the others' results do not depend on it).
__device__ __noinline__ float scaled_any(int sum, float sa, float sb, float bias) {
  return extreme(sa) ? __double2float_rn(fma((double)sum * (double)sa, (double)sb, (double)bias))
                     : scaled(sum, sa, sb, bias);
}

// A channel's (a lane's) sums with 16 tokens, `count` of which exist: sa in
// shared memory (16-byte aligned), o the first token's place, the tokens
// `stride` apart.  A warp writes 32 consecutive channels a token.
template <typename Y>
__device__ __forceinline__ void put16(const uint32_t (&v)[16], const float* sa, float sb,
                                      float bias, bool wide, Y* o, int64_t stride, int count) {
  if (wide) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < count) o[i * stride] = from_float<Y>(scaled_any((int)v[i], sa[i], sb, bias));
  } else if (count >= 16) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const float4 s = *reinterpret_cast<const float4*>(sa + i);
      o[0] = from_float<Y>(scaled((int)v[i], s.x, sb, bias));
      o += stride;
      o[0] = from_float<Y>(scaled((int)v[i + 1], s.y, sb, bias));
      o += stride;
      o[0] = from_float<Y>(scaled((int)v[i + 2], s.z, sb, bias));
      o += stride;
      o[0] = from_float<Y>(scaled((int)v[i + 3], s.w, sb, bias));
      o += stride;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < count) o[i * stride] = from_float<Y>(scaled((int)v[i], sa[i], sb, bias));
  }
}

// Grid: x = cluster (a tile's K parts) fastest, then channel tiles; y = token
// tiles.
template <int kN, typename Y>
__global__ void __launch_bounds__(kThreads, 1)
    int8_matmul_kernel(const __grid_constant__ CUtensorMap tokens,
                       const __grid_constant__ CUtensorMap weights, int64_t M, int64_t N,
                       int64_t K, int stages, Epilogue e) {
  using S = Shape<kN>;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                             ~(uintptr_t)1023);
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], done;
  __shared__ uint32_t tmem_slot, failed;
  __shared__ __align__(16) float a_scale[kN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t parts = cluster_size(), part = cluster_rank();
  const int64_t n0 = (int64_t)(blockIdx.x / parts) * kChannels, m0 = (int64_t)blockIdx.y * kN;
  const int all = (int)ceil_div(K, kStepK);
  const int k0 = (int)((int64_t)all * part / parts), k1 = (int)((int64_t)all * (part + 1) / parts);
  const int steps = k1 - k0;

  const auto weights_of = [&](int i, int s) {
    mbar_arrive_expect_tx(&full[s], S::kStage);
    tma_load_2d(ring + s * S::kStage, &weights, &full[s], (k0 + i) * kStepK, (int)n0);
  };
  int first = 0;  // steps whose weights are on the way
  if (warp == 4 && lane == 0) {
    prefetch_map(&weights);
    prefetch_map(&tokens);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&done, 1);
    failed = 0;
    fence_mbar_init();
    // the weights wait neither for this CTA's other warps nor for the kernel
    // that quantises the tokens
    for (; first < steps && first < stages; ++first) weights_of(first, first);
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(S::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;

  if (warp == 4 && lane == 0) {
    const auto tokens_of = [&](int i, int s) {
      tma_load_2d(ring + s * S::kStage + kWeightBytes, &tokens, &full[s], (k0 + i) * kStepK,
                  (int)m0);
    };
    int i = first;
    grid_dependency_wait();
    for (int f = 0; f < i; ++f) tokens_of(f, f);
    int s = i == stages ? 0 : i;
    uint32_t phase = 0;
    for (; i < steps; ++i) {
      if (!mbar_wait(&empty[s], phase)) {
        atomicExch(&failed, 1u);
        break;
      }
      weights_of(i, s);
      tokens_of(i, s);
      if (++s == stages) s = 0, phase ^= 1u;
    }
    // every load has landed before the CTA can exit or reuse the ring
    for (int f = max(0, i - stages); f < i; ++f)
      if (!mbar_wait(&full[f % stages], (uint32_t)((f / stages) & 1))) atomicExch(&failed, 1u);
  } else if (warp == 5 && lane == 0) {
    int s = 0;
    uint32_t phase = 0;
    for (int i = 0; i < steps; ++i) {
      if (!mbar_wait(&full[s], phase)) {
        atomicExch(&failed, 1u);
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t w = smem_u32(ring + s * S::kStage), t = w + kWeightBytes;
#pragma unroll
      for (int k = 0; k < kStepK / 32; ++k)
        umma_i8(tmem, umma_desc_k_sw128(w + 32 * k), umma_desc_k_sw128(t + 32 * k),
                int8_idesc(kN), (i > 0 || k > 0) ? 1u : 0u);
      umma_commit(&empty[s]);
      if (++s == stages) s = 0, phase ^= 1u;
    }
    umma_commit(&done);
  }
  __syncwarp();
  const int64_t n = n0 + 32 * warp + lane;  // warps 0-3: this thread's channel
  const bool live = warp < 4 && n < N;
  float sb = live ? e.b_scales[n] : 0.0f;
  const float bias = live ? bias_at(e, n) : 0.0f;
  grid_dependency_wait();
  bool wide = false;
  if (warp < 4)
    for (int i = threadIdx.x; i < kN; i += 128) {
      const float sa = m0 + i < M ? e.a_scales[m0 + i] : 0.0f;
      a_scale[i] = sa;
      wide |= extreme(sa);
    }
  if (!mbar_wait(&done, 0)) atomicExch(&failed, 1u);
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  wide = __syncthreads_or(wide) != 0;  // `failed` is final; the ring is free

  const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
  const int columns = (int)min64(kN, M - m0);
  Y* o = static_cast<Y*>(e.out) + m0 * e.out_stride + n;
  if (parts == 1) {
    if (failed) sb = __uint_as_float(0x7FC00000u);
    if (warp < 4) {
#pragma unroll 1
      for (int c = 0; c < columns; c += 16) {
        uint32_t v[16];
        __syncwarp();
        tmem_ld16(lanes + c, v);
        if (live)
          put16<Y>(v, a_scale + c, sb, bias, wide, o + c * e.out_stride, e.out_stride,
                   columns - c);
      }
    }
  } else {
    // a channel's sums in a row; the rows' length keeps 16-byte accesses of
    // neighbouring channels apart
    constexpr int kRow = kN + 4;
    int* own = reinterpret_cast<int*>(ring) + (32 * (warp & 3) + lane) * kRow;
    if (warp < 4) {
#pragma unroll 1
      for (int c = 0; c < columns; c += 16) {
        uint32_t v[16];
        tmem_ld16(lanes + c, v);
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<int4*>(own + c + i) =
              make_int4((int)v[i], (int)v[i + 1], (int)v[i + 2], (int)v[i + 3]);
      }
    }
    cluster_sync();
    const uint32_t base = smem_u32(own), fail = smem_u32(&failed);
    for (uint32_t r = 0; r < parts; ++r)
      if (load_cluster(cluster_address(fail, r)) != 0) sb = __uint_as_float(0x7FC00000u);
    // this CTA's share of the tile's tokens, four at a time, a channel a thread
    if (live) {
      for (int c = 4 * (int)part; c < columns; c += 4 * (int)parts) {
        int4 v[kMostParts];
#pragma unroll
        for (uint32_t r = 0; r < kMostParts; ++r)
          if (r < parts) v[r] = load_cluster4(cluster_address(base + 4 * c, r));
        int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll
        for (uint32_t r = 0; r < kMostParts; ++r)
          if (r < parts) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
        const float4 sa = *reinterpret_cast<const float4*>(a_scale + c);
        Y* to = o + c * e.out_stride;
        const auto y = [&](int x, float s) {
          return from_float<Y>(wide ? scaled_any(x, s, sb, bias) : scaled(x, s, sb, bias));
        };
        to[0] = y(sum.x, sa.x);
        if (c + 1 < columns) to[e.out_stride] = y(sum.y, sa.y);
        if (c + 2 < columns) to[2 * e.out_stride] = y(sum.z, sa.z);
        if (c + 3 < columns) to[3 * e.out_stride] = y(sum.w, sa.w);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its part
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(S::kTmem));
}

// ---------------------------------------------------------------------------
// Many tokens: pairs of CTAs (tcgen05 cta_group::2), persistent.
// ---------------------------------------------------------------------------
// A pair's tile is 256 channels by 256 tokens; each CTA loads its 128
// channels and half of the tokens, and keeps the sums of its channels with
// all 256 tokens (256 TMEM columns, twice: the products of the next tile run
// while the last one is drained).  A stage is 32 KB a CTA instead of the 48
// KB of a lone CTA's 128 x 256 tile: shared memory is read 8 KB (the 128
// weights' 32 bytes, half the tokens') instead of 12 for the same products.
constexpr int kPairTokens = 256;                       // tokens a tile
constexpr int kPairStage = kWeightBytes + kPairTokens / 2 * kStepK;  // of one CTA
constexpr int kPairStages = 6;
// All that a CTA can have, although its ring needs less: see kMostSmem.
constexpr int kPairSmem = kMostSmem - 2048;
static_assert(kPairSmem >= kPairStages * kPairStage + 1024, "the ring does not fit");
constexpr int kPairGroup = 8;                          // token tiles taken together

__host__ __device__ constexpr uint32_t pair_idesc() {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kPairTokens >> 3) << 17) |
         ((uint32_t)(2 * kChannels >> 4) << 24);
}

// A load whose bytes count on the pair's first CTA's barrier.
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, uint32_t bar, int x,
                                          int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void pair_umma_i8(uint32_t tmem_d, uint64_t a, uint64_t b,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(a), "l"(b), "r"(pair_idesc()), "r"(accumulate));
}

// Arrives on the barrier of both CTAs once the products issued so far are done.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

// Barrier of the four warps that drain; whether any of their threads says so.
__device__ __forceinline__ bool drain_warps_or(bool x) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)x)
      : "memory");
  return any != 0;
}

// Tile -> (channel tile, token tile): kPairGroup token tiles by all channel
// tiles, tokens fastest, so that the tiles in flight share operands in L2.
__device__ __forceinline__ void pair_tile(uint32_t t, uint32_t channel_tiles, uint32_t token_tiles,
                                          uint32_t& cn, uint32_t& cm) {
  const uint32_t per = channel_tiles * kPairGroup, group = t / per, in = t - group * per;
  const uint32_t first = group * kPairGroup, high = min(token_tiles - first, (uint32_t)kPairGroup);
  cn = in / high;
  cm = first + in - cn * high;
}

template <typename Y>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    int8_matmul_pair_kernel(const __grid_constant__ CUtensorMap tokens,
                            const __grid_constant__ CUtensorMap weights, int64_t M, int64_t N,
                            int64_t K, Epilogue e) {
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) &
                                             ~(uintptr_t)1023);
  __shared__ uint64_t full[kPairStages], empty[kPairStages], drain[2], drained[2];
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(16) float a_scale[2][kPairTokens];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t channel_tiles = (uint32_t)ceil_div(N, 2 * kChannels);
  const uint32_t token_tiles = (uint32_t)ceil_div(M, kPairTokens);
  const uint32_t tiles = channel_tiles * token_tiles;
  const uint32_t first = blockIdx.x / 2, stride = gridDim.x / 2;
  const int steps = (int)ceil_div(K, kStepK);

  if (threadIdx.x == 0) {
    prefetch_map(&weights);
    prefetch_map(&tokens);
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&drain[i], 1);
      mbar_init(&drained[i], 8);  // four warps of both CTAs
    }
    fence_mbar_init();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&tmem_slot)),
                 "r"(2 * kPairTokens));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;

  grid_dependency_wait();
  if (warp == 4 && lane == 0) {
    int i = 0;
    bool ok = true;
    for (uint32_t t = first; t < tiles && ok; t += stride) {
      uint32_t cn, cm;
      pair_tile(t, channel_tiles, token_tiles, cn, cm);
      const int n0 = (int)(cn * 2 + rank) * kChannels;
      const int m0 = (int)(cm * kPairTokens + rank * (kPairTokens / 2));
      for (int k = 0; k < steps; ++k, ++i) {
        const int s = i % kPairStages;
        if (i >= kPairStages && !mbar_wait(&empty[s], (uint32_t)((i / kPairStages - 1) & 1))) {
          ok = false;
          break;
        }
        uint8_t* at = ring + s * kPairStage;
        const uint32_t bar = cluster_address(smem_u32(&full[s]), 0);
        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStage);
        pair_load(at, &weights, bar, k * kStepK, n0);
        pair_load(at + kWeightBytes, &tokens, bar, k * kStepK, m0);
      }
    }
    // Both CTAs' last loads are read by products before anyone leaves.
    for (int b = i > kPairStages ? i - kPairStages : 0; b < i; ++b)
      mbar_wait(&empty[b % kPairStages], (uint32_t)((b / kPairStages) & 1));
  } else if (warp == 5 && lane == 0 && rank == 0) {
    int i = 0, a = 0;
    bool ok = true;
    for (uint32_t t = first; t < tiles && ok; t += stride, ++a) {
      const int buf = a & 1;
      if (a >= 2 && !mbar_wait(&drained[buf], (uint32_t)((a / 2 - 1) & 1))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int k = 0; k < steps; ++k, ++i) {
        const int s = i % kPairStages;
        if (!mbar_wait(&full[s], (uint32_t)((i / kPairStages) & 1))) {
          ok = false;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t w = smem_u32(ring + s * kPairStage), x = w + kWeightBytes;
#pragma unroll
        for (int q = 0; q < kStepK / 32; ++q)
          pair_umma_i8(tmem + buf * kPairTokens, umma_desc_k_sw128(w + 32 * q),
                       umma_desc_k_sw128(x + 32 * q), (k > 0 || q > 0) ? 1u : 0u);
        pair_commit(&empty[s]);
      }
      if (ok) pair_commit(&drain[buf]);
    }
  } else if (warp < 4) {
    int a = 0;
    bool ok = true;
    for (uint32_t t = first; t < tiles; t += stride, ++a) {
      const int buf = a & 1;
      uint32_t cn, cm;
      pair_tile(t, channel_tiles, token_tiles, cn, cm);
      const int64_t n = (int64_t)(cn * 2 + rank) * kChannels + 32 * warp + lane;
      const int64_t m0 = (int64_t)cm * kPairTokens;
      const bool live = n < N;
      float sb = live ? e.b_scales[n] : 0.0f;
      const float bias = live ? bias_at(e, n) : 0.0f;
      bool wide = false;
      for (int i = threadIdx.x; i < kPairTokens; i += 128) {
        const float sa = m0 + i < M ? e.a_scales[m0 + i] : 0.0f;
        a_scale[buf][i] = sa;
        wide |= extreme(sa);
      }
      // the four warps: the scales are there; those of two tiles ago are read
      wide = drain_warps_or(wide);
      ok = ok && mbar_wait(&drain[buf], (uint32_t)((a / 2) & 1));
      if (!ok) sb = __uint_as_float(0x7FC00000u);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t at = tmem + buf * kPairTokens + ((uint32_t)(32 * warp) << 16);
      const int columns = (int)min64(kPairTokens, M - m0);
      Y* o = static_cast<Y*>(e.out) + m0 * e.out_stride + n;
#pragma unroll 1
      for (int c = 0; c < columns; c += 16) {
        uint32_t v[16];
        __syncwarp();
        tmem_ld16(at + c, v);
        if (live)
          put16<Y>(v, a_scale[buf] + c, sb, bias, wide, o + c * e.out_stride, e.out_stride,
                   columns - c);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_cluster(cluster_address(smem_u32(&drained[buf]), 0));
    }
  }
  __syncwarp();
  __syncthreads();
  cluster_sync();  // no CTA leaves while the other's barriers or products need it
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(2 * kPairTokens));
}

// [rows, K] codes, boxes of 128 bytes by box_rows.
bool codes_map(CUtensorMap* map, const int8_t* codes, int64_t stride, int64_t rows, int64_t K,
               uint32_t box_rows) {
  auto enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  std::memset(map, 0, sizeof(*map));
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride};
  const cuuint32_t box[2] = {kStepK, box_rows};
  const cuuint32_t ones[2] = {1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t*>(codes), dims, strides, box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// A product: its operands and how it is launched.
struct Product {
  const int8_t* a_codes;
  int64_t a_stride, M;
  const int8_t* b_codes;
  int64_t b_stride, N, K;
  Epilogue e;
  bool chained;  // right behind the kernel that writes the tokens' codes
  cudaStream_t stream;
};

template <int kN, typename Y>
mb_status launch_tiles(const Product& p, int parts, int stages, int smem) {
  static std::atomic<uint64_t> attr_done{0};
  MB_CUDA_TRY(set_smem_limit_once(int8_matmul_kernel<kN, Y>, kMostSmem, attr_done));
  CUtensorMap tokens, weights;
  if (!codes_map(&tokens, p.a_codes, p.a_stride, p.M, p.K, kN) ||
      !codes_map(&weights, p.b_codes, p.b_stride, p.N, p.K, kChannels))
    return set_error(MB_ERR_CUDA, "cuTensorMapEncodeTiled rejected the codes");
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ceil_div(p.N, kChannels) * parts), (unsigned)ceil_div(p.M, kN));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = p.stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.chained ? 2 : 1;
  MB_CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_matmul_kernel<kN, Y>, tokens, weights, p.M, p.N, p.K,
                                 stages, p.e));
  return MB_OK;
}

template <typename Y>
mb_status launch_pairs(const Product& p) {
  static std::atomic<uint64_t> attr_done{0};
  MB_CUDA_TRY(set_smem_limit_once(int8_matmul_pair_kernel<Y>, kPairSmem, attr_done));
  CUtensorMap tokens, weights;
  if (!codes_map(&tokens, p.a_codes, p.a_stride, p.M, p.K, kPairTokens / 2) ||
      !codes_map(&weights, p.b_codes, p.b_stride, p.N, p.K, kChannels))
    return set_error(MB_ERR_CUDA, "cuTensorMapEncodeTiled rejected the codes");
  const int64_t tiles = ceil_div(p.N, 2 * kChannels) * ceil_div(p.M, kPairTokens);
  MB_REQUIRE(tiles < (int64_t(1) << 31), "M or N too large");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * min64(tiles, kSms / 2)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kPairSmem;
  cfg.stream = p.stream;
  cfg.attrs = attr;
  cfg.numAttrs = p.chained ? 1 : 0;
  MB_CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_matmul_pair_kernel<Y>, tokens, weights, p.M, p.N, p.K,
                                 p.e));
  return MB_OK;
}

// Tokens a tile and K parts of a product too small for the pairs: the least of
// an estimate, in us, of what a CTA streams (75 GB a second of operands an SM,
// 9 TB of all from L2), what draining a tile costs (0.01 a token) and what
// joining parts costs (1, and their sums at 15 GB a second).  Measured against
// it, whole calls: 64 x 4096 x 4096: 64 tokens in 4 parts 11.9 us, in 1 14.3;
// 256 x 4096 x 4096: 64 tokens in 1 part 15.0, 256 tokens in 4 20.4; 300 x 300
// x 300: 32 tokens 4.9, 256 tokens 8.1; 1000 x 1000 x 1000: 64 tokens 7.9, 256
// tokens 10.8; 1 x 4096 x 4096: 4 parts 8.3, 1 part 13.8.
struct Tiling {
  int tokens, parts;
};
inline Tiling tiling_for(int64_t M, int64_t N, int64_t K) {
  const int64_t steps = ceil_div(K, kStepK), channel_tiles = ceil_div(N, kChannels);
  Tiling best{16, 1};
  double least = 0.0;
  for (int tokens = 16; tokens <= 256; tokens *= 2) {
    if (tokens > 16 && tokens >= 2 * M) break;
    const int64_t tiles = channel_tiles * ceil_div(M, tokens);
    for (int parts = 1; parts <= (int)kMostParts && parts <= steps; ++parts) {
      const int64_t ctas = tiles * parts, rounds = ceil_div(ctas, kSms);
      if (parts > 1 && ctas > 2 * kSms) break;
      const double bytes = (double)ceil_div(steps, parts) * (kWeightBytes + tokens * kStepK);
      const double stream =
          std::max((double)rounds * bytes / 75e3, (double)ctas * bytes / 9e6);
      const double join = parts > 1 ? 1.0 + tokens * kChannels * 4 / 15e3 : 0.0;
      const double cost = stream + join + 0.01 * tokens * (double)rounds;
      if (least == 0.0 || cost < least) least = cost, best = Tiling{tokens, parts};
    }
  }
  return best;
}

template <int kN, typename Y>
mb_status split_tiles(const Product& p, int parts) {
  using S = Shape<kN>;
  const int64_t ctas = ceil_div(p.N, kChannels) * ceil_div(p.M, kN) * parts;
  // as deep a ring as fits (with two CTAs an SM where there are that many and
  // four stages fit), but not deeper than a part has steps
  constexpr int kHalf = (kMostSmem - 2048) / 2;
  constexpr bool kTwo = S::smem(std::max(4, S::kLeast)) <= kHalf;
  int stages = ((kTwo && ctas > kSms ? kHalf : kMostSmem) - 1024) / S::kStage;
  stages = (int)min64(std::min(stages, kMaxStages), ceil_div(ceil_div(p.K, kStepK), parts));
  if (parts > 1) stages = std::max(stages, S::kLeast);
  return launch_tiles<kN, Y>(p, parts, stages,
                             parts > 1 ? std::max(kHalf, S::smem(stages)) : S::smem(stages));
}

template <typename Y>
mb_status dispatch(const Product& p) {
  // pairs where their tiles give every pair of SMs work (1500 x 4096 x 4096:
  // 30.4 us either way; 1024: 19.2 with pairs, 18.1 without), unless most of
  // their 256 columns are empty (a wide N and few tokens, weights from HBM, with
  // pairs and without: 28672 x 8192 1 token 66.5 and 41.6 us, 64 56.1 and 44.1, 128
  // 58.3 and 56.1, 256 61.9 and 70.2; 32000 x 4096 43.8 and 26.6, 35.8 and 26.9, 37.1
  // and 38.7, 37.9 and 46.0)
  if (p.M > 64 &&
      ceil_div(p.N, 2 * kChannels) * ceil_div(p.M, kPairTokens) >= kSms / 2)
    return launch_pairs<Y>(p);
  const Tiling t = tiling_for(p.M, p.N, p.K);
  switch (t.tokens) {
    case 16: return split_tiles<16, Y>(p, t.parts);
    case 32: return split_tiles<32, Y>(p, t.parts);
    case 64: return split_tiles<64, Y>(p, t.parts);
    case 128: return split_tiles<128, Y>(p, t.parts);
    default: return split_tiles<256, Y>(p, t.parts);
  }
}

mb_status multiply(const int8_t* a_codes, int64_t a_stride, const float* a_scales, int64_t M,
                   const int8_t* b_codes, int64_t b_stride, const float* b_scales, int64_t N,
                   int64_t K, const void* bias, mb_dtype bias_type, void* out, mb_dtype out_type,
                   int64_t out_stride, bool chained, mb_stream_t stream) {
  // the stride of a single row is not read, but TMA wants one
  if (M == 1) a_stride = ceil_div(K, 16) * 16;
  if (N == 1) b_stride = ceil_div(K, 16) * 16;
  const Product p{a_codes, a_stride, M, b_codes, b_stride, N, K,
                  Epilogue{a_scales, b_scales, bias, out, out_stride, (int)bias_type},
                  chained, reinterpret_cast<cudaStream_t>(stream)};
  switch (out_type) {
    case MB_FP16: return dispatch<__half>(p);
    case MB_BF16: return dispatch<__nv_bfloat16>(p);
    default: return dispatch<float>(p);
  }
}

// What mb_int8_matmul and mb_int8_linear ask of the weights and the output.
mb_status check_product(int64_t M, const int8_t* b_codes, int64_t b_stride, const float* b_scales,
                        int64_t N, int64_t K, const void* bias, mb_dtype bias_type, void* out,
                        mb_dtype out_type, int64_t out_stride) {
  MB_REQUIRE(b_codes && b_scales && out, "int8_matmul pointers must not be null");
  MB_REQUIRE(dtype_known(out_type) && (bias == nullptr || dtype_known(bias_type)),
             "unknown type of out or bias");
  MB_REQUIRE(M > 0 && N > 0 && K > 0, "M, N and K must be positive");
  MB_REQUIRE(K <= MB_INT8_MAX_K, "K too large: the int32 sums would not be exact");
  MB_REQUIRE(M <= (int64_t(1) << 23) && N < (int64_t(1) << 31) - 256, "M or N too large");
  MB_REQUIRE((N == 1 || b_stride >= K) && (M == 1 || out_stride >= N),
             "strides must be at least the length of a row");
  MB_REQUIRE(aligned(b_codes, 16) && b_stride % 16 == 0, "codes must begin on 16-byte boundaries");
  MB_REQUIRE(aligned(out, dtype_size(out_type)) && aligned(b_scales, 4) &&
                 (bias == nullptr || aligned(bias, dtype_size(bias_type))),
             "misaligned out, scales or bias");
  return MB_OK;
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" mb_status mb_int8_matmul(const int8_t* a_codes, int64_t a_stride, const float* a_scales,
                                    int64_t M, const int8_t* b_codes, int64_t b_stride,
                                    const float* b_scales, int64_t N, int64_t K, const void* bias,
                                    mb_dtype bias_type, void* out, mb_dtype out_type,
                                    int64_t out_stride, mb_stream_t stream) {
  clear_error();
  if (const mb_status st = check_product(M, b_codes, b_stride, b_scales, N, K, bias, bias_type,
                                         out, out_type, out_stride);
      st != MB_OK)
    return st;
  MB_REQUIRE(a_codes && a_scales, "int8_matmul pointers must not be null");
  MB_REQUIRE(M == 1 || a_stride >= K, "strides must be at least the length of a row");
  MB_REQUIRE(aligned(a_codes, 16) && a_stride % 16 == 0, "codes must begin on 16-byte boundaries");
  MB_REQUIRE(aligned(a_scales, 4), "misaligned out, scales or bias");
  return multiply(a_codes, a_stride, a_scales, M, b_codes, b_stride, b_scales, N, K, bias,
                  bias_type, out, out_type, out_stride, false, stream);
}

extern "C" size_t mb_int8_linear_workspace_size(int64_t M, int64_t K) {
  if (M <= 0 || K <= 0) return 0;
  return (size_t)M * ((size_t)ceil_div(K, 16) * 16 + sizeof(float));
}

extern "C" mb_status mb_int8_linear(const void* x, mb_dtype x_type, int64_t x_stride, int64_t M,
                                    const int8_t* b_codes, int64_t b_stride, const float* b_scales,
                                    int64_t N, int64_t K, const void* bias, mb_dtype bias_type,
                                    void* out, mb_dtype out_type, int64_t out_stride,
                                    void* workspace, size_t workspace_bytes, mb_stream_t stream) {
  clear_error();
  if (const mb_status st = check_product(M, b_codes, b_stride, b_scales, N, K, bias, bias_type,
                                         out, out_type, out_stride);
      st != MB_OK)
    return st;
  if (workspace == nullptr || !aligned(workspace, 16) ||
      workspace_bytes < mb_int8_linear_workspace_size(M, K))
    return set_error(MB_ERR_WORKSPACE, "int8_linear workspace missing, misaligned or too small");
  const int64_t pitch = ceil_div(K, 16) * 16;
  int8_t* codes = static_cast<int8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + M * pitch);
  const mb_status st = mb_int8_quantize(x, x_type, M, K, x_stride, codes, pitch, scales, stream);
  if (st != MB_OK) return st;
  return multiply(codes, pitch, scales, M, b_codes, b_stride, b_scales, N, K, bias, bias_type, out,
                  out_type, out_stride, true, stream);
}
