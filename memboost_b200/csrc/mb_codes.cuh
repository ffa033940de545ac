// 8- and 4-bit codes of activations, weights, keys and values: conversions
// between the floating types and the exact rounding of x / scale to a code.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "mb_common.cuh"

namespace mb {

inline size_t dtype_size(mb_dtype t) { return t == MB_FP32 ? 4 : 2; }
inline bool dtype_known(mb_dtype t) { return t == MB_FP16 || t == MB_BF16 || t == MB_FP32; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Eight consecutive values of a 16-bit type: one 16-byte load (`vec`: the address
// is 16-byte aligned), else one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, bool vec, float (&v)[8]) {
  static_assert(sizeof(T) == 2, "16-bit types");
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float<T>(p[i]);
  }
}

// Eight consecutive values to a 16-byte aligned address.
template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// Eight consecutive values as they are held (16 or 32 bytes), by 16-byte loads
// (`vec`: the address is 16-byte aligned) where n is 8; 0 past n.
template <typename T>
struct Raw8 {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* __restrict__ p, bool vec, int n) {
    if (vec && n >= 8) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = u.x; w[4 * i + 1] = u.y; w[4 * i + 2] = u.z; w[4 * i + 3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= n) break;
        if constexpr (sizeof(T) == 4)
          w[i] = __float_as_uint(p[i]);
        else
          w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
      }
    }
  }

  // load of a 16-bit type from any address, by the 16-byte blocks that hold the
  // values where those lie inside [begin, end), else one by one.
  __device__ __forceinline__ void load_any(const T* __restrict__ p, int n, uintptr_t begin,
                                           uintptr_t end) {
    static_assert(sizeof(T) == 2, "16-bit types");
    n = min(n, 8);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), low = at & ~(uintptr_t)15;
    const uint32_t skip = (uint32_t)(at - low);  // bytes of the first block before the values
    const bool two = skip + 2 * n > 16;
    if (low < begin || low + (two ? 32 : 16) > end) {
      load(p, false, n);
      return;
    }
    const uint4 a = reinterpret_cast<const uint4*>(low)[0];
    uint4 b = make_uint4(0u, 0u, 0u, 0u);
    if (two) b = reinterpret_cast<const uint4*>(low)[1];
    uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (skip & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) x[i] = x[i + 2];
    }
    if (skip & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) x[i] = x[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = skip & 2 ? __funnelshift_r(x[i], x[i + 1], 16) : x[i];
      // past n: 0
      if (2 * i >= n) w[i] = 0u;
      if (2 * i + 1 == n) w[i] &= 0xFFFFu;
    }
  }

  __device__ __forceinline__ void floats(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4)
        v[i] = __uint_as_float(w[i]);
      else if constexpr (std::is_same_v<T, __half>)
        v[i] = __half2float(__ushort_as_half((uint16_t)(w[i / 2] >> (16 * (i & 1)))));
      else  // bf16 is the upper half of an fp32
        v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
  }

  // max(m, |values|), two 16-bit magnitudes a word for the 16-bit types: as
  // bits, finite < infinity < NaN, so a NaN is not lost
  __device__ __forceinline__ uint32_t abs_max(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4)
        m = max(m, w[i] & 0x7FFFFFFFu);
      else
        m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    }
    return m;
  }

  // what abs_max gathered, as the bits of an fp32
  __device__ __forceinline__ static uint32_t abs_max_bits(uint32_t m) {
    if constexpr (sizeof(T) == 4) return m;
    const uint32_t h = max(m & 0xFFFFu, m >> 16);
    return __float_as_uint(std::is_same_v<T, __half> ? __half2float(__ushort_as_half((uint16_t)h))
                                                     : __uint_as_float(h << 16)) &
           0x7FFFFFFFu;
  }
};

// max of |v| as bits: finite < infinity < NaN, so a NaN is not lost.
__device__ __forceinline__ uint32_t abs_bits_max(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// A row's scale from the bits of its largest magnitude, and what its codes
// are computed with: inv = 1 / scale, or 0 where the quotient in fp32 is not
// good enough to round from (a scale so small that 1 / scale overflows or
// scale is subnormal, a scale of 0, a row that is not finite).
struct RowScale {
  float scale, inv;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  RowScale r;
  if (amax_bits >= 0x7F800000u) {
    r.scale = __uint_as_float(0x7FC00000u);
    r.inv = 0.0f;
  } else {
    r.scale = __fdiv_rn(__uint_as_float(amax_bits), 127.0f);
    r.inv = r.scale >= 0x1p-100f ? __fdiv_rn(1.0f, r.scale) : 0.0f;
  }
  return r;
}

constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23: x + magic rounds x to an integer
// Distance from the rounded value up to which the fp32 quotient decides: its
// error is below 127 * 2^-23 = 1.6e-5.
constexpr float kRoundSafe = 0.49998f;

// Codes of eight values, x / scale to the nearest integer, ties to even, of
// the exact quotient.  The product x * inv (inv rounds once, the sum with the
// magic number once) decides, unless one of the eight comes within 2e-5 of a
// border (one in a hundred warps' steps or so).  Then the remainder x - t * scale
// says for each whether t is the nearest: it is exact for |t| >= 2 (a
// multiple of scale's last place, below 2^24 of them) and for t = 0; for
// |t| = 1 its rounding can at most turn a remainder just above scale / 2 into
// the tie, which leaves the odd t as well.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], RowScale r) {
  uint32_t y[8];
  if (r.inv != 0.0f) {
    float far = 0.0f;
    const uint64_t inv = f2_pack(r.inv, r.inv), magic = f2_pack(kRoundMagic, kRoundMagic);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint64_t v = f2_pack(x[i], x[i + 1]);
      const uint64_t m = f2_fma(v, inv, magic);
      // magic - m = -(the rounded value), exactly
      float d0, d1, m0, m1;
      f2_unpack(f2_fma(v, inv, f2_sub(magic, m)), d0, d1);
      f2_unpack(m, m0, m1);
      far = fmaxf(far, fmaxf(fabsf(d0), fabsf(d1)));
      y[i] = __float_as_uint(m0);
      y[i + 1] = __float_as_uint(m1);
    }
    if (far > kRoundSafe) {
      const float half = 0.5f * r.scale;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float t = __uint_as_float(y[i]) - kRoundMagic;
        const float rest = fmaf(-t, r.scale, x[i]);
        if (fabsf(rest) > half || (fabsf(rest) == half && (y[i] & 1u)))
          y[i] += rest > 0.0f ? 1u : ~0u;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double q = 0.0;
      if (r.scale > 0.0f) {
        q = rint((double)x[i] / (double)r.scale);
        q = fmin(fmax(q, -127.0), 127.0);
      }
      y[i] = (uint32_t)(int)q;
    }
  }
  uint2 c;
  c.x = __byte_perm(__byte_perm(y[0], y[1], 0x0040), __byte_perm(y[2], y[3], 0x0040), 0x5410);
  c.y = __byte_perm(__byte_perm(y[4], y[5], 0x0040), __byte_perm(y[6], y[7], 0x0040), 0x5410);
  return c;
}

// Scale and minimum of 32 channels in 4 bits from their minimum and maximum
// (NaN if either is): (maximum - minimum) / 15 in 64 bits, rounded to fp32
// and to fp16.  Not finite in fp16: both NaN.
struct GroupScale {
  __half scale, low;
  float inv;
};
__device__ __forceinline__ GroupScale group_scale(float lo, float hi) {
  GroupScale g;
  g.low = __float2half_rn(lo);
  // where the difference is exact in fp32 so is the division's rounding: d / 15
  // is never within 2^-53 of the middle between two fp32 numbers
  const float d = hi - lo;
  float s = __fdiv_rn(d, 15.0f);
  if ((hi - d) - lo != 0.0f) s = __double2float_rn(((double)hi - (double)lo) / 15.0);
  g.scale = __float2half_rn(s);
  if (!isfinite(__half2float(g.low)) || !isfinite(__half2float(g.scale))) {
    g.low = g.scale = __ushort_as_half(0x7E00);
  }
  s = __half2float(g.scale);
  g.inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  return g;
}

// 4-bit codes of eight values of a group, (x - minimum) / scale to the
// nearest, ties to even, in [0, 15]; value i at bits [4 i, 4 i + 4).  As
// codes8: fp32 decides (error below 16 * 2^-22) unless a border is near.  Then
// x - minimum is taken with its rounding error e; t * scale (4 + 11 bits) is
// exact, and so, where a border is near, are the remainder and its distance
// from scale / 2, to which e is added: the sign is that of the exact distance.
__device__ __forceinline__ uint32_t codes4(const float (&x)[8], GroupScale g) {
  const float low = __half2float(g.low), scale = __half2float(g.scale);
  uint32_t y[8];
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = fminf(fmaxf((x[i] - low) * g.inv, 0.0f), 15.0f);
    const float m = q + kRoundMagic;
    far = fmaxf(far, fabsf(q - (m - kRoundMagic)));
    y[i] = __float_as_uint(m);
  }
  if (far > kRoundSafe) {
    const float half = 0.5f * scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float z = x[i] - low;
      const float q = fminf(fmaxf(z * g.inv, 0.0f), 15.0f);
      const float t = __uint_as_float(y[i]) - kRoundMagic;
      if (fabsf(q - t) <= kRoundSafe) continue;
      // z + e = x - low exactly
      const float back = z + low;
      const float e = (x[i] - back) + ((back - z) - low);
      const float rest = fmaf(-t, scale, z);
      const float over = (fabsf(rest) - half) + (rest > 0.0f ? e : -e);
      if (over > 0.0f || (over == 0.0f && (y[i] & 1u))) y[i] += rest > 0.0f ? 1u : ~0u;
    }
  }
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) c |= (y[i] & 0xFu) << (4 * i);
  return c;
}

}  // namespace mb
