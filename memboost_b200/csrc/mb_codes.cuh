// 8- and 4-bit codes of activations, weights, keys and values: conversions
// between the floating types and the exact rounding of x / scale to a code.
#pragma once

#include <cuda_bf16.h>

#include "mb_common.cuh"

namespace mb {

inline size_t dtype_size(mb_dtype t) { return t == MB_FP32 ? 4 : 2; }
inline bool dtype_known(mb_dtype t) { return t == MB_FP16 || t == MB_BF16 || t == MB_FP32; }
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
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

// Eight consecutive values: two 16-byte loads or stores for fp32, one for the
// 16-bit types (`vec`: the address is 16-byte aligned and n is 8), else one by
// one, 0 past n.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ p, bool vec, int n, float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0];
      const float4 b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_float<T>(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, bool vec, int n, const float (&v)[8]) {
  if (vec && n >= 8) {
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
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_float<T>(v[i]);
  }
}

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
constexpr float kRoundSafe = 0.4999f;

// Codes of eight values, x / scale to the nearest integer, ties to even, of
// the exact quotient.  The product x * inv (one rounding of inv, the sum with
// the magic number rounds once) decides unless some value comes within 1e-4
// of a border: those eight take the 64-bit quotient, whose error (2^-46 of a
// code) no 24-bit x and scale can turn into a wrong side.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], RowScale r) {
  uint32_t y[8];
  float far = 1.0f;
  if (r.inv != 0.0f) {
    far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float m = fmaf(x[i], r.inv, kRoundMagic);
      const float t = m - kRoundMagic;
      far = fmaxf(far, fabsf(fmaf(x[i], r.inv, -t)));
      y[i] = __float_as_uint(m);
    }
  }
  if (far > kRoundSafe) {
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
  g.scale = __float2half_rn(__double2float_rn(((double)hi - (double)lo) / 15.0));
  if (!isfinite(__half2float(g.low)) || !isfinite(__half2float(g.scale))) {
    g.low = g.scale = __ushort_as_half(0x7E00);
  }
  const float s = __half2float(g.scale);
  g.inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
  return g;
}

// 4-bit codes of eight values of a group, (x - minimum) / scale to the
// nearest, ties to even, in [0, 15]; value i at bits [4 i, 4 i + 4).  As
// codes8: fp32 decides (error below 16 * 2^-22) unless a border is near.
__device__ __forceinline__ uint32_t codes4(const float (&x)[8], GroupScale g) {
  const float low = __half2float(g.low);
  uint32_t c = 0;
  float far = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = fminf(fmaxf((x[i] - low) * g.inv, 0.0f), 15.0f);
    const float m = q + kRoundMagic;
    far = fmaxf(far, fabsf(q - (m - kRoundMagic)));
    c |= (__float_as_uint(m) & 0xFu) << (4 * i);
  }
  if (far > kRoundSafe) {
    c = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double q = rint(((double)x[i] - (double)low) / (double)__half2float(g.scale));
      q = fmin(fmax(q, 0.0), 15.0);
      c |= (uint32_t)(int)q << (4 * i);
    }
  }
  return c;
}

}  // namespace mb
