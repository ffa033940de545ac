// Rows to 8-bit codes with one fp32 scale each, and back (no counterpart in
// the reference): scale = max|x| / 127, code = x / scale to the nearest.
//
// Both directions are bound by memory: 3 bytes a value for the 16-bit types
// (8192 x 11008 bf16: 46 us = 5.9 TB/s to codes).  A row is read once: its
// threads keep what they loaded in registers between the maximum and the
// codes, 4 or 6 16-byte loads each in flight (with 16 the registers leave too
// few warps: 70 us).  A row too long for 1024 threads' registers is read a
// second time past them, from L2.
#include <algorithm>

#include "mb_codes.cuh"
#include "mb_tma.cuh"

namespace mb {
namespace {

// T threads a row, kPieces pieces of 8 values a thread kept in registers;
// CTAs of max(T, 128) threads.  kWhole: rows of whole 8-value pieces that begin
// on 16-byte boundaries.
template <typename X, int T, int kPieces, bool kWhole>
__global__ void __launch_bounds__(T < 128 ? 128 : T)
    int8_quantize_kernel(const X* __restrict__ x, int64_t rows, int64_t K, int64_t x_stride,
                         int8_t* __restrict__ codes, int64_t codes_stride,
                         float* __restrict__ scales) {
  // in this order: a product behind this may begin with its weights, which the
  // kernel before may have written
  grid_dependency_wait();
  grid_launch_dependents();
  constexpr int kRows = T < 128 ? 128 / T : 1;
  const int tid = threadIdx.x % T, sub = threadIdx.x / T;
  const int64_t row = (int64_t)blockIdx.x * kRows + sub;
  const X* xr = x + row * x_stride;
  const int k = row < rows ? (int)K : 0, n8 = (k + 7) / 8;

  // x as a whole, which a row that begins anywhere may read from
  const uintptr_t begin = reinterpret_cast<uintptr_t>(x);
  const uintptr_t end = begin + ((rows - 1) * x_stride + K) * (int64_t)sizeof(X);
  const auto fetch = [&](Raw8<X>& to, int c) {
    if constexpr (kWhole || sizeof(X) == 4)
      to.load(xr + 8 * c, kWhole, k - 8 * c);
    else
      to.load_any(xr + 8 * c, k - 8 * c, begin, end);
  };
  Raw8<X> v[kPieces];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int c = tid + j * T;
    if (c < n8) fetch(v[j], c);
  }
#pragma unroll
  for (int j = 0; j < kPieces; ++j)
    if (tid + j * T < n8) m = v[j].abs_max(m);
  for (int c = tid + kPieces * T; c < n8; c += T) {
    Raw8<X> u;
    fetch(u, c);
    m = u.abs_max(m);
  }
  m = Raw8<X>::abs_max_bits(m);
  if constexpr (T < 32) {
#pragma unroll
    for (int o = 1; o < T; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  } else {
    m = __reduce_max_sync(0xffffffffu, m);
  }
  if constexpr (T > 32) {
    __shared__ uint32_t part[kRows][T / 32];
    if ((threadIdx.x & 31) == 0) part[sub][tid / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 32; ++w) m = max(m, part[sub][w]);
  }
  if (row >= rows) return;
  const RowScale r = row_scale(m);
  if (tid == 0) scales[row] = r.scale;
  int8_t* cr = codes + row * codes_stride;
  const auto put = [&](int c, const Raw8<X>& u) {
    float f[8];
    u.floats(f);
    const uint2 q = codes8(f, r);
    if (kWhole || 8 * c + 8 <= k) {
      *reinterpret_cast<uint2*>(cr + 8 * c) = q;
    } else {
      for (int i = 0; i < k - 8 * c; ++i)
        cr[8 * c + i] = (int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
    }
  };
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const int c = tid + j * T;
    if (c < n8) put(c, v[j]);
  }
  for (int c = tid + kPieces * T; c < n8; c += T) {
    Raw8<X> u;
    fetch(u, c);
    put(c, u);
  }
}

// A thread decodes two pieces of 8 codes, 256 pieces apart: neighbouring
// lanes store neighbouring 16 bytes.
constexpr uint32_t kDecodeThreads = 256, kDecodePieces = 2 * kDecodeThreads;

template <typename Y>
__global__ void __launch_bounds__(kDecodeThreads)
    int8_dequantize_kernel(const int8_t* __restrict__ codes, int64_t codes_stride,
                           const float* __restrict__ scales, uint32_t pieces, uint32_t total,
                           Y* __restrict__ out, int64_t out_stride) {
  grid_dependency_wait();
  const uint32_t i0 = blockIdx.x * kDecodePieces + threadIdx.x;
  uint2 q[2];
  float s[2];
  uint32_t row[2], c0[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t i = i0 + h * kDecodeThreads;
    if (i >= total) break;
    row[h] = i / pieces;
    c0[h] = 8 * (i - row[h] * pieces);
    q[h] = *reinterpret_cast<const uint2*>(codes + row[h] * codes_stride + c0[h]);
    s[h] = scales[row[h]];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (i0 + h * kDecodeThreads >= total) break;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = __fmul_rn((float)(int)(int8_t)((e < 4 ? q[h].x : q[h].y) >> (8 * (e & 3))), s[h]);
    store8(out + row[h] * out_stride + c0[h], v);
  }
}

// Rows whose outputs begin anywhere, or that end inside a piece: a warp takes
// 256 values of a row, neighbouring lanes neighbouring values.
constexpr int kDecodeValues = 8;
template <typename Y>
__global__ void __launch_bounds__(kDecodeThreads)
    int8_dequantize_any_kernel(const int8_t* __restrict__ codes, int64_t codes_stride,
                               const float* __restrict__ scales, uint32_t K, uint32_t pieces,
                               uint32_t total, Y* __restrict__ out, int64_t out_stride) {
  grid_dependency_wait();
  // warps counted, not threads: 32 times as many pass 32 bits
  const uint32_t i = blockIdx.x * (kDecodeThreads / 32) + threadIdx.x / 32;
  if (i >= total) return;
  const uint32_t row = i / pieces;
  const uint32_t c0 = (i - row * pieces) * (32 * kDecodeValues) + threadIdx.x % 32;
  const int8_t* from = codes + row * codes_stride + c0;
  Y* to = out + row * out_stride + c0;
  const float s = scales[row];
  int8_t q[kDecodeValues];
#pragma unroll
  for (int e = 0; e < kDecodeValues; ++e)
    if (c0 + 32 * e < K) q[e] = from[32 * e];
#pragma unroll
  for (int e = 0; e < kDecodeValues; ++e)
    if (c0 + 32 * e < K) to[32 * e] = from_float<Y>(__fmul_rn((float)(int)q[e], s));
}

template <typename X, int T, int kPieces>
void launch_quantize(const void* x, int64_t rows, int64_t K, int64_t x_stride, bool whole,
                     int8_t* codes, int64_t codes_stride, float* scales, cudaStream_t stream) {
  constexpr int kThreads = T < 128 ? 128 : T;
  const unsigned grid = (unsigned)ceil_div(rows, kThreads / T);
  const auto go = [&](auto kernel) {
    launch_dependent(kernel, grid, kThreads, 0, stream, static_cast<const X*>(x), rows, K, x_stride,
                     codes, codes_stride, scales);
  };
  whole ? go(int8_quantize_kernel<X, T, kPieces, true>)
        : go(int8_quantize_kernel<X, T, kPieces, false>);
}

template <typename X>
void dispatch_quantize(const void* x, int64_t rows, int64_t K, int64_t x_stride, bool whole,
                       int8_t* codes, int64_t codes_stride, float* scales, cudaStream_t stream) {
  const auto go = [&](auto threads, auto pieces) {
    launch_quantize<X, decltype(threads)::value, decltype(pieces)::value>(
        x, rows, K, x_stride, whole, codes, codes_stride, scales, stream);
  };
  using std::integral_constant;
  const auto kept = [&](auto threads, int64_t pieces) {
    pieces <= 4 ? go(threads, integral_constant<int, 4>{})
                : go(threads, integral_constant<int, 6>{});
  };
  // As few threads as hold the row in 6 pieces each; for fewer rows than fill
  // the GPU up to 256, which shorten the call (8 x 4096: 1.6 us against 4.3
  // with 32, 8192 x 4096: 18.4 us with 128, 23.4 with 256, 28.9 with 32).
  const int64_t n8 = ceil_div(K, 8);
  int threads = n8 <= 32 ? 8 : 32;
  while (threads < 1024 && ceil_div(n8, threads) > 6) threads *= 2;
  if (rows < 4 * 148)
    while (threads < 256 && n8 > threads) threads *= 2;
  const int64_t pieces = ceil_div(n8, threads);
  switch (threads) {
    case 8: return kept(integral_constant<int, 8>{}, pieces);
    case 16: return kept(integral_constant<int, 16>{}, pieces);
    case 32: return kept(integral_constant<int, 32>{}, pieces);
    case 64: return kept(integral_constant<int, 64>{}, pieces);
    case 128: return kept(integral_constant<int, 128>{}, pieces);
    case 256: return kept(integral_constant<int, 256>{}, pieces);
    case 512: return kept(integral_constant<int, 512>{}, pieces);
    default: return kept(integral_constant<int, 1024>{}, pieces);
  }
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" mb_status mb_int8_quantize(const void* x, mb_dtype x_type, int64_t rows, int64_t K,
                                      int64_t x_stride, int8_t* codes, int64_t codes_stride,
                                      float* scales, mb_stream_t stream_) {
  clear_error();
  MB_REQUIRE(x && codes && scales, "int8_quantize pointers must not be null");
  MB_REQUIRE(dtype_known(x_type), "unknown type of x");
  MB_REQUIRE(rows > 0 && K > 0, "rows and K must be positive");
  MB_REQUIRE(rows < (int64_t(1) << 31), "too many rows");
  MB_REQUIRE(K < (int64_t(1) << 31) - 8192, "K too large");
  MB_REQUIRE(rows == 1 || codes_stride >= K, "codes_stride must be at least K");
  MB_REQUIRE(rows == 1 || x_stride >= 0, "x_stride must not be negative");
  MB_REQUIRE(aligned(codes, 16) && codes_stride % 16 == 0,
             "codes must begin on 16-byte boundaries");
  MB_REQUIRE(aligned(x, dtype_size(x_type)) && aligned(scales, 4), "misaligned x or scales");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const bool vec = K % 8 == 0 && aligned(x, 16) &&
                   (rows == 1 || x_stride * dtype_size(x_type) % 16 == 0);
  switch (x_type) {
    case MB_FP16:
      dispatch_quantize<__half>(x, rows, K, x_stride, vec, codes, codes_stride, scales, stream);
      break;
    case MB_BF16:
      dispatch_quantize<__nv_bfloat16>(x, rows, K, x_stride, vec, codes, codes_stride, scales,
                                       stream);
      break;
    default:
      dispatch_quantize<float>(x, rows, K, x_stride, vec, codes, codes_stride, scales, stream);
  }
  MB_LAUNCH_CHECK("int8_quantize_kernel");
  return MB_OK;
}

extern "C" mb_status mb_int8_dequantize(const int8_t* codes, int64_t codes_stride,
                                        const float* scales, int64_t rows, int64_t K, void* out,
                                        mb_dtype out_type, int64_t out_stride,
                                        mb_stream_t stream_) {
  clear_error();
  MB_REQUIRE(codes && scales && out, "int8_dequantize pointers must not be null");
  MB_REQUIRE(dtype_known(out_type), "unknown type of out");
  MB_REQUIRE(rows > 0 && K > 0, "rows and K must be positive");
  MB_REQUIRE(K < (int64_t(1) << 31), "K too large");
  MB_REQUIRE(rows == 1 || (codes_stride >= K && out_stride >= K),
             "strides must be at least K");
  MB_REQUIRE(aligned(codes, 16) && codes_stride % 16 == 0,
             "codes must begin on 16-byte boundaries");
  MB_REQUIRE(aligned(out, dtype_size(out_type)) && aligned(scales, 4), "misaligned out or scales");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const size_t size = dtype_size(out_type);
  const bool whole =
      K % 8 == 0 && aligned(out, 16) && (rows == 1 || out_stride * size % 16 == 0);
  // a launch counts its pieces (8 values, or a warp's 256) in 32 bits; its CTAs,
  // of 512 pieces or 8 warps, are 2^27 at most
  const int64_t per_row = whole ? K / 8 : ceil_div(K, 32 * kDecodeValues);
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 30) / per_row);
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    const int64_t n = min64(most, rows - r0);
    const uint32_t total = (uint32_t)(n * per_row);
    const int8_t* c = codes + r0 * codes_stride;
    uint8_t* o = static_cast<uint8_t*>(out) + (size_t)(r0 * out_stride) * size;
    const auto go = [&](auto* typed) {
      if (whole)
        launch_dependent(int8_dequantize_kernel<std::remove_pointer_t<decltype(typed)>>,
                         (unsigned)ceil_div(total, kDecodePieces), kDecodeThreads, 0, stream, c,
                         codes_stride, scales + r0, (uint32_t)per_row, total, typed, out_stride);
      else
        launch_dependent(int8_dequantize_any_kernel<std::remove_pointer_t<decltype(typed)>>,
                         (unsigned)ceil_div((int64_t)total * 32, kDecodeThreads), kDecodeThreads, 0,
                         stream, c, codes_stride, scales + r0, (uint32_t)K, (uint32_t)per_row,
                         total, typed, out_stride);
    };
    if (out_type == MB_FP16)
      go(reinterpret_cast<__half*>(o));
    else if (out_type == MB_BF16)
      go(reinterpret_cast<__nv_bfloat16*>(o));
    else
      go(reinterpret_cast<float*>(o));
    MB_LAUNCH_CHECK("int8_dequantize_kernel");
  }
  return MB_OK;
}
