// out = (a_scales b_scales^T) o (A B^T) + bias for 8-bit codes A (tokens) and
// B (weights, an output channel a row): the sums are whole numbers, exact in
// int32 (127^2 K < 2^31), scaled once at the end.
//
// 64 x 64 outputs a CTA, 64-byte pieces of both operands in shared memory,
// four products an instruction.
#include "mb_codes.cuh"

namespace mb {
namespace {

constexpr int kTile = 64, kStep = 64;

template <typename T>
__device__ __forceinline__ float load_as_float(const void* p, int64_t i) {
  return to_float<T>(static_cast<const T*>(p)[i]);
}

__device__ __forceinline__ float bias_at(const void* bias, int type, int64_t n) {
  if (bias == nullptr) return 0.0f;
  return type == MB_FP16 ? load_as_float<__half>(bias, n)
         : type == MB_BF16 ? load_as_float<__nv_bfloat16>(bias, n)
                           : load_as_float<float>(bias, n);
}

template <typename Y>
__global__ void __launch_bounds__(256)
    int8_matmul_kernel(const int8_t* __restrict__ a, int64_t a_stride,
                       const float* __restrict__ a_scales, int64_t M,
                       const int8_t* __restrict__ b, int64_t b_stride,
                       const float* __restrict__ b_scales, int64_t N, int64_t K,
                       const void* __restrict__ bias, int bias_type, Y* __restrict__ out,
                       int64_t out_stride) {
  __shared__ int sa[kStep / 4][kTile + 1], sb[kStep / 4][kTile + 1];
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int64_t k0 = 0; k0 < K; k0 += kStep) {
    // a thread brings 16 bytes of one row of each operand
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    const auto fetch = [&](const int8_t* p, int64_t stride, int64_t row, int64_t rows,
                           int(*s)[kTile + 1]) {
      int w[4] = {0, 0, 0, 0};
      if (row < rows) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k0 + c + e < K)
            w[e / 4] |= (int)(uint8_t)p[row * stride + k0 + c + e] << (8 * (e & 3));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[c / 4 + e][r] = w[e];
    };
    fetch(a, a_stride, m0 + r, M, sa);
    fetch(b, b_stride, n0 + r, N, sb);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep / 4; ++k) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __dp4a(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= N) continue;
      const float y = __fmul_rn(__fmul_rn((float)acc[i][j], a_scales[m]), b_scales[n]);
      out[m * out_stride + n] = from_float<Y>(__fadd_rn(y, bias_at(bias, bias_type, n)));
    }
  }
}

}  // namespace
}  // namespace mb

using namespace mb;

extern "C" mb_status mb_int8_matmul(const int8_t* a_codes, int64_t a_stride, const float* a_scales,
                                    int64_t M, const int8_t* b_codes, int64_t b_stride,
                                    const float* b_scales, int64_t N, int64_t K, const void* bias,
                                    mb_dtype bias_type, void* out, mb_dtype out_type,
                                    int64_t out_stride, mb_stream_t stream_) {
  clear_error();
  MB_REQUIRE(a_codes && a_scales && b_codes && b_scales && out,
             "int8_matmul pointers must not be null");
  MB_REQUIRE(dtype_known(out_type) && (bias == nullptr || dtype_known(bias_type)),
             "unknown type of out or bias");
  MB_REQUIRE(M > 0 && N > 0 && K > 0, "M, N and K must be positive");
  MB_REQUIRE(K <= MB_INT8_MAX_K, "K too large: the int32 sums would not be exact");
  MB_REQUIRE(M < (int64_t(1) << 31) && N < (int64_t(1) << 31), "M or N too large");
  MB_REQUIRE((M == 1 || a_stride >= K) && (N == 1 || b_stride >= K) && (M == 1 || out_stride >= N),
             "strides must be at least the length of a row");
  MB_REQUIRE(aligned(a_codes, 16) && aligned(b_codes, 16) && a_stride % 16 == 0 &&
                 b_stride % 16 == 0,
             "codes must begin on 16-byte boundaries");
  MB_REQUIRE(aligned(out, dtype_size(out_type)) && aligned(a_scales, 4) && aligned(b_scales, 4) &&
                 (bias == nullptr || aligned(bias, dtype_size(bias_type))),
             "misaligned out, scales or bias");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const dim3 grid((unsigned)ceil_div(N, kTile), (unsigned)ceil_div(M, kTile));
  MB_REQUIRE(grid.y <= 65535u, "M too large");
  const auto go = [&](auto* typed) {
    int8_matmul_kernel<<<grid, 256, 0, stream>>>(a_codes, a_stride, a_scales, M, b_codes, b_stride,
                                                 b_scales, N, K, bias, (int)bias_type, typed,
                                                 out_stride);
  };
  if (out_type == MB_FP16)
    go(static_cast<__half*>(out));
  else if (out_type == MB_BF16)
    go(static_cast<__nv_bfloat16*>(out));
  else
    go(static_cast<float*>(out));
  MB_LAUNCH_CHECK("int8_matmul_kernel");
  return MB_OK;
}
