// out[m, n] = (sum_k x[m, k] * w[n, k]) * sx[m] * sw[n] + bias[n] for 8-bit integers: the sums are exact in 32-bit integers (K up
// to 131,071: 128 * 128 * K < 2^31), so no order of addition matters; then float(sum) * sx * sw + bias in float32, in that
// order, and one rounding to the output's type.
#include "oi_api.h"

namespace {

constexpr int kTile = 64, kWords = 16;     // 64 x 64 results a block, 64 bytes of K at a time

template <typename TOut>
__global__ void __launch_bounds__(256)
linear_int8_kernel(TOut* out, long long ldo, const signed char* x, long long ldx, const float* sx, const signed char* w, long long ldw,
                   const float* sw, const float* bias, int M, int N, int K) {
  pdl_start();
  __shared__ int xs[kWords][kTile + 1], ws[kWords][kTile + 1];
  const int n0 = blockIdx.x * kTile, m0 = blockIdx.y * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 4 * kWords) {
    for (int i = threadIdx.x; i < kTile * kWords; i += 256) {
      const int r = i / kWords, c = i % kWords, k = k0 + 4 * c;
      const int left = K - k;                                      // bytes of this word that count
      const unsigned keep = left >= 4 ? 0xffffffffu : left > 0 ? (1u << 8 * left) - 1u : 0u;
      xs[c][r] = m0 + r < M && left > 0 ? *reinterpret_cast<const int*>(x + (m0 + r) * ldx + k) & keep : 0;
      ws[c][r] = n0 + r < N && left > 0 ? *reinterpret_cast<const int*>(w + (n0 + r) * ldw + k) & keep : 0;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kWords; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(xs[c][ty * 4 + i], ws[c][tx + 16 * j], acc[i][j]);
    }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m < M && n < N) {
        float y = __fmul_rn(__fmul_rn((float)acc[i][j], sx[m]), sw[n]);
        if (bias) y = __fadd_rn(y, bias[n]);
        out[(size_t)m * ldo + n] = from_f32<TOut>(y);
      }
    }
}

}  // namespace

// x [M, K], w [N, K]: 8-bit integers, row strides in bytes; rows start on 16-byte borders. sx [M], sw [N], bias [N] or null: float32.
OI_API int oi_linear_int8(void* out, int out_dtype, long long ldo, const void* x, long long ldx, const float* sx, const void* w,
                          long long ldw, const float* sw, const float* bias, int M, int N, int K, void* stream) {
  OI_REQUIRE(M >= 0 && N >= 0 && K >= 1 && K <= 131071, "linear_int8: bad sizes M=%d N=%d K=%d (K: 1 to 131071)", M, N, K);
  OI_REQUIRE(out_dtype == OI_F32 || out_dtype == OI_BF16, "linear_int8: unknown output dtype code %d", out_dtype);
  if (M == 0 || N == 0) return OI_OK;
  OI_REQUIRE(ldx % 16 == 0 && ldw % 16 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && ldx >= K && ldw >= K,
             "linear_int8: rows of x and w must start on 16-byte borders");
  OI_REQUIRE(M == 1 || ldo >= N, "linear_int8: result rows of %d that start %lld apart", N, ldo);
  OI_REQUIRE(ceil_div(M, kTile) <= 65535, "linear_int8: %d rows are too many", M);
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid(ceil_div(N, kTile), ceil_div(M, kTile));
  if (out_dtype == OI_F32)
    oi_launch(linear_int8_kernel<float>, grid, 256, 0, s, (float*)out, ldo, (const signed char*)x, ldx, sx, (const signed char*)w, ldw, sw, bias, M, N, K);
  else
    oi_launch(linear_int8_kernel<bf16>, grid, 256, 0, s, (bf16*)out, ldo, (const signed char*)x, ldx, sx, (const signed char*)w, ldw, sw, bias, M, N, K);
  OI_CHECK_LAUNCH();
  return OI_OK;
}
