// Rows of numbers as 8-bit integers with one float32 scale a row: plain rows, a norm's output (with the residual's
// addition), a gated activation's; and back.
//
// For a row y with m = max |y|:  q = round(y * (127 / m)) to the nearest, ties to even;  scale = m / 127.
//   zeros only:             q = 0, scale 0
//   an infinity or a NaN:   q = 0, scale NaN, so that what is made of the row is NaN and other rows are not touched
// All arithmetic in float32; y is not rounded to the stored type of its input before it becomes an integer.
#include "oi_api.h"

namespace {

// |y| as bits: ordered like the numbers, infinities above all finite ones and NaNs above those
__device__ __forceinline__ unsigned magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

struct RowScale {
  float pre, inv, scale;
  // `m`: the largest magnitude of the row. Below 2^-100 the row is taken times 2^80 first, or 127 / m would overflow.
  __device__ __forceinline__ explicit RowScale(unsigned m) {
    const float most = __uint_as_float(m);
    if (m >= 0x7f800000u) {
      pre = inv = 0.f;
      scale = __uint_as_float(0x7fffffffu);
    } else if (m == 0u) {
      pre = inv = scale = 0.f;
    } else {
      const bool tiny = most < 7.888609e-31f;
      pre = tiny ? 1.2089258e24f : 1.f;
      inv = 127.f / (most * pre);
      scale = tiny ? most * pre / 127.f / pre : most / 127.f;
    }
  }
  __device__ __forceinline__ int quantise(float y) const { return __float2int_rn(y * pre * inv); }   // (NaN: 0)
};

// What a row's numbers are made of. get(d) may be called more than once for the same d by the same thread.
template <typename T>
struct PlainRow {
  const T* x;
  long long ldx;
  static constexpr bool kNorm = false;
  __device__ __forceinline__ void begin(long long r) { x += r * ldx; }
  __device__ __forceinline__ float get(int d) const { return to_f32(x[d]); }
};

template <typename T>
struct NormRow {
  T* x;                 // x <- round(x + delta) is stored where there is a delta
  const T* delta;
  const void* w;
  long long ldx, ldd;
  int w_dtype;
  float eps, w_offset, inv;
  static constexpr bool kNorm = true;
  __device__ __forceinline__ void begin(long long r) {
    x += r * ldx;
    if (delta) delta += r * ldd;
  }
  __device__ __forceinline__ float add(int d) {
    float v = to_f32(x[d]);
    if (delta) {
      const T sum = from_f32<T>(v + to_f32(delta[d]));
      x[d] = sum;
      v = to_f32(sum);
    }
    return v;
  }
  __device__ __forceinline__ float get(int d) const { return to_f32(x[d]) * inv * (w_offset + load_as_f32(w, w_dtype, d)); }
};

template <typename T>
struct GateRow {
  const T* x;
  long long ldx;
  int block, act;
  static constexpr bool kNorm = false;
  __device__ __forceinline__ void begin(long long r) { x += r * ldx; }
  __device__ __forceinline__ float get(int d) const {
    const int at = d / block * (2 * block) + d % block;
    return glu_act<false>(to_f32(x[at]), to_f32(x[at + block]), act, 0.f);
  }
};

// One block a row, any length and any alignment: the row is read once for each thing that is asked of all of it.
template <typename Row>
__global__ void rows_int8_kernel(Row row, signed char* q, long long ldq, float* scales, int cols) {
  pdl_start();
  __shared__ float sums[32];
  __shared__ unsigned most;
  const long long r = blockIdx.x;
  row.begin(r);
  q += r * ldq;
  if (threadIdx.x == 0) most = 0u;
  if constexpr (Row::kNorm) {
    float ss = 0.f;
    for (int d = threadIdx.x; d < cols; d += blockDim.x) {
      const float v = row.add(d);
      ss += v * v;
    }
    ss = block_sum(ss, sums);
    row.inv = rsqrtf(ss / (float)cols + row.eps);
  }
  unsigned m = 0u;
  for (int d = threadIdx.x; d < cols; d += blockDim.x) m = max(m, magnitude(row.get(d)));
  m = __reduce_max_sync(0xffffffffu, m);
  __syncthreads();                       // `most` is zero
  if ((threadIdx.x & 31) == 0) atomicMax(&most, m);
  __syncthreads();
  const RowScale s(most);
  for (int d = threadIdx.x; d < cols; d += blockDim.x) q[d] = (signed char)s.quantise(row.get(d));
  if (threadIdx.x == 0) scales[r] = s.scale;
}

template <typename Row>
int launch_rows(const Row& row, void* q, long long ldq, float* scales, int rows, int cols, cudaStream_t s) {
  oi_launch(rows_int8_kernel<Row>, rows, 256, 0, s, row, (signed char*)q, ldq, scales, cols);
  OI_CHECK_LAUNCH();
  return OI_OK;
}

template <typename T>
__global__ void dequantize_kernel(T* out, long long ldo, const signed char* q, long long ldq, const float* scales, int cols) {
  pdl_start();
  const long long r = blockIdx.x;
  const float scale = scales[r];
  for (int d = threadIdx.x; d < cols; d += blockDim.x) out[r * ldo + d] = from_f32<T>((float)q[r * ldq + d] * scale);
}

int check_rows(const char* what, const void* q, long long ldq, const float* scales, int rows, int cols) {
  OI_REQUIRE(rows >= 0 && cols >= 1, "%s: bad sizes rows=%d cols=%d", what, rows, cols);
  OI_REQUIRE(rows == 0 || (q && scales), "%s: a pointer is missing", what);
  OI_REQUIRE(rows <= 1 || ldq >= cols, "%s: rows of %d that start %lld apart", what, cols, ldq);
  return OI_OK;
}

}  // namespace

// q[r, :] (row stride ldq bytes) and scales[r] of x[r, :] (row stride ldx elements)
OI_API int oi_quantize_int8(void* q, long long ldq, float* scales, const void* x, int dtype, long long ldx, int rows, int cols, void* stream) {
  if (int rc = check_rows("quantize_int8", q, ldq, scales, rows, cols)) return rc;
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "quantize_int8: unknown dtype code %d", dtype);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == OI_F32) return launch_rows(PlainRow<float>{(const float*)x, ldx}, q, ldq, scales, rows, cols, s);
  return launch_rows(PlainRow<bf16>{(const bf16*)x, ldx}, q, ldq, scales, rows, cols, s);
}

// The rows of oi_rmsnorm's output, not rounded: x <- round(x + delta) (stored; delta may be null), then
// x * rsqrt(mean(x^2) + eps) * (w_offset + w). Row strides ldx, ldd in elements.
OI_API int oi_rmsnorm_int8(void* q, long long ldq, float* scales, void* x, long long ldx, const void* delta, long long ldd, int dtype,
                           const void* w, int w_dtype, int rows, int cols, float eps, float w_offset, void* stream) {
  if (int rc = check_rows("rmsnorm_int8", q, ldq, scales, rows, cols)) return rc;
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "rmsnorm_int8: unknown dtype code %d", dtype);
  OI_REQUIRE(w_dtype == OI_F32 || w_dtype == OI_BF16, "rmsnorm_int8: unknown weight dtype code %d", w_dtype);
  OI_REQUIRE(!delta || rows <= 1 || ldx >= cols, "rmsnorm_int8: rows of %d that start %lld apart cannot take a sum", cols, ldx);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == OI_F32)
    return launch_rows(NormRow<float>{(float*)x, (const float*)delta, w, ldx, ldd, w_dtype, eps, w_offset, 0.f}, q, ldq, scales, rows, cols, s);
  return launch_rows(NormRow<bf16>{(bf16*)x, (const bf16*)delta, w, ldx, ldd, w_dtype, eps, w_offset, 0.f}, q, ldq, scales, rows, cols, s);
}

// The rows of oi_silu_mul's output, not rounded: act(gate) * up of gate_up [rows, 2 inter] (row stride ldx elements), which lies
// in blocks of `block` gate values followed by their up values.
OI_API int oi_silu_mul_int8(void* q, long long ldq, float* scales, const void* gate_up, int dtype, long long ldx, int rows, int inter,
                            int block, int act, void* stream) {
  if (int rc = check_rows("silu_mul_int8", q, ldq, scales, rows, inter)) return rc;
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "silu_mul_int8: unknown dtype code %d", dtype);
  OI_REQUIRE(inter <= (1 << 30) && block >= 1 && inter % block == 0, "silu_mul_int8: %d values in blocks of %d", inter, block);
  OI_REQUIRE(act == OI_ACT_SILU || act == OI_ACT_GELU_TANH, "silu_mul_int8: unknown activation code %d", act);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == OI_F32) return launch_rows(GateRow<float>{(const float*)gate_up, ldx, block, act}, q, ldq, scales, rows, inter, s);
  return launch_rows(GateRow<bf16>{(const bf16*)gate_up, ldx, block, act}, q, ldq, scales, rows, inter, s);
}

// out[r, :] = round(q[r, :] * scales[r]) (row stride ldo elements)
OI_API int oi_dequantize_int8(void* out, int dtype, long long ldo, const void* q, long long ldq, const float* scales, int rows, int cols,
                              void* stream) {
  OI_REQUIRE(rows >= 0 && cols >= 1, "dequantize_int8: bad sizes rows=%d cols=%d", rows, cols);
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "dequantize_int8: unknown dtype code %d", dtype);
  OI_REQUIRE(rows <= 1 || ldo >= cols, "dequantize_int8: rows of %d that start %lld apart", cols, ldo);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == OI_F32) oi_launch(dequantize_kernel<float>, rows, 256, 0, s, (float*)out, ldo, (const signed char*)q, ldq, scales, cols);
  else oi_launch(dequantize_kernel<bf16>, rows, 256, 0, s, (bf16*)out, ldo, (const signed char*)q, ldq, scales, cols);
  OI_CHECK_LAUNCH();
  return OI_OK;
}
