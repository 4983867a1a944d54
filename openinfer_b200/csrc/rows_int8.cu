// Rows of numbers as 8-bit integers with one float32 scale a row: plain rows, a norm's output (with the residual's
// addition), a gated activation's; and back. What a layer of 8-bit products needs between them.
//
// For a row y with m = max |y|:  q = round(y * (127 / m)) to the nearest, ties to even;  scale = m / 127.
//   zeros only:             q = 0, scale 0
//   an infinity or a NaN:   q = 0, scale NaN, so that what is made of the row is NaN and other rows are not touched
// All arithmetic in float32; y is not rounded to the stored type of its input before it becomes an integer.
#include "oi_api.h"
#include "tcgen05.cuh"

namespace {

__device__ int g_rows_int8_error = 0;       // set to a non-zero code when a bounded wait ran out

// |y| as bits: ordered like the numbers, infinities above all finite ones and NaNs above those
__device__ __forceinline__ unsigned magnitude(float y) { return __float_as_uint(y) & 0x7fffffffu; }

// act(gate) * up by the special-function unit's exponential and reciprocal: what follows is a rounding to 8 bits. They are within 2 units
// in the last place each, but the exponent is rounded before them: e^-t is off by up to |t| roundings more (some 30 units at 60). Where it
// passes 2^126 (t below -87.3) its reciprocal is below the normal numbers, and the result a zero.
template <int ACT>
__device__ __forceinline__ float gated(float g, float u) {
  const float t = ACT == OI_ACT_GELU_TANH ? 1.5957691216057308f * (g + 0.044715f * g * g * g) : g;
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(e) : "f"(-1.4426950408889634f * t));
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(1.f + e));
  return g * r * u;
}

// What a row is multiplied by, from the largest magnitude of its numbers. A norm's rows come without the reciprocal root mean
// square `common`, which all of a row shares: q does not depend on it, the scale takes it up.
struct RowScale {
  float inv, scale;
  bool tiny;            // m below 2^-100: the row is taken times 2^80 first, or 127 / m would overflow
  unsigned keep;        // a row with an infinity or a NaN: all its bytes become zeros
  __device__ __forceinline__ RowScale(unsigned m, float common) {
    float most = __uint_as_float(m);
    keep = m < 0x7f800000u ? ~0u : 0u;
    tiny = most < 0x1p-100f;
    if (tiny) most *= 0x1p80f;
    inv = m ? 127.f / most : 0.f;
    scale = keep ? (most * common) / 127.f : __uint_as_float(0x7fffffffu);
    if (tiny) scale *= 0x1p-80f;
  }
  // round(y * inv) in the low byte: added to 1.5 * 2^23, the sum's last bit stands for one (ties to even, as the sum is rounded).
  // Of a tiny row: y times 2^80.
  __device__ __forceinline__ unsigned byte(float y) const { return __float_as_uint(__fadd_rn(__fmul_rn(y, inv), 12582912.f)); }
  __device__ __forceinline__ unsigned four(float a, float b, float c, float d) const {
    return __byte_perm(__byte_perm(byte(a), byte(b), 0x0040), __byte_perm(byte(c), byte(d), 0x0040), 0x5410) & keep;
  }
};

// Eight numbers of a row as they lie in memory, 16 bytes a load
template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(reinterpret_cast<const unsigned*>(v)[e]);
    } else {
      const unsigned w = reinterpret_cast<const unsigned*>(v)[e >> 1];
      return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
    }
  }
  // each number plus the other's, rounded once
  __device__ __forceinline__ void add(const Eight& other) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) set(e, get(e) + other.get(e));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        reinterpret_cast<__nv_bfloat162*>(v)[i] = __hadd2(reinterpret_cast<const __nv_bfloat162*>(v)[i], reinterpret_cast<const __nv_bfloat162*>(other.v)[i]);
    }
  }
  __device__ __forceinline__ void set_pair(int e, float a, float b) {      // e even
    if constexpr (sizeof(T) == 4) set(e, a), set(e + 1, b);
    else reinterpret_cast<__nv_bfloat162*>(v)[e >> 1] = __floats2bfloat162_rn(a, b);
  }
  __device__ __forceinline__ void set(int e, T x) {
    if constexpr (sizeof(T) == 4) reinterpret_cast<unsigned*>(v)[e] = __float_as_uint(x);
    else {
      unsigned& w = reinterpret_cast<unsigned*>(v)[e >> 1];
      const unsigned b = __bfloat16_as_ushort(x);
      w = e & 1 ? (w & 0xffffu) | b << 16 : (w & 0xffff0000u) | b;
    }
  }
};

// What a row's numbers are made of. fetch(d) asks for eight of them (d a multiple of 8, aligned, all within the row), make() turns them
// into numbers; fetch_one(d) and make_one() do so with one number anywhere. Both add up in `squares` what a norm needs; again(d) is
// the number without. (All that is asked for together is asked for before a sum is stored: no load waits for a store it might meet.)
template <typename T>
struct PlainRow {
  const T* x;
  long long ldx;
  static constexpr bool kNorm = false, kRing = sizeof(T) == 2;
  struct Raw { Eight<T> x; };
  struct Kept {};
  __host__ __device__ __forceinline__ int bytes(int cols) const { return cols * (int)sizeof(T); }
  __device__ __forceinline__ void copy(unsigned dst, long long r, int cols, unsigned bar) const { tc::bulk_load(dst, x + r * ldx, bytes(cols), bar); }
  __device__ __forceinline__ void lies_at(const unsigned char* held, int cols) { x = reinterpret_cast<const T*>(held); }
  __device__ __forceinline__ void begin(long long r) { x += r * ldx; }
  __device__ __forceinline__ void keep(int d, Kept& kept) const {}
  __device__ __forceinline__ void fetch(int d, Raw& raw) const { raw.x.load(x + d); }
  __device__ __forceinline__ void make(int d, Raw& raw, const Kept& kept, float (&y)[8], float& squares) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = raw.x.get(e);
  }
  struct RawOne { T x; };
  __device__ __forceinline__ void fetch_one(int d, RawOne& raw) const { raw.x = x[d]; }
  __device__ __forceinline__ float make_one(int d, const RawOne& raw, float& squares) const { return to_f32(raw.x); }
  __device__ __forceinline__ float again(int d) const { return to_f32(x[d]); }
};

// x <- round(x + delta) is stored where there is a delta; the numbers are x * (w_offset + w), without the reciprocal root mean square
template <typename T>
struct NormRow {
  T* x;
  const T* delta;
  const void* w;
  long long ldx, ldd;
  int w_dtype;
  float eps, w_offset;
  static constexpr bool kNorm = true, kRing = true;
  struct Raw { Eight<T> x, delta; };
  struct Kept { Eight<float> w; };
  __host__ __device__ __forceinline__ int bytes(int cols) const { return cols * (int)sizeof(T) * (delta ? 2 : 1); }
  __device__ __forceinline__ void copy(unsigned dst, long long r, int cols, unsigned bar) const {
    const unsigned each = cols * (unsigned)sizeof(T);
    tc::bulk_load(dst, x + r * ldx, each, bar);
    if (delta) tc::bulk_load(dst + each, delta + r * ldd, each, bar);
  }
  __device__ __forceinline__ void lies_at(unsigned char* held, int cols) {
    x = reinterpret_cast<T*>(held);
    if (delta) delta = x + cols;
  }
  __device__ __forceinline__ void begin(long long r) {
    x += r * ldx;
    if (delta) delta += r * ldd;
  }
  __device__ __forceinline__ void keep(int d, Kept& kept) const {
    if (w_dtype == OI_F32) kept.w.load(reinterpret_cast<const float*>(w) + d);
    else kept.w.v[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(w) + d);
  }
  __device__ __forceinline__ void fetch(int d, Raw& raw) const {
    raw.x.load(x + d);
    if (delta) raw.delta.load(delta + d);
  }
  __device__ __forceinline__ void make(int d, Raw& raw, const Kept& kept, float (&y)[8], float& squares) const {
    if (delta) {
      raw.x.add(raw.delta);
      raw.x.store(x + d);
    }
    float wv[8];
    if (w_dtype == OI_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) wv[e] = kept.w.get(e);
    } else {
      Eight<bf16> wb;
      wb.v[0] = kept.w.v[0];
#pragma unroll
      for (int e = 0; e < 8; ++e) wv[e] = wb.get(e);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = raw.x.get(e);
      squares += v * v;
      y[e] = v * (w_offset + wv[e]);
    }
  }
  struct RawOne { T x, delta; float w; };
  __device__ __forceinline__ void fetch_one(int d, RawOne& raw) const {
    raw.x = x[d];
    if (delta) raw.delta = delta[d];
    raw.w = load_as_f32(w, w_dtype, d);
  }
  __device__ __forceinline__ float make_one(int d, const RawOne& raw, float& squares) const {
    float v = to_f32(raw.x);
    if (delta) {
      const T sum = from_f32<T>(v + to_f32(raw.delta));
      x[d] = sum;
      v = to_f32(sum);
    }
    squares += v * v;
    return v * (w_offset + raw.w);
  }
  __device__ __forceinline__ float again(int d) const { return to_f32(x[d]) * (w_offset + load_as_f32(w, w_dtype, d)); }
};

template <typename T, int ACT>
struct GateRow {
  const T* x;
  long long ldx;
  int block, shift;     // shift: of a block that is a power of two; -1: all gates, then all ups; -2: any other
  static constexpr bool kNorm = false, kRing = false;
  struct Raw { Eight<T> gate, up; };
  struct Kept {};
  __device__ __forceinline__ void keep(int d, Kept& kept) const {}
  __device__ __forceinline__ void begin(long long r) { x += r * ldx; }
  __device__ __forceinline__ const T* at(int d) const { return x + d + (shift >= 0 ? d >> shift << shift : shift == -1 ? 0 : d / block * block); }
  __device__ __forceinline__ void fetch(int d, Raw& raw) const {
    raw.gate.load(at(d));
    raw.up.load(at(d) + block);
  }
  __device__ __forceinline__ void make(int d, Raw& raw, const Kept& kept, float (&y)[8], float& squares) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = gated<ACT>(raw.gate.get(e), raw.up.get(e));
  }
  struct RawOne { T gate, up; };
  __device__ __forceinline__ void fetch_one(int d, RawOne& raw) const { raw.gate = at(d)[0], raw.up = at(d)[block]; }
  __device__ __forceinline__ float make_one(int d, const RawOne& raw, float& squares) const { return gated<ACT>(to_f32(raw.gate), to_f32(raw.up)); }
  __device__ __forceinline__ float again(int d) const { return gated<ACT>(to_f32(at(d)[0]), to_f32(at(d)[block])); }
};

// A row in registers, UNITS times eight numbers a thread, read once: by LANES of a warp (short rows, several a block) or, LANES 0, by
// a block. kVec: 16 bytes a load, eight neighbours a thread; else neighbours lie in neighbouring threads and the bytes are put
// together in shared memory. One exchange between the warps, of the largest magnitude and a norm's sum of squares at once; so a norm's
// integers are made of x * w alone, and its reciprocal root mean square goes into the scale. How a norm's row is shared out goes by
// its length, and by whether its operands and the rows behind them start on 16-byte borders, so that its result does not depend on how many
// there are. early: the next kernel may be scheduled while this one runs (not where the rows may be those of a weight: a product fetches
// its weight before it waits).
//
// Bound by memory, or at few rows by the chain load, exchange, store; beside memory by instructions (issue slots 64 to 69 % busy at
// 16384 x 4096). Measured (bytes read and written, each once): norm with residual of 8192 x 4096 39.6 us (5.9 TB/s; read once for each thing
// asked of the row 150), 4096 x 8192 42 (5.6), 65536 x 128 9.9, one row of 4,096 1.8; gate of 4096 x 12288 46.5 (5.4; four units a thread in 384
// threads 60, two in 768 so; wider ones than 768 threads hold by two have four: 12,296 65, 14,336 66, 16,384 71), plain rows of 8192 x 4096
// 19.4 (5.2), 6144 x 4097 in float32 off every border 33 (3.8), 333 x 5001 so 5.8: four bytes a load there.
template <typename Row, bool kVec, int UNITS, int LANES>
__global__ void __launch_bounds__(LANES || UNITS == 1 ? 256 : UNITS == 2 ? 768 : 512)
rows_int8_kernel(Row row, signed char* q, long long ldq, float* scales, int rows, int cols, int early) {
  if (early) pdl_trigger();
  pdl_wait();
  extern __shared__ __align__(16) unsigned char bytes[];
  __shared__ float part_squares[32];
  __shared__ unsigned part_most[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kRows = LANES ? 256 / LANES : 1;
  long long r = (long long)blockIdx.x * kRows + (LANES ? threadIdx.x / (LANES ? LANES : 1) : 0);
  const bool live = r < rows;
  if (LANES && !live) r = rows - 1;                  // reads and writes nothing, but takes part in what its warp does together
  const int me = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x, step = LANES ? LANES : blockDim.x;
  const int row_cols = cols;
  if (LANES && !live) cols = 0;
  row.begin(r);
  q += r * ldq;

  float y[UNITS][8], squares = 0.f;
  unsigned most = 0u;
  auto one = [&](int d) {
    typename Row::RawOne raw;
    row.fetch_one(d, raw);
    return row.make_one(d, raw, squares);
  };
  if constexpr (kVec) {
    constexpr int kAhead = UNITS < 4 ? UNITS : 2;      // units asked for before the first is used
#pragma unroll
    for (int u0 = 0; u0 < UNITS; u0 += kAhead) {
      typename Row::Raw raw[kAhead];
      typename Row::Kept kept[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int d = (me + (u0 + u) * step) * 8;
        if (d + 8 <= cols) row.fetch(d, raw[u]), row.keep(d, kept[u]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int d = (me + (u0 + u) * step) * 8;
        if (d + 8 <= cols) row.make(d, raw[u], kept[u], y[u0 + u], squares);
        else {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[u0 + u][e] = d + e < cols ? one(d + e) : 0.f;
        }
      }
    }
  } else {
    constexpr int kAhead = 8;                          // sixteen: rows of 5,001 in float32 6.1 -> 9.5 us (fewer rows on an SM)
#pragma unroll
    for (int i0 = 0; i0 < UNITS * 8; i0 += kAhead) {
      typename Row::RawOne raw[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int d = me + (i0 + i) * step;
        if (d < cols) row.fetch_one(d, raw[i]);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int d = me + (i0 + i) * step;
        y[(i0 + i) / 8][(i0 + i) % 8] = d < cols ? row.make_one(d, raw[i], squares) : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS * 8; i += 2) most = __vimax3_u32(most, magnitude(y[i / 8][i % 8]), magnitude(y[i / 8][i % 8 + 1]));
  if constexpr (LANES > 0 && LANES < 32) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if constexpr (Row::kNorm) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    }
  } else {
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (Row::kNorm) squares = warp_sum(squares);
  }
  if constexpr (LANES == 0) {
    if (lane == 0) {
      part_most[warp] = most;
      part_squares[warp] = squares;
    }
    __syncthreads();
    const int warps = blockDim.x >> 5;
    most = __reduce_max_sync(0xffffffffu, lane < warps ? part_most[lane] : 0u);
    if constexpr (Row::kNorm) squares = warp_sum(lane < warps ? part_squares[lane] : 0.f);
  }
  float common = 1.f;
  if constexpr (Row::kNorm) common = rsqrtf(squares / (float)row_cols + row.eps);
  const RowScale s(most, common);
  if (me == 0 && (!LANES || live)) scales[r] = s.scale;
  if (s.tiny) {
#pragma unroll
    for (int i = 0; i < UNITS * 8; ++i) y[i / 8][i % 8] *= 0x1p80f;
  }
  if constexpr (kVec) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int d = (me + u * step) * 8;
      const uint2 o = {s.four(y[u][0], y[u][1], y[u][2], y[u][3]), s.four(y[u][4], y[u][5], y[u][6], y[u][7])};
      if (d + 8 <= cols) *reinterpret_cast<uint2*>(q + d) = o;
      else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (d + e < cols) q[d + e] = (signed char)((e < 4 ? o.x : o.y) >> 8 * (e & 3));
      }
    }
  } else {
    unsigned char* mine = bytes + (LANES ? threadIdx.x / (LANES ? LANES : 1) * (LANES * UNITS * 8) : 0);
#pragma unroll
    for (int i = 0; i < UNITS * 8; ++i) {
      const int d = me + i * step;
      if (d < cols) mine[d] = (unsigned char)(s.byte(y[i / 8][i % 8]) & s.keep);
    }
    if constexpr (LANES > 0) __syncwarp();
    else __syncthreads();
    for (int d = me * 16; d < cols; d += step * 16) {
      if (d + 16 <= cols) *reinterpret_cast<uint4*>(q + d) = *reinterpret_cast<const uint4*>(mine + d);
      else
        for (int e = d; e < cols; ++e) q[e] = (signed char)mine[e];
    }
  }
}

// Many wide rows. What bounds the kernel above there is that registers hold what is on the way as well as what is at hand: of a norm's
// row of 12,288 with its residual one block fits an SM, and nothing is on the way while it exchanges and stores. Here rows come into
// shared memory by bulk copies, two or more ahead, one or two blocks an SM take them in turn, and a norm's weights stay in registers. A
// row is shared out as above, so its bits are the same. Measured (us, above -> this; bfloat16 norm with residual, without, plain rows):
//   4096 x 8704   58.0 -> 49.3, 47.3 -> 44.1, 28.4 -> 23.3        1200 x 12288, from L2   21.9 -> 18.1, 19.3 -> 16.3, 9.0 -> 9.4
//   4096 x 12288  97.2 -> 57.0 (6.2 TB/s), 83.6 -> 46.1, 34.7 -> 28.7        300 x 12288, from L2   7.5 -> 8.1, 7.1 -> 7.5, 3.8 -> 4.5
//   4096 x 16384  110 -> 86, 93 -> 53, 46.6 -> 35.6
// Without a residual that is 1.7 to 2.7 times the bytes' time (16.3, 23.1, 30.8). Shared memory is given out for two blocks an SM, but of a
// norm, with 97 registers a thread, one fits (of plain rows, with 57, two): the second half of the blocks runs behind the first, 14 % of an
// SM's warps are there, and the exchange of a row is overlapped by nothing.
// Gates and rows of up to 8,192 are faster above, and so are float32's plain rows (4096 x 12288 38 -> 43). Bound by memory; with a ring of
// two or three rows for one block (16384 with residual) by the wait for the next.
constexpr int kRingMost = 8, kRingUnits = 4, kRingBytes = 208 * 1024;

template <typename Row>
__global__ void __launch_bounds__(512)
ring_rows_int8_kernel(const Row row, signed char* q, long long ldq, float* scales, int rows, int cols, int stages, int early) {
  if (early) pdl_trigger();
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(8) unsigned long long bars[kRingMost];
  __shared__ float part_squares[2][32];
  __shared__ unsigned part_most[2][32];
  __shared__ int aborted;
  volatile int* abort_flag = &aborted;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, me = threadIdx.x, step = blockDim.x;
  const unsigned ring_base = tc::smem_u32(ring), bar_base = tc::smem_u32(bars), stage_bytes = row.bytes(cols);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) tc::mbar_init(bar_base + 8u * s, 1);
    aborted = 0;
    tc::mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  const int count = (rows - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  auto ask = [&](int i, int s) {                     // thread 0
    tc::mbar_expect_tx(bar_base + 8u * s, stage_bytes);
    row.copy(ring_base + s * stage_bytes, blockIdx.x + (long long)i * gridDim.x, cols, bar_base + 8u * s);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && i < count; ++i) ask(i, i);
  typename Row::Kept kept[kRingUnits];
#pragma unroll
  for (int u = 0; u < kRingUnits; ++u)
    if ((me + u * step) * 8 < cols) row.keep((me + u * step) * 8, kept[u]);
  int s = 0;
  unsigned parity = 0;
  bool ok = true;
  for (int i = 0; i < count; ++i) {
    const long long r = blockIdx.x + (long long)i * gridDim.x;
    Row mine = row, held = row;
    mine.begin(r);
    held.lies_at(ring + s * stage_bytes, cols);
    if (ok) ok = tc::mbar_wait(bar_base + 8u * s, parity, abort_flag, &g_rows_int8_error, 31);
    float y[kRingUnits][8], squares = 0.f;
    unsigned most = 0u;
#pragma unroll
    for (int u = 0; u < kRingUnits; ++u) {
      const int d = (me + u * step) * 8;
      typename Row::Raw raw;
      if (ok && d < cols) {
        held.fetch(d, raw);
        mine.make(d, raw, kept[u], y[u], squares);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[u][e] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < kRingUnits * 8; k += 2) most = __vimax3_u32(most, magnitude(y[k / 8][k % 8]), magnitude(y[k / 8][k % 8 + 1]));
    if (!ok) most = 0x7fffffffu;                     // what did not come is no number
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (Row::kNorm) squares = warp_sum(squares);
    if (lane == 0) {
      part_most[i & 1][warp] = most;
      part_squares[i & 1][warp] = squares;
    }
    __syncthreads();                                 // the stage is read; the other part may be written again
    if (threadIdx.x == 0 && i + stages < count && ok) ask(i + stages, s);
    most = __reduce_max_sync(0xffffffffu, lane < warps ? part_most[i & 1][lane] : 0u);
    if constexpr (Row::kNorm) squares = warp_sum(lane < warps ? part_squares[i & 1][lane] : 0.f);
    float common = 1.f;
    if constexpr (Row::kNorm) common = rsqrtf(squares / (float)cols + row.eps);
    const RowScale sc(most, common);
    if (me == 0) scales[r] = sc.scale;
    if (sc.tiny) {
#pragma unroll
      for (int k = 0; k < kRingUnits * 8; ++k) y[k / 8][k % 8] *= 0x1p80f;
    }
    signed char* to = q + r * ldq;
#pragma unroll
    for (int u = 0; u < kRingUnits; ++u) {
      const int d = (me + u * step) * 8;
      const uint2 o = {sc.four(y[u][0], y[u][1], y[u][2], y[u][3]), sc.four(y[u][4], y[u][5], y[u][6], y[u][7])};
      if (d < cols) *reinterpret_cast<uint2*>(to + d) = o;
    }
    if (++s == stages) s = 0, parity ^= 1;
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);      // copies still landing in this block's shared memory
  __syncthreads();
}

// Rows longer than 512 threads hold in registers: one block a row, read once for each thing that is asked of all of it.
template <typename Row>
__global__ void __launch_bounds__(1024) long_rows_int8_kernel(Row row, signed char* q, long long ldq, float* scales, int cols, int early) {
  if (early) pdl_trigger();
  pdl_wait();
  __shared__ float part_squares[32];
  __shared__ unsigned part_most[32];
  const long long r = blockIdx.x;
  row.begin(r);
  q += r * ldq;
  float squares = 0.f;
  unsigned most = 0u;
  for (int d = threadIdx.x; d < cols; d += 1024) {
    typename Row::RawOne raw;
    row.fetch_one(d, raw);
    most = max(most, magnitude(row.make_one(d, raw, squares)));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if constexpr (Row::kNorm) squares = warp_sum(squares);
  if ((threadIdx.x & 31) == 0) {
    part_most[threadIdx.x >> 5] = most;
    part_squares[threadIdx.x >> 5] = squares;
  }
  __syncthreads();
  most = __reduce_max_sync(0xffffffffu, part_most[threadIdx.x & 31]);
  float common = 1.f;
  if constexpr (Row::kNorm) common = rsqrtf(warp_sum(part_squares[threadIdx.x & 31]) / (float)cols + row.eps);
  const RowScale s(most, common);
  for (int d = threadIdx.x; d < cols; d += 1024) q[d] = (signed char)(s.byte(s.tiny ? row.again(d) * 0x1p80f : row.again(d)) & s.keep);
  if (threadIdx.x == 0) scales[r] = s.scale;
}

template <typename Row, bool kVec>
void launch_rows(const Row& row, signed char* q, long long ldq, float* scales, int rows, int cols, int early, cudaStream_t s) {
  const int units = ceil_div(cols, 8);
  if (units <= 64) {
    auto go = [&](auto kernel, int lanes) { oi_launch(kernel, ceil_div(rows, 256 / lanes), 256, kVec ? 0 : 8 * 512, s, row, q, ldq, scales, rows, cols, early); };
    if (units <= 16) go(rows_int8_kernel<Row, kVec, 1, 16>, 16);
    else if (units <= 32) go(rows_int8_kernel<Row, kVec, 1, 32>, 32);
    else go(rows_int8_kernel<Row, kVec, 2, 32>, 32);
    return;
  }
  // Rows of up to 1,024 in a block are back sooner (one row, us: norm 3.7 in a warp, 1.8 so), in a warp there are more of them on the way
  // (8,192 rows: 5.1, and 6.2 in blocks; 8192 x 640 5.7 -> 4.2, its gates 8.1 -> 7.3, float32 gates 7.7 -> 8.2 and so left in blocks, 2048 x 640
  // 3.1 -> 3.5). A norm's sum has one order whatever the number of rows; without one, either will do.
  if constexpr (!Row::kNorm) {
    constexpr bool kThree = !kVec || sizeof(typename Row::Raw) <= 32;
    if (units <= 128 && (units > 96 ? rows >= 2048 : kThree && rows >= 2560)) {
      auto go = [&](auto kernel) { oi_launch(kernel, ceil_div(rows, 8), 256, kVec ? 0 : 8 * 1024, s, row, q, ldq, scales, rows, cols, early); };
      if constexpr (kThree) {
        if (units <= 96) {
          go(rows_int8_kernel<Row, kVec, 3, 32>);
          return;
        }
      }
      go(rows_int8_kernel<Row, kVec, 4, 32>);
      return;
    }
  }
  auto go = [&](auto kernel, int each) {
    oi_launch(kernel, rows, ceil_div(ceil_div(units, each), 32) * 32, kVec ? 0 : ceil_div(cols, 16) * 16, s, row, q, ldq, scales, rows, cols, early);
  };
  if (units <= 256) go(rows_int8_kernel<Row, kVec, 1, 0>, 1);
  else if (units <= (Row::kNorm ? 1024 : 1536)) go(rows_int8_kernel<Row, kVec, 2, 0>, 2);
  else if (units <= 2048) go(rows_int8_kernel<Row, kVec, 4, 0>, 4);
  else if (units <= 4096) go(rows_int8_kernel<Row, kVec, 8, 0>, 8);
  else oi_launch(long_rows_int8_kernel<Row>, rows, 1024, 0, s, row, q, ldq, scales, cols, early);
}

// Where rows are more than what L2 holds for the kernel ahead and this one or, of a norm, where the kernel above has one block on an SM
// (320 threads or fewer of bfloat16 are two) and there are three for each.
template <typename Row>
bool ring_takes(const Row& row, int esize, int rows, int cols) {
  if (cols % 8 != 0 || cols <= 8192 || cols > 8 * kRingUnits * 512 || 2 * row.bytes(cols) > kRingBytes) return false;
  return (long long)rows * row.bytes(cols) >= 64 << 20 || (Row::kNorm && rows >= 3 * oi_sm_count() && (esize == 4 || cols > 10240));
}
template <typename Row>
int launch_ring(const Row& row, signed char* q, long long ldq, float* scales, int rows, int cols, int early, cudaStream_t s) {
  const int bytes = row.bytes(cols), blocks = 4 * bytes <= kRingBytes ? 2 : 1, fit = kRingBytes / blocks / bytes;
  const int stages = fit < kRingMost ? fit : kRingMost, most = oi_sm_count() * blocks;
  auto kernel = ring_rows_int8_kernel<Row>;
  static bool allowed[64];
  if (int bad = tc::allow_smem(kernel, kRingBytes, allowed)) return bad;
  oi_launch(kernel, rows < most ? rows : most, ceil_div(cols, 8 * kRingUnits * 32) * 32, stages * bytes, s, row, q, ldq, scales, rows, cols, stages, early);
  OI_CHECK_LAUNCH();
  return OI_OK;
}

// vec: everything that a row is read from starts on 16-byte borders, and the next row's too, whether there is one or not: one row
// of a matrix is shared out among the threads as it is among others
template <typename Row>
int launch(const Row& row, bool vec, void* q, long long ldq, float* scales, int rows, int cols, int early, cudaStream_t s) {
  if constexpr (Row::kRing) {
    if (vec && ring_takes(row, (int)sizeof(*row.x), rows, cols)) return launch_ring(row, (signed char*)q, ldq, scales, rows, cols, early, s);
  }
  if (vec) launch_rows<Row, true>(row, (signed char*)q, ldq, scales, rows, cols, early, s);
  else launch_rows<Row, false>(row, (signed char*)q, ldq, scales, rows, cols, early, s);
  OI_CHECK_LAUNCH();
  return OI_OK;
}

bool on_borders(const void* p, long long ld, int esize) { return (uintptr_t)p % 16 == 0 && ld * esize % 16 == 0; }

// Sixteen numbers a thread: neighbours where rows start on 16-byte borders, else one of each 1 << lanes_log; 256 >> lanes_log rows a
// block (65536 x 128 with a block a row 69 us, 5.9 so). Bound by memory: many long rows give a thread both its loads (kTimes 2) before
// it stores (the same buffers each time, some of them in L2: 8192 x 4096 16.2 us for 18.9 with one; 8 x 4096 1.5 for 1.3 and 8192 x 640 4.8
// for 3.8, so one there). From memory 8192 x 4096 takes 19.1 us (5.3 TB/s), 4096 x 12288 30.1; 6144 x 4097 into rows off every border 21, one
// byte a load and two a store.
// A byte becomes a number without a conversion: with its sign turned it is the last byte of 2^23 + 128 + q.
template <typename T, bool kVec, bool kWide, int kTimes>
__global__ void __launch_bounds__(256) dequantize_kernel(T* out, long long ldo, const signed char* q, long long ldq, const float* scales, int rows,
                                                         int cols, int lanes_log) {
  pdl_wait();                    // and no early trigger: see launch_dequantize
  if constexpr (kWide) lanes_log = 8;
  const int lanes = 1 << lanes_log, lane = threadIdx.x & (lanes - 1), step = kVec ? 1 : lanes;
  const long long r = ((long long)blockIdx.x << (8 - lanes_log)) + (threadIdx.x >> lanes_log);
  const int first = blockIdx.y * (lanes * 16 * kTimes) + (kVec ? lane * 16 : lane);
  if (r >= rows || first >= cols) return;
  const float scale = scales[r];
  out += r * ldo;
  q += r * ldq;
  uint4 v[kTimes];
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kTimes; ++i)
      if (first + i * lanes * 16 + 16 <= cols) v[i] = *reinterpret_cast<const uint4*>(q + first + i * lanes * 16);
  }
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int d = first + i * lanes * 16;
    if (kVec && d + 16 <= cols) {
      const unsigned words[4] = {v[i].x ^ 0x80808080u, v[i].y ^ 0x80808080u, v[i].z ^ 0x80808080u, v[i].w ^ 0x80808080u};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Eight<T> o;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const unsigned word = words[2 * h + e / 4];
          const float f0 = (__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7650 + e % 4)) - 8388736.f) * scale;
          const float f1 = (__uint_as_float(__byte_perm(word, 0x4b000000u, 0x7651 + e % 4)) - 8388736.f) * scale;
          o.set_pair(e, f0, f1);
        }
        o.store(out + d + 8 * h);
      }
    } else {
      signed char one[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) one[e] = d + e * step < cols ? q[d + e * step] : 0;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (d + e * step < cols) out[d + e * step] = from_f32<T>((float)one[e] * scale);
    }
  }
}

// What is written may be a weight or a cache that later kernels read before their wait (a weight brought back for a bfloat16 product):
// the kernel behind it on its stream starts when it has finished, whatever thread launches that one and whatever runs on other streams.
template <typename T>
int launch_dequantize(T* out, long long ldo, const signed char* q, long long ldq, const float* scales, int rows, int cols, cudaStream_t s) {
  const bool vec = on_borders(out, rows > 1 ? ldo : 0, sizeof(T));
  const bool two = vec && cols > 2048 && (long long)rows * cols >= 1 << 22;
  const int each = two ? 32 : 16;
  int lanes_log = 0;
  while (lanes_log < 8 && each << lanes_log < cols) ++lanes_log;
  const bool wide = lanes_log == 8;
  constexpr int kMostColumns = 1 << 27;          // of a launch: a grid has 65,535 blocks along a row at most
  auto go = [&](auto kernel) {
    for (int c0 = 0; c0 < cols; c0 += kMostColumns) {
      const int n = cols - c0 < kMostColumns ? cols - c0 : kMostColumns;
      const dim3 grid(ceil_div(rows, 256 >> lanes_log), ceil_div(n, each << lanes_log));
      oi_launch(kernel, grid, 256, 0, s, out + c0, ldo, q + c0, ldq, scales, rows, n, lanes_log);
    }
  };
  if (two) wide ? go(dequantize_kernel<T, true, true, 2>) : go(dequantize_kernel<T, true, false, 2>);
  else if (vec) wide ? go(dequantize_kernel<T, true, true, 1>) : go(dequantize_kernel<T, true, false, 1>);
  else wide ? go(dequantize_kernel<T, false, true, 1>) : go(dequantize_kernel<T, false, false, 1>);
  oi_fence_stream(s);
  OI_CHECK_LAUNCH();
  return OI_OK;
}

int check_rows(const char* what, const void* q, long long ldq, const float* scales, int rows, int cols) {
  OI_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 30), "%s: bad sizes rows=%d cols=%d", what, rows, cols);
  OI_REQUIRE(rows == 0 || (q && scales), "%s: a pointer is missing", what);
  OI_REQUIRE(rows <= 1 || ldq >= cols, "%s: rows of %d that start %lld apart", what, cols, ldq);
  return OI_OK;
}

}  // namespace

// q[r, :] (row stride ldq bytes) and scales[r] of x[r, :] (row stride ldx elements). early 0: what is written may be a weight, which
// kernels behind this one read before their wait.
OI_API int oi_quantize_int8(void* q, long long ldq, float* scales, const void* x, int dtype, long long ldx, int rows, int cols, int early,
                            void* stream) {
  if (int rc = check_rows("quantize_int8", q, ldq, scales, rows, cols)) return rc;
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "quantize_int8: unknown dtype code %d", dtype);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  const bool vec = on_borders(x, ldx, dtype == OI_F32 ? 4 : 2);
  if (dtype == OI_F32) return launch(PlainRow<float>{(const float*)x, ldx}, vec, q, ldq, scales, rows, cols, early, s);
  return launch(PlainRow<bf16>{(const bf16*)x, ldx}, vec, q, ldq, scales, rows, cols, early, s);
}

// The rows of oi_rmsnorm's output, not rounded: x <- round(x + delta) (stored; delta may be null), then
// x * rsqrt(mean(x^2) + eps) * (w_offset + w). Row strides ldx, ldd in elements.
OI_API int oi_rmsnorm_int8(void* q, long long ldq, float* scales, void* x, long long ldx, const void* delta, long long ldd, int dtype,
                           const void* w, int w_dtype, int rows, int cols, float eps, float w_offset, int early, void* stream) {
  if (int rc = check_rows("rmsnorm_int8", q, ldq, scales, rows, cols)) return rc;
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "rmsnorm_int8: unknown dtype code %d", dtype);
  OI_REQUIRE(w_dtype == OI_F32 || w_dtype == OI_BF16, "rmsnorm_int8: unknown weight dtype code %d", w_dtype);
  OI_REQUIRE(!delta || rows <= 1 || ldx >= cols, "rmsnorm_int8: rows of %d that start %lld apart cannot take a sum", cols, ldx);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  const int esize = dtype == OI_F32 ? 4 : 2;
  const bool vec = on_borders(x, ldx, esize) && (!delta || on_borders(delta, ldd, esize)) && (uintptr_t)w % 16 == 0;
  if (dtype == OI_F32)
    return launch(NormRow<float>{(float*)x, (const float*)delta, w, ldx, ldd, w_dtype, eps, w_offset}, vec, q, ldq, scales, rows, cols, early, s);
  return launch(NormRow<bf16>{(bf16*)x, (const bf16*)delta, w, ldx, ldd, w_dtype, eps, w_offset}, vec, q, ldq, scales, rows, cols, early, s);
}

// The rows of oi_silu_mul's output, not rounded: act(gate) * up of gate_up [rows, 2 inter] (row stride ldx elements), which lies
// in blocks of `block` gate values followed by their up values.
OI_API int oi_silu_mul_int8(void* q, long long ldq, float* scales, const void* gate_up, int dtype, long long ldx, int rows, int inter,
                            int block, int act, int early, void* stream) {
  if (int rc = check_rows("silu_mul_int8", q, ldq, scales, rows, inter)) return rc;
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "silu_mul_int8: unknown dtype code %d", dtype);
  OI_REQUIRE(block >= 1 && inter % block == 0, "silu_mul_int8: %d values in blocks of %d", inter, block);
  OI_REQUIRE(act == OI_ACT_SILU || act == OI_ACT_GELU_TANH, "silu_mul_int8: unknown activation code %d", act);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  int shift = block == inter ? -1 : -2;
  if (shift == -2 && (block & (block - 1)) == 0)
    for (shift = 0; 1 << shift < block; ++shift) {}
  const bool vec = block % 8 == 0 && on_borders(gate_up, ldx, dtype == OI_F32 ? 4 : 2);
  auto go = [&](auto row) { return launch(row, vec, q, ldq, scales, rows, inter, early, s); };
  if (dtype == OI_F32)
    return act == OI_ACT_SILU ? go(GateRow<float, OI_ACT_SILU>{(const float*)gate_up, ldx, block, shift})
                              : go(GateRow<float, OI_ACT_GELU_TANH>{(const float*)gate_up, ldx, block, shift});
  return act == OI_ACT_SILU ? go(GateRow<bf16, OI_ACT_SILU>{(const bf16*)gate_up, ldx, block, shift})
                            : go(GateRow<bf16, OI_ACT_GELU_TANH>{(const bf16*)gate_up, ldx, block, shift});
}

// out[r, :] = round(q[r, :] * scales[r]) (row stride ldo elements)
OI_API int oi_dequantize_int8(void* out, int dtype, long long ldo, const void* q, long long ldq, const float* scales, int rows, int cols,
                              void* stream) {
  OI_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 30), "dequantize_int8: bad sizes rows=%d cols=%d", rows, cols);
  OI_REQUIRE(dtype == OI_F32 || dtype == OI_BF16, "dequantize_int8: unknown dtype code %d", dtype);
  OI_REQUIRE(rows <= 1 || ldo >= cols, "dequantize_int8: rows of %d that start %lld apart", cols, ldo);
  if (rows == 0) return OI_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == OI_F32) return launch_dequantize((float*)out, ldo, (const signed char*)q, ldq, scales, rows, cols, s);
  return launch_dequantize((bf16*)out, ldo, (const signed char*)q, ldq, scales, rows, cols, s);
}

int oi_take_rows_int8_error(int* error) {
  OI_CHECK_CUDA(cudaMemcpyFromSymbol(error, g_rows_int8_error, sizeof(int)));
  if (*error != 0) {
    const int zero = 0;
    OI_CHECK_CUDA(cudaMemcpyToSymbol(g_rows_int8_error, &zero, sizeof(int)));
  }
  return OI_OK;
}
