// out[m, n] = (sum_k x[m, k] * w[n, k]) * sx[m] * sw[n] + bias[n] for 8-bit integers on the 5th-generation tensor cores
// (tcgen05.mma kind::i8). The sums are exact in 32-bit integers (K up to 131,071: 128 * 128 * K < 2^31), so no order of
// addition, tile or slice of K matters to a result; then float(sum) * sx * sw + bias in float32, in that order, and one
// rounding to the output's type.
//
// Three kernels: for up to 16 rows on mma.sync, for few and for many rows on tcgen05. The operands of the latter two are staged by TMA as
// rows of 128 bytes (128-byte swizzle); bytes beyond K or beyond the last row are zeros of the copy. Every wait on an mbarrier is
// bounded: one that runs out sets an error word and a flag that ends all roles of the CTA, which writes NaN for the results that it did
// not come to (of a cluster that adds up sums, all its CTAs do), still joins its cluster's barriers, frees its tensor memory and
// returns. No load uses cluster multicast.
#include <limits.h>

#include <atomic>

#include "oi_api.h"
#include "tcgen05.cuh"

int oi_take_rows_int8_error(int* error);    // rows_int8.cu

namespace {

constexpr int BM = 128;                     // rows of an operand's box
constexpr int BK = 128;                     // bytes of K a stage
constexpr int kBoxBytes = BM * BK;

__device__ int g_int8_error = 0;            // set to a non-zero code when a bounded wait ran out

// `runs_out`: the code of the wait that is taken as having run out, 0: none (oi_linear_int8_run_out, for tests)
std::atomic<int> g_runs_out{0};
__device__ __forceinline__ bool run_out(volatile int* abort_flag, int code) {
  *abort_flag = 1;
  atomicCAS(&g_int8_error, 0, code);
  return false;
}
__device__ __forceinline__ bool wait_on(unsigned bar, unsigned parity, volatile int* abort_flag, int code, int runs_out) {
  if (code == runs_out) return run_out(abort_flag, code);
  return tc::mbar_wait(bar, parity, abort_flag, &g_int8_error, code);
}
__device__ __forceinline__ float finish(int sum, float sx, float sw, float b, bool biased) {
  const float y = __fmul_rn(__fmul_rn((float)sum, sx), sw);
  return biased ? __fadd_rn(y, b) : y;
}

// A place in a ring of stages and the parity of its turn. (A division a stage by each of the threads that issue copies and products
// is on the path of every stage.)
struct Ring {
  int stage = 0;
  unsigned parity = 0;
  __device__ __forceinline__ void next(int stages) {
    if (++stage == stages) stage = 0, parity ^= 1;
  }
};

struct Scales {
  const float *sx, *sw, *bias;
};

// ------------------------------------------------------------------------------------------------
// Few rows. The product is formed transposed: 128 rows of w are the M side of tcgen05.mma, up to 256 rows of x (a multiple of
// 16, `bn`) its N side, so a weight byte goes HBM -> TMA -> shared memory -> tensor core, and the accumulator [128 rows of
// w x bn] lies in tensor memory. Grid (c, tiles of x, tiles of w; those that share a tile of w run together): a cluster of c CTAs (a
// power of two) shares one tile, CTA r streaming k blocks [r * kb_per_rank, ...) of it. Columns of the accumulator (rows of x) belong to the CTAs by fours in turn: each
// deposits what it has of the others' columns in their shared memory, 16 bytes a channel, and adds to its own, which stay in tensor
// memory, what the others left there. (All of a channel's columns to one CTA, its own part through shared memory too, us, weights from L2: 264 x
// 4096 x 12288 19.2 for 18.3, 400 x 2048 x 8192 14.5 for 12.5, 256 x 512 x 16384 10.2 for 9.2, 24 x 1024 x 1024 3.7 for 3.55.)
//   warp 0     one thread issues the copies; the first ring-full of WEIGHT boxes is requested before the wait for the kernel
//              ahead (programmatic dependent launch), which may still be writing x
//   warp 1     allocates tensor memory (behind that wait: a kernel ahead that needs all of it may not have taken its own
//              yet), one thread issues four products (K = 32) a stage
//   the others (four to sixteen) read the accumulator (one row of w a thread), deposit and add up, scale and store
// What the results cost shows in the instructions per column: with a column at a time, a branch and a cluster address each, and
// six warps, 128 columns took 8,000 cycles to deposit and 8,700 to store (N 1024, K 1024, c 1); stored two channels a lane, by lanes that
// trade halves, 4.6 us instead of 4.3 (500 x 4095 x 512).
// Measured (us, weights in turn, so from memory; in brackets what its bytes at the copy rate or its operations at twice the bfloat16 rate
// take): 32 x 24576 x 4096 18.5 (15.7), 64 x 6144 x 4096 8.8 (4.0), 512 x 4096 x 4096 10.6 (5.2), 264 x 4096 x 12288 18.4 (8.5; from L2 17.4),
// 777 x 5003 x 2001 into float32 11.8 (4.7).
// Bound by what one SM takes in (some 110 GB/s, 32 KB a stage of 128 rows) and, short sums, by launch, x, results.
constexpr int kFewColumns = 32, kMoreColumns = 64;      // up to so many rows of x a tile four warps read results, or eight, else sixteen

struct Shape {
  int M, N, num_kb, kb_per_rank, bn, stages, tmem_cols;
  int recv_offset;          // where deposits go: behind the ring, or over the drained ring (0)
  int scale_offset;         // scales of the tile's rows of x [bn]
  int bar_offset;
  int runs_out;
};

template <typename TOut, int kReaders>
__global__ void __launch_bounds__(64 + 32 * kReaders)
linear_int8_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, TOut* out, long long ldo,
                        const Scales scales, const Shape g) {
  pdl_trigger();
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned smem_base = tc::smem_u32(smem);
  const bool misaligned = (smem_base & 1023u) != 0;   // never seen; refuse rather than compute garbage
  const unsigned stage_bytes = kBoxBytes + g.bn * BK;
  const unsigned bar_base = smem_base + g.bar_offset;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (g.stages + s); };
  const unsigned acc_full = bar_base + 8u * (2 * g.stages);
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + g.bar_offset + 8 * (2 * g.stages + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x, csize = gridDim.x;
  const int n0 = blockIdx.z * BM, m0 = blockIdx.y * g.bn;
  const int kb0 = rank * g.kb_per_rank;
  int nkb = min(g.num_kb - kb0, g.kb_per_rank);
  nkb = nkb > 0 ? nkb : 0;
  if (misaligned) {
    nkb = 0;
    if (threadIdx.x == 0) atomicCAS(&g_int8_error, 0, 9);
  }

  if (threadIdx.x == 64) {
    tc::prefetch_map(&map_w);
    tc::prefetch_map(&map_x);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < g.stages; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), 1);
    }
    tc::mbar_init(acc_full, 1);
    *abort_flag = 0;
    tc::mbar_fence_init();
    const int pre = min(nkb, g.stages);
    for (int s = 0; s < pre; ++s) {
      tc::mbar_expect_tx(full_bar(s), stage_bytes);
      tc::tma_load_2d(smem_base + s * stage_bytes, &map_w, (kb0 + s) * BK, n0, full_bar(s));
    }
  }
  pdl_wait();
  if (warp == 1) {
    tc::tmem_alloc(tc::smem_u32(tmem_slot), g.tmem_cols);
    tc::tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    const int pre = min(nkb, g.stages);
    for (int s = 0; s < pre; ++s)
      tc::tma_load_2d(smem_base + s * stage_bytes + kBoxBytes, &map_x, (kb0 + s) * BK, m0, full_bar(s));
  }
  // what the sums are multiplied by is fetched under the copies: a channel's scale in its thread, later every row's in shared memory
  const int cols = min(g.bn, g.M - m0);  // rows of x in this tile
  const int quarter = warp & 3;          // a warp may only touch lanes [32 * (warp % 4), +32) of tensor memory
  const int row = quarter * 32 + lane, n = n0 + row;
  float sw = n < g.N ? scales.sw[n] : 0.f;
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const unsigned tmem_base = *tmem_slot;
  if (csize > 1) tc::cluster_arrive();   // phase 0: "this CTA runs"; waited for before anyone writes into it

  float* sx_s = reinterpret_cast<float*>(smem + g.scale_offset);
  if (warp >= 2) {
    for (int c = threadIdx.x - 64; c < g.bn; c += 32 * kReaders) sx_s[c] = c < cols ? scales.sx[m0 + c] : 0.f;
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * kReaders) : "memory");      // the warps that read results
  }
  const bool biased = scales.bias != nullptr;
  const float b = biased && n < g.N ? scales.bias[n] : 0.f;

  bool ok = !misaligned;
  if (warp == 0) {
    const bool leader = tc::elect_one();
    Ring at;
    for (int kb = g.stages; kb < nkb; ++kb, at.next(g.stages)) {
      const int s = at.stage;
      if (!wait_on(empty_bar(s), at.parity, abort_flag, 1, g.runs_out)) break;
      if (leader) {
        tc::mbar_expect_tx(full_bar(s), stage_bytes);
        const unsigned dst = smem_base + s * stage_bytes;
        tc::tma_load_2d(dst, &map_w, (kb0 + kb) * BK, n0, full_bar(s));
        tc::tma_load_2d(dst + kBoxBytes, &map_x, (kb0 + kb) * BK, m0, full_bar(s));
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    const bool leader = tc::elect_one();
    const unsigned idesc = tc::idesc_i8_s32(BM, g.bn);
    Ring at;
    for (int kb = 0; kb < nkb; ++kb, at.next(g.stages)) {
      const int s = at.stage;
      ok = wait_on(full_bar(s), at.parity, abort_flag, 2, g.runs_out);
      if (!ok) break;
      tc::fence_after();
      const unsigned a_addr = smem_base + s * stage_bytes;
      const unsigned long long da = tc::desc_k_major_sw128(a_addr), db = tc::desc_k_major_sw128(a_addr + kBoxBytes);
      if (leader) {
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)   // 32 bytes further along K inside the swizzle row: +2 in the address field
          tc::umma_i8(tmem_base, da + 2ull * k, db + 2ull * k, idesc, (kb | k) != 0 ? 1u : 0u);
        tc::umma_commit(empty_bar(s));
      }
      __syncwarp();
    }
    if (leader && ok && nkb > 0) tc::umma_commit(acc_full);
  } else if (nkb > 0) {
    ok = __all_sync(0xffffffffu, wait_on(acc_full, 0, abort_flag, 3, g.runs_out));
    tc::fence_after();
  }
  const float nan = __int_as_float(0x7fffffff);
  if (!ok) sw = nan;                     // of a sum that did not come
  if (csize > 1) {
    __syncwarp();
    tc::cluster_wait();                  // phase 0
    if (g.recv_offset == 0) {            // deposits go over the ring: every CTA's products have read theirs first
      __syncthreads();                   // (warps 0 and 1 come here before the products are done, the others after)
      tc::cluster_arrive();
      tc::cluster_wait();
    }
  }
  const unsigned tmem_row = tmem_base + ((unsigned)(quarter * 32) << 16);
  auto read = [&](int c0, unsigned (&v)[16]) {                // sixteen columns of this thread's channel
    if (nkb > 0 && ok) {
      tc::tmem_ld16(tmem_row + (unsigned)c0, v);
      tc::tmem_ld_wait();
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0u;
    }
  };
  // Four columns are a piece; piece p belongs to CTA p % c, which gets 16 bytes a channel from each of the others.
  const int first = 16 * ((warp - 2) >> 2), last_rank = csize - 1, shift = __popc(last_rank);
  const unsigned recv = smem_base + g.recv_offset + (unsigned)row * 16;
  if (warp >= 2) {
#pragma unroll 1
    for (int c0 = first; c0 < cols; c0 += 4 * kReaders) {
      unsigned v[16];
      read(c0, v);
      if (csize > 1) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int piece = (c0 + e) >> 2, owner = piece & last_rank;
          if (c0 + e < cols && owner != rank)
            asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};\n"
                         ::"r"(tc::map_to_rank(recv, owner) + (unsigned)((piece >> shift) * last_rank + rank - (rank > owner)) * (BM * 16)),
                           "r"(v[e]), "r"(v[e + 1]), "r"(v[e + 2]), "r"(v[e + 3]) : "memory");
        }
      } else {
        float y[16];
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 sx = *reinterpret_cast<const float4*>(sx_s + c0 + e);
          y[e] = finish((int)v[e], sx.x, sw, b, biased), y[e + 1] = finish((int)v[e + 1], sx.y, sw, b, biased);
          y[e + 2] = finish((int)v[e + 2], sx.z, sw, b, biased), y[e + 3] = finish((int)v[e + 3], sx.w, sw, b, biased);
        }
        TOut* at = out + (size_t)(m0 + c0) * ldo + n;
        if (n < g.N) {
#pragma unroll
          for (int e = 0; e < 16; ++e, at += ldo)
            if (c0 + e < cols) *at = from_f32<TOut>(y[e]);
        }
      }
    }
  }
  if (csize > 1) {
    if (warp >= 2 && !ok && lane < csize)  // the CTAs that add up hear of a part that did not come
      asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(tc::map_to_rank(tc::smem_u32((const void*)abort_flag), lane)), "r"(1) : "memory");
    __syncwarp();
    tc::cluster_arrive();                // this CTA's deposits are made ...
    tc::cluster_wait();                  // ... and so are everybody's; nothing remote is touched after this
    if (*abort_flag) sw = nan;
    if (warp >= 2) {
      const unsigned char* mine = smem + g.recv_offset + (size_t)row * 16;
#pragma unroll 1
      for (int c0 = first; c0 < cols; c0 += 4 * kReaders) {
        if (csize == 8 && ((c0 >> 4) & 1) != rank >> 2) continue;       // none of these four pieces
        unsigned v[16];
        read(c0, v);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int piece = (c0 + e) >> 2;
          if ((piece & last_rank) != rank || c0 + e >= cols) continue;
          int4 sum = make_int4((int)v[e], (int)v[e + 1], (int)v[e + 2], (int)v[e + 3]);
          for (int q = 0; q < last_rank; ++q) {
            const int4 part = *reinterpret_cast<const int4*>(mine + (size_t)((piece >> shift) * last_rank + q) * (BM * 16));
            sum.x += part.x, sum.y += part.y, sum.z += part.z, sum.w += part.w;
          }
          const float4 sx = *reinterpret_cast<const float4*>(sx_s + c0 + e);
          TOut* at = out + (size_t)(m0 + c0 + e) * ldo + n;
          if (n < g.N) {
            *at = from_f32<TOut>(finish(sum.x, sx.x, sw, b, biased));
            if (c0 + e + 1 < cols) at[ldo] = from_f32<TOut>(finish(sum.y, sx.y, sw, b, biased));
            if (c0 + e + 2 < cols) at[2 * ldo] = from_f32<TOut>(finish(sum.z, sx.z, sw, b, biased));
            if (c0 + e + 3 < cols) at[3 * ldo] = from_f32<TOut>(finish(sum.w, sx.w, sw, b, biased));
          }
        }
      }
    }
  }
  tc::fence_before();
  if (*abort_flag && threadIdx.x == 0) {
    // copies that were issued may still be landing in this CTA's shared memory: give them time
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_dealloc(tmem_base, g.tmem_cols);
  }
}

// ------------------------------------------------------------------------------------------------
// Many rows, transposed as above. Pairs of CTAs (a cluster of two, cta_group::2) compute tiles of 256 channels x `bn` rows of x (a
// multiple of 32 up to 256: rows are shared out evenly over the tiles, so 777 of them need not be 1,024), persistent: pair p
// works on tiles p, p + pairs, ... (tiles of x fastest, so that pairs that run at the same time share tiles of w through L2).
// The CTA of rank r holds 128 of the tile's rows of w and half of its rows of x in its shared memory, so a byte of x is fetched
// once for 256 channels, and the accumulator of its 128 channels x bn columns in its tensor memory, double buffered: while the
// other warps drain one tile the next is formed.
//   warp 0      of both CTAs loads its own halves, counted on the even CTA's "full" barrier
//   warp 1      of the even CTA issues the products (M = 256, N = bn, K = 32) for both
//   warps 2-17  of both CTAs drain their own tensor memory (32 channels a warp, every fourth group of rows) and arrive on the even
//               CTA's "drained" barrier. A warp scales 32 channels of a few rows, turns them in shared memory, and a TMA store carries
//               them out: 4096 x 4096 x 512 takes 18.5 us so (float32 21; 16.5 with channels across the tile, whose rows need
//               no turning, but then tiles are 256 rows high), with 16-byte stores by the warps 3 and 8 more.
// Measured (us, by the clock that power leaves; at twice the bfloat16 rate): 8192 x 24576 x 4096 480 to 590 (502; 3.4 POP/s at best, the
// library's bfloat16 product 1017), 2048 x 4096 x 4096 26 to 29 (21), 777 x 24576 x 4096 62 (48; tiles of 256 rows 71), 264 x 24576 x 4096 31 to 34
// (17.5; 36), a head of 151936 x 4096 with 64 rows 102 (98). Bound by the tensor cores and their power
// where tiles fill the pairs evenly, else by the last round of them; with K of 512 by the results.
constexpr int kEpilogueWarps = 16;
constexpr int kParts = kEpilogueWarps / 4;                          // the warps of a quarter of the lanes share the rows of x
constexpr int kPairThreads = 64 + 32 * kEpilogueWarps;
constexpr int kBufferBytes = 2048;                                  // a warp's results on their way out: 32 channels of 32 or (float32) 16 rows
constexpr int kPairMostStages = 8;
constexpr int kPairRingBytes = 180 * 1024;
constexpr int kPairBufferOffset = kPairRingBytes;
constexpr int kPairScaleOffset = kPairBufferOffset + kEpilogueWarps * kBufferBytes;      // per warp the scales of its rows of x
constexpr int kPairBarOffset = kPairScaleOffset + kEpilogueWarps * (256 / kParts) * 4;   // full, empty, acc_full[2], acc_empty[2], tmem slot, abort
constexpr int kPairSmem = kPairBarOffset + (2 * kPairMostStages + 4) * 8 + 16 + 1024;
static_assert(kPairSmem <= 227 * 1024, "more shared memory than a CTA may have");

template <typename TOut>
__global__ void __launch_bounds__(kPairThreads)
linear_int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                        const __grid_constant__ CUtensorMap map_out, TOut* out, long long ldo, const Scales scales, int M, int N, int num_kb,
                        int bn, int stages, int tma_out, int runs_out) {
  pdl_start();
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const unsigned smem_base = tc::smem_u32(smem);
  const unsigned bar_base = smem_base + kPairBarOffset;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kPairMostStages + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (2 * kPairMostStages + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (2 * kPairMostStages + 2 + a); };
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + kPairBarOffset + (2 * kPairMostStages + 4) * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = tc::cluster_ctarank();
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int m_tiles = (M + bn - 1) / bn, num_tiles = m_tiles * ((N + 255) / 256);
  const unsigned stage_bytes = kBoxBytes + (bn / 2) * BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      tc::mbar_init(acc_full_bar(a), 1);
      tc::mbar_init(acc_empty_bar(a), 2 * kEpilogueWarps);      // one arrival per epilogue warp of both CTAs
    }
    *abort_flag = 0;
    tc::mbar_fence_init();
  }
  if (warp == 1) {
    tc::tmem_alloc_pair(tc::smem_u32(tmem_slot), 512);
    tc::tmem_relinquish_pair();
  }
  tc::fence_before();
  tc::cluster_arrive();                        // barriers and tensor memory of both CTAs are ready
  tc::cluster_wait();
  tc::fence_after();
  const unsigned tmem_base = *tmem_slot;

  if (warp == 0) {
    const bool leader = tc::elect_one();
    Ring at;
    int ahead = stages;                              // stages that have not been used yet
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      const int m0 = (tile % m_tiles) * bn + (int)rank * (bn / 2), n0 = (tile / m_tiles) * 256 + (int)rank * 128;
      for (int kb = 0; kb < num_kb; ++kb, at.next(stages)) {
        const int s = at.stage;
        if (ahead > 0) --ahead;
        else if (!wait_on(empty_bar(s), at.parity ^ 1, abort_flag, 11, runs_out)) { ok = false; break; }
        if (leader) {
          if (rank == 0) tc::mbar_expect_tx(full_bar(s), 2 * stage_bytes);
          const unsigned counted_on = tc::map_to_rank(full_bar(s), 0);
          const unsigned dst = smem_base + s * stage_bytes;
          tc::tma_load_2d_pair(dst, &map_w, kb * BK, n0, counted_on);
          tc::tma_load_2d_pair(dst + kBoxBytes, &map_x, kb * BK, m0, counted_on);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = tc::elect_one();
      const unsigned idesc = tc::idesc_i8_s32(256, bn);
      Ring at;
      int local = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs, ++local) {
        const int a = local & 1;
        if (local >= 2) {
          ok = runs_out == 14 ? run_out(abort_flag, 14)
                              : tc::mbar_wait_cluster(acc_empty_bar(a), (unsigned)((local >> 1) - 1) & 1, abort_flag, &g_int8_error, 14);
          if (!ok) break;
          tc::fence_after();
        }
        const unsigned tmem_acc = tmem_base + (unsigned)(a * 256);
        for (int kb = 0; kb < num_kb; ++kb, at.next(stages)) {
          const int s = at.stage;
          ok = wait_on(full_bar(s), at.parity, abort_flag, 12, runs_out);
          if (!ok) break;
          tc::fence_after();
          const unsigned a_addr = smem_base + s * stage_bytes;
          const unsigned long long da = tc::desc_k_major_sw128(a_addr), db = tc::desc_k_major_sw128(a_addr + kBoxBytes);
          if (leader) {
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              tc::umma_i8_pair(tmem_acc, da + 2ull * k, db + 2ull * k, idesc, (kb | k) != 0 ? 1u : 0u);
            tc::umma_commit_pair(empty_bar(s), 3);
          }
          __syncwarp();
        }
        if (leader && ok) tc::umma_commit_pair(acc_full_bar(a), 3);
        __syncwarp();
      }
    }
  } else {
    const int quarter = warp & 3;                    // a warp may only touch lanes [32 * (warp % 4), +32)
    const int part = (warp - 2) >> 2;
    constexpr int kTake = kBufferBytes / 32 / (int)sizeof(TOut);      // rows of x at a time
    constexpr int kTurns = 256 / kTake / kParts;                      // of this warp in a tile
    unsigned char* buffer = smem + kPairBufferOffset + (warp - 2) * kBufferBytes;
    float* sx_s = reinterpret_cast<float*>(smem + kPairScaleOffset) + (warp - 2) * (256 / kParts);
    const bool biased = scales.bias != nullptr;
    int local = 0;
    // the next tile's scales are asked for a tile ahead: where sums are short the results, not the products, take the time
    float next_sw, next_b, next_sx[2];
    auto ask = [&](int tile) {
      const bool there = tile < num_tiles;
      const int n = (tile / m_tiles) * 256 + (int)rank * 128 + quarter * 32 + lane;
      next_sw = there && n < N ? scales.sw[n] : 0.f;
      next_b = there && biased && n < N ? scales.bias[n] : 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = 32 * i + lane, row = (at / kTake * kParts + part) * kTake + at % kTake, m = (tile % m_tiles) * bn + row;
        next_sx[i] = there && row < bn && m < M ? scales.sx[m] : 0.f;
      }
    };
    ask(pair);
    bool ok = true;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++local) {
      const int a = local & 1;
      const int m0 = (tile % m_tiles) * bn, n0 = (tile / m_tiles) * 256 + (int)rank * 128 + quarter * 32;
      float sw = next_sw, b = next_b;
      sx_s[lane] = next_sx[0];
      sx_s[32 + lane] = next_sx[1];
      __syncwarp();
      ask(tile + num_pairs);
      if (ok) ok = __all_sync(0xffffffffu, wait_on(acc_full_bar(a), (unsigned)(local >> 1) & 1, abort_flag, 13, runs_out));
      tc::fence_after();
      if (!ok) sw = __int_as_float(0x7fffffff);      // of sums that did not come
      const unsigned tmem_acc = tmem_base + (unsigned)(a * 256) + ((unsigned)(quarter * 32) << 16);
      const int turns = ((min(bn, M - m0) + kTake - 1) / kTake - part + kParts - 1) / kParts;      // groups of rows that are this warp's
#pragma unroll 1
      for (int i = 0; i < kTurns; ++i) {
        unsigned v[kTake];
        const int row0 = (i * kParts + part) * kTake;
        if (i < turns && ok) {
          if constexpr (kTake == 32) tc::tmem_ld32(tmem_acc + (unsigned)row0, v);
          else tc::tmem_ld16(tmem_acc + (unsigned)row0, v);
          tc::tmem_ld_wait();
        }
        if (i >= turns - 1) {                        // all of this warp's part is read: the products may fill it again
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(tc::map_to_rank(acc_empty_bar(a), 0));
        }
        if (i < turns && n0 < N) {
          TOut y[kTake];
#pragma unroll
          for (int e = 0; e < kTake; e += 4) {
            const float4 sx = *reinterpret_cast<const float4*>(sx_s + i * kTake + e);
            y[e] = from_f32<TOut>(finish((int)v[e], sx.x, sw, b, biased)), y[e + 1] = from_f32<TOut>(finish((int)v[e + 1], sx.y, sw, b, biased));
            y[e + 2] = from_f32<TOut>(finish((int)v[e + 2], sx.z, sw, b, biased)), y[e + 3] = from_f32<TOut>(finish((int)v[e + 3], sx.w, sw, b, biased));
          }
          if (lane == 0) tc::bulk_wait<0>();         // the buffer's last contents are on their way
          __syncwarp();
          TOut* held = reinterpret_cast<TOut*>(buffer) + lane;      // a row of x: 32 channels next to each other
#pragma unroll
          for (int e = 0; e < kTake; ++e) held[e * 32] = y[e];
          if (tma_out) {
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tc::tma_store_2d(&map_out, tc::smem_u32(buffer), n0, m0 + row0);
              tc::bulk_commit();
            }
          } else {
            // Result rows that do not start on 16-byte borders: four bytes a lane. A row of bfloat16 may start between two four-byte
            // borders: its pairs are then put together from neighbours' words, its first and last number stored alone.
            __syncwarp();
            constexpr int kWords = 32 * (int)sizeof(TOut) / 4, kRowsAtOnce = 32 / kWords;
            const int own_row = lane / kWords, word = lane % kWords, left = min(32, N - n0), live_rows = min(kTake, M - m0 - row0);
            TOut* dst = out + (size_t)(m0 + row0 + own_row) * ldo + n0;
#pragma unroll 4
            for (int r = own_row; r < kTake; r += kRowsAtOnce, dst += kRowsAtOnce * ldo) {
              const unsigned own = reinterpret_cast<const unsigned*>(buffer)[r * kWords + word];
              const bool live = r < live_rows;
              if constexpr (sizeof(TOut) == 4) {
                if (live && word < left) dst[word] = __uint_as_float(own);
              } else {
                const unsigned next = __shfl_down_sync(0xffffffffu, own, 1);
                const int odd = (int)((uintptr_t)dst >> 1) & 1, at = 2 * word + odd;
                const unsigned two = odd ? __byte_perm(own, next, 0x5432) : own;
                if (live && at + 1 < left) *reinterpret_cast<unsigned*>(dst + at) = two;
                else if (live && at < left) dst[at] = __ushort_as_bfloat16((unsigned short)two);
                if (live && odd && word == 0) dst[0] = __ushort_as_bfloat16((unsigned short)own);
              }
            }
            __syncwarp();
          }
        }
        if (i >= turns - 1) break;
      }
    }
    if (lane == 0) tc::bulk_wait<0, true>();
  }

  tc::fence_before();
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  tc::cluster_arrive();                        // neither CTA reads or is read by the other from here on
  tc::cluster_wait();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------
// Up to 16 rows, on mma.sync: what counts is the chain behind the wait for x, and the kernel above has a TMA copy of x, a
// tensor-memory round trip, deposits and a cluster barrier there. One CTA per SM owns whole rows of w, 16 at a time, so no sums cross
// CTAs:
//   warp 8     copies rows into shared memory (cp.async.bulk, one copy per row of a stage, counted on an mbarrier), as many as the
//              ring holds before the kernel ahead on the stream has finished; it waits for that one, however long it takes, before
//              it waits for a free stage, which is bounded
//   warps 0-7  share out K (blocks of 128 bytes in turn). After the wait a warp reads its part of x straight into the registers that
//              mma.sync takes as operand B (rows of x on the 8-column side); 16 rows of w are operand A. The k index inside a block is
//              permuted alike for both, so 32 contiguous bytes of a row are a lane's fragments of four products. The eight warps'
//              sums meet in shared memory.
// Rows of a stage are 2,048 + 16 bytes apart, so that the eight lanes that a 16-byte shared load serves at once hit different banks.
// Bytes of x behind K are made zeros; whatever lies there in w then does not count. Sixteen lanes that each ask for a row fill the ring
// sooner, one elected lane that asks for all keeps up a longer stream (with a norm ahead, us: N 9216 K 2048 5.1 and 5.6, N 24576 K 4096
// 18.7 and 17.7), so the one is taken where the ring holds all of a CTA's rows, the other where it does not.
//
// Measured (us, one row, a norm and the product in turn inside a graph; the kernel above at its best -> this one; the norm alone 1.7
// to 1.9): N 4096 K 4096 6.9 -> 5.6, N 6144 K 4096 8.9 -> 6.8, N 9216 K 2048 7.3 -> 5.1, N 24576 K 4096 20.5 -> 17.7 (its bytes: 15.4). With
// eight rows 7.5 -> 5.9, 9.2 -> 7.3, 7.4 -> 5.5, 21.0 -> 18.2. What bounds it: the stream where the ring is shorter than a CTA's rows, else
// the chain behind the wait; many short rows are a barrier for each 32 of them (N 16384 K 1024 7.7 above, 8.1 here).
constexpr int kFewWarps = 8, kFewThreads = (kFewWarps + 1) * 32;
constexpr int kChunkBlocks = 2, kChunk = kChunkBlocks * kFewWarps * 128;     // bytes of a row in a stage
constexpr int kFewRowBytes = kChunk + 16, kFewStage = 16 * kFewRowBytes, kFewMostStages = 6;
constexpr int kFewPart = 8192;                 // the warps' sums: 8 x 16 x 16, or twice 8 x 16 x 8

struct FewArgs {
  const signed char *x, *w;
  void* out;
  long long ldx, ldw, ldo;
  Scales scales;
  int M, N, K, groups, stages;
  int at_once;              // the ring holds all of a CTA's rows
  int runs_out;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(unsigned addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// 16 bytes of a row of x from byte k on, past L1 (other SMs have just written them); what lies at K and behind is zero. The 16 bytes that
// hold byte K - 1 belong to the row: rows start on 16-byte borders.
__device__ __forceinline__ uint4 load_x16(const signed char* row, int k, int K) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (k < K) {
    v = __ldcg(reinterpret_cast<const uint4*>(row + k));
    if (K - k < 16) {
      unsigned* words = reinterpret_cast<unsigned*>(&v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int left = K - k - 4 * i;
        words[i] &= left >= 4 ? 0xffffffffu : left > 0 ? (1u << 8 * left) - 1u : 0u;
      }
    }
  }
  return v;
}
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(kFewWarps * 32) : "memory"); }

// NT: groups of eight rows of x; B: blocks of a warp over the whole row
template <int NT, int B, typename TOut>
__global__ void __launch_bounds__(kFewThreads)
linear_int8_few_kernel(const __grid_constant__ FewArgs a) {
  pdl_trigger();
  constexpr int kHeld = 2 / NT, kTokens = 8 * NT, kEach = 16 * kTokens;          // groups whose sums wait for one barrier: 256 sums
  static_assert(kHeld * kFewWarps * kEach * 4 == kFewPart && kHeld * kEach == kFewWarps * 32, "one sum a thread");
  extern __shared__ __align__(1024) unsigned char smem[];
  int* part = reinterpret_cast<int*>(smem);                  // [held][warp][rows of w][rows of x]
  const unsigned ring = tc::smem_u32(smem) + kFewPart, bars = ring + a.stages * kFewStage;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kFewPart + a.stages * (kFewStage + 16));
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (a.stages + s); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunks = (a.K + kChunk - 1) / kChunk, blocks = (a.K + 127) / 128;
  const int turn = blockIdx.x % chunks;                      // the chunk of a row that this CTA begins with: not all read the same of x at once
  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      tc::mbar_init(full_bar(s), 1);
      tc::mbar_init(empty_bar(s), kFewWarps);
    }
    *abort_flag = 0;
    tc::mbar_fence_init();
  }
  __syncthreads();

  if (warp == kFewWarps) {
    const bool leader = tc::elect_one();
    const unsigned long long once = tc::policy_evict_first();
    Ring at;
    int ahead = a.stages;
    bool ok = true, waited = false;
    for (int grp = blockIdx.x; grp < a.groups && ok; grp += gridDim.x) {
      const int rows = min(16, a.N - grp * 16);
      const signed char* from = a.w + (size_t)grp * 16 * a.ldw;
      for (int c = 0; c < chunks; ++c, at.next(a.stages)) {
        if (ahead > 0) --ahead;
        else {
          if (!waited) pdl_wait(), waited = true;
          if (!wait_on(empty_bar(at.stage), at.parity ^ 1, abort_flag, 21, a.runs_out)) { ok = false; break; }
        }
        const int k0 = (c + turn < chunks ? c + turn : c + turn - chunks) * kChunk;
        const unsigned len = (unsigned)min((a.K - k0 + 15) & ~15, kChunk), dst = ring + at.stage * kFewStage;
        if (leader) tc::mbar_expect_tx(full_bar(at.stage), rows * len);
        __syncwarp();
        if (a.at_once) {
          if (lane < rows) tc::bulk_load_hint(dst + lane * kFewRowBytes, from + k0 + lane * a.ldw, len, full_bar(at.stage), once);
        } else if (leader) {
          const signed char* src = from + k0;
#pragma unroll 4
          for (int r = 0; r < rows; ++r, src += a.ldw) tc::bulk_load_hint(dst + r * kFewRowBytes, src, len, full_bar(at.stage), once);
        }
        __syncwarp();
      }
    }
  } else {
    const int g = lane >> 2, c4 = lane & 3;
    auto block_of = [&](int i) {                             // the i-th block of this warp
      const int c = i / kChunkBlocks + turn;
      return ((c < chunks ? c : c - chunks) * kChunkBlocks + (i & 1)) * kFewWarps + warp;
    };
    const unsigned my_w = ring + g * kFewRowBytes + warp * 128 + c4 * 32;
    // this thread's sum of every batch of groups: row m of x, channel `col` of group `f`
    const int f = threadIdx.x / kEach, m = threadIdx.x / 16 % kTokens, col = threadIdx.x % 16;
    const bool biased = a.scales.bias != nullptr;
    auto channel = [&](int first) { return ((long long)first + f * (int)gridDim.x) * 16 + col; };
    auto asked = [&](const float* of, int first) { return channel(first) < a.N ? of[channel(first)] : 0.f; };
    bool ok = wait_on(full_bar(0), 0, abort_flag, 22, a.runs_out);       // weights: not waited for behind x
    pdl_wait();
    uint4 xr[B][NT][2];
#pragma unroll
    for (int i = 0; i < B; ++i) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int k = i / kChunkBlocks < chunks ? block_of(i) * 128 + c4 * 32 : a.K, m = g + 8 * t;
#pragma unroll
        for (int h = 0; h < 2; ++h) xr[i][t][h] = m < a.M ? load_x16(a.x + (size_t)m * a.ldx, k + 16 * h, a.K) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
    const float sx = m < a.M ? a.scales.sx[m] : 0.f;
    float next_sw = asked(a.scales.sw, blockIdx.x);          // a batch ahead
    float next_b = biased ? asked(a.scales.bias, blockIdx.x) : 0.f, sw = 0.f, b = 0.f;

    Ring at;
    int held = 0, first = blockIdx.x;
    for (int grp = blockIdx.x; grp < a.groups; grp += gridDim.x) {
      if (held == 0) {
        sw = next_sw, b = next_b;
        next_sw = asked(a.scales.sw, first + kHeld * gridDim.x);
        if (biased) next_b = asked(a.scales.bias, first + kHeld * gridDim.x);
      }
      int acc[NT][2][4] = {};
#pragma unroll
      for (int c = 0; c < B / kChunkBlocks; ++c) {
        if (c < chunks) {
          if (ok) ok = wait_on(full_bar(at.stage), at.parity, abort_flag, 22, a.runs_out);
          const unsigned src = my_w + at.stage * kFewStage;
#pragma unroll
          for (int j = 0; j < kChunkBlocks; ++j) {
            const int i = c * kChunkBlocks + j;
            if (block_of(i) < blocks) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const unsigned at16 = src + j * kFewWarps * 128 + h * 16;
                const uint4 lo = lds128(at16), hi = lds128(at16 + 8 * kFewRowBytes);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                  mma_s8(acc[t][0], lo.x, hi.x, lo.y, hi.y, xr[i][t][h].x, xr[i][t][h].y);
                  mma_s8(acc[t][1], lo.z, hi.z, lo.w, hi.w, xr[i][t][h].z, xr[i][t][h].w);
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(empty_bar(at.stage));
          at.next(a.stages);
        }
      }
      int* dst = part + (held * kFewWarps + warp) * kEach;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          *reinterpret_cast<int2*>(dst + (q * 8 + g) * kTokens + t * 8 + c4 * 2) =
              make_int2(acc[t][0][2 * q] + acc[t][1][2 * q], acc[t][0][2 * q + 1] + acc[t][1][2 * q + 1]);
      }
      const bool last = grp + (int)gridDim.x >= a.groups;
      if (++held == kHeld || last) {
        few_sync();
        if (*abort_flag) sw = __int_as_float(0x7fffffff);    // of sums that did not come
        const long long n = channel(first);
        if (f < held && m < a.M && n < a.N) {
          const int* src = part + f * kFewWarps * kEach + col * kTokens + m;
          int sum = 0;
#pragma unroll
          for (int q = 0; q < kFewWarps; ++q) sum += src[q * kEach];
          reinterpret_cast<TOut*>(a.out)[(size_t)m * a.ldo + n] = from_f32<TOut>(finish(sum, sx, sw, b, biased));
        }
        held = 0;
        first = grp + gridDim.x;
        if (!last) few_sync();
      }
    }
  }
  __syncthreads();
  if (*abort_flag && threadIdx.x == 0)
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);        // copies still landing in this CTA's shared memory
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------ host side
constexpr int kMostStages = 12, kSmemOfTwo = 110 * 1024, kSmemOfOne = 208 * 1024;

// Result rows that start and end on 16-byte borders can be copied out by TMA. (Of a row that ends inside 16 bytes the copy writes
// what is behind the end, too.)
template <typename TOut>
bool rows_on_borders(const TOut* out, long long ldo, int N) {
  return (uintptr_t)out % 16 == 0 && ldo * sizeof(TOut) % 16 == 0 && N * sizeof(TOut) % 16 == 0;
}

// The height of z tiles of x, of equal size. (In sixteens: fewer of that height may hold all rows, and only those are launched. The
// estimate below goes by the z that was asked for: so its constants were measured. Over 24 sizes where that makes a difference: 50 x 2816
// x 2304 7.3 us with the empty tiles, 6.95 without; 125 x 640 x 7424 7.9 and 7.7; others the same. Of a choice among full tiles alone
// 551 x 128 x 1792 took 5.9 us instead of 5.4.)
int few_rows_height(int M, int z) { return ceil_div(ceil_div(M, z), 16) * 16; }

// What a launch for c slices of K and tiles of bn rows of x needs, and its shared memory
Shape few_rows_shape(int M, int N, int K, int c, int bn, int& smem) {
  const int z = ceil_div(M, bn);
  Shape g = {};
  g.M = M, g.N = N, g.runs_out = g_runs_out, g.bn = bn;
  g.num_kb = ceil_div(K, BK);
  g.kb_per_rank = ceil_div(g.num_kb, c);
  g.tmem_cols = g.bn <= 32 ? 32 : g.bn <= 64 ? 64 : g.bn <= 128 ? 128 : 256;
  const int stage = kBoxBytes + g.bn * BK, recv = ceil_div(g.bn / 4, c) * (c - 1) * BM * 16;
  // two CTAs on an SM, where there are more than SMs: one streams while the other ends, the next kernel's included
  const int budget = (long long)c * z * ceil_div(N, BM) <= (c == 8 ? 96 : oi_sm_count()) || g.bn > 128 ? kSmemOfOne : kSmemOfTwo;
  // deposits beside the ring, or over it when it is drained (a cluster's barrier more) where a ring beside them would have fewer than five
  // stages and a CTA has more (us, beside and over: 100 x 18984 x 17386, two stages and three, 97.1 and 81.0; 65 x 19024 x 20234, three and
  // four, 92.5 and 86.3; 264 x 4096 x 12288, five and six, 18.6 and 18.6; 128 x 4096 x 8192, seven and eight, 12.0 and 12.8)
  const bool own_room = recv <= budget - 256 - g.bn * 4 - (g.kb_per_rank < 5 ? g.kb_per_rank : 5) * stage;
  g.stages = (budget - 256 - g.bn * 4 - (own_room ? recv : 0)) / stage;
  if (g.stages > kMostStages) g.stages = kMostStages;
  g.recv_offset = own_room ? g.stages * stage : 0;
  g.scale_offset = own_room ? g.recv_offset + recv : (g.stages * stage > recv ? g.stages * stage : recv);
  g.bar_offset = g.scale_offset + g.bn * 4;
  smem = g.bar_offset + 8 * (2 * g.stages + 1) + 16;
  return g;
}

template <typename TOut>
int launch_rows(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
                int c, int bn, cudaStream_t s) {
  int smem = 0;
  const Shape g = few_rows_shape(M, N, K, c, bn, smem);
  const int z = ceil_div(M, bn);
  OI_REQUIRE(ceil_div(N, BM) <= 65535, "linear_int8: %d channels are too many for %d rows", N, M);
  CUtensorMap mw, mx;
  int rc = tc::make_map_2d_i8(&mw, w, N, K, ldw, BM);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for the weight failed (%d; -1: cuTensorMapEncodeTiled is not available)", rc);
  rc = tc::make_map_2d_i8(&mx, x, M, K, ldx, g.bn);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for x failed (%d)", rc);
  auto go = [&](auto kernel, int threads, bool (&allowed)[64]) {
    if (int bad = tc::allow_smem(kernel, 227 * 1024, allowed)) return bad;
    oi_launch_cluster(kernel, dim3(c, z, ceil_div(N, BM)), threads, smem, s, c, mw, mx, out, ldo, scales, g);
    return (int)OI_OK;
  };
  static bool few[64], more[64], most[64];
  rc = g.bn <= kFewColumns ? go(linear_int8_rows_kernel<TOut, 4>, 192, few)
       : g.bn <= kMoreColumns ? go(linear_int8_rows_kernel<TOut, 8>, 320, more) : go(linear_int8_rows_kernel<TOut, 16>, 576, most);
  if (rc) return rc;
  OI_CHECK_LAUNCH();
  return OI_OK;
}

int pair_stages(int bn) {
  const int fit = kPairRingBytes / (kBoxBytes + bn / 2 * BK);
  return fit < kPairMostStages ? fit : kPairMostStages;
}

template <typename TOut>
int launch_pair(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
                int bn, cudaStream_t s) {
  CUtensorMap mw, mx;
  int rc = tc::make_map_2d_i8(&mw, w, N, K, ldw, BM);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for the weight failed (%d; -1: cuTensorMapEncodeTiled is not available)", rc);
  rc = tc::make_map_2d_i8(&mx, x, M, K, ldx, bn / 2);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for x failed (%d)", rc);
  const bool tma_out = rows_on_borders(out, ldo, N);
  CUtensorMap mo = mx;
  if (tma_out && (rc = tc::make_map_2d_out(&mo, out, sizeof(TOut) == 4, M, N, ldo, 32, kBufferBytes / 32 / (int)sizeof(TOut))))
    OI_REQUIRE(false, "linear_int8: tensor map for the result failed (%d)", rc);
  auto kernel = linear_int8_pair_kernel<TOut>;
  static bool allowed[64];
  if ((rc = tc::allow_smem(kernel, kPairSmem, allowed))) return rc;
  const long long tiles = (long long)ceil_div(M, bn) * ceil_div(N, 256);
  OI_REQUIRE(tiles < (1LL << 30), "linear_int8: %d rows of %d results are too many", M, N);
  const int most = oi_sm_count() / 2, pairs = tiles < most ? (int)tiles : most;
  const int stages = pair_stages(bn);
  oi_launch_cluster(kernel, 2 * pairs, kPairThreads, kPairSmem, s, 2, mw, mx, mo, out, ldo, scales, M, N, ceil_div(K, BK), bn, stages, (int)tma_out,
                    g_runs_out.load());
  OI_CHECK_LAUNCH();
  return OI_OK;
}

// The longest row of w beside M rows of x, which lie in registers; 0: too many rows
int few_longest(int M) { return M <= 8 ? 12288 : M <= 16 ? 8192 : 0; }

// Stages of all the rows of w of a CTA, and of its ring
long long few_wanted(int N, int K) {
  const int groups = ceil_div(N, 16);
  return (long long)ceil_div(groups, groups < oi_sm_count() ? groups : oi_sm_count()) * ceil_div(K, kChunk);
}
int few_stages(int N, int K) {
  const long long wanted = few_wanted(N, K);
  return wanted < kFewMostStages ? (int)wanted : kFewMostStages;
}

template <typename TOut>
int launch_few(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
               cudaStream_t s) {
  FewArgs f = {(const signed char*)x, (const signed char*)w, out, ldx, ldw, ldo, scales, M, N, K, ceil_div(N, 16), 0, 0, g_runs_out};
  const int chunks = ceil_div(K, kChunk), grid = f.groups < oi_sm_count() ? f.groups : oi_sm_count();
  f.stages = few_stages(N, K);
  f.at_once = few_wanted(N, K) <= kFewMostStages;
  const int smem = kFewPart + f.stages * (kFewStage + 16) + 16;
  auto go = [&](auto kernel, bool (&allowed)[64]) {
    if (int bad = tc::allow_smem(kernel, kFewPart + kFewMostStages * (kFewStage + 16) + 16, allowed)) return bad;
    oi_launch(kernel, grid, kFewThreads, smem, s, f);
    return (int)OI_OK;
  };
  static bool allowed[8][64];
  int rc;
  if (M <= 8)
    rc = chunks <= 1 ? go(linear_int8_few_kernel<1, 2, TOut>, allowed[0]) : chunks <= 2 ? go(linear_int8_few_kernel<1, 4, TOut>, allowed[1])
         : chunks <= 4 ? go(linear_int8_few_kernel<1, 8, TOut>, allowed[2]) : go(linear_int8_few_kernel<1, 12, TOut>, allowed[3]);
  else
    rc = chunks <= 1 ? go(linear_int8_few_kernel<2, 2, TOut>, allowed[4]) : chunks <= 2 ? go(linear_int8_few_kernel<2, 4, TOut>, allowed[5])
         : go(linear_int8_few_kernel<2, 8, TOut>, allowed[6]);
  if (rc) return rc;
  OI_CHECK_LAUNCH();
  return OI_OK;
}

// What a product takes in us, from what was measured (B200; N 32 to 152,000, K 128 to 16,000, 1 to 8,192 rows), to choose a kernel, its
// tiles of x and the slices of K. Over 170 sizes, most of them drawn, the choice took at most 1.16 times the fastest choice's time, in the
// median 1.00.
// Few rows: a stage of 128 bytes of K is 16 KB of w and `cols` rows of x at what one SM takes in, for as many CTAs as an SM has to
// run; the weight's bytes come from memory and all copies through L2 (21 TB/s, less beside memory's). Every round of CTAs costs 2.2 around
// its first copy and its results, 0.004 to 0.009 a column of the accumulator, or added up over a cluster 1.4 and 0.025 to 0.034 a column
// sent. Clusters of four and eight do not fill the SMs (35 of four: two rounds).
// Many rows: 4.5, and for each round of tiles its stages (16 KB of w and half the tile's rows of x for each CTA) or, where sums are
// short, its results, which take longer where result rows do not start and end on 16-byte borders.
float few_rows_us(int M, int N, int num_kb, int c, int z, int sms) {
  const int cols = ceil_div(M, z), bn = ceil_div(cols, 16) * 16, kb = ceil_div(num_kb, c), at_once = c == 8 ? sms * 2 / 3 : c == 4 ? sms - 20 : sms;
  const long long ctas = (long long)ceil_div(N, BM) * z * c;
  const int on_an_sm = ctas <= at_once || bn > 128 ? 1 : 2;
  const float rounds = (float)((ctas + at_once * on_an_sm - 1) / (at_once * on_an_sm));
  const float products = (float)((ctas + at_once - 1) / at_once) * kb * (0.171f + 0.00064f * cols);
  const float memory = (float)N * num_kb * BK / 6.4e6f, l2 = (float)ctas * kb * BK * (BM + cols) / 20.8e6f + 0.6f * memory;
  const float sent = cols * (c - 1.f) / c, added = 0.38f + (sent < 32.f ? 0.025f * sent : 0.8f + 0.034f * (sent - 32.f));
  const float results = c > 1 ? added : (bn > 128 ? 0.0086f : 0.004f) * bn;
  const float around = (c > 1 ? 3.26f : 2.23f) + results * on_an_sm, copies = memory > l2 ? memory : l2, work = products + (rounds - 1.f) * around;
  return around + (work > copies ? work : copies);
}
// Up to 16 rows on mma.sync: 16 rows of w after another, a stage of 2,048 bytes of each at the copy rate or the barrier behind them; x
// into registers.
float few_us(int M, int N, int K, int sms) {
  const int groups = ceil_div(ceil_div(N, 16), sms), chunks = ceil_div(K, kChunk);
  const float bytes = (float)K / (chunks * kChunk);
  const float stage = M <= 8 ? (0.72f * bytes > 0.58f / chunks ? 0.72f * bytes : 0.58f / chunks) : (0.9f * bytes > 0.7f / chunks ? 0.9f * bytes : 0.7f / chunks);
  return (M <= 8 ? 1.4f : 1.6f + 0.0002f * K) + groups * chunks * stage;
}
float many_rows_us(int M, int N, int num_kb, int bn, bool f32, bool on_borders, int sms) {
  const long long tiles = (long long)ceil_div(M, bn) * ceil_div(N, 256);
  const float products = (0.14f + 0.00074f * bn) * num_kb;
  const float results = (on_borders ? (f32 ? 1.0f + 0.0105f * bn : 1.4f + 0.0066f * bn) : (f32 ? 1.5f + 0.0165f * bn : 2.5f + 0.019f * bn)) + 0.4f * products;
  const float rounds = (float)((tiles + sms / 2 - 1) / (sms / 2)), work = rounds * (products > results ? products : results);
  const float memory = (float)N * num_kb * BK / 6.4e6f;
  return 4.5f + (work > memory ? work : memory + 0.05f * work);      // (of equal ones that with the least to do)
}

enum { kFew, kRows, kPairs };
struct Choice {
  int kernel, bn, c;          // bn: rows of x a tile; c: slices of K
};

Choice choose(int M, int N, int K, bool f32, bool on_borders) {
  const int num_kb = ceil_div(K, BK), sms = oi_sm_count(), least = ceil_div(M, 256);
  Choice best = {kPairs, 256, 1};
  float best_us = 3.4e38f;
  for (int bn = 32; bn <= 256; bn += 32) {
    const float us = many_rows_us(M, N, num_kb, bn, f32, on_borders, sms);
    if (us <= best_us) best_us = us, best.bn = bn;
  }
  if (least <= 16 && ceil_div(N, BM) <= 65535) {
    for (int z = least; z <= 4 * least + 4 && z <= ceil_div(M, 16); ++z)
      for (int c = 1; c <= 8 && (c == 1 || (c - 1) * ceil_div(num_kb, c) < num_kb); c *= 2) {     // no slice without a stage
        const float us = few_rows_us(M, N, num_kb, c, z, sms);
        if (us < best_us) best_us = us, best = {kRows, few_rows_height(M, z), c};
      }
  }
  if (M <= 16 && K <= few_longest(M) && few_us(M, N, K, sms) < best_us) best = {kFew, 16, 1};
  return best;
}

template <typename TOut>
int launch(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
           cudaStream_t s) {
  const Choice by = choose(M, N, K, sizeof(TOut) == 4, rows_on_borders(out, ldo, N));
  if (by.kernel == kFew) return launch_few(out, ldo, x, ldx, w, ldw, scales, M, N, K, s);
  if (by.kernel == kRows) return launch_rows(out, ldo, x, ldx, w, ldw, scales, M, N, K, by.c, by.bn, s);
  return launch_pair(out, ldo, x, ldx, w, ldw, scales, M, N, K, by.bn, s);
}

}  // namespace

// x [M, K], w [N, K]: 8-bit integers, row strides in bytes; rows start on 16-byte borders. sx [M], sw [N], bias [N] or null: float32.
// w is read before the kernels ahead on the stream have finished: the library's kernels must not have written it since the last
// launch in plain stream order (oi_launch_fence).
OI_API int oi_linear_int8(void* out, int out_dtype, long long ldo, const void* x, long long ldx, const float* sx, const void* w,
                          long long ldw, const float* sw, const float* bias, int M, int N, int K, void* stream) {
  constexpr int kMost = (1 << 30);
  OI_REQUIRE(M >= 0 && M <= kMost && N >= 0 && N <= kMost && K >= 1 && K <= 131071, "linear_int8: bad sizes M=%d N=%d K=%d (K: 1 to 131071)", M, N, K);
  OI_REQUIRE(out_dtype == OI_F32 || out_dtype == OI_BF16, "linear_int8: unknown output dtype code %d", out_dtype);
  if (M == 0 || N == 0) return OI_OK;
  OI_REQUIRE(ldx % 16 == 0 && ldw % 16 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && ldx >= K && ldw >= K,
             "linear_int8: rows of x and w must start on 16-byte borders");
  OI_REQUIRE(M == 1 || ldo >= N, "linear_int8: result rows of %d that start %lld apart", N, ldo);
  if (M == 1) ldo = ceil_div(N, 16) * 16LL;      // one row's stride means nothing
  const Scales scales = {sx, sw, bias};
  cudaStream_t s = (cudaStream_t)stream;
  if (out_dtype == OI_F32) return launch((float*)out, ldo, x, ldx, w, ldw, scales, M, N, K, s);
  return launch((bf16*)out, ldo, x, ldx, w, ldw, scales, M, N, K, s);
}

// 0 when no bounded wait has run out since the last call; otherwise which role gave up (few rows: 1 copies, 2 products, 3
// results; many rows: 11 to 13 the same, 14 products waiting for drained results; up to 16 rows: 21, 22) or that a row kernel's copies did
// not come (31). Synchronises the device; clears the words.
OI_API int oi_linear_int8_status(int* status) {
  int v = 0;
  OI_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_int8_error, sizeof(int)));
  if (v != 0) {
    int zero = 0;
    OI_CHECK_CUDA(cudaMemcpyToSymbol(g_int8_error, &zero, sizeof(int)));
  }
  if (int rc = oi_take_rows_int8_error(status)) return rc;
  if (v != 0) *status = v;
  return OI_OK;
}

// For tests: products launched from now on take the wait of this code as having run out (0: none).
OI_API int oi_linear_int8_run_out(int code) {
  g_runs_out = code;
  return OI_OK;
}

// For tests: which kernel takes a product of these sizes (0: up to 16 rows, 1: few, 2: many), rows of x a tile, slices of K, tiles,
// stages, and of few rows whether partial sums go over the ring. on_borders: result rows start and end on 16-byte borders.
OI_API int oi_linear_int8_choice(int out_dtype, int on_borders, int M, int N, int K, int* choice) {
  OI_REQUIRE(M >= 1 && N >= 1 && K >= 1 && K <= 131071, "linear_int8_choice: bad sizes M=%d N=%d K=%d", M, N, K);
  const Choice by = choose(M, N, K, out_dtype == OI_F32, on_borders != 0);
  int smem = 0;
  const Shape g = by.kernel == kRows ? few_rows_shape(M, N, K, by.c, by.bn, smem) : Shape{};
  choice[0] = by.kernel, choice[1] = by.bn, choice[2] = by.c;
  const long long tiles = (long long)ceil_div(M, by.bn) * ceil_div(N, by.kernel == kFew ? 16 : by.kernel == kRows ? BM : 256);
  choice[3] = tiles < INT_MAX ? (int)tiles : INT_MAX;
  choice[4] = by.kernel == kRows ? g.stages : by.kernel == kPairs ? pair_stages(by.bn) : few_stages(N, K);
  choice[5] = by.kernel == kRows && by.c > 1 && g.recv_offset == 0;
  return OI_OK;
}
