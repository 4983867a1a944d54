// out[m, n] = (sum_k x[m, k] * w[n, k]) * sx[m] * sw[n] + bias[n] for 8-bit integers on the 5th-generation tensor cores
// (tcgen05.mma kind::i8). The sums are exact in 32-bit integers (K up to 131,071: 128 * 128 * K < 2^31), so no order of
// addition, tile or slice of K matters to a result; then float(sum) * sx * sw + bias in float32, in that order, and one
// rounding to the output's type.
//
// Two kernels. Operands are staged by TMA as rows of 128 bytes (128-byte swizzle); bytes beyond K or beyond the last row are
// zeros of the copy. Every wait on an mbarrier is bounded: one that runs out sets an error word and a flag that ends all roles
// of the CTA, which still joins its cluster's barriers, frees its tensor memory and returns. No load uses cluster multicast.
#include "oi_api.h"
#include "tcgen05.cuh"

namespace {

constexpr int BM = 128;                     // rows of an operand's box
constexpr int BK = 128;                     // bytes of K a stage
constexpr int kBoxBytes = BM * BK;

__device__ int g_int8_error = 0;            // set to a non-zero code when a bounded wait ran out

__device__ __forceinline__ bool wait_on(unsigned bar, unsigned parity, volatile int* abort_flag, int code) {
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
// w x bn] lies in tensor memory. Grid (c, tiles of x, tiles of w; those that share a tile of w run together): a cluster of c CTAs (a power of two) shares one tile, CTA r
// streaming k blocks [r * kb_per_rank, ...) of it, and adds up: row i of the accumulator (a row of w) belongs to CTA i / (128 / c),
// into whose shared memory every CTA deposits its partial sums of it.
//   warp 0     one thread issues the copies; the first ring-full of WEIGHT boxes is requested before the wait for the kernel
//              ahead (programmatic dependent launch), which may still be writing x
//   warp 1     allocates tensor memory (behind that wait: a kernel ahead that needs all of it may not have taken its own
//              yet), one thread issues four products (K = 32) a stage
//   the others (four to sixteen) read the accumulator (one row of w a thread) and deposit, or with c = 1 scale and store; then
//              all warps add up, scale and store.
// What the results cost shows in the instructions per column: with a column at a time, a branch and a cluster address each, and
// six warps, 128 columns took 8,000 cycles to deposit and 8,700 to store (N 1024, K 1024, c 1).
constexpr int kFewColumns = 32, kMoreColumns = 64;      // up to so many rows of x a tile four warps read results, or eight, else sixteen

struct Shape {
  int M, N, num_kb, kb_per_rank, bn, stages, tmem_cols;
  int recv_offset;          // where deposits go: behind the ring, or over the drained ring (0)
  int scale_offset;         // scales of the tile's rows of x [bn]
  int bar_offset;
};

template <typename TOut, int kReaders>
__global__ void __launch_bounds__(64 + 32 * kReaders)
linear_int8_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, TOut* out, long long ldo,
                        const Scales scales, const Shape g) {
  pdl_trigger();
  constexpr int kThreads = 64 + 32 * kReaders;
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
  // what the sums are multiplied by is fetched under the copies: a channel's scale in its thread, later every row's in shared memory
  const int cols = min(g.bn, g.M - m0);  // rows of x in this tile
  const int quarter = warp & 3;          // a warp may only touch lanes [32 * (warp % 4), +32) of tensor memory
  const int rows_mine = BM / csize;      // channels that this CTA adds up
  const int n = n0 + (csize > 1 ? rank * rows_mine + (int)threadIdx.x % rows_mine : quarter * 32 + lane);
  const float sw = n < g.N ? scales.sw[n] : 0.f;
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

  bool ok = true;
  if (warp == 0) {
    const bool leader = tc::elect_one();
    Ring at;
    for (int kb = g.stages; kb < nkb; ++kb, at.next(g.stages)) {
      const int s = at.stage;
      if (!wait_on(empty_bar(s), at.parity, abort_flag, 1)) break;
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
      ok = wait_on(full_bar(s), at.parity, abort_flag, 2);
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
    ok = wait_on(acc_full, 0, abort_flag, 3);
    tc::fence_after();
  }
  if (csize > 1) {
    __syncwarp();
    tc::cluster_wait();                  // phase 0
    if (g.recv_offset == 0) {            // deposits go over the ring: every CTA's products have read theirs first
      __syncthreads();                   // (warps 0 and 1 come here before the products are done, the others after)
      tc::cluster_arrive();
      tc::cluster_wait();
    }
  }
  const int ld = g.bn + 4;               // words of a row of deposits: eight lanes' 16 bytes then lie in different banks
  if (warp >= 2) {
    const unsigned tmem_row = tmem_base + ((unsigned)(quarter * 32) << 16);
    const int row = quarter * 32 + lane;
    unsigned dst = 0;
    if (csize > 1)
      dst = tc::map_to_rank(smem_base + g.recv_offset, row / rows_mine) + (unsigned)((rank * rows_mine + row % rows_mine) * ld) * 4;
#pragma unroll 1
    for (int c0 = 16 * ((warp - 2) >> 2); c0 < cols; c0 += 4 * kReaders) {
      unsigned v[16];
      if (nkb > 0 && ok) {
        tc::tmem_ld16(tmem_row + (unsigned)c0, v);
        tc::tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0u;
      }
      if (csize > 1) {
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (c0 + e < cols) asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};\n"
                       ::"r"(dst + (unsigned)(c0 + e) * 4), "r"(v[e]), "r"(v[e + 1]), "r"(v[e + 2]), "r"(v[e + 3]) : "memory");
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
  tc::fence_before();
  if (csize > 1) {
    __syncwarp();
    tc::cluster_arrive();                // this CTA's deposits are made ...
    tc::cluster_wait();                  // ... and so are everybody's; nothing remote is touched after this
    // a channel and four rows of x a thread (rows_mine divides the threads: its channel stays)
    const int local = (int)threadIdx.x % rows_mine, step = kThreads / rows_mine;
    const unsigned char* mine = smem + g.recv_offset + (size_t)local * ld * 4;
    if (n < g.N) {
#pragma unroll 2
      for (int c = (int)threadIdx.x / rows_mine * 4; c < cols; c += step * 4) {
        int4 sum = make_int4(0, 0, 0, 0);
        for (int q = 0; q < csize; ++q) {
          const int4 part = *reinterpret_cast<const int4*>(mine + ((size_t)q * rows_mine * ld + c) * 4);
          sum.x += part.x, sum.y += part.y, sum.z += part.z, sum.w += part.w;
        }
        const float4 sx = *reinterpret_cast<const float4*>(sx_s + c);
        TOut* at = out + (size_t)(m0 + c) * ldo + n;
        *at = from_f32<TOut>(finish(sum.x, sx.x, sw, b, biased));
        if (c + 1 < cols) at[ldo] = from_f32<TOut>(finish(sum.y, sx.y, sw, b, biased));
        if (c + 2 < cols) at[2 * ldo] = from_f32<TOut>(finish(sum.z, sx.z, sw, b, biased));
        if (c + 3 < cols) at[3 * ldo] = from_f32<TOut>(finish(sum.w, sx.w, sw, b, biased));
      }
    }
  }
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
// Many rows. Pairs of CTAs (a cluster of two, cta_group::2) compute 256 x 256 tiles, persistent: pair p works on tiles p, p +
// pairs, ... (row tiles fastest, so that pairs that run at the same time share tiles of w through L2). The CTA of rank r holds
// rows [128 r, +128) of the tile's rows of x and of w in its shared memory, and the accumulator of its 128 rows x 256 columns
// in its tensor memory, double buffered (512 columns): while the epilogue warps drain one tile the next is formed.
//   warp 0     of both CTAs loads its own halves, counted on the even CTA's "full" barrier
//   warp 1     of the even CTA issues the products (M = 256, N = 256, K = 32) for both
//   warps 2-17 of both CTAs drain their own tensor memory and arrive on the even CTA's "drained" barrier
constexpr int kEpilogueWarps = 16;
constexpr int kParts = kEpilogueWarps / 4;                          // the warps of a quarter of the lanes share its columns
constexpr int kPartCols = 256 / kParts;
constexpr int kPairThreads = 64 + 32 * kEpilogueWarps;
constexpr int kPairStages = 5;
constexpr int kPairStageBytes = 2 * kBoxBytes;
constexpr int kBufferBytes = 32 * 64;                               // a warp's results on their way out: 32 rows of 64 bytes
constexpr int kPairBufferOffset = kPairStages * kPairStageBytes;
constexpr int kPairScaleOffset = kPairBufferOffset + kEpilogueWarps * kBufferBytes;      // per warp its channels' scales, then biases
constexpr int kPairBarOffset = kPairScaleOffset + kEpilogueWarps * 2 * kPartCols * 4;  // full, empty, acc_full[2], acc_empty[2], tmem slot, abort
constexpr int kPairSmem = kPairBarOffset + (2 * kPairStages + 4) * 8 + 16 + 1024;
static_assert(kPairSmem <= 227 * 1024, "more shared memory than a CTA may have");

template <typename TOut>
__global__ void __launch_bounds__(kPairThreads)
linear_int8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                        const __grid_constant__ CUtensorMap map_out, TOut* out, long long ldo, const Scales scales, int M, int N, int num_kb,
                        int tma_out) {
  pdl_start();
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const unsigned smem_base = tc::smem_u32(smem);
  const unsigned bar_base = smem_base + kPairBarOffset;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kPairStages + s); };
  auto acc_full_bar = [&](int a) { return bar_base + 8u * (2 * kPairStages + a); };
  auto acc_empty_bar = [&](int a) { return bar_base + 8u * (2 * kPairStages + 2 + a); };
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(smem + kPairBarOffset + (2 * kPairStages + 4) * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = tc::cluster_ctarank();
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int m_tiles = (M + 255) / 256, num_tiles = m_tiles * ((N + 255) / 256);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
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
    int ahead = kPairStages;                         // stages that have not been used yet
    bool ok = true;
    for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
      const int m0 = (tile % m_tiles) * 256 + (int)rank * 128, n0 = (tile / m_tiles) * 256 + (int)rank * 128;
      for (int kb = 0; kb < num_kb; ++kb, at.next(kPairStages)) {
        const int s = at.stage;
        if (ahead > 0) --ahead;
        else if (!wait_on(empty_bar(s), at.parity ^ 1, abort_flag, 11)) { ok = false; break; }
        if (leader) {
          if (rank == 0) tc::mbar_expect_tx(full_bar(s), 2 * kPairStageBytes);
          const unsigned counted_on = tc::map_to_rank(full_bar(s), 0);
          const unsigned dst = smem_base + s * kPairStageBytes;
          tc::tma_load_2d_pair(dst, &map_x, kb * BK, m0, counted_on);
          tc::tma_load_2d_pair(dst + kBoxBytes, &map_w, kb * BK, n0, counted_on);
        }
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leader = tc::elect_one();
      constexpr unsigned idesc = tc::idesc_i8_s32(256, 256);
      Ring at;
      int local = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs, ++local) {
        const int a = local & 1;
        if (local >= 2) {
          ok = tc::mbar_wait_cluster(acc_empty_bar(a), (unsigned)((local >> 1) - 1) & 1, abort_flag, &g_int8_error, 14);
          if (!ok) break;
          tc::fence_after();
        }
        const unsigned tmem_acc = tmem_base + (unsigned)(a * 256);
        for (int kb = 0; kb < num_kb; ++kb, at.next(kPairStages)) {
          const int s = at.stage;
          ok = wait_on(full_bar(s), at.parity, abort_flag, 12);
          if (!ok) break;
          tc::fence_after();
          const unsigned a_addr = smem_base + s * kPairStageBytes;
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
    const int quarter = warp & 3;            // a warp may only touch lanes [32 * (warp % 4), +32)
    const int part = (warp - 2) >> 2;
    constexpr int kCols = 64 / (int)sizeof(TOut);             // columns of a row of the buffer
    unsigned char* buffer = smem + kPairBufferOffset + (warp - 2) * kBufferBytes;
    float* sw_s = reinterpret_cast<float*>(smem + kPairScaleOffset) + (warp - 2) * 2 * kPartCols;
    float* b_s = sw_s + kPartCols;
    const bool biased = scales.bias != nullptr;
    int local = 0;
    // the next tile's scales are asked for a tile ahead: where sums are short the results, not the products, take the time
    float next_sx, next_sw[kPartCols / 32], next_b[kPartCols / 32];
    auto ask = [&](int tile) {
      const int m = (tile % m_tiles) * 256 + (int)rank * 128 + quarter * 32 + lane, n0 = (tile / m_tiles) * 256 + part * kPartCols + lane;
      next_sx = tile < num_tiles && m < M ? scales.sx[m] : 0.f;
#pragma unroll
      for (int i = 0; i < kPartCols / 32; ++i) {
        const bool there = tile < num_tiles && n0 + 32 * i < N;
        next_sw[i] = there ? scales.sw[n0 + 32 * i] : 0.f;
        next_b[i] = there && biased ? scales.bias[n0 + 32 * i] : 0.f;
      }
    };
    ask(pair);
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++local) {
      const int a = local & 1;
      const int m0 = (tile % m_tiles) * 256 + (int)rank * 128 + quarter * 32, n0 = (tile / m_tiles) * 256 + part * kPartCols;
      const float sx = next_sx;
#pragma unroll
      for (int i = 0; i < kPartCols / 32; ++i) {
        sw_s[32 * i + lane] = next_sw[i];
        b_s[32 * i + lane] = next_b[i];
      }
      __syncwarp();
      ask(tile + num_pairs);
      if (!wait_on(acc_full_bar(a), (unsigned)(local >> 1) & 1, abort_flag, 13)) break;
      tc::fence_after();
      const unsigned tmem_acc = tmem_base + (unsigned)(a * 256 + part * kPartCols) + ((unsigned)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < kPartCols; c += kCols) {
        unsigned v[kCols];
        if constexpr (kCols == 32) tc::tmem_ld32(tmem_acc + (unsigned)c, v);
        else tc::tmem_ld16(tmem_acc + (unsigned)c, v);
        tc::tmem_ld_wait();
        if (c + kCols == kPartCols) {                // all of this warp's part is read: the products may fill it again
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive_cluster(tc::map_to_rank(acc_empty_bar(a), 0));
        }
        if (n0 + c >= N || m0 >= M) continue;        // the same for the whole warp
        float y[kCols];
#pragma unroll
        for (int e = 0; e < kCols; e += 4) {
          const float4 sw = *reinterpret_cast<const float4*>(sw_s + c + e);
          y[e] = __fmul_rn(__fmul_rn((float)(int)v[e], sx), sw.x), y[e + 1] = __fmul_rn(__fmul_rn((float)(int)v[e + 1], sx), sw.y);
          y[e + 2] = __fmul_rn(__fmul_rn((float)(int)v[e + 2], sx), sw.z), y[e + 3] = __fmul_rn(__fmul_rn((float)(int)v[e + 3], sx), sw.w);
        }
        if (biased) {
#pragma unroll
          for (int e = 0; e < kCols; e += 4) {
            const float4 b = *reinterpret_cast<const float4*>(b_s + c + e);
            y[e] = __fadd_rn(y[e], b.x), y[e + 1] = __fadd_rn(y[e + 1], b.y), y[e + 2] = __fadd_rn(y[e + 2], b.z), y[e + 3] = __fadd_rn(y[e + 3], b.w);
          }
        }
        if (lane == 0) tc::bulk_wait<0>();           // the buffer's last contents are on their way
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {                // 16 bytes at a time, their place turned by the row (the copy's swizzle)
          uint4 o;
          if constexpr (sizeof(TOut) == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<__nv_bfloat162*>(&o)[e] = __floats2bfloat162_rn(y[8 * j + 2 * e], y[8 * j + 2 * e + 1]);
          } else {
            o = make_uint4(__float_as_uint(y[4 * j]), __float_as_uint(y[4 * j + 1]), __float_as_uint(y[4 * j + 2]), __float_as_uint(y[4 * j + 3]));
          }
          *reinterpret_cast<uint4*>(buffer + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = o;
        }
        if (tma_out) {
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tc::tma_store_2d(&map_out, tc::smem_u32(buffer), n0 + c, m0);
            tc::bulk_commit();
          }
        } else {
          // Rows that do not start on 16-byte borders: two rows at a time, four bytes a lane. A row of bfloat16 may start between two
          // four-byte borders: its pairs are then put together from neighbours' words, its first and last number stored alone.
          __syncwarp();
          const int half = lane >> 4, word = lane & 15, left = min(kCols, N - (n0 + c));
          const unsigned char* from = buffer + half * 64 + (word & 3) * 4;
          TOut* dst = out + (size_t)(m0 + half) * ldo + n0 + c;
#pragma unroll 4
          for (int i = 0; i < 16; ++i, dst += 2 * ldo) {
            const unsigned own = *reinterpret_cast<const unsigned*>(from + i * 128 + (((word >> 2) ^ (i & 3)) << 4));
            const bool live = m0 + 2 * i + half < M;
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

// ------------------------------------------------------------------------------------------------ host side
// The shared memory that a kernel may ask for, allowed once for each device that it runs on.
template <typename Kernel>
int allow_smem(Kernel kernel, int bytes, bool (&done)[64]) {
  int dev = 0;
  OI_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !done[dev]) {
    OI_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return OI_OK;
}

constexpr int kMostStages = 12, kSmemOfTwo = 110 * 1024, kSmemOfOne = 208 * 1024;

// result rows that start on 16-byte borders can be copied out by TMA
template <typename TOut>
bool rows_on_borders(const TOut* out, long long ldo) { return (uintptr_t)out % 16 == 0 && ldo * sizeof(TOut) % 16 == 0; }

template <typename TOut>
int launch_rows(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
                int c, int z, cudaStream_t s) {
  Shape g = {};
  g.M = M, g.N = N;
  g.bn = ceil_div(ceil_div(M, z), 16) * 16;                            // z tiles of x, of equal size
  g.num_kb = ceil_div(K, BK);
  g.kb_per_rank = ceil_div(g.num_kb, c);
  g.tmem_cols = g.bn <= 32 ? 32 : g.bn <= 64 ? 64 : g.bn <= 128 ? 128 : 256;
  const int stage = kBoxBytes + g.bn * BK, recv = c > 1 ? BM * (g.bn + 4) * 4 : 0;
  // two CTAs on an SM, where there are more than SMs: one streams while the other ends, the next kernel's included
  const int budget = (long long)c * z * ceil_div(N, BM) <= (c == 8 ? 96 : oi_sm_count()) || g.bn > 128 ? kSmemOfOne : kSmemOfTwo;
  // deposits beside the ring, or over it when it is drained (a cluster's barrier more) where a ring beside them would be short (264 rows, N
  // 4096, K 12288, c 2: three stages beside them 23.4 us, six under them 19.7)
  const bool own_room = recv <= budget - 256 - g.bn * 4 - (g.kb_per_rank < 5 ? g.kb_per_rank : 5) * stage;
  g.stages = (budget - 256 - g.bn * 4 - (own_room ? recv : 0)) / stage;
  if (g.stages > kMostStages) g.stages = kMostStages;
  g.recv_offset = own_room ? g.stages * stage : 0;
  g.scale_offset = own_room ? g.recv_offset + recv : (g.stages * stage > recv ? g.stages * stage : recv);
  g.bar_offset = g.scale_offset + g.bn * 4;
  const int smem = g.bar_offset + 8 * (2 * g.stages + 1) + 16;
  OI_REQUIRE(ceil_div(N, BM) <= 65535, "linear_int8: %d channels are too many for %d rows", N, M);
  CUtensorMap mw, mx;
  int rc = tc::make_map_2d_i8(&mw, w, N, K, ldw, BM);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for the weight failed (%d; -1: cuTensorMapEncodeTiled is not available)", rc);
  rc = tc::make_map_2d_i8(&mx, x, M, K, ldx, g.bn);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for x failed (%d)", rc);
  auto go = [&](auto kernel, int threads, bool (&allowed)[64]) {
    if (int bad = allow_smem(kernel, 227 * 1024, allowed)) return bad;
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

template <typename TOut>
int launch_pair(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
                cudaStream_t s) {
  CUtensorMap mx, mw;
  int rc = tc::make_map_2d_i8(&mx, x, M, K, ldx, BM);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for x failed (%d; -1: cuTensorMapEncodeTiled is not available)", rc);
  rc = tc::make_map_2d_i8(&mw, w, N, K, ldw, BM);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for the weight failed (%d)", rc);
  const bool tma_out = rows_on_borders(out, ldo);
  CUtensorMap mo = mx;
  if (tma_out && (rc = tc::make_map_2d_out(&mo, out, sizeof(TOut) == 4, M, N, ldo, 32))) OI_REQUIRE(false, "linear_int8: tensor map for the result failed (%d)", rc);
  auto kernel = linear_int8_pair_kernel<TOut>;
  static bool allowed[64];
  if ((rc = allow_smem(kernel, kPairSmem, allowed))) return rc;
  const long long tiles = (long long)ceil_div(M, 256) * ceil_div(N, 256);
  OI_REQUIRE(tiles < (1LL << 30), "linear_int8: %d rows of %d results are too many", M, N);
  const int most = oi_sm_count() / 2, pairs = tiles < most ? (int)tiles : most;
  oi_launch_cluster(kernel, 2 * pairs, kPairThreads, kPairSmem, s, 2, mx, mw, mo, out, ldo, scales, M, N, ceil_div(K, BK), (int)tma_out);
  OI_CHECK_LAUNCH();
  return OI_OK;
}

// What a product takes in us, from what was measured (B200; N 128 to 32,000, K 128 to 16,000, 1 to 4,096 rows), to choose a kernel, the
// tiles of x and the slices of K.
// Few rows: a stage of 128 bytes of K is 16 KB of w and `cols` rows of x at what one SM takes in, for as many CTAs as an SM has to
// run; the weight's bytes come from memory; every round of CTAs costs 2.3 around its first copy and its results, 0.006 to 0.008 a column
// of the accumulator, or added up over a cluster 0.7 and 0.028 a column. Clusters of four and eight do not fill the SMs (35 of four: two
// rounds). Many rows: 4.5, and for each round of tiles 0.33 a stage, or what a tile's results take: 3.2, and 6.5 where result rows do
// not start on 16-byte borders.
float few_rows_us(int M, int N, int num_kb, int c, int z, int sms) {
  const int cols = ceil_div(M, z), bn = ceil_div(cols, 16) * 16, kb = ceil_div(num_kb, c), at_once = c == 8 ? sms * 2 / 3 : c == 4 ? sms - 20 : sms;
  const long long ctas = (long long)ceil_div(N, BM) * z * c;
  const int on_an_sm = ctas <= at_once || bn > 128 ? 1 : 2;
  const float rounds = (float)((ctas + at_once * on_an_sm - 1) / (at_once * on_an_sm));
  const float stream = (float)((ctas + at_once - 1) / at_once) * kb * (0.185f + 0.0005f * cols), memory = (float)N * num_kb * BK / 6.4e6f;
  const float results = c > 1 ? 0.7f + 0.028f * (cols < bn - 12 ? cols : bn) : (bn > 128 ? 0.008f : 0.006f) * bn;
  return rounds * (2.3f + results * on_an_sm) + (stream > memory ? stream : memory);
}
float many_rows_us(int M, int N, int num_kb, bool on_borders, int sms) {
  const long long tiles = (long long)ceil_div(M, 256) * ceil_div(N, 256);
  const float products = 0.33f * num_kb, results = on_borders ? 3.2f : 6.5f, a_round = products > results ? products : results;
  return 4.5f + (float)((tiles + sms / 2 - 1) / (sms / 2)) * a_round;
}

template <typename TOut>
int launch(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
           cudaStream_t s) {
  const int num_kb = ceil_div(K, BK), sms = oi_sm_count(), least = ceil_div(M, 256);
  int best_c = 0, best_z = 0;
  float best = many_rows_us(M, N, num_kb, rows_on_borders(out, ldo), sms);
  if (least <= 16 && ceil_div(N, BM) <= 65535) {
    for (int z = least; z <= 4 * least + 4 && z <= ceil_div(M, 16); ++z)
      for (int c = 1; c <= 8 && (c == 1 || (c - 1) * ceil_div(num_kb, c) < num_kb); c *= 2) {     // no slice without a stage
        const float us = few_rows_us(M, N, num_kb, c, z, sms);
        if (us < best) best = us, best_c = c, best_z = z;
      }
  }
  return best_c ? launch_rows(out, ldo, x, ldx, w, ldw, scales, M, N, K, best_c, best_z, s) : launch_pair(out, ldo, x, ldx, w, ldw, scales, M, N, K, s);
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
// results; many rows: 11 to 13 the same, 14 products waiting for drained results). Synchronises the device; clears the word.
OI_API int oi_linear_int8_status(int* status) {
  int v = 0;
  OI_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_int8_error, sizeof(int)));
  if (v != 0) {
    int zero = 0;
    OI_CHECK_CUDA(cudaMemcpyToSymbol(g_int8_error, &zero, sizeof(int)));
  }
  *status = v;
  return OI_OK;
}
