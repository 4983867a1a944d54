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
__device__ __forceinline__ float finish(int sum, float sx, float sw) { return __fmul_rn(__fmul_rn((float)sum, sx), sw); }

struct Scales {
  const float *sx, *sw, *bias;
};

// ------------------------------------------------------------------------------------------------
// Few rows. The product is formed transposed: 128 rows of w are the M side of tcgen05.mma, up to 256 rows of x (a multiple of
// 16, `bn`) its N side, so a weight byte goes HBM -> TMA -> shared memory -> tensor core, and the accumulator [128 rows of
// w x bn] lies in tensor memory. Grid (c, tiles of w, tiles of x): a cluster of c CTAs shares one tile, CTA r streaming k blocks
// [r * kb_per_rank, ...) of it, and adds up: column j of the accumulator (a row of x) belongs to CTA j / cols_per_owner, into
// whose shared memory every CTA deposits its partial sums of it.
//   warp 0     one thread issues the copies; the first ring-full of WEIGHT boxes is requested before the wait for the kernel
//              ahead (programmatic dependent launch), which may still be writing x
//   warp 1     allocates tensor memory (behind that wait: a kernel ahead that needs all of it may not have taken its own
//              yet), one thread issues four products (K = 32) a stage
//   warps 2-5  read the accumulator (one weight row a thread) and deposit; then all six warps add up, scale and store.
constexpr int kThreads = 192;

struct Shape {
  int M, N, num_kb, kb_per_rank, bn, stages, cols_per_owner, tmem_cols;
  int recv_offset;          // where deposits go: behind the ring, or over the drained ring (0)
  int bar_offset;
  int vec;                  // result rows may be stored four numbers at a time
};

template <typename TOut>
__device__ __forceinline__ void store4(TOut* dst, const float (&y)[4], int valid, int vec) {
  if (vec && valid >= 4) {
    if constexpr (sizeof(TOut) == 2) {
      uint2 o;
      reinterpret_cast<__nv_bfloat162*>(&o)[0] = __floats2bfloat162_rn(y[0], y[1]);
      reinterpret_cast<__nv_bfloat162*>(&o)[1] = __floats2bfloat162_rn(y[2], y[3]);
      *reinterpret_cast<uint2*>(dst) = o;
    } else {
      *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) dst[e] = from_f32<TOut>(y[e]);
  }
}

template <typename TOut>
__global__ void __launch_bounds__(kThreads)
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
  const int n0 = blockIdx.y * BM, m0 = blockIdx.z * g.bn;
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
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const unsigned tmem_base = *tmem_slot;
  if (csize > 1) tc::cluster_arrive();   // phase 0: "this CTA runs"; waited for before anyone writes into it

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      for (int kb = g.stages; kb < nkb; ++kb) {
        const int s = kb % g.stages;
        if (!wait_on(empty_bar(s), (unsigned)((kb / g.stages) - 1) & 1, abort_flag, 1)) break;
        tc::mbar_expect_tx(full_bar(s), stage_bytes);
        const unsigned dst = smem_base + s * stage_bytes;
        tc::tma_load_2d(dst, &map_w, (kb0 + kb) * BK, n0, full_bar(s));
        tc::tma_load_2d(dst + kBoxBytes, &map_x, (kb0 + kb) * BK, m0, full_bar(s));
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const unsigned idesc = tc::idesc_i8_s32(BM, g.bn);
      for (int kb = 0; kb < nkb; ++kb) {
        const int s = kb % g.stages;
        ok = wait_on(full_bar(s), (unsigned)(kb / g.stages) & 1, abort_flag, 2);
        if (!ok) break;
        tc::fence_after();
        const unsigned a_addr = smem_base + s * stage_bytes;
        const unsigned long long da = tc::desc_k_major_sw128(a_addr), db = tc::desc_k_major_sw128(a_addr + kBoxBytes);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)   // 32 bytes further along K inside the swizzle row: +2 in the address field
          tc::umma_i8(tmem_base, da + 2ull * k, db + 2ull * k, idesc, (kb | k) != 0 ? 1u : 0u);
        tc::umma_commit(empty_bar(s));
      }
      if (ok && nkb > 0) tc::umma_commit(acc_full);
    }
  } else if (nkb > 0) {
    ok = wait_on(acc_full, 0, abort_flag, 3);
    tc::fence_after();
  }
  if (csize > 1) {
    __syncwarp();
    tc::cluster_wait();                  // phase 0
    if (g.recv_offset == 0) {            // deposits go over the ring: every CTA's products have read theirs first
      __syncthreads();                   // (warps 0 and 1 come here before the products are done, warps 2-5 after)
      tc::cluster_arrive();
      tc::cluster_wait();
    }
  } else if (g.recv_offset == 0) {
    __syncthreads();
  }
  const int cols = min(g.bn, g.M - m0);  // rows of x in this tile
  const unsigned recv = smem_base + g.recv_offset;
  if (warp >= 2) {
    const int quarter = warp & 3;        // a warp may only touch lanes [32 * (warp % 4), +32)
    const unsigned tmem_row = tmem_base + ((unsigned)(quarter * 32) << 16);
    const unsigned mine = (unsigned)(rank * g.cols_per_owner) * (BM * 4) + (quarter * 32 + lane) * 4;
    int owner = 0, local = 0;
    unsigned dst = csize > 1 ? tc::map_to_rank(recv, 0) : recv;
#pragma unroll 1
    for (int c0 = 0; c0 < cols; c0 += 16) {
      unsigned v[16];
      if (nkb > 0 && ok) {
        tc::tmem_ld16(tmem_row + (unsigned)c0, v);
        tc::tmem_ld_wait();
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0u;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (c0 + e >= cols) break;
        asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(dst + mine + (unsigned)local * (BM * 4)), "r"(v[e]) : "memory");
        if (++local == g.cols_per_owner) {
          local = 0;
          ++owner;
          if (owner < csize) dst = tc::map_to_rank(recv, owner);
        }
      }
    }
  }
  tc::fence_before();
  if (csize > 1) {
    __syncwarp();
    tc::cluster_arrive();                // this CTA's deposits are made ...
    tc::cluster_wait();                  // ... and so are everybody's; nothing remote is touched after this
  } else {
    __syncthreads();
  }
  // a warp a column, four rows of w a lane
  const int n = n0 + 4 * lane, valid = g.N - n;
  if (valid > 0) {
    float sw[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sw[e] = e < valid ? scales.sw[n + e] : 0.f;
      b[e] = scales.bias && e < valid ? scales.bias[n + e] : 0.f;
    }
    const int first = rank * g.cols_per_owner, last = min(first + g.cols_per_owner, cols);
    for (int c = first + warp; c < last; c += kThreads / 32) {
      int4 sum = make_int4(0, 0, 0, 0);
      for (int q = 0; q < csize; ++q) {
        const int4 part = *reinterpret_cast<const int4*>(smem + g.recv_offset + (size_t)(q * g.cols_per_owner + c - first) * (BM * 4) + 16 * lane);
        sum.x += part.x, sum.y += part.y, sum.z += part.z, sum.w += part.w;
      }
      const float sx = scales.sx[m0 + c];
      float y[4] = {finish(sum.x, sx, sw[0]), finish(sum.y, sx, sw[1]), finish(sum.z, sx, sw[2]), finish(sum.w, sx, sw[3])};
      if (scales.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __fadd_rn(y[e], b[e]);
      }
      store4(out + (size_t)(m0 + c) * ldo + n, y, valid, g.vec);
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
//   warps 2-9  of both CTAs drain their own tensor memory and arrive on the even CTA's "drained" barrier
constexpr int kEpilogueWarps = 8;
constexpr int kPairThreads = 64 + 32 * kEpilogueWarps;
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * kBoxBytes;
constexpr int kPairBarOffset = kPairStages * kPairStageBytes;       // full, empty, acc_full[2], acc_empty[2], tmem slot, abort
constexpr int kPairSmem = kPairBarOffset + (2 * kPairStages + 4) * 8 + 16 + 1024;

template <typename TOut>
__device__ __forceinline__ void store32(TOut* dst, const float (&a)[32], int valid) {
  if (valid >= 32 && (((uintptr_t)dst) & 15) == 0) {
    if constexpr (sizeof(TOut) == 2) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint4 o;
        __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
        for (int e = 0; e < 4; ++e) o2[e] = __floats2bfloat162_rn(a[q * 8 + 2 * e], a[q * 8 + 2 * e + 1]);
        reinterpret_cast<uint4*>(dst)[q] = o;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) reinterpret_cast<float4*>(dst)[q] = make_float4(a[q * 4], a[q * 4 + 1], a[q * 4 + 2], a[q * 4 + 3]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 32; ++e)
      if (e < valid) dst[e] = from_f32<TOut>(a[e]);
  }
}

template <typename TOut>
__global__ void __launch_bounds__(kPairThreads)
linear_int8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, TOut* out, long long ldo,
                        const Scales scales, int M, int N, int num_kb) {
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
    if (lane == 0) {
      long long it = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
        const int m0 = (tile % m_tiles) * 256 + (int)rank * 128, n0 = (tile / m_tiles) * 256 + (int)rank * 128;
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = (int)(it % kPairStages);
          if (it >= kPairStages && !wait_on(empty_bar(s), (unsigned)((it / kPairStages) - 1) & 1, abort_flag, 11)) { ok = false; break; }
          if (rank == 0) tc::mbar_expect_tx(full_bar(s), 2 * kPairStageBytes);
          const unsigned counted_on = tc::map_to_rank(full_bar(s), 0);
          const unsigned dst = smem_base + s * kPairStageBytes;
          tc::tma_load_2d_pair(dst, &map_x, kb * BK, m0, counted_on);
          tc::tma_load_2d_pair(dst + kBoxBytes, &map_w, kb * BK, n0, counted_on);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr unsigned idesc = tc::idesc_i8_s32(256, 256);
      long long it = 0;
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
        for (int kb = 0; kb < num_kb; ++kb, ++it) {
          const int s = (int)(it % kPairStages);
          ok = wait_on(full_bar(s), (unsigned)(it / kPairStages) & 1, abort_flag, 12);
          if (!ok) break;
          tc::fence_after();
          const unsigned a_addr = smem_base + s * kPairStageBytes;
          const unsigned long long da = tc::desc_k_major_sw128(a_addr), db = tc::desc_k_major_sw128(a_addr + kBoxBytes);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            tc::umma_i8_pair(tmem_acc, da + 2ull * k, db + 2ull * k, idesc, (kb | k) != 0 ? 1u : 0u);
          tc::umma_commit_pair(empty_bar(s), 3);
        }
        if (ok) tc::umma_commit_pair(acc_full_bar(a), 3);
      }
    }
  } else {
    const int quarter = warp & 3;            // a warp may only touch lanes [32 * (warp % 4), +32)
    const int part = (warp - 2) >> 2;        // the two warps of a quarter take half of the columns each
    int local = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++local) {
      const int a = local & 1;
      const int row = (tile % m_tiles) * 256 + (int)rank * 128 + quarter * 32 + lane, n0 = (tile / m_tiles) * 256 + part * 128;
      const float sx = row < M ? scales.sx[row] : 0.f;
      if (!wait_on(acc_full_bar(a), (unsigned)(local >> 1) & 1, abort_flag, 13)) break;
      tc::fence_after();
      const unsigned tmem_acc = tmem_base + (unsigned)(a * 256 + part * 128) + ((unsigned)(quarter * 32) << 16);
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        if (n0 + c >= N) break;                      // the same for the whole warp
        unsigned v[32];
        float y[32];
        tc::tmem_ld32(tmem_acc + (unsigned)c, v);
        tc::tmem_ld_wait();
        if (n0 + c + 32 <= N) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            y[e] = finish((int)v[e], sx, scales.sw[n0 + c + e]);
            if (scales.bias) y[e] = __fadd_rn(y[e], scales.bias[n0 + c + e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const int n = n0 + c + e < N ? n0 + c + e : N - 1;
            y[e] = finish((int)v[e], sx, scales.sw[n]);
            if (scales.bias) y[e] = __fadd_rn(y[e], scales.bias[n]);
          }
        }
        if (row < M) store32(out + (size_t)row * ldo + n0 + c, y, N - (n0 + c));
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive_cluster(tc::map_to_rank(acc_empty_bar(a), 0));
    }
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

constexpr int kSmemOfTwo = 110 * 1024, kSmemOfOne = 208 * 1024;      // two CTAs on an SM, or one

template <typename TOut>
int launch_rows(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
                int c, int z, cudaStream_t s) {
  Shape g = {};
  g.M = M, g.N = N;
  g.bn = ceil_div(ceil_div(M, z), 16) * 16;                            // z tiles of x, of equal size
  g.num_kb = ceil_div(K, BK);
  g.kb_per_rank = ceil_div(g.num_kb, c);
  g.cols_per_owner = ceil_div(g.bn, c);
  g.tmem_cols = g.bn <= 32 ? 32 : g.bn <= 64 ? 64 : g.bn <= 128 ? 128 : 256;
  const int stage = kBoxBytes + g.bn * BK, recv = c * g.cols_per_owner * BM * 4, budget = g.bn <= 128 ? kSmemOfTwo : kSmemOfOne;
  const bool own_room = g.bn <= 64;                                    // deposits beside the ring, or over it when it is drained
  g.stages = (budget - 256 - (own_room ? recv : 0)) / stage;
  if (g.stages > 8) g.stages = 8;
  g.recv_offset = own_room ? g.stages * stage : 0;
  g.bar_offset = own_room ? g.recv_offset + recv : (g.stages * stage > recv ? g.stages * stage : recv);
  g.vec = (uintptr_t)out % (4 * sizeof(TOut)) == 0 && (M == 1 || ldo % 4 == 0);
  const int smem = g.bar_offset + 8 * (2 * g.stages + 1) + 16;
  OI_REQUIRE(ceil_div(N, BM) <= 65535, "linear_int8: %d channels are too many for %d rows", N, M);
  CUtensorMap mw, mx;
  int rc = tc::make_map_2d_i8(&mw, w, N, K, ldw, BM);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for the weight failed (%d; -1: cuTensorMapEncodeTiled is not available)", rc);
  rc = tc::make_map_2d_i8(&mx, x, M, K, ldx, g.bn);
  OI_REQUIRE(rc == 0, "linear_int8: tensor map for x failed (%d)", rc);
  auto kernel = linear_int8_rows_kernel<TOut>;
  static bool allowed[64];
  if ((rc = allow_smem(kernel, 227 * 1024, allowed))) return rc;
  oi_launch_cluster(kernel, dim3(c, ceil_div(N, BM), z), kThreads, smem, s, c, mw, mx, out, ldo, scales, g);
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
  auto kernel = linear_int8_pair_kernel<TOut>;
  static bool allowed[64];
  if ((rc = allow_smem(kernel, kPairSmem, allowed))) return rc;
  const long long tiles = (long long)ceil_div(M, 256) * ceil_div(N, 256);
  OI_REQUIRE(tiles < (1LL << 31), "linear_int8: %d rows of %d results are too many", M, N);
  const int most = oi_sm_count() / 2, pairs = tiles < most ? (int)tiles : most;
  oi_launch_cluster(kernel, 2 * pairs, kPairThreads, kPairSmem, s, 2, mx, mw, out, ldo, scales, M, N, ceil_div(K, BK));
  OI_CHECK_LAUNCH();
  return OI_OK;
}

constexpr int kRowsMost = 512;

template <typename TOut>
int launch(TOut* out, long long ldo, const void* x, long long ldx, const void* w, long long ldw, const Scales& scales, int M, int N, int K,
           cudaStream_t s) {
  if (M > kRowsMost) return launch_pair(out, ldo, x, ldx, w, ldw, scales, M, N, K, s);
  // slices of K: as many as run at once, each of two stages at least, none empty
  const int num_kb = ceil_div(K, BK), tiles = ceil_div(N, BM) * ceil_div(M, 256);
  const int at_once = ceil_div(M, ceil_div(M, 256)) <= 128 ? 264 : 132;     // two CTAs on an SM, or one
  int c = 1;
  while (c < 8 && tiles * c < oi_sm_count() && tiles * 2 * c <= at_once && num_kb / (2 * c) >= 2) c *= 2;
  while (c > 1 && (c - 1) * ((num_kb + c - 1) / c) >= num_kb) c /= 2;
  return launch_rows(out, ldo, x, ldx, w, ldw, scales, M, N, K, c, ceil_div(M, 256), s);
}

}  // namespace

// x [M, K], w [N, K]: 8-bit integers, row strides in bytes; rows start on 16-byte borders. sx [M], sw [N], bias [N] or null: float32.
// w is read before the kernels ahead on the stream have finished: the library's kernels must not have written it since the last
// launch in plain stream order (oi_launch_fence).
OI_API int oi_linear_int8(void* out, int out_dtype, long long ldo, const void* x, long long ldx, const float* sx, const void* w,
                          long long ldw, const float* sw, const float* bias, int M, int N, int K, void* stream) {
  OI_REQUIRE(M >= 0 && N >= 0 && K >= 1 && K <= 131071, "linear_int8: bad sizes M=%d N=%d K=%d (K: 1 to 131071)", M, N, K);
  OI_REQUIRE(out_dtype == OI_F32 || out_dtype == OI_BF16, "linear_int8: unknown output dtype code %d", out_dtype);
  if (M == 0 || N == 0) return OI_OK;
  OI_REQUIRE(ldx % 16 == 0 && ldw % 16 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)w % 16 == 0 && ldx >= K && ldw >= K,
             "linear_int8: rows of x and w must start on 16-byte borders");
  OI_REQUIRE(M == 1 || ldo >= N, "linear_int8: result rows of %d that start %lld apart", N, ldo);
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
