// Matrix product of the linear layer on the 5th-generation tensor cores:
//   C[m, n] = sum_k A(m, k) B(n, k)
// A and B are 16-bit, each either K-major (a row of the matrix is contiguous
// along k) or MN-major (contiguous along m or n): the forward's x and W are
// K-major, the input gradient reads W MN-major, the weight gradient reads dz
// and x MN-major, so no operand is ever transposed in memory.
//
// fp32 operands come as three bf16 planes whose sum is the value (8 + 8 + 8
// bits; exact from 2^-110 up, to 2^-134 below).  Each is rounded to nearest, so the second and third are at most
// 2^-8 and 2^-17 of the value's leading power of two.  Six of the nine plane
// products are formed; the three left out are at most 2 * 2^-25 + 2^-34 of the
// product, half a unit of its last place, with either sign.
//
// One persistent block per SM (or a pair of blocks on two SMs, CG = 2, sharing
// a 256-row tile: each holds half of A's rows and half of B's, which halves
// what is read from L2 per product).  Warp 0 copies tiles by TMA into a ring
// of shared-memory stages, warp 1 issues the products into TMEM, warps 4-19
// read finished accumulators back while the next tile's products run.
#pragma once

#include <cuda.h>

#include "ls_common.cuh"
#include "ls_epilogue.cuh"

namespace nnue_ls {

constexpr int kEpilogueWarp0 = 4, kEpilogueWarps = 16;
constexpr int kGemmThreads = 32 * (kEpilogueWarp0 + kEpilogueWarps);
constexpr int kColumnGroups = kEpilogueWarps / 4;  // a warp reaches a quarter of the accumulators' lanes
constexpr int kTileM = 128;          // rows of C per block
// The last wait of a block, for what it has in flight: at least so long, or this after a wait ran out (a copy or product
// that has not ended by then will not).
constexpr uint64_t kDrainNs = 4000000000ull, kDrainAfterTimeoutNs = 250000000ull;

// Shared memory: stages of A and B tiles, one transpose buffer per epilogue
// warp, barriers.  Planes = 1: 64 k values per stage; 3: 32.
template <int PLANES, int CG>
struct GemmShape {
  static constexpr int kBK = PLANES == 1 ? 64 : 32;
  static constexpr int kMaxBN = PLANES == 3 && CG == 1 ? 128 : 256;   // columns of C per tile
  static constexpr int kAccs = 512 / kMaxBN;                          // accumulators that TMEM holds
  static constexpr int kRowsB = kMaxBN / CG;                         // rows of B held by one block
  static constexpr int kPlaneA = kTileM * kBK * 2, kPlaneB = kRowsB * kBK * 2;
  static constexpr int kStage = PLANES * (kPlaneA + kPlaneB);
  static constexpr int kStages = PLANES == 1 && CG == 2 ? 5 : 3;
  static constexpr int kTranspose = kEpilogueWarps * 32 * 32 * 4;
  static constexpr int kTail = 384;  // barriers and parameters
  static constexpr int kSmem = 1024 + kStages * kStage + kTranspose + kTail;
  // k blocks summed in TMEM before the epilogue warps take the sum into
  // registers.  The tensor cores' running sums lose up to a unit of the last
  // place per instruction; with fp32 operands that would show, so there a
  // chain is 2 blocks x 2 steps x 6 products long.  0: all of the item's.
  static constexpr int kChunk = PLANES == 1 ? 0 : 2;
};

struct GemmParams {
  int64_t M, N;
  int32_t k_blocks, splits;      // k blocks in all; pieces the k range is cut into
  int32_t m_tiles, n_tiles, bn;  // bn: columns of C per tile, a multiple of 16
  int32_t a_mn, b_mn;            // 1: MN-major
  uint32_t idesc;
  float* partial;  // splits > 1: [splits, M, N] sums, joined by another kernel
  int64_t items;           // tiles times pieces; 0 where wait_limit_ns is
  uint64_t wait_limit_ns;  // 0: no product is formed, as if every wait had run out
  EpilogueParams e;
};

// ---- PTX ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Arrives on the barrier at the same offset in the pair's first block.
__device__ __forceinline__ void mbar_arrive_leader(uint32_t bar) {
  asm volatile(
      "{\n .reg .b32 ra;\n mapa.shared::cluster.u32 ra, %0, 0;\n"
      " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [ra];\n}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for the phase, for limit_ns at most; a wait that runs out raises the
// device flag and ends every other wait of the block.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, uint64_t limit_ns) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t i = 1; !mbar_try(bar, parity); ++i) {
    if (i % 16) continue;
    if (*gave_up) return false;
    if (global_ns() - t0 > limit_ns) {
      *gave_up = 1;
      flag_error(kErrWaitTimeout);
      return false;
    }
  }
  return true;
}

// The same for a whole warp, whose lanes could run out on either side of the phase's end: they go on together or give
// up together, as the collective reads of TMEM that follow need.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* gave_up,
                                               uint64_t limit_ns) {
  return __all_sync(kFull, mbar_wait(bar, parity, gave_up, limit_ns));
}

// The epilogue's warps say that they are done, one more warp waits for that (named barrier 1).
__device__ __forceinline__ void epilogue_done_arrive() {
  __syncwarp();
  asm volatile("bar.arrive 1, %0;" ::"n"(32 * (kEpilogueWarps + 1)) : "memory");
}
__device__ __forceinline__ void epilogue_done_wait() {
  asm volatile("bar.sync 1, %0;" ::"n"(32 * (kEpilogueWarps + 1)) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Copies one box; in a pair both blocks' copies count on the first block's barrier.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar & 0xfeffffffu)  // bit 24 selects the block within the pair
        : "memory");
  }
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

template <int CG>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// The barrier's phase ends when the products issued so far are done; in a pair
// the barrier at this offset in both blocks.
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  }
}
__device__ __forceinline__ void tcgen_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// 32 lanes x 16 columns of accumulators: this thread's lane, 16 columns.
__device__ __forceinline__ void tmem_load16(uint32_t addr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared-memory operand descriptors.  K-major: rows of BK values, 8-row groups
// `8 * BK * 2` bytes apart, 128-byte swizzle for 64 values and 64-byte for 32.
// MN-major: rows of 64 m (or n) values under the 128-byte swizzle, one row per
// k; 8-k groups 1024 bytes apart, blocks of 64 values BK rows apart.
template <int BK>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, int mn_major) {
  const uint64_t swizzle = mn_major || BK == 64 ? 2 : 4;
  const uint64_t sbo = mn_major ? 1024 : 8 * BK * 2;
  const uint64_t lbo = mn_major ? BK * 128 : 16;
  return (uint64_t)((addr & 0x3ffff) >> 4) | (lbo >> 4) << 16 | (sbo >> 4) << 32 | (uint64_t)1 << 46 | swizzle << 61;
}

// By one warp: NaN in all that its block owns.  Nothing here is known to the rest of the kernel: parameters come from
// their copy in shared memory and the block's place from opaque reads.  Otherwise the compiler keeps values for it in
// registers that the epilogue's loops need (bf16 65536 x 1040 x 1024 with GELU and residual, forward: 175 us against 162).
template <typename T, int CG>
__device__ __forceinline__ void store_nan(const volatile GemmParams* q) {
  using D = Derivative<T>;
  const float nan = __int_as_float(0x7fffffff);
  uint32_t block, blocks, lane;
  asm volatile("mov.u32 %0, %%ctaid.x;\nmov.u32 %1, %%nctaid.x;\nmov.u32 %2, %%laneid;" : "=r"(block), "=r"(blocks), "=r"(lane));
  const uint32_t n_tiles = q->n_tiles, tiles = q->m_tiles * n_tiles;
#pragma unroll 1
  for (uint32_t item = block / CG; item < tiles * q->splits; item += blocks / CG) {
    const uint32_t tile = item % tiles;
#pragma unroll 1
    for (int r = 0; r < kTileM; ++r) {
      const int64_t m = (int64_t)(tile / n_tiles * CG + block % CG) * kTileM + r;
      if (m >= q->M) break;
#pragma unroll 1
      for (int c = (int)lane; c < q->bn; c += 32) {
        const int64_t n = (int64_t)(tile % n_tiles) * q->bn + c;
        if (n >= q->N) break;
        const int64_t at = m * q->N + n;
        if (q->splits > 1) {
          q->partial[item / tiles * q->M * q->N + at] = nan;
        } else {
          static_cast<T*>(q->e.out)[at] = from_f<T>(nan);
          if (q->e.act_grad) static_cast<typename D::Code*>(q->e.act_grad)[at] = D::encode(nan);
        }
      }
    }
  }
}

// map_a, map_b: [planes][rows][columns], the contiguous direction first.  They are parameters of their own because
// their address is taken: parameters whose address is not are read as constants.
// ---- the kernel -----------------------------------------------------------------
template <typename T, int CG>
__global__ void __launch_bounds__(kGemmThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const GemmParams p) {
  constexpr int PLANES = sizeof(T) == 4 ? 3 : 1;
  using S = GemmShape<PLANES, CG>;
  constexpr int BK = S::kBK;
  extern __shared__ uint8_t smem_raw[];
  // the same offset in both blocks of a pair: the dynamic shared memory starts at the same address there
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float4* transpose = reinterpret_cast<float4*>(smem + S::kStages * S::kStage);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStage + S::kTranspose);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * S::kStages;
  const uint32_t acc_full0 = empty0 + 8 * S::kStages, acc_empty0 = acc_full0 + 8 * S::kAccs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * (S::kStages + S::kAccs));
  volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
  GemmParams* shared = reinterpret_cast<GemmParams*>(tmem_slot + 2);
  static_assert(8 * (2 * (S::kStages + S::kAccs) + 1) + sizeof(GemmParams) <= S::kTail, "barriers and parameters");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 1 ? 0 : (int)cluster_rank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < S::kAccs; ++i) {
      mbar_init(acc_full0 + 8 * i, 1);
      mbar_init(acc_empty0 + 8 * i, kEpilogueWarps * CG);
    }
    *gave_up = p.wait_limit_ns == 0;
    if (p.wait_limit_ns == 0) flag_error(kErrWaitTimeout);
    *shared = p;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async;" ::: "memory");
  }
  if (warp == 2) tmem_alloc<CG>(smem_u32(tmem_slot));
  tcgen_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tcgen_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int worker = blockIdx.x / CG, workers = gridDim.x / CG;
  const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles, items = p.items;
  const int rows_b = p.bn / CG;  // rows of B this block holds
  const int blocks_b = (rows_b + 63) / 64;

  if (warp == 0 && lane == 0) {
    // ---- copies ----
    const uint32_t bytes =
        CG * PLANES * (S::kPlaneA + (p.b_mn ? blocks_b * 64 * BK * 2 : rows_b * BK * 2));
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    for (int64_t item = worker; item < items && ok; item += workers) {
      const int64_t tile = item % tiles;
      const int split = (int)(item / tiles);
      const int m0 = (int)(tile / p.n_tiles) * (kTileM * CG) + rank * kTileM;
      const int n0 = (int)(tile % p.n_tiles) * p.bn + rank * rows_b;
      const int k0 = (int)((int64_t)p.k_blocks * split / p.splits), k1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
      for (int k = k0; k < k1; ++k) {
        if (!(ok = mbar_wait(empty0 + 8 * stage, phase ^ 1, gave_up, p.wait_limit_ns))) break;
        const uint32_t bar = full0 + 8 * stage;
        if (rank == 0) mbar_expect(bar, bytes);
        const uint32_t sa = smem_u32(smem + stage * S::kStage), sb = sa + PLANES * S::kPlaneA;
        for (int q = 0; q < PLANES; ++q) {
          if (p.a_mn) {
            for (int i = 0; i < kTileM / 64; ++i)
              tma_load<CG>(sa + q * S::kPlaneA + i * 64 * BK * 2, &map_a, m0 + 64 * i, k * BK, q, bar);
          } else {
            tma_load<CG>(sa + q * S::kPlaneA, &map_a, k * BK, m0, q, bar);
          }
          if (p.b_mn) {
            for (int i = 0; i < blocks_b; ++i)
              tma_load<CG>(sb + q * S::kPlaneB + i * 64 * BK * 2, &map_b, n0 + 64 * i, k * BK, q, bar);
          } else {
            tma_load<CG>(sb + q * S::kPlaneB, &map_b, k * BK, n0, q, bar);
          }
        }
        if (++stage == S::kStages) stage = 0, phase ^= 1;
      }
    }
    // the last copies and products have to land before the block ends: wait for every stage to be free again
    for (int i = 0; i < S::kStages; ++i) {
      const uint64_t t0 = global_ns();
      while (!mbar_try(empty0 + 8 * stage, phase ^ 1) &&
             global_ns() - t0 < (ok && !*gave_up ? max(kDrainNs, p.wait_limit_ns) : kDrainAfterTimeoutNs)) {
      }
      if (++stage == S::kStages) stage = 0, phase ^= 1;
    }
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ---- products ----
    const uint32_t step_a = (p.a_mn ? 16 * 128 : 32) >> 4, step_b = (p.b_mn ? 16 * 128 : 32) >> 4;
    uint32_t stage = 0, phase = 0, chunk = 0;
    bool ok = true;
    for (int64_t item = worker; item < items && ok; item += workers) {
      const int split = (int)(item / tiles);
      const int k0 = (int)((int64_t)p.k_blocks * split / p.splits), k1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
      const int per_chunk = S::kChunk ? S::kChunk : k1 - k0;
      for (int kc = k0; kc < k1 && ok; kc += per_chunk, ++chunk) {
        const uint32_t acc = chunk % S::kAccs, d = tmem + acc * S::kMaxBN;
        if (!(ok = mbar_wait(acc_empty0 + 8 * acc, ((chunk / S::kAccs) & 1) ^ 1, gave_up, p.wait_limit_ns))) break;
        tcgen_fence_after();
        uint32_t accumulate = 0;
        for (int k = kc; k < min(kc + per_chunk, k1); ++k) {
          if (!(ok = mbar_wait(full0 + 8 * stage, phase, gave_up, p.wait_limit_ns))) break;
          tcgen_fence_after();
          const uint32_t sa = smem_u32(smem + stage * S::kStage), sb = sa + PLANES * S::kPlaneA;
          uint64_t da[PLANES], db[PLANES];
#pragma unroll
          for (int q = 0; q < PLANES; ++q) {
            da[q] = operand_desc<BK>(sa + q * S::kPlaneA, p.a_mn);
            db[q] = operand_desc<BK>(sb + q * S::kPlaneB, p.b_mn);
          }
#pragma unroll
          for (int i = 0; i < BK / 16; ++i) {
            // small products first
#pragma unroll
            for (int s = PLANES == 1 ? 0 : 2; s >= 0; --s)
#pragma unroll
              for (int q = 0; q <= s; ++q) {
                mma<CG>(d, da[q] + i * step_a, db[s - q] + i * step_b, p.idesc, accumulate);
                accumulate = 1;
              }
          }
          mma_commit<CG>(empty0 + 8 * stage);
          if (++stage == S::kStages) stage = 0, phase ^= 1;
        }
        if (ok) mma_commit<CG>(acc_full0 + 8 * acc);
      }
    }
  } else if (warp >= kEpilogueWarp0) {
    // ---- epilogue: warp's quarter of the lanes, every fourth block of 32 columns ----
    const int quarter = warp & 3, group = (warp - kEpilogueWarp0) >> 2;
    const int64_t M = p.M, N = p.N;
    Block32 block{transpose + (warp - kEpilogueWarp0) * 256};
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int col_blocks = (p.bn + 31) / 32;
    uint32_t chunk = 0;
    bool ok = true;
    for (int64_t item = worker; item < items && ok; item += workers) {
      const int64_t tile = item % tiles;
      const int split = (int)(item / tiles);
      const int64_t m0 = (tile / p.n_tiles) * (kTileM * CG) + rank * kTileM + quarter * 32;
      const int64_t n0 = (tile % p.n_tiles) * p.bn, n1 = min(N, n0 + p.bn);
      const int rows = (int)max((int64_t)0, min((int64_t)32, M - m0));
      float* partial = p.splits > 1 ? p.partial + (int64_t)split * M * N : nullptr;
      if (p.e.residual && !partial && lane < rows) {
        // the residual's rows come from HBM while the tile's products run
        const char* r = reinterpret_cast<const char*>(static_cast<const T*>(p.e.residual) + (m0 + lane) * p.e.ldr);
        for (int cb = group; cb < col_blocks; cb += kColumnGroups)
          if (n0 + cb * 32 < n1) prefetch_l2(r + (n0 + cb * 32) * sizeof(T));
      }
      if constexpr (S::kChunk == 0) {
        const uint32_t acc = chunk % S::kAccs;
        if (!(ok = mbar_wait_warp(acc_full0 + 8 * acc, (chunk / S::kAccs) & 1, gave_up, p.wait_limit_ns))) break;
        tcgen_fence_after();
        for (int cb = group; cb < col_blocks; cb += kColumnGroups) {
          const int64_t n = n0 + cb * 32;
          BlockWriter<T> writer(p.e, m0, partial ? 0 : rows, n, n1, N, lane);
          float v[32];
          tmem_load16(lanes + acc * S::kMaxBN + cb * 32, v);
          tmem_load16(lanes + acc * S::kMaxBN + cb * 32 + 16, v + 16);
          if (cb + kColumnGroups >= col_blocks) {  // this warp's last read: the accumulator may be written again
            tcgen_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 1) mbar_arrive(acc_empty0 + 8 * acc);
              else mbar_arrive_leader(acc_empty0 + 8 * acc);
            }
          }
          block.put(v, lane);
          if (partial) store_partial(block, partial, N % 4 == 0, m0, rows, n, n1, N, lane);
          else writer.write(block);
        }
        if (group >= col_blocks && lane == 0) {  // a narrow tile leaves this warp nothing to read
          if constexpr (CG == 1) mbar_arrive(acc_empty0 + 8 * acc);
          else mbar_arrive_leader(acc_empty0 + 8 * acc);
        }
        ++chunk;
      } else {
        constexpr int kMine = S::kMaxBN / (32 * kColumnGroups);  // column blocks per warp
        float sum[kMine][32];
#pragma unroll
        for (int i = 0; i < kMine; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[i][j] = 0.f;
        const int k0 = (int)((int64_t)p.k_blocks * split / p.splits),
                  k1 = (int)((int64_t)p.k_blocks * (split + 1) / p.splits);
        for (int kc = k0; kc < k1; kc += S::kChunk, ++chunk) {
          const uint32_t acc = chunk % S::kAccs;
          if (!(ok = mbar_wait_warp(acc_full0 + 8 * acc, (chunk / S::kAccs) & 1, gave_up, p.wait_limit_ns))) break;
          tcgen_fence_after();
#pragma unroll
          for (int i = 0; i < kMine; ++i) {
            const int cb = group + kColumnGroups * i;
            if (cb < col_blocks) {
#pragma unroll
              for (int h = 0; h < 32; h += 16) {
                float v[16];
                tmem_load16(lanes + acc * S::kMaxBN + cb * 32 + h, v);
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[i][h + j] += v[j];
              }
            }
          }
          tcgen_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 1) mbar_arrive(acc_empty0 + 8 * acc);
            else mbar_arrive_leader(acc_empty0 + 8 * acc);
          }
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (group + kColumnGroups * i < col_blocks) {
            const int64_t n = n0 + (group + kColumnGroups * i) * 32;
            block.put(sum[i], lane);
            if (partial) store_partial(block, partial, N % 4 == 0, m0, rows, n, n1, N, lane);
            else store_block_f32(block.s, &shared->e, m0, rows, n, n1, N, lane);
          }
      }
    }
    epilogue_done_arrive();
  } else if (warp == 3) {
    // ---- after a wait ran out: NaN in place of whatever the memory held ----
    epilogue_done_wait();
    if (*gave_up) store_nan<T, CG>(shared);
  }
  __syncwarp();
  tcgen_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the other block may still signal barriers here
  if (warp == 2) {
    tcgen_fence_after();
    tmem_free<CG>(tmem);
  }
}

}  // namespace nnue_ls
