// Product of e4m3 operands with a scale for each block of 128
// (b200k_scaled_mm, include/b200k.h):
//
//   out[m, n] = sum_g sa[m, g] sb[g, n / 128] sum_{k in block g} a[m, k] b[k, n]
//
// No reference counterpart (its GEMM is 16-bit).  The inner sum is a 128-deep
// tcgen05 product (kind::f8f6f4, fp32 accumulators in tensor memory).  The
// scales differ from block to block, so it cannot run on over k: each block's
// product goes to one of several tensor-memory buffers, and while the tensor
// pipe fills the next ones the epilogue warps read it and add it, times its
// scale, to fp32 sums in registers.
//
// Warps of a CTA:
//   warp 0      TMA producer (128-byte swizzled tiles of 128 k);
//   warps 1, 3  MMA issuers, of every other block: the waits and the issue of a
//               block take one warp 600 clocks, more than a block of few rows
//               takes to arrive;
//   warp 2      brings the scales of kScaleBlocks blocks at a time to shared
//               memory, transposed (and owns tensor memory);
//   warps 4..   epilogue.
// Two kinds of tile:
//   wide        256 rows of a x 256 columns of b on a pair of CTAs (cta_group::2),
//               each with 128 of the rows.  A thread has one row and 128 columns,
//               of one scale block, so a block costs it one scale and 64 packed
//               FMAs.  (128 x 256 on one CTA: the operands' way from L2 to shared
//               memory, 12 TB/s, held it at 2050 TFLOP/s.)
//   turned      128 columns of b as the product's rows x 16 to 128 rows of a as
//               its columns, on a cluster of `split` CTAs that share the blocks
//               of k out among them and add their sums over distributed shared
//               memory in the order of the ranks.  For few rows, where b's
//               bytes are the bound: every SM fetches some of them, and the
//               tensor-memory lanes are full whatever the number of rows.
// Measured: [16384, 4096] x [4096, 14336] 980-1040 us = 1.9 PFLOP/s in long runs, at 1.5
// GHz under the power limit (870-910 us in four calls after a pause).  No unit is
// full (8192 rows: tensor pipe 60 %, issue 42 %, L2 37 %): the tensor pipe waits for
// the sums, a buffer's way from the MMAs' issue over the epilogue back takes 1700
// clocks, of which two buffers hide half (MMAs of 128 columns, which would give
// four, cost more than they hide: 1010 us with an earlier version).  64 rows of
// [4096, 14336] 17.8 us = 3.4 TB/s, a row of [8192, 2048] 7.4 us.
#include <type_traits>

#include "gemm_kernel.cuh"

namespace b200k {
namespace mm8 {
namespace {

using namespace gemm;

constexpr int kBlk = 128;  // k of a block, one swizzle row of bytes
// Registers of a thread of wide tiles: launched with 168, 128 control threads
// leave theirs to 256 epilogue threads (128 sums each).
constexpr int kCtlRegs = 56, kEpiRegs = 224;
// Blocks of k whose scales are fetched together, a 32-byte sector of a row.  (A
// load by each epilogue thread touched 32 lines for each block and kept all eight
// epilogue warps 1500 clocks for four blocks.)
constexpr int kScaleBlocks = 8;
constexpr int kScaleRow = 132;                                        // floats: 128 rows of a block, turned banks
constexpr uint32_t kScaleBytes = kScaleBlocks * (kScaleRow + 4) * 4;  // with two scales of b a block
constexpr uint32_t kStgBox = 32 * 128;    // 32 rows x 128 bytes of the output
constexpr int kStgBoxes = 2;              // of an epilogue warp: its tile in 16 bits
constexpr int kMaxSplit = 8;

struct MmParams {
  int32_t M, N;
  int32_t tiles_m, tiles_n, num_tiles, k_blocks;
  int32_t split;            // CTAs that share a tile's blocks (turned)
  int32_t tma_out;          // the output's rows can be stored by TMA (wide)
  const float* sa;          // [M, k_blocks]
  int64_t sa_m, sa_k;
  int32_t sa_vec;           // four neighbouring blocks' scales lie 16-byte aligned
  const float* sb;          // [k_blocks, ceil(N / 128)]
  int64_t sb_k, sb_n;
  void* out;                // [M, N] contiguous
  int32_t out_dt;
  int32_t test_flags;
  int32_t* status;
  int64_t timeout_ns;
};

// BN: columns of the product in tensor memory (256: wide).
template <int BN>
struct Cfg8 {
  static constexpr bool kWide = BN == 256;
  static constexpr int kGroups = BN >= 128 ? 2 : 1;        // column groups, four epilogue warps each
  static constexpr int kCols = BN / kGroups;               // of an epilogue thread
  static constexpr int kBufs = kWide ? 2 : 4;
  static constexpr uint32_t kTmemCols = BN * kBufs;
  static constexpr int kThreads = 128 + 128 * kGroups;
  static constexpr uint32_t kRowBytes = 128 * kBlk;        // the product's 128 rows (of this CTA)
  static constexpr uint32_t kStage = kRowBytes + (kWide ? BN / 2 : BN) * kBlk;
  // Few rows: two CTAs an SM, so that one's waits, start and end lie under the
  // other's (64 rows of [4096, 14336] with one: 20.7 us).
  static constexpr int kCtas = BN <= 64 ? 2 : 1;
  static constexpr int kStages = BN >= 128 ? (kWide ? 4 : 6) : 4;
  static constexpr uint32_t kOffStg = kStages * kStage;
  static constexpr uint32_t kOffSc = kOffStg + (kWide ? 4 * kGroups * kStgBoxes * kStgBox : 0);  // two chunks of scales
  static constexpr uint32_t kOffBar = kOffSc + 2 * kScaleBytes;
  static constexpr uint32_t kSmem = 1024 + kOffBar + 512;
  static constexpr int kPartRow = 132;  // floats: 128 sums of a split tile's column
  static_assert(kTmemCols >= 32 && kTmemCols <= 512, "tensor memory");
  static_assert(kSmem <= (kCtas == 1 ? 232448u : 115712u) && kCtas * kTmemCols <= 512, "fits the SM");
  static_assert(kCtas > 1 || kSmem > 232448 / 2, "one CTA per SM");
  static_assert(kWide || BN * kPartRow * 4 <= kOffStg, "the sums of a split tile fit the ring");
};

// The four MMAs of a block (32 k each, 32 bytes apart in the swizzled rows).
// Called by a whole warp and issued by one elected lane: in warp-uniform code the
// descriptors stay in uniform registers (from a lane's branch the MMAs of a block
// and its commits took 390 clocks to issue, a block's product itself 512).
template <bool PAIR>
__device__ __forceinline__ void umma_block(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
#define B200K_UMMA_BLOCK(GROUP)                                                                            \
  asm volatile(                                                                                            \
      "{\n\t.reg .pred e, no, yes;\n\t"                                                                    \
      "elect.sync _|e, 0xffffffff;\n\t"                                                                    \
      "setp.ne.b32 no, 0, 0;\n\t"                                                                          \
      "setp.eq.b32 yes, 0, 0;\n\t"                                                                         \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], %1, %5, %9, no;\n\t"                         \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], %2, %6, %9, yes;\n\t"                        \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], %3, %7, %9, yes;\n\t"                        \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], %4, %8, %9, yes;\n\t}\n" ::"r"(d_tmem),      \
      "l"(adesc), "l"(adesc + 2), "l"(adesc + 4), "l"(adesc + 6), "l"(bdesc), "l"(bdesc + 2), "l"(bdesc + 4), \
      "l"(bdesc + 6), "r"(idesc)                                                                           \
      : "memory")
  if constexpr (PAIR) B200K_UMMA_BLOCK("2");
  else B200K_UMMA_BLOCK("1");
#undef B200K_UMMA_BLOCK
}
// Arrives on a barrier (a pair: on both CTAs') when the MMAs so far have completed.
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred e;\n\t.reg .b16 both;\n\t"
        "mov.b16 both, 3;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n\t}\n" ::"r"(
            smem_u32(bar))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
        : "memory");
}
// Arrival at a barrier of the pair's even CTA.
__device__ __forceinline__ void arrive_even(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(bar, 0)) : "memory");
}
// A phase that has completed costs a test (the wait alone took 30 clocks more).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Ctl& c) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  if (__all_sync(0xffffffffu, done)) return true;
  return __all_sync(0xffffffffu, wait_bar(bar, parity, c));
}
// 16 or 32 columns of this thread's tensor-memory row, and the wait for them,
// which names the registers so that no use of them is scheduled before it.
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) { tmem_wait_ld_regs(r); }
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Tile t: wide ones go kGroupM tile rows down before they move on, so that
// CTAs side by side share operands in L2; turned ones along the rows of a.
template <bool WIDE>
__device__ __forceinline__ void tile_at(int t, const MmParams& p, int& tm, int& tn) {
  if (WIDE) {
    const int per_group = kGroupM * p.tiles_n;
    const int g = t / per_group, first = g * kGroupM;
    const int rows = min(p.tiles_m - first, kGroupM), r = t - g * per_group;
    tm = first + r % rows;
    tn = r / rows;
  } else {
    tn = t / p.tiles_m;
    tm = t - tn * p.tiles_m;
  }
}

template <int BN>
__global__ void __launch_bounds__(Cfg8<BN>::kThreads, Cfg8<BN>::kCtas)
    mm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
              const __grid_constant__ CUtensorMap tmO, const __grid_constant__ MmParams p) {
  using C = Cfg8<BN>;
  constexpr bool WIDE = C::kWide;
  constexpr int S = C::kStages, COLS = C::kCols, BUFS = C::kBufs;
  constexpr int kTileM = WIDE ? 256 : BN, kTileN = WIDE ? BN : 128;  // rows of a and columns of b of a tile
  constexpr int kRowsM = WIDE ? 128 : BN;                            // rows of a of a CTA
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sbase = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint64_t* full = reinterpret_cast<uint64_t*>(sbase + C::kOffBar);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + BUFS;
  uint64_t* sc_full = tempty + BUFS;  // [2]
  uint64_t* sc_empty = sc_full + 2;
  uint64_t* drain = sc_empty + 2;     // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int split = WIDE ? 1 : p.split, cluster = WIDE ? 2 : split;
  const uint32_t rank = cluster > 1 ? cluster_rank() : 0;
  const int part = WIDE ? 0 : static_cast<int>(rank);     // of the blocks of k
  const int rows_at = WIDE ? static_cast<int>(rank) * 128 : 0;  // of a tile's rows
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < BUFS; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4 * C::kGroups * (WIDE ? 2 : 1));  // a pair's arrive at the even CTA's
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sc_full[a], 1);
      mbar_init(&drain[a], 1);
      mbar_init(&sc_empty[a], 4 * C::kGroups);
    }
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_map(&tmA);
    prefetch_map(&tmB);
    if (WIDE) prefetch_map(&tmO);
  }
  // Launched under the end of the kernel before, whose writes are waited for here.
  // Tensor memory is taken behind the wait and what follows in the stream launched
  // when all CTAs have theirs: of two kernels that overlap neither holds tensor
  // memory that the other, for which it waits, has still to take.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == 2) {
    if (WIDE) {
      tmem_alloc_pair(tmem_slot, C::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (WIDE) cluster_sync();  // the other CTA's barriers are there too
  else __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  const Ctl ctl{abort_flag, p.status, static_cast<uint64_t>(p.timeout_ns)};
  const int cid = static_cast<int>(blockIdx.x) / cluster, ncl = static_cast<int>(gridDim.x) / cluster;
  // this CTA's blocks of k
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * part / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (part + 1) / split);

  if (warp < 4) {
    if (WIDE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtlRegs));
    if (warp == 0 && lane == 0) {
      // -------------------------------------------------------------- producer
      int s = 0;
      uint32_t ph = 0;
      int64_t issued = 0;
      bool ok = true;
      for (int t = cid; t < p.num_tiles && ok; t += ncl) {
        int tm, tn;
        tile_at<WIDE>(t, p, tm, tn);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = wait_bar(&empty[s], ph ^ 1u, ctl))) break;
          uint8_t* rows = sbase + s * C::kStage;
          if (WIDE) {  // both CTAs' bytes are counted on the even one's barrier
            const uint32_t bar = cluster_addr(&full[s], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStage);
            tma_load_2d_pair(rows, &tmA, bar, kb * kBlk, tm * kTileM + rows_at);
            tma_load_2d_pair(rows + C::kRowBytes, &tmB, bar, kb * kBlk, tn * kTileN + static_cast<int>(rank) * (BN / 2));
          } else {
            mbar_arrive_expect_tx(&full[s], C::kStage);
            tma_load_2d(rows + C::kRowBytes, &tmA, &full[s], kb * kBlk, tm * kTileM);
            tma_load_2d(rows, &tmB, &full[s], kb * kBlk, tn * kTileN);
          }
          ++issued;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // No load is in flight when the MMAs have read every stage; after a timeout
      // the loads that no MMA waited for are waited for here.
      for (int x = 0; x < S; ++x)
        if (issued > x) wait_bar_drain(&empty[x], x < s ? ph : (ph ^ 1u), ok ? 100000000ull : 1000000ull);
      if (!ok && rank == 0) {
        for (int64_t k = issued > S ? issued - S : 0; k < issued; ++k)
          wait_bar_drain(&full[k % S], static_cast<uint32_t>((k / S) & 1), 100000000ull);
      }
    } else if (WIDE && (warp & 1) && rank != 0) {
      // The even CTA's commits arrive here too: the last of each issuer, behind all
      // its MMAs, before this CTA's shared memory may become another's.
      wait_bar_drain(&drain[warp >> 1], 0, 100000000ull);
    } else if (warp & 1) {
      // ----------------------------------------------------------- MMA issuers
      // fp32 accumulators, both operands e4m3 (format 0) and K-major
      const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(BN >> 3) << 17) | ((WIDE ? 256u : 128u) >> 4 << 24);
      const uint64_t da0 = sw128_desc(smem_u32(sbase), 16, 1024);
      const uint64_t db0 = sw128_desc(smem_u32(sbase + C::kRowBytes), 16, 1024);
      const int which = warp >> 1;
      bool ok = true, signal = !(p.test_flags & B200K_SCALED_MM_TEST_WITHHOLD_READY);
      const int64_t blocks = static_cast<int64_t>(cid < p.num_tiles ? (p.num_tiles - cid + ncl - 1) / ncl : 0) * (kb1 - kb0);
      static_assert(S % 2 == 0 && BUFS % 2 == 0, "an issuer's blocks have stages and buffers of their own");
      int s = which, buf = which;
      uint32_t ph = 0, bph = 0;
      for (int64_t i = which; i < blocks; i += 2) {
        if (!(ok = warp_wait(&full[s], ph, ctl) && warp_wait(&tempty[buf], bph ^ 1u, ctl))) break;
        tc_fence_after();
        const uint32_t stage = (s * C::kStage) >> 4;
        umma_block<WIDE>(tmem_base + buf * BN, da0 + stage, db0 + stage, idesc);
        if (signal) commit<WIDE>(&tfull[buf]);
        commit<WIDE>(&empty[s]);
        signal = true;
        if ((s += 2) >= S) {
          s = which;
          ph ^= 1u;
        }
        if ((buf += 2) >= BUFS) {
          buf = which;
          bph ^= 1u;
        }
      }
      // every MMA of this warp completes before tensor memory is freed (the odd CTA
      // waits for its arrival as well)
      commit<WIDE>(&drain[which]);
      wait_bar_drain(&drain[which], 0, 100000000ull);
    } else if (warp == 2) {
      // ---------------------------------------------------------------- scales
      // of this CTA's rows of a; turned: multiplied by b's, of which a tile has
      // one.  Two lanes take a row's eight blocks, four each.
      constexpr int kEach = kRowsM / 16, kAtOnce = WIDE ? 2 : kEach;
      const int kb4 = (lane & 1) * 4, r0 = lane >> 1;
      const bool vec = p.sa_vec && kb0 % 4 == 0;
      int c = 0;
      bool ok = true;
      for (int t = cid; t < p.num_tiles && ok; t += ncl) {
        int tm, tn;
        tile_at<WIDE>(t, p, tm, tn);
        for (int kb = kb0; kb < kb1; kb += kScaleBlocks, ++c) {
          const int k0 = kb + kb4, left = kb1 - k0;  // this lane's blocks
          const int n = tn * kTileN + (WIDE ? (lane >> 1 & 1) * 128 : 0);
          float b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = j < left && n < p.N ? fetch<true>(p.sb + (k0 + j) * p.sb_k + n / kBlk * p.sb_n) : 0.0f;
          float* to = reinterpret_cast<float*>(sbase + C::kOffSc + (c & 1) * kScaleBytes) + kb4 * (kScaleRow + 4);
          if (WIDE && !(ok = warp_wait(&sc_empty[c & 1], ((c >> 1) & 1) ^ 1, ctl))) break;
#pragma unroll 1
          for (int i0 = 0; i0 < kEach; i0 += kAtOnce) {
            float a[kAtOnce][4];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
              const int m = tm * kTileM + rows_at + r0 + (i0 + i) * 16;
              const float* pa = p.sa + m * p.sa_m + k0 * p.sa_k;
              if (vec && left > 0 && k0 + 4 <= p.k_blocks && m < p.M) {
                const float4 v = fetch<true>(reinterpret_cast<const float4*>(pa));
                a[i][0] = v.x;
                a[i][1] = v.y;
                a[i][2] = v.z;
                a[i][3] = v.w;
              } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) a[i][j] = j < left && m < p.M ? fetch<true>(pa + j * p.sa_k) : 0.0f;
              }
            }
            if (!WIDE && i0 == 0 && !(ok = warp_wait(&sc_empty[c & 1], ((c >> 1) & 1) ^ 1, ctl))) break;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) to[j * (kScaleRow + 4) + r0 + (i0 + i) * 16] = WIDE ? a[i][j] : a[i][j] * b[j];
          }
          if (!ok) break;
          if (WIDE && lane < 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j * (kScaleRow + 4) + kScaleRow + (lane >> 1)] = b[j];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[c & 1]);
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    if (WIDE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    const int quarter = warp & 3, cg = (warp - 4) >> 2;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + cg * COLS;
    const bool bf16 = p.out_dt == B200K_BF16;
    int buf = 0, c = 0;  // c: chunks of scales
    uint32_t bph = 0;
    bool ok = true;
    for (int t = cid; t < p.num_tiles && ok; t += ncl) {
      int tm, tn;
      tile_at<WIDE>(t, p, tm, tn);
      // wide: this thread's row and first column; turned: its column and first row
      const int row0 = tm * kTileM + rows_at + (WIDE ? quarter * 32 : cg * COLS), n0 = tn * kTileN + (WIDE ? cg * COLS : quarter * 32);
      const bool any = row0 < p.M && n0 < p.N;  // warp-uniform
      float2 acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
      // Block by block, kLd columns a load; a buffer is released when its last
      // load has landed.
      constexpr int kLd = COLS < 32 ? 16 : 32, J = COLS / kLd;
      for (int kb = kb0, in = 0; kb < kb1; ++kb) {
        const float* sc = reinterpret_cast<const float*>(sbase + C::kOffSc + (c & 1) * kScaleBytes) + in * (kScaleRow + 4);
        ok = (in != 0 || warp_wait(&sc_full[c & 1], (c >> 1) & 1, ctl)) && warp_wait(&tfull[buf], bph, ctl);
        if (!ok) break;
        tc_fence_after();
        uint32_t raw[2][kLd];
        tmem_get(t_row + buf * BN, raw[0]);
        const float scale = WIDE ? sc[quarter * 32 + lane] * sc[kScaleRow + cg] : 0.0f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          tmem_wait(raw[j & 1]);
          if (j + 1 < J) {
            tmem_get(t_row + buf * BN + (j + 1) * kLd, raw[(j + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (WIDE && rank != 0) arrive_even(&tempty[buf]);
              else mbar_arrive(&tempty[buf]);
            }
          }
#pragma unroll
          for (int k = 0; k < kLd / 2; ++k) {
            const float2 v = make_float2(__uint_as_float(raw[j & 1][2 * k]), __uint_as_float(raw[j & 1][2 * k + 1]));
            const float2 f = WIDE ? make_float2(scale, scale) : *reinterpret_cast<const float2*>(sc + cg * COLS + j * kLd + 2 * k);
            acc[j * (kLd / 2) + k] = __ffma2_rn(v, f, acc[j * (kLd / 2) + k]);
          }
        }
        if (++in == kScaleBlocks || kb + 1 == kb1) {  // done with the chunk of scales
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_empty[c & 1]);
          ++c;
          in = 0;
        }
        if (++buf == BUFS) {
          buf = 0;
          bph ^= 1u;
        }
      }
      if (!WIDE && split > 1) {
        // every load has landed and been read: the ring holds the sums, [BN][128]
        float* part = reinterpret_cast<float*>(sbase) + cg * COLS * C::kPartRow + quarter * 32 + lane;
        if (ok && any) {
#pragma unroll
          for (int i = 0; i < COLS / 2; ++i) {
            part[2 * i * C::kPartRow] = acc[i].x;
            part[(2 * i + 1) * C::kPartRow] = acc[i].y;
          }
        }
        break;  // one tile a cluster; joined below
      }
      if (!ok || !any) continue;
      if constexpr (!WIDE) {
        // a warp's lanes are neighbouring columns of the output
        const int n = n0 + lane;
#pragma unroll
        for (int i = 0; i < COLS; ++i)
          if (row0 + i < p.M && n < p.N)
            store_scalar(p.out, static_cast<int64_t>(row0 + i) * p.N + n, p.out_dt, i & 1 ? acc[i / 2].y : acc[i / 2].x);
      } else {
        uint8_t* stg = sbase + C::kOffStg + (warp - 4) * kStgBoxes * kStgBox;
        if (p.tma_out) {
          // staged as boxes of 32 rows x 128 bytes (128-byte swizzle), stored by
          // TMA under the next tile; fp32 takes two rounds
          const bool f32 = p.out_dt == B200K_F32;
          const int step = f32 ? 32 : 64;  // columns of a box
#pragma unroll
          for (int h = 0; h < COLS / 32; ++h) {  // 32 columns: a box of fp32, half of one of 16 bits
            if (h == 0 || (f32 && h == 2)) {
              if (lane == 0) bulk_wait_read_all();  // the stores before have read the boxes
              __syncwarp();
            }
            const float2* v = acc + h * 16;
            uint8_t* row = stg + (f32 ? h & 1 : h >> 1) * kStgBox + lane * 128;
            if (f32) {
#pragma unroll
              for (int g = 0; g < 8; ++g)
                *reinterpret_cast<float4*>(row + ((g ^ (lane & 7)) << 4)) = make_float4(v[2 * g].x, v[2 * g].y, v[2 * g + 1].x, v[2 * g + 1].y);
            } else {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint4*>(row + ((((h & 1) * 4 + g) ^ (lane & 7)) << 4)) =
                    make_uint4(pack16(v[4 * g].x, v[4 * g].y, bf16), pack16(v[4 * g + 1].x, v[4 * g + 1].y, bf16),
                               pack16(v[4 * g + 2].x, v[4 * g + 2].y, bf16), pack16(v[4 * g + 3].x, v[4 * g + 3].y, bf16));
            }
            if (f32 ? h & 1 : h == COLS / 32 - 1) {
              fence_async_smem();
              __syncwarp();
              if (lane == 0) {
                const int first = f32 ? n0 + (h - 1) * 32 : n0;
                if (first < p.N) tma_store_2d(&tmO, stg, first, row0);
                if (first + step < p.N) tma_store_2d(&tmO, stg + kStgBox, first + step, row0);
                bulk_commit();
              }
            }
          }
        } else {
          // Rows that TMA cannot store (N no multiple of 16 bytes): 256 bytes of 32
          // rows through shared memory (chunks of 16 turned by the row), then a warp
          // a row, eight bytes a lane, in pieces as large as N's alignment.
          const bool f32 = p.out_dt == B200K_F32;
          const int per = f32 ? 2 : 4;                             // columns of eight bytes
          const int fit = p.N % per == 0 ? 8 : f32 || p.N % 2 ? (f32 ? 4 : 2) : 4;
          // (the sums stay in registers: each of the three fills has its own constants)
          auto fill = [&](auto wide_type, auto first) {
#pragma unroll
            for (int g = 0; g < 16; ++g) {
              uint4 u;
              if constexpr (decltype(wide_type)::value) {
                const float2 x = acc[decltype(first)::value + 2 * g], y = acc[decltype(first)::value + 2 * g + 1];
                u = make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
              } else {
                u = make_uint4(pack16(acc[4 * g].x, acc[4 * g].y, bf16), pack16(acc[4 * g + 1].x, acc[4 * g + 1].y, bf16),
                               pack16(acc[4 * g + 2].x, acc[4 * g + 2].y, bf16), pack16(acc[4 * g + 3].x, acc[4 * g + 3].y, bf16));
              }
              *reinterpret_cast<uint4*>(stg + lane * 256 + ((g ^ (lane & 15)) << 4)) = u;
            }
          };
          auto empty_out = [&](int h) {
            __syncwarp();
            const int n = n0 + h * 64 + lane * per;
            for (int r = 0; r < 32 && row0 + r < p.M; ++r) {
              const uint2 u = *reinterpret_cast<const uint2*>(stg + r * 256 + (((lane >> 1) ^ (r & 15)) << 4) + (lane & 1) * 8);
              uint8_t* dst = static_cast<uint8_t*>(p.out) + (static_cast<int64_t>(row0 + r) * p.N + n) * (f32 ? 4 : 2);
              if (fit == 8) {
                if (n < p.N) *reinterpret_cast<uint2*>(dst) = u;
              } else if (fit == 4) {
                if (n < p.N) *reinterpret_cast<uint32_t*>(dst) = u.x;
                if (n + per / 2 < p.N) *reinterpret_cast<uint32_t*>(dst + 4) = u.y;
              } else {
                const uint32_t w[2] = {u.x, u.y};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (n + k < p.N) reinterpret_cast<uint16_t*>(dst)[k] = static_cast<uint16_t>(w[k >> 1] >> (k & 1) * 16);
              }
            }
            __syncwarp();
          };
          const std::integral_constant<int, 0> front;
          const std::integral_constant<int, 32> back;
          if (f32) {
            fill(std::true_type(), front);
            empty_out(0);
            fill(std::true_type(), back);
            empty_out(1);
          } else {
            fill(std::false_type(), front);
            empty_out(0);
          }
          __syncwarp();
        }
      }
    }
    if (WIDE && p.tma_out) {
      if (lane == 0) bulk_wait_all();
      __syncwarp();
    }
  }

  if (!WIDE && split > 1) {
    // Every CTA of the cluster adds up a share of the rows, in the ranks' order.
    cluster_sync();
    int tm, tn;
    tile_at<WIDE>(cid, p, tm, tn);
    const int rows = min(kTileM, p.M - tm * kTileM), cols = min(kTileN, p.N - tn * kTileN);
    const bool bf16 = p.out_dt == B200K_BF16, vec = p.N % 4 == 0;
    const int n = lane * 4;
    if (!*abort_flag && n < cols) {
      for (int r = static_cast<int>(rank) + split * warp; r < rows; r += split * (C::kThreads / 32)) {
        const float* mine = reinterpret_cast<const float*>(sbase) + r * C::kPartRow + n;
        float4 v[kMaxSplit];
#pragma unroll
        for (int k = 0; k < kMaxSplit; ++k)
          if (k < split) v[k] = ld_cluster4(cluster_addr(mine, k));
        float4 sum = v[0];
#pragma unroll
        for (int k = 1; k < kMaxSplit; ++k)
          if (k < split) {
            sum.x += v[k].x;
            sum.y += v[k].y;
            sum.z += v[k].z;
            sum.w += v[k].w;
          }
        const int64_t at = static_cast<int64_t>(tm * kTileM + r) * p.N + tn * kTileN + n;
        if (vec && p.out_dt == B200K_F32) {
          *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = sum;
        } else if (vec) {
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(pack16(sum.x, sum.y, bf16), pack16(sum.z, sum.w, bf16));
        } else {
          const float x[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < cols) store_scalar(p.out, at + j, p.out_dt, x[j]);
        }
      }
    }
    cluster_sync();  // no CTA leaves while another may read its shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (WIDE) cluster_sync();  // no CTA leaves while the other may still signal its barriers
  if (warp == 2) {
    tc_fence_after();
    if (WIDE) tmem_dealloc_pair(tmem_base, C::kTmemCols);
    else tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

// 2-d map of rows of `inner` elements, `row_bytes` apart; 128-byte swizzle.
bool make_map2(CUtensorMap* map, CUtensorMapDataType dt, const void* ptr, uint64_t inner, uint64_t outer, uint64_t row_bytes,
               uint32_t box_inner, uint32_t box_outer) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {inner, outer};
  const cuuint64_t strides[1] = {row_bytes};
  const cuuint32_t box[2] = {box_inner, box_outer};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, dt, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
int launch(MmParams p, const B200kScaledMmArgs* a, int sms, cudaStream_t st) {
  using C = Cfg8<BN>;
  auto kernel = mm_kernel<BN>;
  static std::atomic<uint64_t> done{0};
  if (!attributes_set(done)) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return B200K_ERR_LAUNCH;
    // the epilogue's registers come out of what the launch has: with fewer, setmaxnreg would wait
    if (C::kWide && fa.numRegs * C::kThreads < kCtlRegs * 128 + kEpiRegs * 256) return B200K_ERR_LAUNCH;
    attributes_done(done);
  }
  CUtensorMap ta, tb, to;
  const uint64_t K = static_cast<uint64_t>(a->K), one_row = (K + 15) / 16 * 16;  // the stride of a single row is never stepped
  constexpr int kTileM = C::kWide ? 256 : BN, kTileN = C::kWide ? BN : 128;
  const int ob = a->out_dtype == B200K_F32 ? 4 : 2;
  if (!make_map2(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->a, K, a->M, a->M == 1 ? one_row : a->a_stride_m, kBlk, C::kWide ? 128 : BN) ||
      !make_map2(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->b, K, a->N, a->N == 1 ? one_row : a->b_stride_n, kBlk, 128))
    return B200K_ERR_LAUNCH;
  std::memset(&to, 0, sizeof(to));
  p.tma_out = C::kWide && a->N * ob % 16 == 0;
  if (p.tma_out && !make_map2(&to, tma_dtype(a->out_dtype), a->out, a->N, a->M, a->N * ob, 128 / ob, 32))
    return B200K_ERR_LAUNCH;
  const int64_t tm = (a->M + kTileM - 1) / kTileM, tn = (a->N + kTileN - 1) / kTileN;
  if (tm * tn > 0x7fffffffLL / kMaxSplit) return B200K_ERR_SHAPE;
  p.tiles_m = static_cast<int32_t>(tm);
  p.tiles_n = static_cast<int32_t>(tn);
  p.num_tiles = static_cast<int32_t>(tm * tn);
  const int cluster = C::kWide ? 2 : p.split;
  const int64_t clusters = !C::kWide && p.split > 1 ? tm * tn : std::min<int64_t>(tm * tn, sms * C::kCtas / cluster);
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, ta, tb, to, p) == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
}

}  // namespace
}  // namespace mm8
}  // namespace b200k

using namespace b200k;

extern "C" int b200k_scaled_mm(const B200kScaledMmArgs* a, void* stream_) {
  if (!a) return B200K_ERR_ARG;
  if (a->M < 0 || a->N < 0 || a->K < 0 || a->M > 0x3fffffff || a->N > 0x3fffffff || a->K > 0x3fffffff) return B200K_ERR_SHAPE;
  if (a->out_dtype != B200K_BF16 && a->out_dtype != B200K_F16 && a->out_dtype != B200K_F32) return B200K_ERR_UNSUPPORTED;
  if ((a->tile != 0 && a->tile != 1 && a->tile != 16 && a->tile != 32 && a->tile != 64 && a->tile != 128) || a->split < 0 ||
      a->split > mm8::kMaxSplit)
    return B200K_ERR_ARG;
  if (a->M == 0 || a->N == 0) return B200K_OK;
  if (!a->out) return B200K_ERR_ARG;
  if (!aligned16(a->out)) return B200K_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream_);
  if (a->K == 0) {  // an empty sum
    const size_t n = static_cast<size_t>(a->M) * a->N * dtype_size(a->out_dtype);
    return cudaMemsetAsync(a->out, 0, n, st) == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
  }
  if (!a->a || !a->b || !a->a_scale || !a->b_scale) return B200K_ERR_ARG;
  if (!aligned16(a->a) || !aligned16(a->b) || (a->M > 1 && (a->a_stride_m < a->K || a->a_stride_m % 16)) ||
      (a->N > 1 && (a->b_stride_n < a->K || a->b_stride_n % 16)))
    return B200K_ERR_ALIGN;
  const int sms = device_sm_count();
  if (sms <= 0) return B200K_ERR_DEVICE;
  mm8::MmParams p;
  std::memset(&p, 0, sizeof(p));
  p.M = static_cast<int32_t>(a->M);
  p.N = static_cast<int32_t>(a->N);
  p.k_blocks = static_cast<int32_t>((a->K + 127) / 128);
  p.sa = a->a_scale;
  p.sa_m = a->a_scale_strides[0];
  p.sa_k = a->a_scale_strides[1];
  p.sa_vec = p.sa_k == 1 && p.sa_m % 4 == 0 && aligned16(p.sa);
  p.sb = a->b_scale;
  p.sb_k = a->b_scale_strides[0];
  p.sb_n = a->b_scale_strides[1];
  p.out = a->out;
  p.out_dt = a->out_dtype;
  p.test_flags = a->test_flags;
  p.status = a->status;
  p.timeout_ns = a->timeout_ns > 0 ? a->timeout_ns : 2000000000ll;
  // tile: 0 the choice below, 1 wide, else the turned tiles' rows of a.  Wide
  // tiles pay once they fill half of the GPU: rows x [4096, 4096] as wide and as
  // turned tiles of 128: 512 (32 pairs) 21.9 and 20.1 us, 1024 (64 pairs) 22.9 and
  // 35.2; 512 x [8192, 8192] 37.7 and 55.5.
  int tile = a->tile;
  p.split = 1;
  if (tile == 0) {
    const int64_t wide = (a->M + 255) / 256 * ((a->N + 255) / 256) * 2;
    tile = a->M > 128 && wide * 2 > sms ? 1 : a->M <= 16 ? 16 : a->M <= 32 ? 32 : a->M <= 64 ? 64 : 128;
  }
  if (tile == 1) return mm8::launch<256>(p, a, sms, st);
  // The split with the least rounds x (blocks of a CTA + what its start and,
  // when split, its join cost, in blocks).  64 rows of [4096, 14336] (112 tiles)
  // with 1, 2 and 4: 22, 18 and 25 us; a row of [8192, 2048] (16 tiles) with 4 and
  // 8: 9.7 and 8.0.  Clusters of 8 CTAs that have an SM each do not all find room
  // at once: 128 rows of [8192, 2048] with 4 and 8: 12.5 and 20.6 us.  Of 16 shapes of 1
  // to 128 rows the choice is within 5 % of the best split in 15; in the other it
  // takes 48 clusters of 3, which do not all find room either: 100 rows of [4096,
  // 6144] 19.5 us, 12.5 with 2.
  const int64_t tiles = (a->M + tile - 1) / tile * ((a->N + 127) / 128), slots = static_cast<int64_t>(sms) * (tile <= 64 ? 2 : 1);
  int64_t best = INT64_MAX;
  for (int split = 1; split <= std::min<int32_t>(tile <= 64 ? mm8::kMaxSplit : 4, p.k_blocks); ++split) {
    const int64_t rounds = split == 1 ? 1 : (tiles * split + slots - 1) / slots;
    const int64_t each = split == 1 ? (tiles + slots - 1) / slots * p.k_blocks : (p.k_blocks + split - 1) / split;
    const int64_t cost = rounds * (each + 6 + (split > 1 ? 2 : 0));
    if (cost < best) {
      best = cost;
      p.split = split;
    }
  }
  if (a->split > 0) p.split = a->split;
  switch (tile) {
    case 16: return mm8::launch<16>(p, a, sms, st);
    case 32: return mm8::launch<32>(p, a, sms, st);
    case 64: return mm8::launch<64>(p, a, sms, st);
    default: return mm8::launch<128>(p, a, sms, st);
  }
}
