// Product of e4m3 operands with a scale for each block of 128
// (b200k_scaled_mm, include/b200k.h):
//
//   out[m, n] = sum_g sa[m, g] sb[g, n / 128] sum_{k in block g} a[m, k] b[k, n]
//
// No reference counterpart (its GEMM is 16-bit).  The inner sum is a 128-deep
// tcgen05 product (kind::f8f6f4, fp32 accumulators in tensor memory); the
// scales differ from block to block, so it cannot run on over k: each block's
// product goes to one of two tensor-memory buffers, and while the tensor pipe
// fills the other one the epilogue warps read it and add it, times its scale,
// to fp32 sums in registers.  A thread has one row and up to 128 columns of
// one scale block, so a block costs it one scale and 64 packed FMAs.
//
// One CTA per SM:
//   warp 0      TMA producer (128-byte swizzled tiles of 128 k);
//   warp 1      MMA issuer;
//   warp 2      owns tensor memory;
//   warps 4..   epilogue: four for every 128 (or 64) columns.
// Kinds of tile:
//   pair    256 x 256 on a cluster of two CTAs (cta_group::2), each with its
//           own 128 rows: large products, a third less operand traffic than
//           128 x 256;
//   single  128 x 128 or 128 x 64, on a cluster of `split` CTAs that share
//           the blocks of k out among them and add their sums over distributed
//           shared memory in the order of the ranks: few rows, where the
//           weights' bytes are the bound and every SM has to fetch some.
#include "gemm_kernel.cuh"

namespace b200k {
namespace gemm {
// Host helpers defined with the GEMM's host code (gemm_sm100.cu).
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();
CUtensorMapDataType tma_dtype(int dt);
}  // namespace gemm

namespace mm8 {
namespace {

using namespace gemm;

constexpr int kBlk = 128;  // k of a block, one swizzle row of bytes
// Registers of a thread of 256-wide tiles: launched with 168, 128 control
// threads leave theirs to 256 epilogue threads (128 sums each).
constexpr int kCtlRegs = 40, kEpiRegs = 232;

struct MmParams {
  int32_t M, N;
  int32_t tiles_m, tiles_n, num_tiles, k_blocks;
  int32_t group_m;
  int32_t split;            // CTAs that share a tile's blocks (single)
  int32_t a_rows;           // rows of an A box (single)
  int32_t tma_out;          // the output's rows can be stored by TMA
  const float* sa;          // [M, k_blocks]
  int64_t sa_m, sa_k;
  const float* sb;          // [k_blocks, ceil(N / 128)]
  int64_t sb_k, sb_n;
  void* out;                // [M, N] contiguous
  int32_t out_dt;
  int32_t test_flags;
  int32_t* status;
  int64_t timeout_ns;
};

template <bool PAIR, int BN>
struct Cfg8 {
  static constexpr int kGroups = BN == 256 ? 2 : 1;        // column groups, four warps each
  static constexpr int kCols = BN / kGroups;               // of an epilogue thread
  static constexpr int kThreads = 128 + 128 * kGroups;
  static constexpr uint32_t kABytes = 128 * kBlk;
  static constexpr uint32_t kBBytes = (PAIR ? BN / 2 : BN) * kBlk;
  static constexpr uint32_t kStage = kABytes + kBBytes;
  static constexpr int kStages = PAIR ? 6 : BN == 128 ? 6 : 8;
  static constexpr uint32_t kOffStg = kStages * kStage;
  static constexpr uint32_t kOffBar = kOffStg + 4 * kGroups * kStgBytes;
  static constexpr uint32_t kSmem = 1024 + kOffBar + 256;
  static constexpr int kPartStride = BN + 4;               // floats: rows of 16-byte words fall on other banks
  static_assert(kSmem <= 232448 && kSmem > 232448 / 2, "one CTA per SM");
  static_assert(128 * kPartStride * 4 <= kOffStg, "the sums of a split tile fit the ring");
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
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

__device__ __forceinline__ void tile_at(int t, const MmParams& p, int& tm, int& tn) {
  const int per_group = p.group_m * p.tiles_n;
  const int g = t / per_group, first = g * p.group_m;
  const int rows = min(p.tiles_m - first, p.group_m), r = t - g * per_group;
  tm = first + r % rows;
  tn = r / rows;
}

// Scale products of four blocks of k for one row and column block, 0 outside.
struct Scales {
  float s[4];
  __device__ __forceinline__ void load(const MmParams& p, int m, int nb, int kb, int end) {
    const float* a = p.sa + m * p.sa_m + kb * p.sa_k;
    const float* b = p.sb + kb * p.sb_k + nb * p.sb_n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = 0.0f;
      if (kb + i < end && m < p.M) s[i] = __ldg(a + i * p.sa_k) * __ldg(b + i * p.sb_k);
    }
  }
};

template <bool PAIR, int BN>
__global__ void __launch_bounds__(Cfg8<PAIR, BN>::kThreads, 1)
    mm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
              const __grid_constant__ CUtensorMap tmO, const __grid_constant__ MmParams p) {
  using C = Cfg8<PAIR, BN>;
  constexpr int S = C::kStages, COLS = C::kCols;
  constexpr int kTileM = PAIR ? 256 : 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sbase = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint64_t* full = reinterpret_cast<uint64_t*>(sbase + C::kOffBar);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = PAIR || p.split > 1 ? cluster_rank() : 0;
  const int cluster = PAIR ? 2 : p.split;
  const bool leads = !PAIR || rank == 0;  // issues the MMAs
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], (PAIR ? 8 : 4) * C::kGroups);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_map(&tmA);
    prefetch_map(&tmB);
    prefetch_map(&tmO);
  }
  if (warp == 2) {
    if (PAIR) {
      tmem_alloc_pair(tmem_slot, 2 * BN);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, 2 * BN);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (cluster > 1) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const Ctl ctl{abort_flag, p.status, static_cast<uint64_t>(p.timeout_ns)};
  const int cid = static_cast<int>(blockIdx.x) / cluster, ncl = static_cast<int>(gridDim.x) / cluster;
  // this CTA's blocks of k
  const int kb0 = PAIR ? 0 : static_cast<int>(static_cast<int64_t>(p.k_blocks) * rank / p.split);
  const int kb1 = PAIR ? p.k_blocks : static_cast<int>(static_cast<int64_t>(p.k_blocks) * (rank + 1) / p.split);

  if (warp < 4) {
    if (C::kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtlRegs));
    if (warp == 0 && lane == 0) {
      // -------------------------------------------------------------- producer
      int s = 0;
      uint32_t ph = 0;
      int64_t issued = 0;
      bool ok = true;
      const uint32_t tx = PAIR ? 2 * C::kStage : static_cast<uint32_t>(p.a_rows) * kBlk + C::kBBytes;
      for (int t = cid; t < p.num_tiles && ok; t += ncl) {
        int tm, tn;
        tile_at(t, p, tm, tn);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = wait_bar(&empty[s], ph ^ 1u, ctl))) break;
          uint8_t* sa = sbase + s * C::kStage;
          if (PAIR) {
            const uint32_t fb = cluster_addr(&full[s], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[s], tx);
            tma_load_2d_pair(sa, &tmA, fb, kb * kBlk, tm * kTileM + static_cast<int>(rank) * 128);
            tma_load_2d_pair(sa + C::kABytes, &tmB, fb, kb * kBlk, tn * BN + static_cast<int>(rank) * (BN / 2));
          } else {
            mbar_arrive_expect_tx(&full[s], tx);
            tma_load_2d(sa, &tmA, &full[s], kb * kBlk, tm * kTileM);
            tma_load_2d(sa + C::kABytes, &tmB, &full[s], kb * kBlk, tn * BN);
          }
          ++issued;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // every stage that was filled has been read: no load is in flight, and
      // no commit of the leading CTA targets this CTA's barriers any more
      for (int x = 0; x < S; ++x)
        if (issued > x) wait_bar_drain(&empty[x], x < s ? ph : (ph ^ 1u), 100000000ull);
      if (!ok && !PAIR) {  // after a timeout: the loads that no MMA waited for
        for (int64_t k = issued > S ? issued - S : 0; k < issued; ++k)
          wait_bar_drain(&full[k % S], static_cast<uint32_t>((k / S) & 1), 100000000ull);
      }
    } else if (warp == 1 && lane == 0 && leads) {
      // ------------------------------------------------------------ MMA issuer
      // fp32 accumulators, both operands e4m3 (format 0) and K-major
      const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(kTileM >> 4) << 24);
      int s = 0, buf = 0;
      uint32_t ph = 0, bph = 0;
      bool ok = true, first = true;
      for (int t = cid; t < p.num_tiles && ok; t += ncl) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = wait_bar(&full[s], ph, ctl) && wait_bar(&tempty[buf], bph ^ 1u, ctl))) break;
          tc_fence_after();
          const uint64_t da = sw128_desc(smem_u32(sbase + s * C::kStage), 16, 1024);
          const uint64_t db = sw128_desc(smem_u32(sbase + s * C::kStage + C::kABytes), 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (PAIR) umma_f8_pair(tmem_base + buf * BN, da + 2 * k, db + 2 * k, idesc, k != 0);
            else umma_f8(tmem_base + buf * BN, da + 2 * k, db + 2 * k, idesc, k != 0);
          }
          const bool signal = !(first && (p.test_flags & B200K_SCALED_MM_TEST_WITHHOLD_READY));
          first = false;
          if (PAIR) {
            umma_commit_pair(smem_u32(&empty[s]));
            umma_commit_pair(cluster_addr(&empty[s], 1));
            if (signal) {
              umma_commit_pair(smem_u32(&tfull[buf]));
              umma_commit_pair(cluster_addr(&tfull[buf], 1));
            }
          } else {
            umma_commit(&empty[s]);
            if (signal) umma_commit(&tfull[buf]);
          }
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
          buf ^= 1;
          if (buf == 0) bph ^= 1u;
        }
      }
      // every MMA of this thread completes before tensor memory is freed
      if (PAIR) umma_commit_pair(smem_u32(drain));
      else umma_commit(drain);
      wait_bar_drain(drain, 0, 100000000ull);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    if (C::kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
    const int quarter = warp & 3, cg = (warp - 4) >> 2;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + cg * COLS;
    uint8_t* stg = sbase + C::kOffStg + (warp - 4) * kStgBytes;
    const int rank_rows = PAIR ? static_cast<int>(rank) * 128 : 0;
    const bool bf16 = p.out_dt == B200K_BF16;
    int buf = 0;
    uint32_t bph = 0;
    bool ok = true;
    for (int t = cid; t < p.num_tiles && ok; t += ncl) {
      int tm, tn;
      tile_at(t, p, tm, tn);
      const int row0 = tm * kTileM + rank_rows + quarter * 32, m = row0 + lane;
      const int n0 = tn * BN + cg * COLS;
      const int nb = min(n0, p.N - 1) / kBlk;
      const bool any = row0 < p.M && n0 < p.N;  // warp-uniform
      float2 acc[COLS / 2];
#pragma unroll
      for (int i = 0; i < COLS / 2; ++i) acc[i] = make_float2(0.0f, 0.0f);
      Scales next;
      next.load(p, m, nb, kb0, kb1);
      for (int kb = kb0; ok && kb < kb1; kb += 4) {
        const Scales now = next;
        next.load(p, m, nb, kb + 4, kb1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb + i >= kb1) break;
          ok = __all_sync(0xffffffffu, wait_bar(&tfull[buf], bph, ctl));
          if (!ok) break;
          tc_fence_after();
          if (any) {
            const float2 sc = make_float2(now.s[i], now.s[i]);
            uint32_t raw[2][32];
            tmem_ld32(t_row + buf * BN, raw[0]);
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
              tmem_wait_ld_regs(raw[c & 1]);
              if (c + 1 < COLS / 32) tmem_ld32(t_row + buf * BN + (c + 1) * 32, raw[(c + 1) & 1]);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                acc[c * 16 + j] = __ffma2_rn(make_float2(__uint_as_float(raw[c & 1][2 * j]), __uint_as_float(raw[c & 1][2 * j + 1])),
                                             sc, acc[c * 16 + j]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && rank != 0) mbar_arrive_cluster(cluster_addr(&tempty[buf], 0));
            else mbar_arrive(&tempty[buf]);
          }
          buf ^= 1;
          if (buf == 0) bph ^= 1u;
        }
      }
      if (!PAIR && p.split > 1) {
        // every load has landed and been read: the ring holds the sums
        float* part = reinterpret_cast<float*>(sbase) + (quarter * 32 + lane) * C::kPartStride;
        if (ok && any) {
#pragma unroll
          for (int i = 0; i < COLS / 4; ++i)
            reinterpret_cast<float4*>(part)[i] = make_float4(acc[2 * i].x, acc[2 * i].y, acc[2 * i + 1].x, acc[2 * i + 1].y);
        }
        break;  // one tile a cluster; joined below
      }
      if (!ok || !any) continue;
      if (p.tma_out) {
        // staged as rows of 128 bytes, 128-byte swizzle, and stored by TMA
        const bool f32 = p.out_dt == B200K_F32;
#pragma unroll
        for (int h = 0; h < COLS / 32; ++h) {
          if (n0 + h * 32 >= p.N) break;
          const int half = f32 ? 0 : h & 1;
          if (half == 0) {
            if (lane == 0) bulk_wait_read_all();  // the store before has read the rows
            __syncwarp();
          }
          if (f32) {
#pragma unroll
            for (int g = 0; g < 8; ++g)
              *reinterpret_cast<float4*>(stg + lane * 128 + ((g ^ (lane & 7)) << 4)) =
                  make_float4(acc[h * 16 + 2 * g].x, acc[h * 16 + 2 * g].y, acc[h * 16 + 2 * g + 1].x, acc[h * 16 + 2 * g + 1].y);
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2* v = acc + h * 16 + 4 * g;
              *reinterpret_cast<uint4*>(stg + lane * 128 + (((half * 4 + g) ^ (lane & 7)) << 4)) =
                  make_uint4(pack16(v[0].x, v[0].y, bf16), pack16(v[1].x, v[1].y, bf16), pack16(v[2].x, v[2].y, bf16),
                             pack16(v[3].x, v[3].y, bf16));
            }
          }
          if (f32 || half == 1 || n0 + (h + 1) * 32 >= p.N) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmO, stg, n0 + (f32 ? h : h & ~1) * 32, row0);
              bulk_commit();
            }
          }
        }
      } else {
        // rows that TMA cannot store: 32 columns at a time through shared
        // memory (33 floats a row), a warp's lanes on neighbouring columns
        float* tile = reinterpret_cast<float*>(stg);
#pragma unroll
        for (int h = 0; h < COLS / 16; ++h) {
          if (n0 + h * 16 >= p.N) break;
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            tile[lane * 17 + 2 * j] = acc[h * 8 + j].x;
            tile[lane * 17 + 2 * j + 1] = acc[h * 8 + j].y;
          }
          __syncwarp();
          const int n = n0 + h * 16 + (lane & 15);
          for (int r = lane >> 4; r < 32 && row0 + r < p.M; r += 2)
            if (n < p.N) store_scalar(p.out, static_cast<int64_t>(row0 + r) * p.N + n, p.out_dt, tile[r * 17 + (lane & 15)]);
        }
        __syncwarp();
      }
    }
    if (p.tma_out) {
      if (lane == 0) bulk_wait_all();
      __syncwarp();
    }
  }

  if (!PAIR && p.split > 1) {
    // Every CTA of the cluster adds up a share of the rows, in the ranks' order.
    cluster_sync();
    int tm, tn;
    tile_at(cid, p, tm, tn);
    const int rows = min(128, p.M - tm * 128), cols = min(BN, p.N - tn * BN);
    constexpr int kPer = BN / 4;  // threads of a row
    const bool bf16 = p.out_dt == B200K_BF16, vec = p.N % 4 == 0;
    const int c = (threadIdx.x % kPer) * 4;
    if (!*abort_flag && c < cols) {
      for (int r = static_cast<int>(rank) + p.split * static_cast<int>(threadIdx.x / kPer); r < rows;
           r += p.split * (C::kThreads / kPer)) {
        const float* mine = reinterpret_cast<const float*>(sbase) + r * C::kPartStride + c;
        float4 sum = ld_cluster4(cluster_addr(mine, 0));
        for (int k = 1; k < p.split; ++k) {
          const float4 v = ld_cluster4(cluster_addr(mine, k));
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
        const int64_t at = static_cast<int64_t>(tm * 128 + r) * p.N + tn * BN + c;
        if (vec && p.out_dt == B200K_F32) {
          *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = sum;
        } else if (vec) {
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(pack16(sum.x, sum.y, bf16), pack16(sum.z, sum.w, bf16));
        } else {
          const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (c + j < cols) store_scalar(p.out, at + j, p.out_dt, v[j]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (cluster > 1) cluster_sync();  // no CTA leaves while another may signal or read its shared memory
  if (warp == 2) {
    tc_fence_after();
    if (PAIR) tmem_dealloc_pair(tmem_base, 2 * BN);
    else tmem_dealloc(tmem_base, 2 * BN);
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

template <bool PAIR, int BN>
int launch(MmParams p, const B200kScaledMmArgs* a, int sms, cudaStream_t st) {
  using C = Cfg8<PAIR, BN>;
  auto kernel = mm_kernel<PAIR, BN>;
  static std::atomic<uint64_t> done{0};
  if (!attributes_set(done)) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess ||
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
      return B200K_ERR_LAUNCH;
    // the epilogue's registers come out of what the launch has: with fewer, setmaxnreg would wait
    if (C::kGroups == 2 && fa.numRegs * C::kThreads < kCtlRegs * 128 + kEpiRegs * 256) return B200K_ERR_LAUNCH;
    attributes_done(done);
  }
  CUtensorMap ta, tb, to;
  const uint64_t K = static_cast<uint64_t>(a->K);
  p.a_rows = PAIR ? 128 : static_cast<int32_t>(std::min<int64_t>(128, (a->M + 7) / 8 * 8));
  const int ob = a->out_dtype == B200K_F32 ? 4 : 2;
  if (!make_map2(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->a, K, a->M, a->M == 1 ? (K + 15) / 16 * 16 : a->a_stride_m, kBlk, p.a_rows) ||
      !make_map2(&tb, CU_TENSOR_MAP_DATA_TYPE_UINT8, a->b, K, a->N, a->N == 1 ? (K + 15) / 16 * 16 : a->b_stride_n, kBlk,
                 PAIR ? BN / 2 : BN))
    return B200K_ERR_LAUNCH;
  std::memset(&to, 0, sizeof(to));
  p.tma_out = a->N * ob % 16 == 0 && p.split == 1;
  if (p.tma_out && !make_map2(&to, tma_dtype(a->out_dtype), a->out, a->N, a->M, a->N * ob, 128 / ob, 32)) return B200K_ERR_LAUNCH;
  const int tile_m = PAIR ? 256 : 128;
  const int64_t tm = (a->M + tile_m - 1) / tile_m, tn = (a->N + BN - 1) / BN;
  const int cluster = PAIR ? 2 : p.split;
  if (tm * tn * cluster > 0x7fffffffLL) return B200K_ERR_SHAPE;
  p.tiles_m = static_cast<int32_t>(tm);
  p.tiles_n = static_cast<int32_t>(tn);
  p.num_tiles = static_cast<int32_t>(tm * tn);
  p.group_m = PAIR ? kGroupMPair : kGroupM;
  const int64_t clusters = !PAIR && p.split > 1 ? tm * tn : std::min<int64_t>(tm * tn, sms / cluster);
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = static_cast<unsigned>(cluster);
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
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
  if (a->tile < 0 || a->tile > 3 || a->split < 0 || a->split > 8) return B200K_ERR_ARG;
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
  p.sb = a->b_scale;
  p.sb_k = a->b_scale_strides[0];
  p.sb_n = a->b_scale_strides[1];
  p.out = a->out;
  p.out_dt = a->out_dtype;
  p.test_flags = a->test_flags;
  p.status = a->status;
  p.timeout_ns = a->timeout_ns > 0 ? a->timeout_ns : 2000000000ll;
  p.split = 1;
  const int64_t tiles = (a->M + 255) / 256 * ((a->N + 255) / 256);
  if (a->tile == 1 || (a->tile == 0 && a->M > 128 && tiles * 2 >= sms)) return mm8::launch<true, 256>(p, a, sms, st);
  const bool narrow = a->tile == 3 || (a->tile == 0 && a->M <= 128);
  const int64_t single = (a->M + 127) / 128 * ((a->N + (narrow ? 63 : 127)) / (narrow ? 64 : 128));
  int split = 1;
  while (split < 8 && single * split * 2 <= sms && p.k_blocks >= split * 4) split *= 2;
  if (a->split > 0) split = a->split;
  p.split = split;
  return narrow ? mm8::launch<false, 64>(p, a, sms, st) : mm8::launch<false, 128>(p, a, sms, st);
}
