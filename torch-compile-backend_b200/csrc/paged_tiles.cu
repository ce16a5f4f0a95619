// The tile kernel of b200k_paged_attention (paged_attention.cu): sequences
// with many query rows (prompts, chunks of prompts) on the tcgen05 tensor
// cores.
//
// A unit is 256 query rows (queries x G heads, packed, of one kv head) as two
// tiles of 128, a step one block of 64 keys of a unit, and the steps of all
// units form one list of which every CTA (one per SM) takes an equal run, so
// causal, ragged and single long prompts balance to one step.  A unit that
// is cut leaves fp32 parts in the workspace; tile_join (called from the
// combine kernel) adds them.
//
// A CTA has 14 warps:
//   warps 0-7    softmax of tile 0 (0-3) and 1, one thread a query row: its 64
//                scores from tensor memory, cap and mask, running maximum and
//                sum in fp32, the probabilities as 16-bit pairs back into
//                tensor memory;
//   warps 8, 9   issue S_t = Q_t K^T (M=128, N=64) of tile t = 0, 1;
//   warps 10, 11 issue O_t += P_t V, P_t read from tensor memory (one warp
//                for both products spent longer on its waits than a step has);
//   warps 12, 13 loaders, of queries and keys and of values, into 128-byte
//                swizzled tiles: TMA boxes of as many rows as pages and
//                blocks have in common (8 or more), 16-byte cp.async copies
//                where a block reaches past the sequence's keys (those rows
//                become zeros) or the page size has no such box (8 prompts of
//                2048 with copies alone: 356 us, with boxes 277).
// Tensor memory is full (S 2 x 2 x 64, O 2 x 128 columns): a tile's scores
// alternate between two buffers, P takes the columns of its S, and S of the
// next block is computed under this block's exponentials.  With one buffer of
// 128 keys, S, softmax and P V of a tile one after the other, 128 keys with heads
// of 128 took 4400 clocks (now ~3900).
// Measured: 8 prompts of 2048, 32 / 8 heads of 64, causal, 277 us = 497
// TFLOP/s; 5 chunks of 1024 behind up to 6000 keys, heads of 128, 317 us = 828
// TFLOP/s in calls back to back, which lower the clock under the power limit
// (268 us in a short run).  Heads of 64 are bound by the softmax (per block of
// 64 keys ~1750 clocks of one warp's dependent instructions; the exponential
// unit alone ~770).  With heads of 128 the tensor pipe is active 54 % of the
// time: of a block's ~1950 clocks the two products take ~1540 if one with
// N = 64 costs what one with N = 128 does, the rest is waits between them.
// Every wait is bounded (gemm_kernel.cuh): a timeout sets the status word and
// drains.
#include "gemm_kernel.cuh"
#include "paged.cuh"

namespace b200k {
namespace gemm {
// Host helpers defined with the GEMM's host code (gemm_sm100.cu).
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();
CUtensorMapDataType tma_dtype(int dt);
}  // namespace gemm

namespace paged {
namespace {

using gemm::Ctl;
using gemm::smem_u32;

constexpr int kThreads = 448;
constexpr int kLoaders = 64;               // threads that arrive for a query tile; 32 for a key or value block
constexpr uint32_t kHalfTile = 128 * 128;  // 128 rows of 64 16-bit values: one swizzled column
constexpr uint32_t kHalfBlk = kBlock * 128;
// Of so many probabilities two are computed on the FMA pipe.  8 prompts of
// 2048 (32 heads of 64): 277 us, 291 with none, 286 with half of them.
constexpr int kFmaEvery = 8;
template <int D>
struct Layout {
  static constexpr int kStages = D == 128 ? 4 : 6;         // of K and of V
  static constexpr uint32_t kTile = kHalfTile * (D / 64);  // a query tile
  static constexpr uint32_t kBlk = kHalfBlk * (D / 64);    // a block of keys or values
  static constexpr uint32_t kOffK = 2 * kTile;
  static constexpr uint32_t kOffV = kOffK + kStages * kBlk;
  static constexpr uint32_t kOffBar = kOffV + kStages * kBlk;
  static constexpr uint32_t kSmem = 1024 + kOffBar + 512;
  static_assert(kSmem <= 232448 && kSmem > 116 * 1024, "one CTA per SM");
};
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;
// Tensor-memory columns: scores of block g of tile t at 128 t + 64 (g & 1),
// its probabilities in the first 32 of them, O_t at 256 + D t.

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// The barrier's arrival of this thread, when its copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The products and commits below are called by whole warps and issued by one
// elected lane: in warp-uniform code the descriptors stay in uniform
// registers (issued from a lane's branch, an MMA took ~120 clocks to issue).
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A from tensor memory (16-bit pairs, one row a lane), B from shared memory.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// NaN if any of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^x on the FMA pipe, for a share of the probabilities: the special-function
// unit's 16 a clock bound a step otherwise.  x = n + f with n the nearest
// integer (read off the low bits of x + 1.5 * 2^23), 2^f on [-1/2, 1/2] by
// the polynomial of least relative error (Remez exchange; 7.5e-5 in degree 3
// for bf16 probabilities, 2.6e-6 in degree 4 for f16: below half a step of
// the type), n added to the exponent.  x below -125 gives 2^-125; x is not NaN
// unless the row's maximum is.
template <bool BF16>
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  x.x = fmaxf(x.x, -125.0f);
  x.y = fmaxf(x.y, -125.0f);
  const float big = 12582912.0f;
  const float2 t = __fadd2_rn(x, make_float2(big, big));
  const float2 n = __fadd2_rn(t, make_float2(-big, -big));
  const float2 f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);
  auto both = [](float c) { return make_float2(c, c); };
  float2 r;
  if (BF16) {
    r = __ffma2_rn(both(0.05517167f), f, both(0.24261112f));
    r = __ffma2_rn(r, f, both(0.69326099f));
    r = __ffma2_rn(r, f, both(0.99992807f));
  } else {
    r = __ffma2_rn(both(0.0095701f), f, both(0.05591786f));
    r = __ffma2_rn(r, f, both(0.24024745f));
    r = __ffma2_rn(r, f, both(0.69312181f));
    r = __ffma2_rn(r, f, both(0.99999926f));
  }
  return make_float2(__int_as_float(__float_as_int(r.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(r.y) + (__float_as_int(t.y) << 23)));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Ctl& c) {
  const bool ok = gemm::wait_bar(bar, parity, c);
  return __all_sync(0xffffffffu, ok);
}

// A CTA's consecutive steps of one unit (Walk::u until the next one).
struct Portion {
  int kvh;
  int beg, end;       // key blocks of this portion
  int t_beg[2], t_end[2];  // of each tile (empty: a tile without keys here)
  bool whole;         // the unit's every step
  int slot;           // where its part goes: 0 began in an earlier CTA, 1 ends in a later one
};

// Walks the portions of a CTA's run.
struct Walk {
  int64_t left;    // positions of the list that remain
  int e, kvh, in;  // entry (sequence, 256 rows), kv head, position in its unit
  bool fresh;      // entry e is not loaded
  Unit u;
  __device__ __forceinline__ bool next(const Params& p, Portion& o) {
    while (left > 0) {
      if (fresh) {
        const int2 bq = p.entries[e];
        u = unit_at(p, bq.x, bq.y);
        fresh = false;
      }
      const int n = u.ub1 - u.ub0, len = n + kPortionCost;
      const int take = static_cast<int>(min(left, static_cast<int64_t>(len - in)));
      const int s0 = max(0, in - kPortionCost), s1 = max(0, in + take - kPortionCost);
      left -= take;
      o.kvh = kvh;
      if (s1 > s0) {
        o.beg = u.ub0 + s0;
        o.end = u.ub0 + s1;
        o.whole = s0 == 0 && s1 == n;
        o.slot = s0 == 0 ? 1 : 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          int lo, hi;
          tile_keys(p, u, t, lo, hi);
          o.t_beg[t] = max(o.beg, lo / kBlock);
          o.t_end[t] = hi > 0 ? min(o.end, (hi + kBlock - 1) / kBlock) : o.t_beg[t];
        }
      }
      in += take;
      if (in == len) {
        in = 0;
        if (++kvh == p.Hkv) {
          kvh = 0;
          ++e;
          fresh = true;
        }
      }
      if (s1 > s0) return true;
    }
    return false;
  }
};

template <bool BF16, int D, int CAP>
__global__ void __launch_bounds__(kThreads, 1)
    tiles_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap tm_q,
                 const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using L = Layout<D>;
  constexpr int S = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sbase = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint8_t* sQ = sbase;
  uint8_t* sK = sbase + L::kOffK;
  uint8_t* sV = sbase + L::kOffV;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sbase + L::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + S;
  uint64_t* v_full = k_empty + S;
  uint64_t* v_empty = v_full + S;
  uint64_t* s_full = v_empty + S;  // [4] by tile and buffer
  uint64_t* p_full = s_full + 4;   // [4]
  uint64_t* o_done = p_full + 4;   // [4]
  uint64_t* o_free = o_done + 4;   // [2] by tile
  uint64_t* drain = o_free + 2;    // [4] by issuer
  int* copied = reinterpret_cast<int*>(drain + 4);  // [S] of K, [S] of V: the stage's block came by cp.async
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(copied + 2 * S);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* first_entry = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the plan
  const int64_t total = p.entry_steps[0], run = p.entry_steps[1];
  const int n_entries = static_cast<int>(p.entry_steps[2]);
  const int64_t* before = p.entry_steps + 3;  // list positions before each entry
  const int64_t w0 = run * blockIdx.x;
  if (w0 >= total) return;  // the whole CTA
  if (warp == 0) {  // the last entry with before[e] <= w0, 32 probes at a time
    int lo = 0, hi = n_entries;
    while (hi - lo > 1) {
      const int stride = (hi - lo + 31) / 32;
      const int at = lo + lane * stride;
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && before[at] <= w0);
      lo += (31 - __clz(static_cast<int>(le))) * stride;  // before[lo] <= w0: bit 0 is set
      hi = min(hi, lo + stride);
    }
    if (lane == 0) *first_entry = lo;
  }
  if (threadIdx.x == 256) {
    gemm::mbar_init(q_full, kLoaders);
    gemm::mbar_init(q_empty, 2);
    for (int s = 0; s < S; ++s) {
      gemm::mbar_init(&k_full[s], 32);
      gemm::mbar_init(&k_empty[s], 2);
      gemm::mbar_init(&v_full[s], 32);
      gemm::mbar_init(&v_empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      for (int i = 0; i < 2; ++i) {
        gemm::mbar_init(&s_full[t * 2 + i], 1);
        gemm::mbar_init(&p_full[t * 2 + i], 4);
        gemm::mbar_init(&o_done[t * 2 + i], 1);
        gemm::mbar_init(&drain[t * 2 + i], 1);
      }
      gemm::mbar_init(&o_free[t], 4);
    }
    *abort_flag = 0;
    gemm::fence_mbar_init();
  }
  if (warp == 12) {
    gemm::tmem_alloc(tmem_slot, kTmemCols);
    gemm::tmem_relinquish();
  }
  gemm::tc_fence_before();
  __syncthreads();
  gemm::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  Walk walk;
  walk.left = min(run, total - w0);
  walk.e = *first_entry;
  walk.fresh = false;
  {
    const int2 bq = p.entries[walk.e];
    walk.u = unit_at(p, bq.x, bq.y);
    const int64_t in = w0 - before[walk.e];
    const int len = walk.u.ub1 - walk.u.ub0 + kPortionCost;
    walk.kvh = static_cast<int>(in / len);
    walk.in = static_cast<int>(in - static_cast<int64_t>(walk.kvh) * len);
  }
  const Ctl ctl{abort_flag, p.status, static_cast<uint64_t>(p.timeout_ns)};
  Portion po;

  if (warp >= 8 && warp < 12) {
    // ---------------------------------------------------------------- MMA issuers
    const int t = warp & 1;
    const bool scores = warp < 10;
    const uint32_t fmt = BF16 ? 1u : 0u;
    // fp32 accumulators; B of Q K^T K-major, of P V N-major
    const uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kBlock >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t idesc_pv =
        (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t tS = tmem_base + t * 128, tO = tmem_base + kTmemO + t * D;
    const uint64_t dq = gemm::sw128_desc(smem_u32(sQ) + t * L::kTile, 16, 1024);
    const uint64_t dk = gemm::sw128_desc(smem_u32(sK), 16, 1024);
    const uint64_t dv = gemm::sw128_desc(smem_u32(sV), kHalfBlk, 1024);
    uint64_t* full = scores ? k_full : v_full;
    uint64_t* empty = scores ? k_empty : v_empty;
    const volatile int* by_copy = scores ? copied : copied + S;
    int c = 0;      // key blocks passed, over all portions
    int g = 0;      // of them this tile's
    int done = 0;   // portions in which this tile had steps
    bool ok = true;
    for (int li = 0; ok && walk.next(p, po); ++li) {
      if (scores) {
        ok = warp_wait(q_full, li & 1, ctl);
        if (p.q_box == 0) gemm::fence_async_smem();
      }
      for (int j = po.beg; ok && j < po.end; ++j, ++c) {
        const int st = c % S;
        if (!(ok = warp_wait(&full[st], (c / S) & 1, ctl))) break;
        if (j < po.t_beg[t] || j >= po.t_end[t]) {
          // not a block of this tile (the arrival follows the landing, so it
          // belongs to this phase)
          if (lane == 0) gemm::mbar_arrive(&empty[st]);
          __syncwarp();
          continue;
        }
        if (by_copy[st]) gemm::fence_async_smem();  // cp.async's writes, before the MMA's reads
        const int buf = g & 1;
        if (scores) {
          // P V of the block two before has read P from this buffer
          if (g > 1 && !(ok = warp_wait(&o_done[t * 2 + buf], ((g >> 1) - 1) & 1, ctl))) break;
          gemm::tc_fence_after();
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_ss(tS + buf * 64, dq + (((k >> 2) * kHalfTile + (k & 3) * 32) >> 4),
                    dk + ((st * L::kBlk + (k >> 2) * kHalfBlk + (k & 3) * 32) >> 4), idesc_s, k != 0);
          if (!(t == 0 && g == 0 && (p.test_flags & B200K_PAGED_TEST_WITHHOLD_SCORES))) commit(&s_full[t * 2 + buf]);
          commit(&k_empty[st]);
          if (j + 1 == po.t_end[t]) commit(q_empty);
        } else {
          const bool first = j == po.t_beg[t];
          // the epilogue of the portion before has read O
          if (first && done > 0 && !(ok = warp_wait(&o_free[t], (done - 1) & 1, ctl))) break;
          if (!(ok = warp_wait(&p_full[t * 2 + buf], (g >> 1) & 1, ctl))) break;
          gemm::tc_fence_after();
#pragma unroll
          for (int k = 0; k < kBlock / 16; ++k)
            umma_ts(tO, tS + buf * 64 + k * 8, dv + ((st * L::kBlk + k * 2048) >> 4), idesc_pv, (!first || k != 0) ? 1u : 0u);
          commit(&o_done[t * 2 + buf]);
          commit(&v_empty[st]);
        }
        ++g;
      }
      if (!ok) break;
      if (po.t_end[t] > po.t_beg[t]) ++done;
      else if (scores && lane == 0) gemm::mbar_arrive(q_empty);
      __syncwarp();
    }
    // every MMA of this warp completes before tensor memory is freed
    commit(&drain[warp - 8]);
    gemm::wait_bar_drain(&drain[warp - 8], 0, 100000000ull);
    __syncwarp();
  } else if (warp >= 12) {
      // ------------------------------------------------------------------ loaders
      // warp 12: keys and the queries of tile 0; warp 13: values and tile 1
      const bool is_v = warp == 13;
      constexpr int kChunks = D / 8, kRowsPerCp = 32 / kChunks;
      const int ch = lane % kChunks, sub = lane / kChunks;
      const uint32_t half_off = (ch >> 3) * kHalfTile;
      const int cc = ch & 7;
      const uint32_t ring = smem_u32(is_v ? sV : sK);
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      volatile int* by_copy = is_v ? copied + S : copied;
      const uint16_t* cache = is_v ? p.v : p.k;
      const CUtensorMap* map = is_v ? &tm_v : &tm_k;
      const int box = p.box_rows;                          // 0: no TMA
      const int boxes = box > 0 ? kBlock / box : 0;        // of one 64-element half
      int c = 0;
      bool ok = true;
      for (int li = 0; ok && walk.next(p, po); ++li) {
        const Unit& u = walk.u;
        for (int j = po.beg; j < po.end; ++j, ++c) {
          const int st = c % S;
          const uint32_t par = ((c / S) & 1) ^ 1;
          const uint32_t dst = ring + st * L::kBlk;
          const int key0 = j * kBlock;
          bool tma = box > 0 && key0 >= u.s.lo && key0 + kBlock <= u.s.n;  // every row of the block is a key
          int page = 0, in_page = 0;
          if (tma) {
            const int key = key0 + (lane % max(1, boxes)) * box;
            const uint32_t pi = fdiv(static_cast<uint32_t>(key), p.div_page);
            in_page = key - static_cast<int>(pi) * p.page_size;
            page = __ldg(p.table + u.b * p.table_stride + pi);
            tma = __all_sync(0xffffffffu, page >= 0 && page < p.num_pages);
          }
          int64_t off[kBlock / 32];
          if (!tma) {
            // this lane's keys of the block: lane, lane + 32, ...
#pragma unroll
            for (int i = 0; i < kBlock / 32; ++i) off[i] = key_offset(p, u.b, key0 + i * 32 + lane, u.s.lo, u.s.n, po.kvh);
          }
          if (!(ok = warp_wait(&empty[st], par, ctl))) break;
          if (lane == 0) by_copy[st] = tma ? 0 : 1;
          __syncwarp();  // before this warp's arrivals
          if (tma) {
            // a lane per box (8 of 8 rows, fewer of more), for each half
            if (lane < boxes) {
              gemm::mbar_arrive_expect_tx(&full[st], box * D * 2);
#pragma unroll
              for (int h = 0; h < D / 64; ++h)
                tma_load_4d(dst + h * kHalfBlk + lane * box * 128, map, &full[st], h * 64, in_page, po.kvh, page);
            } else {
              gemm::mbar_arrive(&full[st]);
            }
            __syncwarp();
          } else {
#pragma unroll
            for (int part = 0; part < kBlock / 32; ++part)
#pragma unroll 2
              for (int i = 0; i < 32; i += kRowsPerCp) {
                const int row = part * 32 + i + sub;
                const int64_t o = __shfl_sync(0xffffffffu, off[part], i + sub);
                cp16(dst + (ch >> 3) * kHalfBlk + row * 128 + ((cc ^ (row & 7)) << 4), cache + (o >= 0 ? o : 0) + ch * 8, o >= 0);
              }
            cp_arrive(&full[st]);
          }
          if (j == po.beg) {
            // the portion's queries, when the products of the one before have read theirs
            if (li > 0 && !(ok = warp_wait(q_empty, (li - 1) & 1, ctl))) break;
            if (p.q_box > 0) {
              // tiles of 128 / G tokens
              const int t = is_v ? 1 : 0, r0 = u.r0 + t * 128;
              if (lane < D / 64 && r0 < u.rows) {
                gemm::mbar_arrive_expect_tx(q_full, kHalfTile);
                tma_load_4d(smem_u32(sQ) + t * L::kTile + lane * kHalfTile, &tm_q, q_full, lane * 64, 0, po.kvh,
                            u.s.t0 + static_cast<int>(fdiv(static_cast<uint32_t>(r0), p.div_g)));
              } else {
                gemm::mbar_arrive(q_full);
              }
              __syncwarp();
            } else {
              const int t = is_v ? 1 : 0;
#pragma unroll 4
              for (int i = 0; i < 128 / kRowsPerCp; ++i) {
                const int in = i * kRowsPerCp + sub;  // row of the tile
                const int r = u.r0 + t * 128 + in;
                const bool real = r < u.rows;
                const uint32_t tok = fdiv(static_cast<uint32_t>(real ? r : u.r0), p.div_g);
                const int hg = (real ? r : u.r0) - tok * p.G;
                const uint16_t* src = p.q + static_cast<int64_t>(u.s.t0 + tok) * p.q_t +
                                      static_cast<int64_t>(po.kvh * p.G + hg) * p.q_h + ch * 8;
                cp16(smem_u32(sQ) + t * L::kTile + half_off + in * 128 + ((cc ^ (in & 7)) << 4), src, real);
              }
              cp_arrive(q_full);
            }
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      // The last TMA boxes have landed when the issuers are done with them;
      // after a timeout they are waited for here.
      if (!ok) {
        for (int k = max(0, c - S); k < c; ++k) gemm::wait_bar_drain(&full[k % S], (k / S) & 1, 100000000ull);
      }
      __syncwarp();
  } else {
    // -------------------------------------------------------------------- softmax
    const int t = warp >> 2, quarter = warp & 3;
    const int in_unit = t * 128 + quarter * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t tS = t_lane + t * 128, tO = t_lane + kTmemO + t * D;
    int g = 0;
    bool ok = true;
    while (ok && walk.next(p, po)) {
      if (!po.whole && po.slot == 1 && threadIdx.x == 0) {
        // the run's last unit goes on in the next CTAs, the steps that are left at `run` each
        const int left = walk.u.ub1 - po.end;
        p.joins[blockIdx.x] = Join{static_cast<int>(blockIdx.x + (left + run - 1) / run), walk.u.s.t0, po.kvh, walk.u.r0,
                                   walk.u.rows};
      }
      const int r = walk.u.r0 + in_unit;
      const bool real = r < walk.u.rows;
      const uint32_t tok = fdiv(static_cast<uint32_t>(min(r, walk.u.rows - 1)), p.div_g);
      const int pos = walk.u.s.first + static_cast<int>(tok);
      // positions of the warp's first and last row
      const int w_lo = __shfl_sync(0xffffffffu, pos, 0), w_hi = __shfl_sync(0xffffffffu, pos, 31);
      float m = -INFINITY, l = 0.0f;
      const int jb = po.t_beg[t], je = po.t_end[t];
      for (int j = jb; j < je; ++j, ++g) {
        const uint32_t buf = g & 1;
        if (!(ok = warp_wait(&s_full[t * 2 + buf], (g >> 1) & 1, ctl))) break;
        gemm::tc_fence_after();
        float s[kBlock];
        {
          uint32_t raw[kBlock / 32][32];
#pragma unroll
          for (int c = 0; c < kBlock / 32; ++c) gemm::tmem_ld32(tS + buf * 64 + c * 32, raw[c]);
          gemm::tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < kBlock / 32; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) s[c * 32 + i] = __uint_as_float(raw[c][i]);
        }
        if (CAP != kNoCap) {
#pragma unroll
          for (int c = 0; c < kBlock; ++c) s[c] = score<CAP>(p, s[c]);
        }
        const int key0 = j * kBlock;
        if (key0 + kBlock - 1 > w_lo || (p.window > 0 && key0 <= w_hi - p.window)) {  // warp-uniform
          const int hi = pos - key0, lo = p.window > 0 ? hi - p.window : -1;
#pragma unroll
          for (int c = 0; c < kBlock; ++c)
            if (c > hi || c <= lo) s[c] = -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c + 8 <= kBlock; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], s[c + i], s[c + 4 + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max2(mx[i], s[kBlock - 4 + i]);
        float top = max2(max3(mx[0], mx[1], mx[2]), mx[3]);
        if (CAP == kNoCap) top *= p.mul;
        const float was = m;
        float alpha = 1.0f;
        bool moved = false;
        // A NaN score, and an infinite one (0 * top), makes the maximum NaN and
        // with it every probability and sum of the row from here on.
        if (!(top <= m + kTileLag<BF16>)) {
          m = fmaf(0.0f, top, top);
          alpha = ex2(was - m);
          moved = j > jb;
        }
        // probabilities are rounded to the input type, half a step each, in f16
        // down to 2^-26 of the row's maximum (smaller ones by less than 2^-36 of it)
        const float ref = (m == -INFINITY ? 0.0f : m) - kTileReach<BF16>;
        float2 sum2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 sc2 = CAP != kNoCap ? make_float2(1.0f, 1.0f) : make_float2(p.mul, p.mul), nm2 = make_float2(-ref, -ref);
        uint32_t pk[kBlock / 2];
#pragma unroll
        for (int c = 0; c < kBlock; c += 2) {
          const float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), sc2, nm2);
          const float2 e = c % kFmaEvery == kFmaEvery - 2 ? ex2_fma<BF16>(x) : make_float2(ex2(x.x), ex2(x.y));
          sum2[c / 2 % 2] = __fadd2_rn(sum2[c / 2 % 2], e);
          pk[c / 2] = pack16<BF16>(e.x, e.y);
        }
        l = fmaf(l, alpha, (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
        if (__any_sync(0xffffffffu, moved)) {
          // P V of the block before has written O
          if (!(ok = warp_wait(&o_done[t * 2 + (buf ^ 1)], ((g - 1) >> 1) & 1, ctl))) break;
          gemm::tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            gemm::tmem_ld32(tO + c * 32, o);
            gemm::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
        tmem_st32(tS + buf * 64, pk);
        tmem_wait_st();
        gemm::tc_fence_before();
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&p_full[t * 2 + buf]);
      }
      if (!ok) break;
      const bool had = je > jb;
      if (had && !(ok = warp_wait(&o_done[t * 2 + ((g - 1) & 1)], ((g - 1) >> 1) & 1, ctl))) break;
      gemm::tc_fence_after();
      // a row without keys has m = -inf (and l the sum of its 2^-125)
      const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
      const int64_t part = static_cast<int64_t>(blockIdx.x) * 2 + po.slot;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (had) {
          gemm::tmem_ld32(tO + c * 32, o);
          gemm::tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (real && po.whole) {
          uint16_t* dst = p.out + (static_cast<int64_t>(walk.u.s.t0 + tok) * p.H + po.kvh * p.G + (r - tok * p.G)) * D + c * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 u;
            u.x = pack16<BF16>(__uint_as_float(o[i * 8 + 0]) * inv, __uint_as_float(o[i * 8 + 1]) * inv);
            u.y = pack16<BF16>(__uint_as_float(o[i * 8 + 2]) * inv, __uint_as_float(o[i * 8 + 3]) * inv);
            u.z = pack16<BF16>(__uint_as_float(o[i * 8 + 4]) * inv, __uint_as_float(o[i * 8 + 5]) * inv);
            u.w = pack16<BF16>(__uint_as_float(o[i * 8 + 6]) * inv, __uint_as_float(o[i * 8 + 7]) * inv);
            reinterpret_cast<uint4*>(dst)[i] = u;
          }
        } else if (real) {
          // [4 columns][256 rows]: a warp's rows side by side
#pragma unroll
          for (int i = 0; i < 8; ++i)
            reinterpret_cast<uint4*>(p.tile_o)[(part * (D / 4) + c * 8 + i) * kUnitRows + in_unit] =
                make_uint4(o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]);
        }
        __syncwarp();  // the next load is warp-collective
      }
      if (had) {
        gemm::tc_fence_before();
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&o_free[t]);
      }
      if (!po.whole && real)
        reinterpret_cast<float2*>(p.tile_ml)[part * kUnitRows + in_unit] = make_float2(m, l);
    }
  }

  gemm::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    gemm::tc_fence_after();
    gemm::tmem_dealloc(tmem_base, kTmemCols);
  }
}

// [64 elements, rows, 1, 1] boxes of a 4-d view, inner dim first.
bool make_map(CUtensorMap* map, bool bf16, const void* ptr, const int64_t (&sizes)[4], const int64_t (&strides)[3],
              const cuuint32_t (&box)[4]) {
  auto fn = gemm::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4], gstr[3];
  uint64_t natural = static_cast<uint64_t>(sizes[0]) * 2;
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(sizes[i]);
  for (int i = 0; i < 3; ++i) {  // the stride of a dim of one is never stepped: give it a legal value
    gstr[i] = sizes[i + 1] == 1 ? natural : static_cast<uint64_t>(strides[i]) * 2;
    natural = std::max<uint64_t>(natural, gstr[i]);
    if (gstr[i] == 0 || gstr[i] >= (1ull << 40)) return false;
  }
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, gemm::tma_dtype(bf16 ? B200K_BF16 : B200K_F16), 4, const_cast<void*>(ptr), dims, gstr, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, int D, int CAP>
int launch(Params p, cudaStream_t st) {
  auto kernel = tiles_kernel<BF16, D, CAP>;
  static std::atomic<uint64_t> done{0};
  if (!attributes_set(done)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kSmem) != cudaSuccess)
      return B200K_ERR_LAUNCH;
    attributes_done(done);
  }
  // Boxes of the rows that lie together in a page and in a block: the largest
  // power of two, 8 to 64, that divides the page size.
  CUtensorMap tq, tk, tv;
  std::memset(&tq, 0, sizeof(tq));
  tk = tv = tq;
  p.box_rows = 0;
  const int both = p.page_size & -p.page_size;
  const int rows = std::min(both, kBlock);
  if (rows >= 8) {
    const int64_t sizes[4] = {D, p.page_size, p.Hkv, p.num_pages}, strides[3] = {p.c_slot, p.c_head, p.c_page};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1};
    if (make_map(&tk, BF16, p.k, sizes, strides, box) && make_map(&tv, BF16, p.v, sizes, strides, box)) p.box_rows = rows;
  }
  p.q_box = 0;
  if (p.G <= 128 && (p.G & (p.G - 1)) == 0) {  // a tile is whole tokens
    const int64_t sizes[4] = {D, p.G, p.Hkv, p.T}, strides[3] = {p.q_h, p.q_h * p.G, p.q_t};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(p.G), 1, static_cast<cuuint32_t>(128 / p.G)};
    if (make_map(&tq, BF16, p.q, sizes, strides, box)) p.q_box = 1;
  }
  // launched under the row kernel's end, as the combine kernel is
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(p.tile_ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<D>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, tq, tk, tv) == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
}

template <bool BF16, int D>
int launch_cap(const Params& p, int cap, cudaStream_t st) {
  if (cap == kNoCap) return launch<BF16, D, kNoCap>(p, st);
  return cap == kCapPlain ? launch<BF16, D, kCapPlain>(p, st) : launch<BF16, D, kCapSeries>(p, st);
}

}  // namespace

int launch_tiles(const Params& p, bool bf16, int dim, int cap, cudaStream_t st) {
  if (dim == 64) return bf16 ? launch_cap<true, 64>(p, cap, st) : launch_cap<false, 64>(p, cap, st);
  return bf16 ? launch_cap<true, 128>(p, cap, st) : launch_cap<false, 128>(p, cap, st);
}

}  // namespace paged
}  // namespace b200k
