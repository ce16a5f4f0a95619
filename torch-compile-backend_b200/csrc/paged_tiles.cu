// The tile kernel of b200k_paged_attention (paged_attention.cu): sequences
// with many query rows (prompts, chunks of prompts) on the tcgen05 tensor
// cores.
//
// A unit is 256 query rows (queries x G heads, packed, of one kv head) as two
// tiles of 128, a step one block of 128 keys of a unit, and the steps of all
// units form one list of which every CTA (one per SM) takes an equal run, so
// causal, ragged and single long prompts balance to one step.  A unit that
// is cut leaves fp32 parts in the workspace; tile_join (called from the
// combine kernel) adds them.
//
// A CTA has 384 threads:
//   warps 0, 1   one MMA issuer each, for query tile 0 and 1:
//                S_t = Q_t K^T (M=128, N=128) into tensor memory, then
//                O_t += P_t V with P_t read from tensor memory;
//   warps 2, 3   loaders: 16-byte cp.async copies of Q, K and V rows into
//                128-byte swizzled tiles, each key by its own page (so any
//                page size), completing on mbarriers;
//   warps 4-11   softmax, one thread a query row: its 128 scores from tensor
//                memory, cap and mask, running maximum and sum in fp32, the
//                probabilities as 16-bit pairs back into the columns the
//                scores came from.
// S_t and P_t share columns: S of the next block is issued when P V of this
// one has completed, and the two tiles' chains overlap each other.
// Every wait is bounded (gemm_kernel.cuh): a timeout sets the status word and
// drains.
#include "gemm_kernel.cuh"
#include "paged.cuh"

namespace b200k {
namespace paged {
namespace {

using gemm::Ctl;
using gemm::smem_u32;

constexpr int kThreads = 384;
constexpr int kLoaders = 64;
constexpr uint32_t kHalfTile = 128 * 128;  // 128 rows of 64 16-bit values: one swizzled column
constexpr float kRescaleLog2 = 8.0f;       // a running maximum may lag by a factor of 256
// setmaxnreg split, as in attention.cu: 128 x 104 + 256 x 200 = 384 x 168
constexpr int kLaunchRegs = 168, kCtlRegs = 104, kSoftmaxRegs = 200;
static_assert(128 * kCtlRegs + 256 * kSoftmaxRegs <= kThreads * kLaunchRegs, "register split exceeds the launch");

template <int D>
struct Layout {
  static constexpr int kStages = D == 128 ? 2 : 4;         // of K and of V
  static constexpr uint32_t kTile = kHalfTile * (D / 64);  // a query tile, or a block of keys or values
  static constexpr uint32_t kOffK = 2 * kTile;
  static constexpr uint32_t kOffV = kOffK + kStages * kTile;
  static constexpr uint32_t kOffBar = kOffV + kStages * kTile;
  static constexpr uint32_t kSmem = 1024 + kOffBar + 256;
  static_assert(kSmem <= 232448 && kSmem > 116 * 1024, "one CTA per SM");
};
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// The barrier's arrival of this thread, when its copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A from tensor memory (16-bit pairs, one row a lane), B from shared memory.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
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
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Ctl& c) {
  const bool ok = gemm::wait_bar(bar, parity, c);
  return __all_sync(0xffffffffu, ok);
}

// A CTA's consecutive steps of one unit.
struct Portion {
  Unit u;
  int kvh;
  int beg, end;       // key blocks of this portion
  int t_beg[2], t_end[2];  // of each tile (empty: a tile without keys here)
  bool whole;         // the unit's every step
  int slot;           // where its part goes: 0 began in an earlier CTA, 1 ends in a later one
};

// Walks the portions of the run [w, w1) of steps.
struct Walk {
  int64_t w, w1;
  int e;              // entry (sequence, 256 rows); its kv heads' units follow one another
  int64_t e_steps;    // steps before entry e
  __device__ __forceinline__ bool next(const Params& p, Portion& o) {
    if (w >= w1) return false;
    for (;;) {
      const int2 bq = p.entries[e];
      o.u = unit_at(p, bq.x, bq.y);
      const int64_t n = o.u.ub1 - o.u.ub0;
      const int64_t in = w - e_steps;
      if (in >= n * p.Hkv) {
        e_steps += n * p.Hkv;
        ++e;
        continue;
      }
      o.kvh = static_cast<int>(in / n);
      const int s0 = static_cast<int>(in - o.kvh * n);
      const int64_t left = w1 - w;
      const int s1 = static_cast<int>(min(n, s0 + left));
      o.beg = o.u.ub0 + s0;
      o.end = o.u.ub0 + s1;
      o.whole = s0 == 0 && s1 == n;
      o.slot = s0 == 0 ? 1 : 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        int lo, hi;
        tile_keys(p, o.u, t, lo, hi);
        o.t_beg[t] = max(o.beg, lo / kBlock);
        o.t_end[t] = hi > 0 ? min(o.end, (hi + kBlock - 1) / kBlock) : o.t_beg[t];
      }
      w += s1 - s0;
      return true;
    }
  }
};

template <bool BF16, int D, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) tiles_kernel(const __grid_constant__ Params p) {
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
  uint64_t* s_full = v_empty + S;  // [2] by tile
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* o_free = o_done + 2;
  uint64_t* drain = o_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* first_entry = reinterpret_cast<int*>(tmem_slot + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t total = p.entry_steps[0], run = p.entry_steps[1];
  const int n_entries = static_cast<int>(p.entry_steps[2]);
  const int64_t* before = p.entry_steps + 3;  // steps before each entry
  Walk walk;
  walk.w = run * blockIdx.x;
  walk.w1 = min(total, walk.w + run);
  if (walk.w >= walk.w1) return;  // the whole CTA
  if (warp == 0) {  // the last entry with before[e] <= w, 32 probes at a time
    int lo = 0, hi = n_entries;
    while (hi - lo > 1) {
      const int stride = (hi - lo + 31) / 32;
      const int at = lo + lane * stride;
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && before[at] <= walk.w);
      lo += (31 - __clz(static_cast<int>(le))) * stride;  // before[lo] <= w: bit 0 is set
      hi = min(hi, lo + stride);
    }
    if (lane == 0) *first_entry = lo;
  }
  if (threadIdx.x == 32) {
    gemm::mbar_init(q_full, kLoaders);
    gemm::mbar_init(q_empty, 2);
    for (int s = 0; s < S; ++s) {
      gemm::mbar_init(&k_full[s], kLoaders);
      gemm::mbar_init(&k_empty[s], 2);
      gemm::mbar_init(&v_full[s], kLoaders);
      gemm::mbar_init(&v_empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      gemm::mbar_init(&s_full[t], 1);
      gemm::mbar_init(&p_full[t], 4);
      gemm::mbar_init(&o_done[t], 1);
      gemm::mbar_init(&o_free[t], 4);
      gemm::mbar_init(&drain[t], 1);
    }
    *abort_flag = 0;
    gemm::fence_mbar_init();
  }
  if (warp == 2) {
    gemm::tmem_alloc(tmem_slot, kTmemCols);
    gemm::tmem_relinquish();
  }
  gemm::tc_fence_before();
  __syncthreads();
  gemm::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  walk.e = *first_entry;
  walk.e_steps = before[walk.e];
  const Ctl ctl{abort_flag, p.status, static_cast<uint64_t>(p.timeout_ns)};
  Portion po;

  if (warp < 4) {
    regs_dec<kCtlRegs>();
    if (warp < 2) {
      // -------------------------------------------------------------- MMA issuers
      if (lane == 0) {
        const int t = warp;
        const uint32_t fmt = BF16 ? 1u : 0u;
        // fp32 accumulators; B of Q K^T K-major, of P V N-major
        const uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kBlock >> 3) << 17) | ((128u >> 4) << 24);
        const uint32_t idesc_pv =
            (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17) | ((128u >> 4) << 24);
        const uint32_t tS = tmem_base + t * 128, tO = tmem_base + kTmemO + t * D;
        int c = 0;      // key blocks passed, over all portions
        int g = 0;      // of them this tile's
        int done = 0;   // portions in which this tile had steps
        bool ok = true;
        for (int li = 0; ok && walk.next(p, po); ++li) {
          bool any = false;
          ok = gemm::wait_bar(q_full, li & 1, ctl);
          for (int j = po.beg; ok && j < po.end; ++j, ++c) {
            const int st = c % S;
            const uint32_t par = (c / S) & 1;
            const bool mine = j >= po.t_beg[t] && j < po.t_end[t];
            if (!(ok = gemm::wait_bar(&k_full[st], par, ctl))) break;
            if (!mine) {
              // not before the block has landed: the arrival belongs to this phase
              gemm::mbar_arrive(&k_empty[st]);
              if (!(ok = gemm::wait_bar(&v_full[st], par, ctl))) break;
              gemm::mbar_arrive(&v_empty[st]);
              continue;
            }
            // P V of the block before has read P, which S overwrites
            if (g > 0 && !(ok = gemm::wait_bar(&o_done[t], (g - 1) & 1, ctl))) break;
            gemm::fence_async_smem();  // the loaders' copies, before the MMA's reads
            gemm::tc_fence_after();
            const uint32_t a0 = smem_u32(sQ) + t * L::kTile, b0 = smem_u32(sK) + st * L::kTile;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t at = (k >> 2) * kHalfTile + (k & 3) * 32;
              gemm::umma_f16(tS, gemm::sw128_desc(a0 + at, 16, 1024), gemm::sw128_desc(b0 + at, 16, 1024), idesc_s,
                             k != 0);
            }
            if (!(t == 0 && g == 0 && (p.test_flags & B200K_PAGED_TEST_WITHHOLD_SCORES))) gemm::umma_commit(&s_full[t]);
            gemm::umma_commit(&k_empty[st]);
            if (j + 1 == po.t_end[t]) gemm::umma_commit(q_empty);
            if (!(ok = gemm::wait_bar(&v_full[st], par, ctl))) break;
            // the epilogue of the portion before has read O
            if (!any && done > 0 && !(ok = gemm::wait_bar(&o_free[t], (done - 1) & 1, ctl))) break;
            if (!(ok = gemm::wait_bar(&p_full[t], g & 1, ctl))) break;
            gemm::fence_async_smem();
            gemm::tc_fence_after();
            const uint32_t v0 = smem_u32(sV) + st * L::kTile;
#pragma unroll
            for (int k = 0; k < kBlock / 16; ++k)
              umma_ts(tO, tS + k * 8, gemm::sw128_desc(v0 + k * 2048, kHalfTile, 1024), idesc_pv, (any || k != 0) ? 1u : 0u);
            gemm::umma_commit(&o_done[t]);
            gemm::umma_commit(&v_empty[st]);
            any = true;
            ++g;
          }
          if (!ok) break;
          if (any) ++done;
          else gemm::mbar_arrive(q_empty);
        }
        // every MMA of this thread completes before tensor memory is freed
        gemm::umma_commit(&drain[t]);
        gemm::wait_bar_drain(&drain[t], 0, 100000000ull);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------------ loaders
      const int lw = warp - 2;
      constexpr int kChunks = D / 8, kRowsPerCp = 32 / kChunks;
      const int ch = lane % kChunks, sub = lane / kChunks;
      const uint32_t half_off = (ch >> 3) * kHalfTile;
      const int cc = ch & 7;
      int c = 0;
      bool ok = true;
      for (int li = 0; ok && walk.next(p, po); ++li) {
        for (int j = po.beg; j < po.end; ++j, ++c) {
          const int st = c % S;
          const uint32_t par = ((c / S) & 1) ^ 1;
          // this lane's keys of the warp's 64: lane and lane + 32
          int64_t off[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            off[i] = key_offset(p, po.u.b, j * kBlock + lw * 64 + i * 32 + lane, po.u.lo, po.u.hi, po.kvh);
          if (!(ok = warp_wait(&k_empty[st], par, ctl))) break;
          const uint32_t dk = smem_u32(sK) + st * L::kTile + half_off, dv = smem_u32(sV) + st * L::kTile + half_off;
#pragma unroll
          for (int i = 0; i < 64 / kRowsPerCp; ++i) {
            const int in = i * kRowsPerCp + sub, row = lw * 64 + in;
            const int64_t o = __shfl_sync(0xffffffffu, off[(i * kRowsPerCp) >> 5], in & 31);
            cp16(dk + row * 128 + ((cc ^ (row & 7)) << 4), p.k + (o >= 0 ? o : 0) + ch * 8, o >= 0);
          }
          cp_arrive(&k_full[st]);
          if (j == po.beg) {
            // the portion's queries, when the products of the one before have read theirs
            if (li > 0 && !(ok = warp_wait(q_empty, (li - 1) & 1, ctl))) break;
#pragma unroll 4
            for (int i = 0; i < 128 / kRowsPerCp; ++i) {
              const int in = lw * 128 + i * kRowsPerCp + sub;  // row of the unit; tile lw
              const int r = po.u.r0 + in;
              const bool real = r < po.u.rows;
              const uint32_t tok = fdiv(static_cast<uint32_t>(real ? r : po.u.r0), p.div_g);
              const int hg = (real ? r : po.u.r0) - tok * p.G;
              const uint16_t* src = p.q + static_cast<int64_t>(po.u.s.t0 + tok) * p.q_t +
                                    static_cast<int64_t>(po.kvh * p.G + hg) * p.q_h + ch * 8;
              cp16(smem_u32(sQ) + lw * L::kTile + half_off + (in & 127) * 128 + ((cc ^ (in & 7)) << 4), src, real);
            }
            cp_arrive(q_full);
          }
          if (!(ok = warp_wait(&v_empty[st], par, ctl))) break;
#pragma unroll
          for (int i = 0; i < 64 / kRowsPerCp; ++i) {
            const int in = i * kRowsPerCp + sub, row = lw * 64 + in;
            const int64_t o = __shfl_sync(0xffffffffu, off[(i * kRowsPerCp) >> 5], in & 31);
            cp16(dv + row * 128 + ((cc ^ (row & 7)) << 4), p.v + (o >= 0 ? o : 0) + ch * 8, o >= 0);
          }
          cp_arrive(&v_full[st]);
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else {
    regs_inc<kSoftmaxRegs>();
    // -------------------------------------------------------------------- softmax
    const int t = (warp - 4) >> 2, quarter = warp & 3;
    const int in_unit = t * 128 + quarter * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t tS = t_lane + t * 128, tO = t_lane + kTmemO + t * D;
    int g = 0;
    bool ok = true;
    while (ok && walk.next(p, po)) {
      const int r = po.u.r0 + in_unit;
      const bool real = r < po.u.rows;
      const uint32_t tok = fdiv(static_cast<uint32_t>(min(r, po.u.rows - 1)), p.div_g);
      const int pos = po.u.s.first + static_cast<int>(tok);
      // positions of the warp's first and last row
      const int w_lo = __shfl_sync(0xffffffffu, pos, 0), w_hi = __shfl_sync(0xffffffffu, pos, 31);
      float m = -INFINITY, l = 0.0f;
      const int jb = po.t_beg[t], je = po.t_end[t];
      for (int j = jb; j < je; ++j, ++g) {
        if (!(ok = warp_wait(&s_full[t], g & 1, ctl))) break;
        gemm::tc_fence_after();
        float s[kBlock];
        {
          uint32_t raw[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) gemm::tmem_ld32(tS + c * 32, raw[c]);
          gemm::tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) s[c * 32 + i] = __uint_as_float(raw[c][i]);
        }
        if (CAP) {
#pragma unroll
          for (int c = 0; c < kBlock; ++c) s[c] = score<true>(p, s[c]);
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
        for (int c = 4; c < kBlock; c += 4)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = fmaxf(mx[i], s[c + i]);
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (!CAP) top *= p.mul;
        float alpha = 1.0f;
        bool moved = false;
        if (top > m + kRescaleLog2 || (m == -INFINITY && top > m)) {
          alpha = ex2(m - top);
          m = top;
          moved = j > jb;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float2 sum2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 sc2 = CAP ? make_float2(1.0f, 1.0f) : make_float2(p.mul, p.mul), nm2 = make_float2(-ref, -ref);
        uint32_t pk[kBlock / 2];
#pragma unroll
        for (int c = 0; c < kBlock; c += 4)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 x = __ffma2_rn(make_float2(s[c + 2 * i], s[c + 2 * i + 1]), sc2, nm2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            sum2[i] = __fadd2_rn(sum2[i], e);
            pk[c / 2 + i] = pack16<BF16>(e.x, e.y);
          }
        l = fmaf(l, alpha, (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
        if (__any_sync(0xffffffffu, moved)) {  // P V of the blocks before is complete: S waited for it
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
        tmem_st32(tS, pk);
        tmem_st32(tS + 32, pk + 32);
        tmem_wait_st();
        gemm::tc_fence_before();
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&p_full[t]);
      }
      if (!ok) break;
      const bool had = je > jb;
      if (had && !(ok = warp_wait(&o_done[t], (g - 1) & 1, ctl))) break;
      gemm::tc_fence_after();
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
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
          uint16_t* dst = p.out + (static_cast<int64_t>(po.u.s.t0 + tok) * p.H + po.kvh * p.G + (r - tok * p.G)) * D + c * 32;
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
  if (warp == 2) {
    gemm::tc_fence_after();
    gemm::tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <bool BF16, int D, bool CAP>
int launch(const Params& p, cudaStream_t st) {
  auto kernel = tiles_kernel<BF16, D, CAP>;
  cudaFuncAttributes fa;
  // The register split is sized for kLaunchRegs a thread at launch; with any
  // other count setmaxnreg.inc could wait for registers that do not exist.
  if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs != kLaunchRegs) return B200K_ERR_UNSUPPORTED;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kSmem) != cudaSuccess)
    return B200K_ERR_LAUNCH;
  kernel<<<p.tile_ctas, kThreads, Layout<D>::kSmem, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
}

}  // namespace

int launch_tiles(const Params& p, bool bf16, int dim, bool cap, cudaStream_t st) {
  if (dim == 64) {
    if (bf16) return cap ? launch<true, 64, true>(p, st) : launch<true, 64, false>(p, st);
    return cap ? launch<false, 64, true>(p, st) : launch<false, 64, false>(p, st);
  }
  if (bf16) return cap ? launch<true, 128, true>(p, st) : launch<true, 128, false>(p, st);
  return cap ? launch<false, 128, true>(p, st) : launch<false, 128, false>(p, st);
}

}  // namespace paged
}  // namespace b200k
