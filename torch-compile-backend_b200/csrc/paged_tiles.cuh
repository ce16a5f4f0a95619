// What the tile kernels of b200k_paged_attention (paged_tiles.cu) and
// b200k_paged_attention_quant (paged_tiles8.cu) share: instruction wrappers,
// the walk over a CTA's part of the list, tensor maps.
#pragma once

#include "gemm_kernel.cuh"
#include "paged.cuh"

namespace b200k {
namespace paged {
namespace {

using gemm::Ctl;
using gemm::smem_u32;

constexpr uint32_t kHalfTile = 128 * 128;  // 128 rows of 64 16-bit values: one swizzled column
constexpr uint32_t kHalfBlk = kBlock * 128;
// Of so many probabilities two are computed on the FMA pipe.  8 prompts of
// 2048 (32 heads of 64): 277 us, 291 with none, 286 with half of them.
constexpr int kFmaEvery = 8;

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
// the type), n added to the exponent.  x below -125 gives 2^-125, with ZERO 0 (x from
// -250 on, whose exponents come out as negative integers); x is not NaN unless the
// row's maximum is.
template <bool BF16, bool ZERO>
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  constexpr float kLeast = ZERO ? -250.0f : -125.0f;
  x.x = fmaxf(x.x, kLeast);
  x.y = fmaxf(x.y, kLeast);
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
  int a = __float_as_int(r.x) + (__float_as_int(t.x) << 23), b = __float_as_int(r.y) + (__float_as_int(t.y) << 23);
  if (ZERO) {
    a = max(a, 0);
    b = max(b, 0);
  }
  return make_float2(__int_as_float(a), __int_as_float(b));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Ctl& c) {
  const bool ok = gemm::wait_bar(bar, parity, c);
  return __all_sync(0xffffffffu, ok);
}

// The same for a phase that has nearly always completed: tested first.
__device__ __forceinline__ bool warp_test_wait(uint64_t* bar, uint32_t parity, const Ctl& c) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, done) || warp_wait(bar, parity, c);
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

constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;
// Tensor-memory columns: scores of block g of tile t at 128 t + 64 (g & 1),
// its probabilities in the first 32 of them, O_t at 256 + D t.

// What the roles of a CTA share: barriers, and 16-bit tiles in shared memory.
struct Shared {
  uint64_t *q_full, *q_empty;
  uint64_t *k_full, *k_empty, *v_full, *v_empty;  // [stages]
  uint64_t *s_full, *p_full, *o_done;             // [4] by tile and buffer
  uint64_t *o_free;                               // [2] by tile
  uint64_t *drain;                                // [4] by issuer
  uint8_t *sQ, *sK, *sV;
  const volatile int* copied;                     // [2 stages] of K, of V: the stage's block came by cp.async
  // over e4m3 caches (paged_tiles8.cu)
  uint64_t *sc_full, *sc_empty;                   // [kScaleSlots] by block
  const float* sc;                                // [kScaleSlots][kScaleFloats]: 64 keys' ks, log2 vs, 1 / vs
};
// ks: times the scores' factor, except under a cap
constexpr int kScaleSlots = 8, kScaleFloats = 3 * kBlock;

// The MMA issuers: warps 8, 9 of S_t = Q_t K^T of tile t = 0, 1, warps 10, 11 of
// O_t += P_t V.  S: stages; Q8: codes made 16-bit by warps that fence their writes
// themselves, keys' in q's type, values' in f16.
template <bool BF16, int D, int S, bool Q8>
__device__ __forceinline__ void issue_products(const Params& p, Walk& walk, const Ctl& ctl, const Shared& b, uint32_t tmem_base,
                                               int warp, int lane) {
  constexpr uint32_t kTile = kHalfTile * (D / 64), kBlk = kHalfBlk * (D / 64);
  Portion po;
  const int t = warp & 1;
  const bool scores = warp < 10;
  const uint32_t fmt = BF16 ? 1u : 0u, fmt_pv = BF16 && !Q8 ? 1u : 0u;
  // fp32 accumulators; B of Q K^T K-major, of P V N-major
  const uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kBlock >> 3) << 17) | ((128u >> 4) << 24);
  const uint32_t idesc_pv =
      (1u << 4) | (fmt_pv << 7) | (fmt_pv << 10) | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17) | ((128u >> 4) << 24);
  const uint32_t tS = tmem_base + t * 128, tO = tmem_base + kTmemO + t * D;
  const uint64_t dq = gemm::sw128_desc(smem_u32(b.sQ) + t * kTile, 16, 1024);
  const uint64_t dk = gemm::sw128_desc(smem_u32(b.sK), 16, 1024);
  const uint64_t dv = gemm::sw128_desc(smem_u32(b.sV), kHalfBlk, 1024);
  uint64_t* full = scores ? b.k_full : b.v_full;
  uint64_t* empty = scores ? b.k_empty : b.v_empty;
  const volatile int* by_copy = scores ? b.copied : b.copied + S;
  int c = 0;      // key blocks passed, over all portions
  int g = 0;      // of them this tile's
  int done = 0;   // portions in which this tile had steps
  bool ok = true;
  for (int li = 0; ok && walk.next(p, po); ++li) {
    if (scores) {
      ok = warp_wait(b.q_full, li & 1, ctl);
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
      if (!Q8 && by_copy[st]) gemm::fence_async_smem();  // cp.async's writes, before the MMA's reads
      const int buf = g & 1;
      if (scores) {
        // P V of the block two before has read P from this buffer
        if (g > 1 && !(ok = warp_wait(&b.o_done[t * 2 + buf], ((g >> 1) - 1) & 1, ctl))) break;
        gemm::tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_ss(tS + buf * 64, dq + (((k >> 2) * kHalfTile + (k & 3) * 32) >> 4),
                  dk + ((st * kBlk + (k >> 2) * kHalfBlk + (k & 3) * 32) >> 4), idesc_s, k != 0);
        if (!(t == 0 && g == 0 && (p.test_flags & B200K_PAGED_TEST_WITHHOLD_SCORES))) commit(&b.s_full[t * 2 + buf]);
        commit(&b.k_empty[st]);
        if (j + 1 == po.t_end[t]) commit(b.q_empty);
      } else {
        const bool first = j == po.t_beg[t];
        // the epilogue of the portion before has read O
        if (first && done > 0 && !(ok = warp_wait(&b.o_free[t], (done - 1) & 1, ctl))) break;
        if (!(ok = warp_wait(&b.p_full[t * 2 + buf], (g >> 1) & 1, ctl))) break;
        gemm::tc_fence_after();
#pragma unroll
        for (int k = 0; k < kBlock / 16; ++k)
          umma_ts(tO, tS + buf * 64 + k * 8, dv + ((st * kBlk + k * 2048) >> 4), idesc_pv, (!first || k != 0) ? 1u : 0u);
        commit(&b.o_done[t * 2 + buf]);
        commit(&b.v_empty[st]);
      }
      ++g;
    }
    if (!ok) break;
    if (po.t_end[t] > po.t_beg[t]) ++done;
    else if (scores && lane == 0) gemm::mbar_arrive(b.q_empty);
    __syncwarp();
  }
  // every MMA of this warp completes before tensor memory is freed
  commit(&b.drain[warp - 8]);
  gemm::wait_bar_drain(&b.drain[warp - 8], 0, 100000000ull);
  __syncwarp();
}

// The softmax warps 0-7, one thread a query row.  Q8: both products are of codes, so
// a score is multiplied by its key's scale and has the logarithm of its value's added,
// and a weight enters the sum over its value's scale (paged.cuh).  What a row does
// not see has weight zero there, exactly: 1 / vs may be anything beside it.
template <bool BF16, int D, int CAP, bool Q8>
__device__ __forceinline__ void softmax_rows(const Params& p, Walk& walk, const Ctl& ctl, const Shared& b, uint32_t tmem_base,
                                             int64_t run, int warp, int lane) {
  constexpr bool P16 = BF16 && !Q8;  // weights of the second product in bf16
  Portion po;
  const int t = warp >> 2, quarter = warp & 3;
  const int in_unit = t * 128 + quarter * 32 + lane;
  const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t tS = t_lane + t * 128, tO = t_lane + kTmemO + t * D;
  int g = 0, c = 0;  // c: blocks passed
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
    for (int j = Q8 ? po.beg : jb; j < (Q8 ? po.end : je); ++j) {
      const int slot = c % kScaleSlots;
      if (Q8) {
        if (!(ok = warp_test_wait(&b.sc_full[slot], (c / kScaleSlots) & 1, ctl))) break;
        ++c;
        if (j < jb || j >= je) {  // not a block of this tile
          if (lane == 0) gemm::mbar_arrive(&b.sc_empty[slot]);
          __syncwarp();
          continue;
        }
      }
      const float* scales = b.sc + slot * kScaleFloats;
      const uint32_t buf = g & 1;
      if (!(ok = warp_wait(&b.s_full[t * 2 + buf], (g >> 1) & 1, ctl))) break;
      gemm::tc_fence_after();
      float s[kBlock];
      {
        uint32_t raw[kBlock / 32][32];
#pragma unroll
        for (int c = 0; c < kBlock / 32; ++c) gemm::tmem_ld32(tS + buf * 64 + c * 32, raw[c]);
        // (the waits name the registers, so that no use of them is scheduled ahead)
        gemm::tmem_wait_ld_regs2(raw[0], raw[1]);
#pragma unroll
        for (int c = 0; c < kBlock / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) s[c * 32 + i] = __uint_as_float(raw[c][i]);
      }
      if (Q8) {
#pragma unroll
        for (int c = 0; c < kBlock; c += 4) {
          const float4 k = *reinterpret_cast<const float4*>(scales + c), lv = *reinterpret_cast<const float4*>(scales + kBlock + c);
          float2 x = make_float2(s[c], s[c + 1]), y = make_float2(s[c + 2], s[c + 3]);
          if (CAP == kNoCap) {
            x = __ffma2_rn(x, make_float2(k.x, k.y), make_float2(lv.x, lv.y));
            y = __ffma2_rn(y, make_float2(k.z, k.w), make_float2(lv.z, lv.w));
          } else {
            x = make_float2(score<CAP>(p, x.x * k.x) + lv.x, score<CAP>(p, x.y * k.y) + lv.y);
            y = make_float2(score<CAP>(p, y.x * k.z) + lv.z, score<CAP>(p, y.y * k.w) + lv.w);
          }
          s[c] = x.x;
          s[c + 1] = x.y;
          s[c + 2] = y.x;
          s[c + 3] = y.y;
        }
      } else if (CAP != kNoCap) {
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
      constexpr bool kRaw = CAP == kNoCap && !Q8;  // scores that p.mul is still to be multiplied with
      if (kRaw) top *= p.mul;
      const float was = m;
      float alpha = 1.0f;
      bool moved = false;
      // A NaN score, and an infinite one (0 * top), makes the maximum NaN and
      // with it every probability and sum of the row from here on.
      if (!(top <= m + kTileLag<P16>)) {
        m = fmaf(0.0f, top, top);
        alpha = ex2(was - m);
        moved = j > jb;
      }
      // probabilities are rounded to the input type, half a step each, in f16
      // down to 2^-26 of the row's maximum (smaller ones by less than 2^-36 of it)
      const float ref = (m == -INFINITY ? 0.0f : m) - kTileReach<P16>;
      float2 sum2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
      const float2 sc2 = kRaw ? make_float2(p.mul, p.mul) : make_float2(1.0f, 1.0f), nm2 = make_float2(-ref, -ref);
      uint32_t pk[kBlock / 2];
#pragma unroll
      for (int c = 0; c < kBlock; c += 2) {
        const float2 x = __ffma2_rn(make_float2(s[c], s[c + 1]), sc2, nm2);
        const float2 e = c % kFmaEvery == kFmaEvery - 2 ? ex2_fma<P16, Q8>(x) : make_float2(ex2(x.x), ex2(x.y));
        sum2[c / 2 % 2] = Q8 ? __ffma2_rn(e, *reinterpret_cast<const float2*>(scales + 2 * kBlock + c), sum2[c / 2 % 2])
                             : __fadd2_rn(sum2[c / 2 % 2], e);
        pk[c / 2] = pack16<P16>(e.x, e.y);
      }
      if (Q8) {
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&b.sc_empty[slot]);
      }
      const float sum = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      l = fmaf(l, alpha, sum);
      if (__any_sync(0xffffffffu, moved)) {
        // P V of the block before has written O
        if (!(ok = warp_wait(&b.o_done[t * 2 + (buf ^ 1)], ((g - 1) >> 1) & 1, ctl))) break;
        gemm::tc_fence_after();
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          gemm::tmem_ld32(tO + c * 32, o);
          gemm::tmem_wait_ld_regs(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(tO + c * 32, o);
        }
      }
      tmem_st32(tS + buf * 64, pk);
      tmem_wait_st();
      gemm::tc_fence_before();
      __syncwarp();
      if (lane == 0) gemm::mbar_arrive(&b.p_full[t * 2 + buf]);
      ++g;
    }
    if (!ok) break;
    const bool had = je > jb;
    if (had && !(ok = warp_wait(&b.o_done[t * 2 + ((g - 1) & 1)], ((g - 1) >> 1) & 1, ctl))) break;
    gemm::tc_fence_after();
    // a row without keys has m = -inf (and l the sum of its 2^-125, or 0)
    const float inv = m == -INFINITY ? 0.0f : 1.0f / l;
    const int64_t part = static_cast<int64_t>(blockIdx.x) * 2 + po.slot;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      if (had) {
        gemm::tmem_ld32(tO + c * 32, o);
        gemm::tmem_wait_ld_regs(o);
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
      if (lane == 0) gemm::mbar_arrive(&b.o_free[t]);
    }
    if (!po.whole && real)
      reinterpret_cast<float2*>(p.tile_ml)[part * kUnitRows + in_unit] = make_float2(m, l);
  }
}

// Boxes of a 4-d view, inner dim first; sizes and strides in elements of `bytes`.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, int bytes, CUtensorMapSwizzle swizzle, const void* ptr, const int64_t (&sizes)[4], const int64_t (&strides)[3],
              const cuuint32_t (&box)[4]) {
  auto fn = gemm::encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4], gstr[3];
  uint64_t natural = static_cast<uint64_t>(sizes[0]) * bytes;
  for (int i = 0; i < 4; ++i) dims[i] = static_cast<cuuint64_t>(sizes[i]);
  for (int i = 0; i < 3; ++i) {  // the stride of a dim of one is never stepped: give it a legal value
    gstr[i] = sizes[i + 1] == 1 ? natural : static_cast<uint64_t>(strides[i]) * bytes;
    natural = std::max<uint64_t>(natural, gstr[i]);
    if (gstr[i] == 0 || gstr[i] >= (1ull << 40)) return false;
  }
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, type, 4, const_cast<void*>(ptr), dims, gstr, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace paged
}  // namespace b200k
