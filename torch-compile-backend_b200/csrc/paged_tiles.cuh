// What the tile kernels of b200k_paged_attention (paged_tiles.cu) and
// b200k_paged_attention_quant (paged_tiles8.cu) share: instruction wrappers,
// the walk over a CTA's part of the list, tensor maps.
#pragma once

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

constexpr uint32_t kHalfTile = 128 * 128;  // 128 rows of 64 16-bit values: one swizzled column
constexpr uint32_t kHalfBlk = kBlock * 128;
// Of so many probabilities two are computed on the FMA pipe.  8 prompts of
// 2048 (32 heads of 64): 277 us, 291 with none, 286 with half of them.
constexpr int kFmaEvery = 8;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
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
