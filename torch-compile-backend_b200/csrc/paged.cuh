// What the kernels of b200k_paged_attention share: the launch parameters, how
// a sequence's work is read from the index tensors, and the score transform.
#pragma once

#include "common.cuh"

namespace b200k {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 16;      // keys of one step of the row kernel (one MMA k)
constexpr int kKeys8 = 32;     // ... over e4m3 caches: as many bytes
constexpr int kRows = 16;      // query rows of one unit of the row kernel (one MMA m)
constexpr int kBlock = 64;     // keys of one step of the tile kernel
constexpr int kUnitRows = 256; // query rows of one unit of the tile kernel (two MMA m)
// Probabilities of the second product are rounded to the input type.  f16 ones
// below 2^-14 would lose bits and those below 2^-25 vanish, while their sum
// keeps them (a key 17 nats above the others and of value zero: the output 40 %
// off), so they are computed 2^kF16Reach times too large, the sum with them,
// which the division takes out: f16 reaches 65504.  A tile's maximum may lag
// behind by 2^kLagF16, which its probabilities have to leave free.  8 f16
// prompts of 2048 (32 heads of 64) with a lag of 8, 4, 3 and 2: 279, 275, 278
// and 286 us.  bf16 has fp32's exponents.
constexpr float kF16Reach = 15.0f;
constexpr float kLagF16 = 3.0f, kLagBf16 = 8.0f;
template <bool BF16>
constexpr float kRowReach = BF16 ? 0.0f : kF16Reach;
template <bool BF16>
constexpr float kTileLag = BF16 ? kLagBf16 : kLagF16;
template <bool BF16>
constexpr float kTileReach = BF16 ? 0.0f : kF16Reach - kLagF16;
// What a unit's start and end cost (queries in, output out, pipeline empty),
// in steps: counted in the list that the CTAs share out.  8 prompts of 2048
// (32 heads of 64) with 0, 2, 4 and 8: 387, 300, 277 and 297 us.
constexpr int kPortionCost = 4;

// A unit of the tile kernel whose parts lie in CTAs i (slot 1) to last (slot 0).
struct Join {
  int32_t last;      // 0: none
  int32_t t0, kvh;   // the sequence's first token
  int32_t r0, rows;
};

struct Params {
  int32_t T, B, H, Hkv, G;     // G = H / Hkv
  int32_t page_size, num_pages, table_cols;
  int32_t capacity;            // table_cols * page_size, clamped to int32
  int32_t window;              // 0: none
  int32_t long_rows;           // sequences of more query rows (queries * G) run the tile kernel,
  int64_t mid_steps;           // those of more than kRows too where they have so many steps (0: never)
  int32_t combine_rows;        // tokens of a sequence that the combine grid covers side by side
  int32_t join_mode;           // how the combine kernel's warps share the rows
  FastDiv div_page, div_g;
  int64_t table_stride;
  const uint16_t* q;
  int64_t q_t, q_h;
  const uint16_t *k, *v;
  int64_t c_page, c_slot, c_head;
  // e4m3 caches: codes in place of k and v (same strides), and their scales
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  int64_t s_page, s_slot, s_head;
  uint32_t c16_page, c16_slot, c16_head;  // their strides in 16 bytes
  int32_t far_rows;            // offsets past 2^32 in those, or in scales
  uint16_t* out;               // [T, H, D] contiguous
  const int32_t *table, *q_start, *kv_len;
  // base-2 scores: y = x * mul; with a cap (cap_far) mul = 2 scale log2(e) / cap,
  // lin = scale log2(e), cap2 = cap log2(e)
  float mul, lin, cap2;
  float* part_o;               // [workers][2][16][D]
  float* part_ml;              // [workers][2][16][2]: running max (base 2) and sum
  int64_t* prefix;             // [B + 1] steps before each sequence; [B + 1]: steps a worker takes
  int32_t workers;
  // tile kernel: steps count kPortionCost a unit; [0] all, [1] a CTA's, [2] entries, [3 + e] before entry e
  int64_t* entry_steps;
  int2* entries;               // (sequence, 256-row block), at most max_entries
  int32_t max_entries;
  float* tile_o;               // [CTAs][2][D / 4][256][4]
  float* tile_ml;              // [CTAs][2][256][2]
  Join* joins;                 // [CTAs] the cut unit that begins in each CTA's run
  int32_t tile_ctas;           // 0: not launched
  int32_t box_rows;            // rows of a TMA box of keys or values, 0: copied row by row
  int32_t q_box;               // queries by TMA
  int32_t test_flags;
  int32_t* status;
  int64_t timeout_ns;
};

// One sequence's queries and keys, clamped to the tensors that hold them.
struct Seq {
  int t0, m;     // first token, queries
  int n;         // keys
  int first;     // position of the first query (may be negative: queries without keys)
  int lo;        // first key that any query sees
};

__device__ __forceinline__ Seq seq_at(const Params& p, int b) {
  Seq s;
  // (in the row kernel over e4m3 caches, launched early)
  const int a0 = fetch<true>(p.q_start + b), a1 = fetch<true>(p.q_start + b + 1), n = fetch<true>(p.kv_len + b);
  s.t0 = min(max(a0, 0), p.T);
  s.m = min(max(a1, s.t0), p.T) - s.t0;
  s.n = min(max(n, 0), p.capacity);
  if ((s.t0 != a0 || s.t0 + s.m != a1 || s.n != n) && p.status) atomicCAS(p.status, 0, B200K_ERR_INDEX);
  s.first = s.n - s.m;
  s.lo = p.window > 0 ? max(0, s.first - p.window + 1) : 0;
  return s;
}

// 256 query rows of a sequence, as the tile kernel works on them.
struct Unit {
  Seq s;
  int b, r0, rows;   // first row, rows of the sequence
  int lo, hi;        // keys that its rows see
  int ub0, ub1;      // their blocks: at least one, so that rows without keys are written
};
// Keys that rows [r0, r1) of a sequence see: [lo, hi), hi <= 0 when none.
__device__ __forceinline__ void rows_keys(const Params& p, const Seq& s, int r0, int r1, int& lo, int& hi) {
  const int a = s.first + static_cast<int>(fdiv(static_cast<uint32_t>(r0), p.div_g));
  const int z = s.first + static_cast<int>(fdiv(static_cast<uint32_t>(r1 - 1), p.div_g));
  lo = p.window > 0 ? max(0, a - p.window + 1) : 0;
  hi = z + 1;
}
__device__ __forceinline__ Unit unit_at(const Params& p, int b, int qb) {
  Unit u;
  u.s = seq_at(p, b);
  u.b = b;
  u.r0 = qb * kUnitRows;
  u.rows = u.s.m * p.G;
  rows_keys(p, u.s, u.r0, min(u.r0 + kUnitRows, u.rows), u.lo, u.hi);
  u.ub0 = u.lo / kBlock;
  u.ub1 = max(u.ub0 + 1, (u.hi + kBlock - 1) / kBlock);
  return u;
}
// Keys of tile t (rows r0 + 128 t ...) of a unit; hi <= 0 for a tile without rows.
__device__ __forceinline__ void tile_keys(const Params& p, const Unit& u, int t, int& lo, int& hi) {
  const int a = u.r0 + t * 128;
  lo = hi = 0;
  if (a < u.rows) rows_keys(p, u.s, a, min(a + 128, u.rows), lo, hi);
}

// Launches the tile kernel (paged_tiles.cu, over e4m3 caches paged_tiles8.cu)
// on the plan in p.entries.
int launch_tiles(const Params& p, bool bf16, int dim, int cap, cudaStream_t st);
int launch_tiles8(const Params& p, bool bf16, int dim, int cap, cudaStream_t st);

// Offset of a key's row in the caches, `page` being what the table holds for
// it, or -1: not between lo and n (nothing there is read: the pages may hold
// anything), or a page that does not exist.
__device__ __forceinline__ int64_t page_offset(const Params& p, int page, int key, int lo, int n, int kvh) {
  if (key < lo || key >= n) return -1;
  if (page < 0 || page >= p.num_pages) {
    if (p.status) atomicCAS(p.status, 0, B200K_ERR_INDEX);
    return -1;
  }
  const uint32_t pi = fdiv(static_cast<uint32_t>(key), p.div_page);
  return static_cast<int64_t>(page) * p.c_page +
         static_cast<int64_t>(static_cast<uint32_t>(key) - pi * static_cast<uint32_t>(p.page_size)) * p.c_slot +
         static_cast<int64_t>(kvh) * p.c_head;
}
__device__ __forceinline__ int64_t key_offset(const Params& p, int b, int key, int lo, int n, int kvh) {
  if (key < lo || key >= n) return -1;
  const int page = __ldg(p.table + b * p.table_stride + fdiv(static_cast<uint32_t>(key), p.div_page));
  return page_offset(p, page, key, lo, n, kvh);
}

// ... with the offset of its scales.
struct Place8 {
  int64_t row, scale;
};
__device__ __forceinline__ Place8 place8(const Params& p, int page, int key, int lo, int n, int kvh) {
  Place8 r{-1, -1};
  if (key < lo || key >= n) return r;
  if (page < 0 || page >= p.num_pages) {
    if (p.status) atomicCAS(p.status, 0, B200K_ERR_INDEX);
    return r;
  }
  const uint32_t pi = fdiv(static_cast<uint32_t>(key), p.div_page);
  const int64_t in = static_cast<uint32_t>(key) - pi * static_cast<uint32_t>(p.page_size);
  r.row = static_cast<int64_t>(page) * p.c_page + in * p.c_slot + static_cast<int64_t>(kvh) * p.c_head;
  r.scale = static_cast<int64_t>(page) * p.s_page + in * p.s_slot + static_cast<int64_t>(kvh) * p.s_head;
  return r;
}

// Attention over e4m3 caches: key and value rows are code * scale.  The scales
// stay out of the products: a score is (q . codes) ks_j, and with
//   y_j = f(score_j) log2(e) + log2(vs_j),  w_j = 2^(y_j - max y)
// the output is sum_j w_j codes_j / sum_j w_j / vs_j: one exponential for both
// sums, and no w_j above 1 however far the values' scales lie apart.  Codes are
// exact in f16, so both products are f16 ones whatever q's type.
// Scales of values below kMinVs (that of rows of zeros) count as it.
constexpr float kMinVs = 1e-12f / 448.0f;
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float value_scale(float vs) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(vs), "f"(kMinVs));
  return r;
}
// Two e4m3 codes (the low or high half of a word) as f16.
__device__ __forceinline__ uint32_t codes16(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}
__device__ __forceinline__ uint32_t codes_lo(uint32_t c) { return codes16(static_cast<uint16_t>(c)); }
__device__ __forceinline__ uint32_t codes_hi(uint32_t c) { return codes16(static_cast<uint16_t>(c >> 16)); }
// bf16 queries as f16: a row is divided by a power of two that puts its
// largest magnitude (`top`, as bits) between 2^14 and 2^15, which leaves 28
// binades at full precision below it, and its scores are multiplied by it.
struct RowScale {
  float div, mul;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const uint32_t e = top >> 23;  // biased exponent of the largest magnitude
  RowScale r{1.0f, 1.0f};
  if (e == 255 || top == 0) return r;  // a row with an infinity or NaN, of zeros
  const uint32_t b = max(e, 15u);
  r.div = __uint_as_float((268u - b) << 23);
  r.mul = __uint_as_float((b - 14u) << 23);
  return r;
}
// Two bf16 values times `f` as f16.
__device__ __forceinline__ uint32_t bf16_to_f16(uint32_t w, float f) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(__uint_as_float(w & 0xffff0000u) * f), "f"(__uint_as_float(w << 16) * f));
  return r;
}

// Asynchronous copies of 16 and 4 bytes to shared memory, of zeros where there is nothing to read.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A capped score in base 2: cap2 tanh(u), u = x scale / cap, with t = 2 u log2(e)
// at hand as x mul.  Where the cap is at most kPlainCap, cap2 - 2 cap2 / (1 + 2^t):
// the approximate units' 2^-22 and 2^-23 leave 3.6e-7 of the cap, 3.6e-5.  That
// error stays at small u, where the terms cancel, and grows with the cap (with
// scores of 5 and a cap of 1e6 it was 0.1).  So with larger ones (kCapSeries)
// scores below 0.35 of the cap are the series tanh(u) = u (1 + u^2 P(u^2)) on the
// uncapped score u cap2 = x lin, P by Remez exchange on [0, 0.35^2], 4.1e-8
// relative; above, the first form is within 6.2e-7 of the score.  The series for
// every cap: decode of 64 sequences to 8192 keys 232 us in place of 225, chunks
// whose scores reach the cap 693 in place of 489.
constexpr float kPlainCap = 100.0f;
enum { kNoCap, kCapPlain, kCapSeries };
constexpr float kSmallCap = 0.35f * 2.0f * kLog2e;
__device__ __forceinline__ float cap_far(const Params& p, float t) {
  return fmaf(-2.0f * p.cap2, rcp(1.0f + ex2(t)), p.cap2);
}
__device__ __forceinline__ float cap_near(const Params& p, float x, float t) {
  constexpr float k = 1.0f / (2.0f * kLog2e);  // u = k t
  const float w = x * p.lin, z = t * t;
  float r = fmaf(-4.9148502e-2f * (k * k * k * k * k * k), z, 1.3299825e-1f * (k * k * k * k));
  r = fmaf(r, z, -3.3332663e-1f * (k * k));
  return fmaf(w, z * r, w);
}
template <int CAP>
__device__ __forceinline__ float score(const Params& p, float x) {
  const float t = x * p.mul;
  if (CAP == kNoCap) return t;
  return CAP == kCapSeries && fabsf(t) < kSmallCap ? cap_near(p, x, t) : cap_far(p, t);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace paged
}  // namespace b200k
