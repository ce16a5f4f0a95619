// Attention over a paged key/value cache (b200k_paged_attention,
// include/b200k.h): packed queries of ragged sequences against each
// sequence's pages.
//
//   out[t, h] = sum_j softmax_j(f(scale q[t, h] . k_j)) v_j,  f(s) = s or cap tanh(s / cap),
//   j over the keys max(0, pos - window + 1) .. pos of the token's sequence,
//   pos = kv_len - queries + index of the token among them
//
// No reference counterpart (it leaves attention to ATen and has no cache).
//
// The row kernel (this file), for single tokens and few queries a sequence:
// bound by HBM, it reads each visible key and value once for the G query
// heads that share it.  Work is one long list of steps, a step being 16 keys
// of one unit (sequence, kv head, 16 query rows = queries x G heads); every
// warp takes an equal run of the list, so ragged lengths balance to one step
// whatever their order, and a single long sequence spreads over the GPU.
// A warp streams its steps' rows of K and V into its own shared-memory ring
// with 16-byte cp.async copies (S - 1 steps ahead, across unit boundaries; no
// block-wide barrier while it streams), multiplies with m16n8k16 MMAs (16 rows by 8
// keys, rows beyond the unit's are zero: the tensor pipe has the time, the
// memory does not) and keeps its running maximum, sum and output in fp32.
// A unit inside one run is written at once; a cut one leaves its parts
// (max, sum, unnormalised output, fp32) in the workspace, one for a CTA whose
// warps are all in the unit (one token over 30000 keys of one key head: 20 us,
// with a part a warp 42), and combine_kernel joins them in an order that only
// the lengths decide.
// Measured: one token of 64 sequences to 8192 keys, 32 / 8 heads of 128, 215 us
// = 6.36 TB/s; of 3 sequences to 65536 keys 95 us = 6.05 TB/s.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "host_common.h"
#include "paged.cuh"
#include "rowreduce.cuh"

namespace b200k {
namespace paged {
namespace {

constexpr int kWarps = 4;
// Eight warps an SM with three stages of 8 KB each (heads of 128): decode of
// 64 sequences to 8192 keys 221 us, with twelve warps of two stages 219, with
// four of six 278; a single token over 2574 keys 13.1, 14.8 and 13.9.
constexpr int kCtasPerSm = 2;
constexpr uint32_t kRingBytes = 24576;  // of one warp

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A sequence as the row kernel cuts it: `units` of `tiles` steps each.
struct Work {
  Seq s;
  int base;   // first key of step 0 (lo rounded down to a step)
  int tiles;  // 0: no keys, no queries, or the tile kernel's
  int rts;    // row blocks of a kv head
};
// `limit`: query rows above which a sequence is the tile kernel's; KEYS: of a step,
// ROWS: query rows of a unit.
template <int KEYS, int ROWS>
__device__ __forceinline__ Work work_at(const Params& p, int b, int limit) {
  Work w;
  w.s = seq_at(p, b);
  w.base = w.s.lo & ~(KEYS - 1);
  const int64_t rows = static_cast<int64_t>(w.s.m) * p.G;
  w.rts = static_cast<int>((rows + ROWS - 1) / ROWS);
  w.tiles = (w.s.m > 0 && w.s.n > w.base && rows <= limit) ? (w.s.n - w.base + KEYS - 1) / KEYS : 0;
  return w;
}
__device__ __forceinline__ int64_t steps_of(const Params& p, const Work& w) {
  return static_cast<int64_t>(p.Hkv) * w.rts * w.tiles;
}
__device__ __forceinline__ int64_t warp_scan(int64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// The limit of this call: p.long_rows, or kRows where the sequences between
// the two (two row blocks, so the row kernel reads their keys twice) have
// enough keys for the tile kernel to pay.  Every warp that asks gets the same.
template <int KEYS, int ROWS>
__device__ __forceinline__ int limit_of(const Params& p) {
  if (p.mid_steps == 0) return p.long_rows;
  int64_t steps = 0;
  for (int b = threadIdx.x & 31; b < p.B; b += 32) {
    const Work w = work_at<KEYS, ROWS>(p, b, p.long_rows);
    if (w.rts > 1) steps += static_cast<int64_t>(p.Hkv) * w.tiles;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) steps += __shfl_xor_sync(0xffffffffu, steps, o);
  return steps >= p.mid_steps ? kRows : p.long_rows;
}

// n / d for n >= 0, d > 0: 32-bit where both fit, which every real list does
// (a 64-bit division takes about 0.25 us, on the path to the first load).
__device__ __forceinline__ int64_t div64(int64_t n, int64_t d) {
  if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}
// Steps that a worker takes of a list of `total` whose longest unit has
// `longest`: an equal share, but enough that a unit has at most kMaxParts CTAs.
// One token over 30000, 8000 and 120000 keys of one key head: 14.7, 10.5 and
// 31 us, without the bound 19.8, 13.3 and 32, with 32 in its place 20.3, 10.6
// and 62.
constexpr int kMaxParts = 96;
__device__ __forceinline__ int64_t run_of(const Params& p, int64_t total, int longest) {
  return max(div64(total + p.workers - 1, p.workers),
             static_cast<int64_t>(max(1, (longest + kMaxParts * kWarps - 1) / (kMaxParts * kWarps))));
}

// A position in the list of steps: within a sequence kv head by kv head, row
// block by row block, key by key.
template <int KEYS, int ROWS>
struct Cursor {
  Work w;
  int b, kvh, rt, tile;
  int limit;
  __device__ __forceinline__ void next(const Params& p) {
    if (++tile < w.tiles) return;
    tile = 0;
    if (++rt < w.rts) return;
    rt = 0;
    if (++kvh < p.Hkv) return;
    kvh = 0;
    do {
      if (++b >= p.B) return;
      w = work_at<KEYS, ROWS>(p, b, limit);
    } while (w.tiles == 0 || w.rts == 0);
  }
};

// The tile kernel's list: an entry for every 256 query rows of a sequence
// that is its own, with the steps before it.  One CTA of 128 threads.
template <int KEYS, int ROWS>
__device__ __noinline__ void plan_tiles(const Params& p) {
  __shared__ int starts[kWarps * 32 + 1];   // entries before each of 128 sequences
  __shared__ int64_t sums[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t* before = p.entry_steps + 3;
  for (int i = tid; i < p.tile_ctas; i += kWarps * 32) p.joins[i].last = 0;
  const int limit = limit_of<KEYS, ROWS>(p);
  int64_t steps = 0;
  int entry0 = 0;
  auto block_scan = [&](int64_t v, int64_t& all) {  // inclusive
    int64_t x = warp_scan(v);
    __syncthreads();
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    all = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) x += sums[w];
      all += sums[w];
    }
    return x;
  };
  for (int b0 = 0; b0 < p.B; b0 += kWarps * 32) {
    int n = 0;
    if (b0 + tid < p.B) {
      const int64_t rows = static_cast<int64_t>(seq_at(p, b0 + tid).m) * p.G;
      if (rows > limit) n = static_cast<int>((rows + kUnitRows - 1) / kUnitRows);
    }
    int64_t all;
    const int64_t upto = block_scan(n, all);
    // A q_start that runs backwards gives tokens to several sequences: the
    // list ends where the workspace does (seq_at reports it).
    all = min(all, static_cast<int64_t>(p.max_entries - entry0));
    starts[tid] = static_cast<int>(upto - n);
    if (tid == 0) starts[kWarps * 32] = static_cast<int>(all);
    __syncthreads();
    for (int e0 = 0; e0 < all; e0 += kWarps * 32) {
      const int e = e0 + tid;
      int64_t mine = 0;
      if (e < all) {
        int lo = 0, hi = kWarps * 32;  // the last sequence with starts <= e
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (starts[mid] <= e) lo = mid;
          else hi = mid;
        }
        const Unit u = unit_at(p, b0 + lo, e - starts[lo]);
        p.entries[entry0 + e] = make_int2(b0 + lo, e - starts[lo]);
        mine = static_cast<int64_t>(u.ub1 - u.ub0 + kPortionCost) * p.Hkv;
      }
      int64_t sum;
      const int64_t x = block_scan(mine, sum);
      if (e < all) before[entry0 + e] = steps + x - mine;
      steps += sum;
    }
    entry0 += static_cast<int>(all);
    __syncthreads();
  }
  if (tid == 0) {
    p.entry_steps[0] = steps;
    p.entry_steps[1] = (steps + p.tile_ctas - 1) / p.tile_ctas;
    p.entry_steps[2] = entry0;
    before[entry0] = steps;
  }
}

// A warp's part in shared memory, in its ring: rows of D sums, a maximum and
// a sum, 32 bytes apart modulo the banks.
template <int D>
constexpr int kJointStride = D + 8;
template <int D, uint32_t RING, int ROWS = kRows>
__device__ __forceinline__ float* joint_rows(uint8_t* smem, int warp) {
  static_assert(ROWS * kJointStride<D> * 4 <= RING, "a part fits a ring");
  return reinterpret_cast<float*>(smem + warp * RING);
}
// The CTA's warps' parts of one unit as one: written to `worker`'s slot, or to
// the output where the CTA has the whole unit.  A warp takes every kWarps-th row.
template <bool BF16, int D, uint32_t RING, int ROWS = kRows, typename Out>
__device__ __forceinline__ void join_warps(const Params& p, uint8_t* smem, int warp, int lane, int rows, int worker, int slot,
                                           bool whole, Out out_row) {
  constexpr int V = D / 32;
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  for (int in = warp; in < rows; in += kWarps) {
    float2 ml[kWarps];
    float mx = -INFINITY, sum = 0.0f, acc[V];
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      ml[k] = *reinterpret_cast<const float2*>(joint_rows<D, RING, ROWS>(smem, k) + in * kJointStride<D> + D);
      mx = fmaxf(mx, ml[k].x);
    }
    const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float f = ex2(ml[k].x - ref);
      const Vec x = reinterpret_cast<const Vec*>(joint_rows<D, RING, ROWS>(smem, k) + in * kJointStride<D>)[lane];
      sum = fmaf(ml[k].y, f, sum);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] = fmaf(reinterpret_cast<const float*>(&x)[j], f, acc[j]);
    }
    if (whole) {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      uint32_t* dst = reinterpret_cast<uint32_t*>(out_row(in)) + lane * (V / 2);
#pragma unroll
      for (int j = 0; j < V; j += 2) dst[j / 2] = pack16<BF16>(acc[j] * inv, acc[j + 1] * inv);
    } else {
      const int64_t at = (static_cast<int64_t>(worker) * 2 + slot) * ROWS + in;
      Vec x;
#pragma unroll
      for (int j = 0; j < V; ++j) reinterpret_cast<float*>(&x)[j] = acc[j];
      reinterpret_cast<Vec*>(p.part_o + at * D)[lane] = x;
      if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mx, sum);
    }
  }
}

template <bool BF16, int D, int CAP>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) rows_kernel(const __grid_constant__ Params p) {
  constexpr int S = kRingBytes / (kKeys * D * 4);  // ring stages: K and V rows of a step each
  constexpr uint32_t kRowBytes = D * 2, kTile = kKeys * kRowBytes;
  constexpr int kChunks = D / 8;          // 16-byte chunks of a row
  constexpr int kRowsPerCp = 32 / kChunks;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the first CTA plans the tile kernel's work, when that runs
  const int worker = (static_cast<int>(blockIdx.x) - (p.tile_ctas > 0 ? 1 : 0)) * kWarps + warp;
  const uint32_t ring = smem_addr(smem) + warp * kRingBytes;
  if (worker < 0) {
    plan_tiles<kKeys, kRows>(p);
    return;
  }

  // combine_kernel may be launched from here on: its CTAs find room as this
  // kernel's leave, and wait for its writes themselves.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // The whole list's length and, from it, this worker's run [w0, w1).
  const int limit = limit_of<kKeys, kRows>(p);
  int64_t total = 0, mine0 = 0, upto0 = 0;
  int longest = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int64_t mine = 0;
    if (b0 + lane < p.B) {
      const Work w = work_at<kKeys, kRows>(p, b0 + lane, limit);
      mine = steps_of(p, w);
      longest = max(longest, w.tiles);
    }
    const int64_t upto = warp_scan(mine);
    if (worker == 0 && b0 + lane < p.B) p.prefix[b0 + lane] = total + upto - mine;  // for combine_kernel
    total += __shfl_sync(0xffffffffu, upto, 31);
    mine0 = mine;
    upto0 = upto;
  }
  const int64_t run = run_of(p, total, __reduce_max_sync(0xffffffffu, longest));
  if (worker == 0 && lane == 0) {
    p.prefix[p.B] = total;
    p.prefix[p.B + 1] = run;
  }
  const int64_t w0 = run * worker, w1 = min(total, w0 + run);
  if (w0 >= w1) return;
  Cursor<kKeys, kRows> cur;
  cur.b = 0;
  int64_t seq0 = 0;  // the list's index of cur.b's first step
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int64_t mine = mine0, upto = upto0;  // of the last 32: all there are in a small batch
    if (p.B > 32) {
      mine = b0 + lane < p.B ? steps_of(p, work_at<kKeys, kRows>(p, b0 + lane, limit)) : 0;
      upto = warp_scan(mine);
    }
    const unsigned hit = __ballot_sync(0xffffffffu, seq0 + upto > w0);
    if (hit) {
      const int at = __ffs(hit) - 1;
      cur.b = b0 + at;
      seq0 += __shfl_sync(0xffffffffu, upto - mine, at);
      break;
    }
    seq0 += __shfl_sync(0xffffffffu, upto, 31);
  }
  cur.limit = limit;
  cur.w = work_at<kKeys, kRows>(p, cur.b, limit);
  const int unit = static_cast<int>(div64(w0 - seq0, cur.w.tiles));
  cur.tile = static_cast<int>((w0 - seq0) - static_cast<int64_t>(unit) * cur.w.tiles);
  cur.kvh = unit / cur.w.rts;
  cur.rt = unit - cur.kvh * cur.w.rts;

  Cursor<kKeys, kRows> ld = cur;
  int64_t ld_t = w0;
  // The page that holds this lane's key of a step, -1 for no key: fetched a
  // step before its first use, so that no step waits for the table.
  auto page_of = [&](const Cursor<kKeys, kRows>& c) {
    const int key = c.w.base + c.tile * kKeys + (lane & (kKeys - 1));
    if (key < c.w.s.lo || key >= c.w.s.n) return -1;
    return __ldg(p.table + c.b * p.table_stride + fdiv(static_cast<uint32_t>(key), p.div_page));
  };
  int page = -1;  // of the next step to load
  page = page_of(ld);
  int ld_stage = 0;
  auto issue = [&] {
    if (ld_t < w1) {
      const uint32_t sk = ring + ld_stage * 2 * kTile, sv = sk + kTile;
      const int c = lane % kChunks;
      const int64_t off = page_offset(p, page, ld.w.base + ld.tile * kKeys + (lane & (kKeys - 1)), ld.w.s.lo, ld.w.s.n, ld.kvh);
#pragma unroll
      for (int i = 0; i < kKeys / kRowsPerCp; ++i) {
        const int row = i * kRowsPerCp + lane / kChunks;
        const int64_t o = __shfl_sync(0xffffffffu, off, row);
        const bool real = o >= 0;
        const int64_t e = (real ? o : 0) + c * 8;
        const uint32_t d = row * kRowBytes + ((c ^ (row & 7)) << 4);
        cp16(sk + d, p.k + e, real);
        cp16(sv + d, p.v + e, real);
      }
      if (++ld_t < w1) {
        ld.next(p);
        page = page_of(ld);
      }
    }
    cp_commit();
    ld_stage = ld_stage + 1 == S ? 0 : ld_stage + 1;
  };

  const int g = lane >> 2, quad = lane & 3;
  uint32_t qf[D / 16][4];
  float o[D / 8][4];
  float m[2], l[2];
  int pos[2], row_first = 0, row_last = 0;
  bool fresh = true;
  int stage = 0;
  int64_t unit0 = seq0 + static_cast<int64_t>(unit) * cur.w.tiles;  // the current unit's first step
  // All of this CTA's runs lie in one unit: its warps' parts become one.
  const int64_t c0 = run * (worker & ~(kWarps - 1)), c1 = c0 + run * kWarps;
  const bool joint = unit0 <= c0 && c1 <= unit0 + cur.w.tiles;
  // The first S - 1 rounds only load.  One copy of the loading code: unrolled
  // ahead of the loop, its instructions alone took 2 us to arrive.
#pragma unroll 1
  for (int64_t t = w0 - (S - 1); t < w1; ++t) {
    if (t >= w0) {
      cp_wait<S - 2>();
      __syncwarp();  // step t has landed, and all lanes are done with the stage of step t - 1
    }
    issue();
    if (t < w0) continue;
    if (fresh) {  // a new unit: its query rows as A fragments
      fresh = false;
      const int rows = cur.w.s.m * p.G, r0 = cur.rt * kRows;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + g + 8 * i;
        const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
        const uint16_t* src = p.q + static_cast<int64_t>(cur.w.s.t0 + tok) * p.q_t +
                              static_cast<int64_t>(cur.kvh * p.G + (r - tok * p.G)) * p.q_h + quad * 2;
        pos[i] = cur.w.s.first + static_cast<int>(tok);
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qf[k][i] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16)) : 0u;
          qf[k][2 + i] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + k * 16 + 8)) : 0u;
        }
      }
#pragma unroll
      for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
      row_first = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(r0), p.div_g));
      row_last = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(min(r0 + kRows, rows) - 1), p.div_g));
    }
    const uint32_t sk = ring + stage * 2 * kTile, sv = sk + kTile;
    float s[2][4] = {};
    {
      // matrices: keys 0-7 / 8-15 by halves of the lanes, d chunk by quarters
      const int row = (lane & 7) + ((lane >> 4) << 3), ch = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t kb[4];
        ldm4(kb, sk + row * kRowBytes + (((k * 2 + ch) ^ (row & 7)) << 4));
        mma<BF16>(s[0], qf[k], kb[0], kb[1]);
        mma<BF16>(s[1], qf[k], kb[2], kb[3]);
      }
    }
    const int key0 = cur.w.base + cur.tile * kKeys;
    const bool masked = key0 + kKeys - 1 > row_first || (p.window > 0 && key0 <= row_last - p.window);  // warp-uniform
    uint32_t pa[4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = score<CAP>(p, s[n][i]);
    if (masked) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + n * 8 + quad * 2 + (i & 1), at = pos[i >> 1];
          if (key > at || (p.window > 0 && key <= at - p.window)) s[n][i] = -INFINITY;
        }
    }
    float alpha[2];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      const float was = m[i];
      m[i] = fmaxf(was, x);
      const float top = m[i] == -INFINITY ? 0.0f : m[i], ref = top - kRowReach<BF16>;
      alpha[i] = ex2(was - top);
      moved |= m[i] != was;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][2 * i] = ex2(s[n][2 * i] - ref);
        s[n][2 * i + 1] = ex2(s[n][2 * i + 1] - ref);
      }
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) l[i] *= alpha[i];
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= alpha[0];
        o[n][1] *= alpha[0];
        o[n][2] *= alpha[1];
        o[n][3] *= alpha[1];
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      l[i] += (s[0][2 * i] + s[0][2 * i + 1]) + (s[1][2 * i] + s[1][2 * i + 1]);
    // probabilities rounded to the input type for the second product (the sum
    // keeps fp32): half a step each, in f16 down to 2^-29 of the row's maximum
    // (smaller ones by less than 2^-40 of it)
    pa[0] = pack16<BF16>(s[0][0], s[0][1]);
    pa[1] = pack16<BF16>(s[0][2], s[0][3]);
    pa[2] = pack16<BF16>(s[1][0], s[1][1]);
    pa[3] = pack16<BF16>(s[1][2], s[1][3]);
    {
      const int row = lane & 15, ch = lane >> 4;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t vb[4];
        ldm4t(vb, sv + row * kRowBytes + (((n * 2 + ch) ^ (row & 7)) << 4));
        mma<BF16>(o[2 * n], pa, vb[0], vb[1]);
        mma<BF16>(o[2 * n + 1], pa, vb[2], vb[3]);
      }
    }
    stage = stage + 1 == S ? 0 : stage + 1;

    const bool unit_ends = cur.tile + 1 == cur.w.tiles;
    if (unit_ends || t + 1 == w1) {
      const int rows = cur.w.s.m * p.G, r0 = cur.rt * kRows;
      const bool whole = unit0 >= w0 && unit_ends;
      if (joint) {  // its last step: the rings are free
        cp_wait<0>();
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int in = g + 8 * i, r = r0 + in;
        if (r >= rows) continue;
        if (joint) {
          float* dst = joint_rows<D, kRingBytes>(smem, warp) + in * kJointStride<D>;
          if (quad == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[i], l[i]);
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(dst + n * 8 + quad * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        } else if (whole) {
          const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
          uint32_t* dst = reinterpret_cast<uint32_t*>(
              p.out + (static_cast<int64_t>(cur.w.s.t0 + tok) * p.H + cur.kvh * p.G + (r - tok * p.G)) * D + quad * 2);
          const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
          for (int n = 0; n < D / 8; ++n) dst[n * 4] = pack16<BF16>(o[n][2 * i] * inv, o[n][2 * i + 1] * inv);
        } else {
          const int64_t slot = static_cast<int64_t>(worker) * 2 + (unit0 < w0 ? 0 : 1);
          const int64_t at = slot * kRows + in;
          if (quad == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m[i], l[i]);
          float2* dst = reinterpret_cast<float2*>(p.part_o + at * D + quad * 2);
#pragma unroll
          for (int n = 0; n < D / 8; ++n) dst[n * 4] = make_float2(o[n][2 * i], o[n][2 * i + 1]);
        }
      }
      if (joint) {
        __syncthreads();  // every warp of the CTA comes here once
        join_warps<BF16, D, kRingBytes>(p, smem, warp, lane, min(kRows, rows - r0), worker & ~(kWarps - 1), unit0 < c0 ? 0 : 1,
                            unit0 == c0 && c1 == unit0 + cur.w.tiles, [&](int in) {
                              const int r = r0 + in;
                              const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
                              return p.out + (static_cast<int64_t>(cur.w.s.t0 + tok) * p.H + cur.kvh * p.G + (r - tok * p.G)) * D;
                            });
        return;
      }
      __syncwarp();
      fresh = true;
      unit0 = t + 1;
    }
    if (t + 1 < w1) cur.next(p);
  }
  cp_wait<0>();
}

constexpr int kJoinWarps = 4;

// Joins the tile kernel's parts of the cut unit that begins in CTA i's run:
// block y of 8 takes 32 of its 256 rows, a thread one row and every fourth
// group of 4 columns.
template <bool BF16, int D>
__device__ __forceinline__ void tile_join(const Params& p, int i, int y) {
  const Join u = p.joins[i];
  const int row = y * 32 + (threadIdx.x & 31), r = u.r0 + row, warp = threadIdx.x >> 5;
  if (u.last == 0 || r >= u.rows) return;
  auto part_of = [&](int k) { return k * 2ll + (k == i ? 1 : 0); };
  const float2* ml = reinterpret_cast<const float2*>(p.tile_ml);
  float m = -INFINITY;
#pragma unroll 4
  for (int k = i; k <= u.last; ++k) m = fmaxf(m, ml[part_of(k) * kUnitRows + row].x);
  const float ref = m == -INFINITY ? 0.0f : m;
  constexpr int C = D / 4 / kJoinWarps;  // column groups of a thread
  float sum = 0.0f;
  float4 acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
  for (int k = i; k <= u.last; ++k) {
    const float2 v = ml[part_of(k) * kUnitRows + row];
    const float f = ex2(v.x - ref);
    sum = fmaf(v.y, f, sum);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float4 o = reinterpret_cast<const float4*>(p.tile_o)[(part_of(k) * (D / 4) + c * kJoinWarps + warp) * kUnitRows + row];
      acc[c].x = fmaf(o.x, f, acc[c].x);
      acc[c].y = fmaf(o.y, f, acc[c].y);
      acc[c].z = fmaf(o.z, f, acc[c].z);
      acc[c].w = fmaf(o.w, f, acc[c].w);
    }
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
  uint16_t* dst = p.out + (static_cast<int64_t>(u.t0 + tok) * p.H + u.kvh * p.G + (r - tok * p.G)) * D;
#pragma unroll
  for (int c = 0; c < C; ++c)
    *reinterpret_cast<uint2*>(dst + (c * kJoinWarps + warp) * 4) =
        make_uint2(pack16<BF16>(acc[c].x * inv, acc[c].y * inv), pack16<BF16>(acc[c].z * inv, acc[c].w * inv));
}

// The parts of a query row: one for each worker whose run holds steps of the
// row's unit, or for each CTA whose kWarps runs all lie in it (at its first
// worker's place).  n = 0: no step covers the row (zeros); n = 1: the row
// kernel has written it.
template <int ROWS>
struct RowParts {
  int64_t unit0, run;
  int first, lead, group0, groups, n;  // workers, then groups CTAs, then workers
  __device__ __forceinline__ void find(int64_t begin, int64_t end, int64_t steps) {
    unit0 = begin;
    run = steps;
    first = static_cast<int>(div64(begin, run));
    const int last = static_cast<int>(div64(end - 1, run));
    const int from = first + (begin > first * run ? 1 : 0);             // runs from .. to - 1 lie in the unit
    const int to = last + ((last + 1) * run == end ? 1 : 0);
    group0 = (from + kWarps - 1) / kWarps;
    groups = max(0, to / kWarps - group0);
    lead = groups > 0 ? group0 * kWarps - first : last - first + 1;
    n = groups > 0 ? lead + groups + (last + 1 - (group0 + groups) * kWarps) : lead;
  }
  __device__ __forceinline__ int64_t at(int k, int row) const {
    const int w = k < lead ? first + k : k < lead + groups ? (group0 + k - lead) * kWarps
                                                           : (group0 + groups) * kWarps + (k - lead - groups);
    return (w * 2ll + (unit0 < w * run ? 0 : 1)) * ROWS + row;
  }
};

// Joins a row's parts (`row`: of its 16), SHARE warps together: every warp
// finds the maximum and the sum of all parts, a lane 32 parts apart (the first
// 32 kKept parts' in registers, loaded together), and adds every SHARE-th
// part's output, kBatch loaded together whatever their number; the warps' sums
// meet in shared memory.
template <bool BF16, int D, int SHARE, int ROWS>
__device__ __forceinline__ void join_row(const Params& p, const RowParts<ROWS>& rp, int row, uint32_t* dst,
                                         typename std::conditional<D == 128, float4, float2>::type (*sh_o)[32]) {
  constexpr int V = D / 32;  // columns of a lane, side by side
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  constexpr int kBatch = SHARE > 1 ? 8 : 4;
  constexpr int kKept = SHARE > 1 ? 8 : 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % SHARE;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  const int parts = rp.n;
  float sum = 0.0f, acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.0f;
  if (parts > 0) {
    float2 v[kKept];
#pragma unroll
    for (int c = 0; c < kKept; ++c) {
      v[c] = make_float2(-INFINITY, 0.0f);
      if (lane + 32 * c < parts) v[c] = ml[rp.at(lane + 32 * c, row)];
    }
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < kKept; ++c) mx = fmaxf(mx, v[c].x);
    for (int k = lane + 32 * kKept; k < parts; k += 32) mx = fmaxf(mx, ml[rp.at(k, row)].x);
    mx = warp_max(mx);
    const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
    for (int c = 0; c < kKept; ++c) {
      v[c].x = ex2(v[c].x - ref);  // the part's weight
      sum = fmaf(v[c].y, v[c].x, sum);
    }
    for (int k = lane + 32 * kKept; k < parts; k += 32) {
      const float2 u = ml[rp.at(k, row)];
      sum = fmaf(u.y, ex2(u.x - ref), sum);
    }
    sum = warp_sum(sum);
    for (int k0 = 0; k0 < parts; k0 += 32) {
      float f = v[0].x;
#pragma unroll
      for (int c = 1; c < kKept; ++c)
        if (k0 == 32 * c) f = v[c].x;
      if (k0 >= 32 * kKept) f = k0 + lane < parts ? ex2(ml[rp.at(k0 + lane, row)].x - ref) : 0.0f;
      const int n = min(32, parts - k0);
      for (int k = part; k < n; k += SHARE * kBatch) {
        Vec x[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          x[i] = Vec();
          if (k + i * SHARE < n) x[i] = reinterpret_cast<const Vec*>(p.part_o + rp.at(k0 + k + i * SHARE, row) * D)[lane];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const float c = __shfl_sync(0xffffffffu, f, (k + i * SHARE) & 31);
          if (k + i * SHARE >= n) break;
#pragma unroll
          for (int j = 0; j < V; ++j) acc[j] = fmaf(reinterpret_cast<const float*>(&x[i])[j], c, acc[j]);
        }
      }
    }
  }
  if (SHARE > 1) {  // all warps of the CTA are here
    Vec x;
#pragma unroll
    for (int j = 0; j < V; ++j) reinterpret_cast<float*>(&x)[j] = acc[j];
    __syncthreads();  // the row before has been read
    sh_o[warp][lane] = x;
    __syncthreads();
  }
  if (part == 0) {
#pragma unroll
    for (int k = 1; k < SHARE; ++k) {
      const Vec o = sh_o[k][lane];
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += reinterpret_cast<const float*>(&o)[j];
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int j = 0; j < V; j += 2) dst[lane * (V / 2) + j / 2] = pack16<BF16>(acc[j] * inv, acc[j + 1] * inv);
  }
}

// Joins the parts of the units that were cut, and writes zeros for the rows
// that no step covers: queries without keys and tokens of no sequence, in front
// of the first and behind the last.  An item is a (sequence, token, head); MODE says how the four
// warps of a CTA share them:
//   kRowCta    one item a CTA, all warps together: few items, each of many
//              parts (a single long sequence has one for every worker);
//   kRowWarp   an item a warp: many items, few of them cut;
//   kRowMixed  an item a warp, those of more than kAlone parts all warps
//              together (long sequences among short or empty ones).  A CTA's
//              items lie far apart, so that a long sequence's rows go to many SMs.
// Measured: one token of 16 sequences to 4000 keys with 32 heads 36.4 us with
// kRowCta, 38.0 with kRowWarp; 64 sequences to 8192 keys 217 with kRowCta, 211
// with the other two; one of 16384 keys among 63 of 100 29.4, 30.2 (kRowMixed)
// and 39.7 (kRowWarp); 7 tokens of 70 sequences 76, 51 and 47.
enum { kRowCta, kRowMixed, kRowWarp };
template <bool BF16, int D, int MODE, int KEYS, int ROWS>
__global__ void __launch_bounds__(kJoinWarps * 32) combine_kernel(const __grid_constant__ Params p) {
  using Vec = typename std::conditional<D == 128, float4, float2>::type;
  constexpr int W = kJoinWarps, kPerCta = MODE == kRowCta ? 1 : W;
  constexpr int kAlone = 16;
  __shared__ Vec sh_o[W][32];
  __shared__ int shared_item[W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row_ctas = (p.B * p.combine_rows * p.H + kPerCta - 1) / kPerCta;
  if (static_cast<int>(blockIdx.x) >= row_ctas) {
    const int at = blockIdx.x - row_ctas;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    tile_join<BF16, D>(p, at / 8, at % 8);
    return;
  }
  auto out_row = [&](int64_t tok, int head) { return reinterpret_cast<uint32_t*>(p.out + (tok * p.H + head) * D); };
  // What the index tensors say of an item.  They are older than the row
  // kernel; what else is read here is of the row kernel's.
  struct Item {
    Work w;
    int b, y, h, kvh;
    int64_t seq0, run;
  };
  const int limit = limit_of<KEYS, ROWS>(p);
  auto look = [&](int item) {
    Item it;
    it.h = item % p.H;
    it.y = item / p.H % p.combine_rows;
    it.b = item / p.H / p.combine_rows;
    it.kvh = static_cast<int>(fdiv(static_cast<uint32_t>(it.h), p.div_g));
    it.w = work_at<KEYS, ROWS>(p, min(it.b, p.B - 1), limit);
    it.seq0 = it.run = 0;
    if (p.B <= 32) {  // the list in one scan; else what the row kernel left
      int64_t mine = 0;
      int longest = 0;
      if (lane < p.B) {
        const Work w = work_at<KEYS, ROWS>(p, lane, limit);
        mine = steps_of(p, w);
        longest = w.tiles;
      }
      const int64_t upto = warp_scan(mine);
      it.run = run_of(p, __shfl_sync(0xffffffffu, upto, 31), __reduce_max_sync(0xffffffffu, longest));
      it.seq0 = __shfl_sync(0xffffffffu, upto - mine, min(it.b, 31));
    }
    return it;
  };
  auto finish_look = [&](Item& it) {
    if (p.B > 32) {
      it.seq0 = p.prefix[min(it.b, p.B - 1)];
      it.run = p.prefix[p.B + 1];
    }
  };
  auto parts_of = [&](const Item& it, int r) {
    RowParts<ROWS> rp;
    rp.n = 0;
    if (it.w.tiles > 0) {
      const int64_t begin = it.seq0 + (static_cast<int64_t>(it.kvh) * it.w.rts + r / ROWS) * it.w.tiles;
      rp.find(begin, begin + it.w.tiles, it.run);
    }
    return rp;
  };
  // Every row of an item whose parts `take` accepts, joined by SHARE warps.
  auto join = [&](const Item& it, auto share, auto take) {
    for (int i = it.y; i < it.w.s.m; i += p.combine_rows) {
      const int r = i * p.G + (it.h - it.kvh * p.G);
      const RowParts<ROWS> rp = parts_of(it, r);
      if (rp.n != 1 && take(rp.n))
        join_row<BF16, D, decltype(share)::value, ROWS>(p, rp, r % ROWS, out_row(it.w.s.t0 + i, it.h), sh_o);
    }
  };
  const std::integral_constant<int, 1> alone;
  const std::integral_constant<int, W> together;
  const int cta = static_cast<int>(blockIdx.x);
  const int item = MODE == kRowCta ? cta : MODE == kRowMixed ? warp * row_ctas + cta : cta * W + warp;
  Item it = look(item);
  const int first = min(max(__ldg(p.q_start), 0), p.T), end = min(max(__ldg(p.q_start + p.B), 0), p.T);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto zero = [&](int from, int to) {
    const int64_t words = static_cast<int64_t>(to - from) * p.H * (D / 2);
    uint32_t* dst = out_row(from, 0);
    const int64_t step = static_cast<int64_t>(row_ctas) * (W * 32);
    for (int64_t i = cta * static_cast<int64_t>(W * 32) + threadIdx.x; i < words; i += step) dst[i] = 0u;
  };
  zero(0, first);  // tokens in front of the first sequence, and behind the last
  zero(end, p.T);
  const bool real = it.b < p.B && static_cast<int64_t>(it.w.s.m) * p.G <= limit;  // else the tile kernel's, or none
  if (real) finish_look(it);
  if constexpr (MODE == kRowCta) {
    if (real) join(it, together, [](int) { return true; });
  } else if constexpr (MODE == kRowWarp) {
    if (real) join(it, alone, [](int) { return true; });
  } else {
    bool many = false;
    if (real) {
      join(it, alone, [&](int n) {
        many |= n > kAlone;
        return n <= kAlone;
      });
    }
    if (!__syncthreads_or(many)) return;
    if (lane == 0) shared_item[warp] = many ? item : -1;
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < W; ++k) {
      if (shared_item[k] < 0) continue;
      it = look(shared_item[k]);
      finish_look(it);
      join(it, together, [](int n) { return n > kAlone; });
    }
  }
}

#include "paged_rows8.cuh"

// Q8: over e4m3 caches, in units of ROWS query rows.
template <bool BF16, int D, int CAP, bool Q8, int ROWS>
int launch(const Params& p, int ctas, cudaStream_t st) {
  constexpr uint32_t kSmem = kWarps * (Q8 ? kRing8Bytes<ROWS> : kRingBytes);
  constexpr int KEYS = Q8 ? kKeys8 : kKeys;
  void (*kernel)(const Params);
  if constexpr (Q8) kernel = rows8_kernel<BF16, D, CAP, ROWS>;
  else kernel = rows_kernel<BF16, D, CAP>;
  static std::atomic<uint64_t> done{0};
  if (!attributes_set(done)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
      return B200K_ERR_LAUNCH;
    attributes_done(done);
  }
  const unsigned grid = static_cast<unsigned>(ctas + (p.tile_ctas > 0 ? 1 : 0));
  if (Q8) {
    if (const int rc = launch_early(kernel, grid, kWarps * 32, kSmem, st, p); rc != B200K_OK) return rc;
  } else {
    kernel<<<grid, kWarps * 32, kSmem, st>>>(p);
    if (cudaGetLastError() != cudaSuccess) return B200K_ERR_LAUNCH;
  }
  if (p.tile_ctas > 0) {
    const int rc = Q8 ? launch_tiles8(p, BF16, D, CAP, st) : launch_tiles(p, BF16, D, CAP, st);
    if (rc != B200K_OK) return rc;
  }
  // The combine's launch overlaps the row kernel's end (it waits for the
  // row kernel's writes itself, before it reads or writes anything).
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  const int per_cta = p.join_mode == kRowCta ? 1 : kJoinWarps;
  cfg.gridDim = dim3(static_cast<unsigned>((p.B * p.combine_rows * p.H + per_cta - 1) / per_cta + p.tile_ctas * 8));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  auto combine = p.join_mode == kRowCta     ? combine_kernel<BF16, D, kRowCta, KEYS, ROWS>
                 : p.join_mode == kRowMixed ? combine_kernel<BF16, D, kRowMixed, KEYS, ROWS>
                                            : combine_kernel<BF16, D, kRowWarp, KEYS, ROWS>;
  return cudaLaunchKernelEx(&cfg, combine, p) == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
}

template <bool BF16, int D, bool Q8, int ROWS>
int launch_cap(const Params& p, int cap, int ctas, cudaStream_t st) {
  if (cap == kNoCap) return launch<BF16, D, kNoCap, Q8, ROWS>(p, ctas, st);
  return cap == kCapPlain ? launch<BF16, D, kCapPlain, Q8, ROWS>(p, ctas, st) : launch<BF16, D, kCapSeries, Q8, ROWS>(p, ctas, st);
}
template <bool Q8, int ROWS>
int launch_type(const Params& p, bool bf16, int dim, int cap, int ctas, cudaStream_t st) {
  if (bf16) return dim == 64 ? launch_cap<true, 64, Q8, ROWS>(p, cap, ctas, st) : launch_cap<true, 128, Q8, ROWS>(p, cap, ctas, st);
  return dim == 64 ? launch_cap<false, 64, Q8, ROWS>(p, cap, ctas, st) : launch_cap<false, 128, Q8, ROWS>(p, cap, ctas, st);
}

}  // namespace
}  // namespace paged
}  // namespace b200k

using namespace b200k;
using namespace b200k::paged;

namespace {

int check_shape(const B200kPagedAttentionArgs* a) {
  if (!a) return B200K_ERR_ARG;
  if (a->tokens < 0 || a->seqs < 0 || a->heads < 0 || a->kv_heads < 0 || a->num_pages < 0 || a->page_size < 0 ||
      a->table_cols < 0)
    return B200K_ERR_SHAPE;
  if (a->tokens == 0 || a->heads == 0) return B200K_OK;  // empty output
  if (a->head_dim != 64 && a->head_dim != 128) return B200K_ERR_UNSUPPORTED;
  if (a->kv_heads == 0 || a->heads % a->kv_heads != 0) return B200K_ERR_SHAPE;
  if (a->tokens > 0x3fffffffLL || a->seqs > 0xffffffLL || a->heads > 65536 || a->page_size > 0x3fffffffLL ||
      a->num_pages > 0x3fffffffLL || a->table_cols > 0x3fffffffLL || a->tokens * (a->heads / a->kv_heads) > 0x3fffffffLL)
    return B200K_ERR_SHAPE;
  return B200K_OK;
}

// Sequences of more query rows than this run the tile kernel.  With 16 and 64
// in place of 32: 20 rows of 32 sequences to 4000 keys 82 and 75 us (32: 75),
// 32 rows 85 and 91 (91), 20 rows of 2 sequences to 1000 keys 28 and 12 (12), up
// to 68 rows of 8 sequences to 1500 keys, heads of 64, 22 and 29 (27).  Those are
// figures of 16-bit caches; e4m3 ones take the same limits, which are low for them:
// row and tile kernel, 36 rows of 16 sequences to 4000 keys, 88 and 121 us, 64 rows
// 115 and 121, 68 rows of 8 sequences to 1500 keys, heads of 64, 36 and 38.
constexpr int kLongRows = 32;

// ... and sequences of more rows than one block of the row kernel where all
// such have this many steps of 128 values together.  Five tokens of 16
// sequences, 32 / 8 heads of 128, to 1000 (8000 steps), 2000, 4000 and 8000
// keys: row kernel 30, 52, 90 and 165 us, tile kernel 32, 44, 64 and 108.  Over e4m3
// caches, whose steps are twice the keys, to 2000, 4000 and 8000 keys: row kernel 41,
// 66 and 111, tile kernel 77, 119 and 197, so there the row kernel would do.  Only
// the device knows the lengths; where the page table could hold as many steps
// the tile kernel is launched, which costs 2 to 6 us when it has no work.
constexpr int64_t kMidSteps = 12288;
// Sequences that the limit is worked out for: every warp goes over them.
constexpr int kMidSeqs = 256;

int64_t most_rows(const B200kPagedAttentionArgs* a) {
  const int64_t q = a->max_q_len > 0 ? std::min<int64_t>(a->max_q_len, a->tokens) : a->tokens;
  return q * (a->heads / a->kv_heads);
}
int64_t mid_steps(const B200kPagedAttentionArgs* a, bool q8) {
  const int step = q8 ? kKeys8 : kKeys;
  const int64_t steps = kMidSteps * 128 / a->head_dim * kKeys / step;
  const int64_t keys = std::min<int64_t>(a->table_cols * a->page_size, 0x3fffffff);
  const bool reach = a->seqs <= kMidSeqs && a->seqs * a->kv_heads * (keys / step + 1) >= steps;
  return most_rows(a) > kRows && reach ? steps : 0;
}
bool may_be_long(const B200kPagedAttentionArgs* a, bool q8) { return most_rows(a) > kLongRows || mid_steps(a, q8) > 0; }

// Entries of the tile kernel's list: 256-row blocks of sequences that share the
// tokens out among them.
int64_t max_entries(const B200kPagedAttentionArgs* a) {
  return a->tokens * (a->heads / a->kv_heads) / kUnitRows + a->seqs;
}

// Where each part of the workspace begins; returns its size.
int64_t place(const B200kPagedAttentionArgs* a, bool q8, int sms, uint8_t* ws, Params* p) {
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    uint8_t* r = ws + at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  static_assert(kCtas8<128, 8> * 8 <= kCtasPerSm * kRows, "parts of units of 8 rows");
  const int64_t slots = static_cast<int64_t>(sms) * kCtasPerSm * kWarps * 2 * kRows;
  uint8_t* part_o = take(slots * a->head_dim * 4);
  uint8_t* part_ml = take(slots * 8);
  uint8_t* prefix = take((a->seqs + 2) * 8);
  uint8_t *steps = ws, *entries = ws, *tile_o = ws, *tile_ml = ws, *joins = ws;
  if (may_be_long(a, q8)) {
    const int64_t n = max_entries(a) + 1;
    steps = take((n + 4) * 8);
    entries = take(n * 8);
    tile_o = take(static_cast<int64_t>(sms) * 2 * kUnitRows * a->head_dim * 4);
    tile_ml = take(static_cast<int64_t>(sms) * 2 * kUnitRows * 8);
    joins = take(static_cast<int64_t>(sms) * sizeof(Join));
  }
  if (p) {
    p->part_o = reinterpret_cast<float*>(part_o);
    p->part_ml = reinterpret_cast<float*>(part_ml);
    p->prefix = reinterpret_cast<int64_t*>(prefix);
    p->entry_steps = reinterpret_cast<int64_t*>(steps);
    p->entries = reinterpret_cast<int2*>(entries);
    p->tile_o = reinterpret_cast<float*>(tile_o);
    p->tile_ml = reinterpret_cast<float*>(tile_ml);
    p->joins = reinterpret_cast<Join*>(joins);
  }
  return at;
}

int workspace(const B200kPagedAttentionArgs* a, bool q8, int64_t* bytes) {
  const int rc = check_shape(a);
  if (rc != B200K_OK) return rc;
  if (!bytes) return B200K_ERR_ARG;
  *bytes = 0;
  if (a->tokens == 0 || a->heads == 0) return B200K_OK;
  const int sms = device_sm_count();
  if (sms <= 0) return B200K_ERR_DEVICE;
  *bytes = place(a, q8, sms, nullptr, nullptr);
  return B200K_OK;
}

// `q8` (NULL: 16-bit caches): the scales.
int attend(const B200kPagedAttentionArgs* a, const B200kPagedAttentionQuantArgs* q8, void* stream_) {
  const int rc = check_shape(a);
  if (rc != B200K_OK) return rc;
  if (a->tokens == 0 || a->heads == 0) return B200K_OK;
  if (!a->q || !a->out) return B200K_ERR_ARG;
  if (a->dtype != B200K_BF16 && a->dtype != B200K_F16) return B200K_ERR_UNSUPPORTED;
  if (!(a->softcap >= 0.0f) || !std::isfinite(2.0f * a->softcap * kLog2e) || a->window < 0 || !(a->scale >= 0.0f) ||
      !std::isfinite(a->scale))
    return B200K_ERR_ARG;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->out)) return B200K_ERR_ALIGN;
  for (int d = 0; d < 2; ++d)
    if (a->q_strides[d] < 0 || a->q_strides[d] % 8) return B200K_ERR_ALIGN;
  for (int d = 0; d < 3; ++d)
    if (a->cache_strides[d] < 0 || a->cache_strides[d] % (q8 ? 16 : 8)) return B200K_ERR_ALIGN;
  const int sms = device_sm_count();
  if (sms <= 0) return B200K_ERR_DEVICE;
  cudaStream_t st = static_cast<cudaStream_t>(stream_);
  const int64_t keys = std::min<int64_t>(a->table_cols * a->page_size, 0x3fffffff);
  if (a->seqs == 0 || keys == 0 || a->num_pages == 0) {  // no keys at all: every row is zero
    const size_t n = static_cast<size_t>(a->tokens) * a->heads * a->head_dim * 2;
    return cudaMemsetAsync(a->out, 0, n, st) == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
  }
  if (!a->k_cache || !a->v_cache || !a->page_table || !a->q_start || !a->kv_len) return B200K_ERR_ARG;
  if (q8) {
    if (!q8->k_scale || !q8->v_scale) return B200K_ERR_ARG;
    for (int d = 0; d < 3; ++d)
      if (q8->scale_strides[d] < 0) return B200K_ERR_SHAPE;
  }
  if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < place(a, q8 != nullptr, sms, nullptr, nullptr)) return B200K_ERR_ARG;
  Params p;
  std::memset(&p, 0, sizeof(p));
  p.T = static_cast<int32_t>(a->tokens);
  p.B = static_cast<int32_t>(a->seqs);
  p.H = static_cast<int32_t>(a->heads);
  p.Hkv = static_cast<int32_t>(a->kv_heads);
  p.G = p.H / p.Hkv;
  p.page_size = static_cast<int32_t>(a->page_size);
  p.num_pages = static_cast<int32_t>(a->num_pages);
  p.table_cols = static_cast<int32_t>(a->table_cols);
  p.capacity = static_cast<int32_t>(keys);
  p.window = static_cast<int32_t>(std::min<int64_t>(a->window, 0x3fffffff));
  p.tile_ctas = may_be_long(a, q8 != nullptr) ? sms : 0;
  p.max_entries = static_cast<int32_t>(max_entries(a));
  p.long_rows = p.tile_ctas > 0 ? kLongRows : 0x7fffffff;
  p.mid_steps = mid_steps(a, q8 != nullptr);
  p.test_flags = a->test_flags;
  p.div_page = make_fastdiv(static_cast<uint32_t>(p.page_size));
  p.div_g = make_fastdiv(static_cast<uint32_t>(p.G));
  p.table_stride = a->table_stride;
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_t = a->q_strides[0];
  p.q_h = a->q_strides[1];
  p.k = static_cast<const uint16_t*>(a->k_cache);
  p.v = static_cast<const uint16_t*>(a->v_cache);
  p.c_page = a->cache_strides[0];
  p.c_slot = a->cache_strides[1];
  p.c_head = a->cache_strides[2];
  if (q8) {
    p.k8 = static_cast<const uint8_t*>(a->k_cache);
    p.v8 = static_cast<const uint8_t*>(a->v_cache);
    p.ks = q8->k_scale;
    p.vs = q8->v_scale;
    p.s_page = q8->scale_strides[0];
    p.s_slot = q8->scale_strides[1];
    p.s_head = q8->scale_strides[2];
    p.c16_page = static_cast<uint32_t>(p.c_page / 16);
    p.c16_slot = static_cast<uint32_t>(p.c_slot / 16);
    p.c16_head = static_cast<uint32_t>(p.c_head / 16);
    auto last = [&](int64_t page, int64_t slot, int64_t head) {
      return static_cast<double>(a->num_pages) * page + static_cast<double>(a->page_size) * slot + static_cast<double>(a->kv_heads) * head;
    };
    p.far_rows = last(p.c_page, p.c_slot, p.c_head) / 16 > 4.2e9 || last(p.s_page, p.s_slot, p.s_head) > 4.2e9;
  }
  p.out = static_cast<uint16_t*>(a->out);
  p.table = a->page_table;
  p.q_start = a->q_start;
  p.kv_len = a->kv_len;
  const int cap = a->softcap == 0.0f ? kNoCap : a->softcap <= kPlainCap ? kCapPlain : kCapSeries;
  const float scale = a->scale > 0.0f ? a->scale : 1.0f / std::sqrt(static_cast<float>(a->head_dim));
  p.mul = cap != kNoCap ? 2.0f * scale / a->softcap * kLog2e : scale * kLog2e;
  p.lin = scale * kLog2e;
  p.cap2 = a->softcap * kLog2e;
  if (!std::isfinite(p.mul) || !std::isfinite(p.lin)) return B200K_ERR_ARG;  // a cap too small for its scale
  // Over e4m3 caches, when no sequence is said to have more than 8 query rows,
  // units of so many.
  const bool few = q8 && most_rows(a) <= 8;
  const int ctas = sms * (few ? kCtas8<128, 8> : kCtasPerSm);
  p.workers = ctas * kWarps;
  place(a, q8 != nullptr, sms, static_cast<uint8_t*>(a->workspace), &p);
  p.status = a->status;
  p.timeout_ns = a->timeout_ns > 0 ? a->timeout_ns : 2000000000ll;
  // The combine covers this many tokens of a sequence side by side and the
  // rest in a loop; its grid stays below 2^31 CTAs.
  const int64_t per_token = static_cast<int64_t>(p.B) * p.H;
  if (per_token > 0x1fffffffLL) return B200K_ERR_SHAPE;
  int64_t rows = a->max_q_len > 0 ? std::min<int64_t>(a->max_q_len, a->tokens) : a->tokens;
  if (p.tile_ctas > 0) rows = std::min<int64_t>(rows, kLongRows / p.G);
  p.combine_rows = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(rows, 0x1fffffff / per_token)));
  const int64_t items = per_token * p.combine_rows;
  p.join_mode = items <= 4ll * sms ? kRowCta : items <= 16ll * sms ? kRowMixed : kRowWarp;
  const bool bf16 = a->dtype == B200K_BF16;
  const int dim = static_cast<int>(a->head_dim);
  if (!q8) return launch_type<false, kRows>(p, bf16, dim, cap, ctas, st);
  return few ? launch_type<true, 8>(p, bf16, dim, cap, ctas, st) : launch_type<true, kRows>(p, bf16, dim, cap, ctas, st);
}

}  // namespace

extern "C" int b200k_paged_attention_workspace(const B200kPagedAttentionArgs* a, int64_t* bytes) {
  return workspace(a, false, bytes);
}
extern "C" int b200k_paged_attention(const B200kPagedAttentionArgs* a, void* stream_) { return attend(a, nullptr, stream_); }
extern "C" int b200k_paged_attention_quant_workspace(const B200kPagedAttentionQuantArgs* a, int64_t* bytes) {
  return workspace(a ? &a->base : nullptr, true, bytes);
}
extern "C" int b200k_paged_attention_quant(const B200kPagedAttentionQuantArgs* a, void* stream_) {
  return a ? attend(&a->base, a, stream_) : B200K_ERR_ARG;
}
