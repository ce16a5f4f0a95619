// The tile kernel of b200k_paged_attention_quant: sequences with many query
// rows over e4m3 caches.  The plan, the portions, the products and the parts
// are the 16-bit tile kernel's (paged_tiles.cu); here
//   warps 12, 13 load codes (TMA boxes or 16-byte cp.async copies) and scales,
//   warps 16, 17 and 18, 19 turn a block's key and value codes into f16 tiles in
//                shared memory (a conversion for two codes, exact) and, for
//                bf16, a portion's queries too, each row with its power of two
//                (row_scale); they leave the keys' scales and the values'
//                scales' logarithms and reciprocals for the softmax;
//   warps 0-7    put the scales into the scores: paged.cuh has the formulas.
// Both products are f16 ones.  The registers are shared out by setmaxnreg: five
// warpgroups are launched with 96 a thread.
#include "paged_tiles.cuh"

namespace b200k {
namespace paged {
namespace {

constexpr int kThreads8 = 640;
constexpr int kLaunchRegs = 96, kSoftmaxRegs = 144, kIssueRegs = 56, kConvertRegs = 80;
static_assert(2 * kSoftmaxRegs + 2 * kIssueRegs + kConvertRegs <= 5 * kLaunchRegs, "what the launch has");
constexpr int kScaleSlots = 4;  // blocks whose scales are held for the softmax
template <int D>
struct Layout8 {
  static constexpr int kStages = D == 128 ? 3 : 4;         // of f16 keys and of values
  static constexpr int kRaw = D == 128 ? 3 : 4;            // of codes
  static constexpr uint32_t kTile = kHalfTile * (D / 64);  // a query tile
  static constexpr uint32_t kBlk = kHalfBlk * (D / 64);    // an f16 block
  static constexpr uint32_t kCodes = kBlock * D;           // a block of codes
  static constexpr uint32_t kOffK = 2 * kTile;
  static constexpr uint32_t kOffV = kOffK + kStages * kBlk;
  static constexpr uint32_t kOffRawK = kOffV + kStages * kBlk;
  static constexpr uint32_t kOffRawV = kOffRawK + kRaw * kCodes;
  static constexpr uint32_t kOffRawKs = kOffRawV + kRaw * kCodes;      // [kRaw][64] scales
  static constexpr uint32_t kOffRawVs = kOffRawKs + kRaw * kBlock * 4;
  static constexpr uint32_t kOffSc = kOffRawVs + kRaw * kBlock * 4;    // [kScaleSlots][3][64]: ks, log2 vs, 1 / vs
  static constexpr uint32_t kOffRs = kOffSc + kScaleSlots * 3 * kBlock * 4;  // [2][256]: the rows' powers of two
  static constexpr uint32_t kOffBar = kOffRs + 2 * kUnitRows * 4;
  static constexpr uint32_t kSmem = 1024 + kOffBar + 1024;
  static_assert(kSmem <= 232448 && kSmem > 116 * 1024, "one CTA per SM");
};
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kTmemO = 256;
// Tensor-memory columns as in the 16-bit kernel: scores of block g of tile t at
// 128 t + 64 (g & 1), its weights in the first 32 of them, O_t at 256 + D t.

template <bool BF16, int D, int CAP>
__global__ void __launch_bounds__(kThreads8, 1)
    tiles8_kernel(const __grid_constant__ Params p, const __grid_constant__ CUtensorMap tm_q,
                  const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using L = Layout8<D>;
  constexpr int S = L::kStages, R = L::kRaw;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sbase = smem_raw + (((smem_u32(smem_raw) + 1023u) & ~1023u) - smem_u32(smem_raw));
  uint8_t* sQ = sbase;
  uint8_t* sK = sbase + L::kOffK;
  uint8_t* sV = sbase + L::kOffV;
  float* sc = reinterpret_cast<float*>(sbase + L::kOffSc);
  float* rs = reinterpret_cast<float*>(sbase + L::kOffRs);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sbase + L::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* rk_full = q_empty + 1;   // codes
  uint64_t* rk_empty = rk_full + R;
  uint64_t* rv_full = rk_empty + R;
  uint64_t* rv_empty = rv_full + R;
  uint64_t* k_full = rv_empty + R;   // f16
  uint64_t* k_empty = k_full + S;
  uint64_t* v_full = k_empty + S;
  uint64_t* v_empty = v_full + S;
  uint64_t* s_full = v_empty + S;    // [4] by tile and buffer
  uint64_t* p_full = s_full + 4;     // [4]
  uint64_t* o_done = p_full + 4;     // [4]
  uint64_t* o_free = o_done + 4;     // [2] by tile
  uint64_t* drain = o_free + 2;      // [4] by issuer
  uint64_t* sc_full = drain + 4;     // [kScaleSlots]
  uint64_t* sc_empty = sc_full + kScaleSlots;
  uint64_t* rs_full = sc_empty + kScaleSlots;  // [2] by portion: bf16 queries converted
  uint64_t* rs_empty = rs_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rs_empty + 2);
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
    gemm::mbar_init(q_full, 64);
    gemm::mbar_init(q_empty, 2);
    for (int s = 0; s < R; ++s) {
      gemm::mbar_init(&rk_full[s], 33);
      gemm::mbar_init(&rk_empty[s], 2);
      gemm::mbar_init(&rv_full[s], 33);
      gemm::mbar_init(&rv_empty[s], 2);
    }
    for (int s = 0; s < S; ++s) {
      gemm::mbar_init(&k_full[s], 2);
      gemm::mbar_init(&k_empty[s], 2);
      gemm::mbar_init(&v_full[s], 2);
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
      gemm::mbar_init(&rs_full[t], 4);
      gemm::mbar_init(&rs_empty[t], 8);
    }
    for (int i = 0; i < kScaleSlots; ++i) {
      gemm::mbar_init(&sc_full[i], 2);
      gemm::mbar_init(&sc_empty[i], 8);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    const int t = warp & 1;
    const bool scores = warp < 10;
    // fp32 accumulators of f16; B of Q K^T K-major, of P V N-major
    const uint32_t idesc_s = (1u << 4) | ((kBlock >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17) | ((128u >> 4) << 24);
    const uint32_t tS = tmem_base + t * 128, tO = tmem_base + kTmemO + t * D;
    const uint64_t dq = gemm::sw128_desc(smem_u32(sQ) + t * L::kTile, 16, 1024);
    const uint64_t dk = gemm::sw128_desc(smem_u32(sK), 16, 1024);
    const uint64_t dv = gemm::sw128_desc(smem_u32(sV), kHalfBlk, 1024);
    uint64_t* full = scores ? k_full : v_full;
    uint64_t* empty = scores ? k_empty : v_empty;
    int c = 0;      // key blocks passed, over all portions
    int g = 0;      // of them this tile's
    int done = 0;   // portions in which this tile had steps
    bool ok = true;
    for (int li = 0; ok && walk.next(p, po); ++li) {
      if (scores) {
        ok = BF16 ? warp_wait(&rs_full[li & 1], (li >> 1) & 1, ctl) : warp_wait(q_full, li & 1, ctl);
        if (!BF16 && p.q_box == 0) gemm::fence_async_smem();
      }
      for (int j = po.beg; ok && j < po.end; ++j, ++c) {
        const int st = c % S;
        if (!(ok = warp_wait(&full[st], (c / S) & 1, ctl))) break;
        if (j < po.t_beg[t] || j >= po.t_end[t]) {
          // not a block of this tile
          if (lane == 0) gemm::mbar_arrive(&empty[st]);
          __syncwarp();
          continue;
        }
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
  } else if (warp >= 16) {
    // ----------------------------------------------------------------- converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
    const bool is_v = warp >= 18;
    const int half_of = warp & 1;  // of a block's chunks
    uint8_t* raw = sbase + (is_v ? L::kOffRawV : L::kOffRawK);
    const float* raw_sc = reinterpret_cast<const float*>(sbase + (is_v ? L::kOffRawVs : L::kOffRawKs));
    uint8_t* dst0 = is_v ? sV : sK;
    uint64_t* r_full = is_v ? rv_full : rk_full;
    uint64_t* r_empty = is_v ? rv_empty : rk_empty;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    constexpr int kChunks = D / 16;            // 16-byte chunks of a row of codes
    constexpr int kEach = kBlock * kChunks / 64;
    int c = 0;
    bool ok = true;
    for (int li = 0; ok && walk.next(p, po); ++li) {
      if (BF16) {
        // the portion's queries in place, a row of each tile a thread
        if (!(ok = warp_wait(q_full, li & 1, ctl) && warp_wait(&rs_empty[li & 1], ((li >> 1) & 1) ^ 1, ctl))) break;
        const int row = (warp - 16) * 32 + lane;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (walk.u.r0 + t * 128 >= walk.u.rows) break;
          uint8_t* q = sQ + t * L::kTile + row * 128;
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < D / 8; ++k) {
            const uint4 x = *reinterpret_cast<const uint4*>(q + (k >> 3) * kHalfTile + (((k & 7) ^ (row & 7)) << 4));
#pragma unroll
            for (uint32_t w : {x.x, x.y, x.z, x.w}) top = max(top, max((w << 16) & 0x7fffffffu, w & 0x7fff0000u));
          }
          const RowScale s = row_scale(top);
#pragma unroll
          for (int k = 0; k < D / 8; ++k) {
            uint4* at = reinterpret_cast<uint4*>(q + (k >> 3) * kHalfTile + (((k & 7) ^ (row & 7)) << 4));
            const uint4 x = *at;
            *at = make_uint4(bf16_to_f16(x.x, s.div), bf16_to_f16(x.y, s.div), bf16_to_f16(x.z, s.div), bf16_to_f16(x.w, s.div));
          }
          rs[(li & 1) * kUnitRows + t * 128 + row] = s.mul;
        }
        gemm::fence_async_smem();
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&rs_full[li & 1]);
      }
      for (int j = po.beg; j < po.end; ++j, ++c) {
        const int rst = c % R, st = c % S, slot = c % kScaleSlots;
        if (!(ok = warp_wait(&r_full[rst], (c / R) & 1, ctl))) break;
        if (!(ok = warp_wait(&empty[st], ((c / S) & 1) ^ 1, ctl))) break;
        const uint4* src = reinterpret_cast<const uint4*>(raw + rst * L::kCodes) + half_of * 32 + lane;
        uint8_t* dst = dst0 + st * L::kBlk;
#pragma unroll 4
        for (int i = 0; i < kEach; ++i) {
          const int idx = i * 64 + half_of * 32 + lane, row = idx / kChunks, ch = idx % kChunks;
          const uint4 x = src[i * 64];
          const uint4 a = make_uint4(codes_lo(x.x), codes_hi(x.x), codes_lo(x.y), codes_hi(x.y));
          const uint4 b = make_uint4(codes_lo(x.z), codes_hi(x.z), codes_lo(x.w), codes_hi(x.w));
          // two 16-byte chunks of f16; the upper half's lanes write theirs the
          // other way round, so that eight lanes cover all banks
          uint8_t* to = dst + (ch >> 2) * kHalfBlk + row * 128;
          const int c0 = (ch & 3) * 2, turn = (ch >> 2) & 1;
          *reinterpret_cast<uint4*>(to + (((c0 + turn) ^ (row & 7)) << 4)) = turn ? b : a;
          *reinterpret_cast<uint4*>(to + (((c0 + 1 - turn) ^ (row & 7)) << 4)) = turn ? a : b;
        }
        if (half_of == 0) {
          if (!(ok = warp_wait(&sc_empty[slot], ((c / kScaleSlots) & 1) ^ 1, ctl))) break;
          float* to = sc + slot * 3 * kBlock;
#pragma unroll
          for (int i = lane; i < kBlock; i += 32) {
            const float x = raw_sc[rst * kBlock + i];
            if (is_v) {
              const float v = value_scale(x);
              to[kBlock + i] = lg2(v);
              to[2 * kBlock + i] = 1.0f / v;
            } else {
              to[i] = x;
            }
          }
        }
        gemm::fence_async_smem();  // the tile's writes, before the MMA's reads
        __syncwarp();
        if (lane == 0) {
          gemm::mbar_arrive(&full[st]);
          gemm::mbar_arrive(&r_empty[rst]);
          if (half_of == 0) gemm::mbar_arrive(&sc_full[slot]);
        }
      }
    }
    __syncwarp();
  } else if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp < 14) {
      // ------------------------------------------------------------------ loaders
      // warp 12: keys and the queries of tile 0; warp 13: values and tile 1
      const bool is_v = warp == 13;
      constexpr int kChunks = D / 16, kRowsPerCp = 32 / kChunks;
      const int ch = lane % kChunks, sub = lane / kChunks;
      const uint32_t ring = smem_u32(sbase + (is_v ? L::kOffRawV : L::kOffRawK));
      const uint32_t ring_sc = smem_u32(sbase + (is_v ? L::kOffRawVs : L::kOffRawKs));
      uint64_t* full = is_v ? rv_full : rk_full;
      uint64_t* empty = is_v ? rv_empty : rk_empty;
      const uint8_t* cache = is_v ? p.v8 : p.k8;
      const float* scales = is_v ? p.vs : p.ks;
      const CUtensorMap* map = is_v ? &tm_v : &tm_k;
      const int box = p.box_rows;                    // 0: no TMA
      const int boxes = box > 0 ? kBlock / box : 0;
      int c = 0;
      bool ok = true;
      for (int li = 0; ok && walk.next(p, po); ++li) {
        const Unit& u = walk.u;
        for (int j = po.beg; j < po.end; ++j, ++c) {
          const int st = c % R, key0 = j * kBlock;
          const uint32_t dst = ring + st * L::kCodes;
          // this lane's keys: lane and lane + 32
          Place8 at[2];
          int pages[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int key = key0 + i * 32 + lane;
            pages[i] = -1;
            if (key >= u.s.lo && key < u.s.n)
              pages[i] = __ldg(p.table + u.b * p.table_stride + fdiv(static_cast<uint32_t>(key), p.div_page));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) at[i] = place8(p, pages[i], key0 + i * 32 + lane, u.s.lo, u.s.n, po.kvh);
          const bool tma = box > 0 && __all_sync(0xffffffffu, at[0].row >= 0 && at[1].row >= 0);  // every row is a key
          if (!(ok = warp_wait(&empty[st], ((c / R) & 1) ^ 1, ctl))) break;
          if (lane == 0) {
            if (tma) gemm::mbar_arrive_expect_tx(&full[st], L::kCodes);
            else gemm::mbar_arrive(&full[st]);
          }
          __syncwarp();
          if (tma) {
            const int key = key0 + lane * box;  // of box `lane`: its page is with another lane
            const int in = (lane * box) & 63;
            const int pa = __shfl_sync(0xffffffffu, pages[0], in & 31), pb = __shfl_sync(0xffffffffu, pages[1], in & 31);
            if (lane < boxes) {
              const uint32_t pi = fdiv(static_cast<uint32_t>(key), p.div_page);
              tma_load_4d(dst + lane * box * D, map, &full[st], 0, key - static_cast<int>(pi) * p.page_size, po.kvh,
                          in < 32 ? pa : pb);
            }
            __syncwarp();
          } else {
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll 2
              for (int i = 0; i < 32; i += kRowsPerCp) {
                const int64_t o = __shfl_sync(0xffffffffu, at[part].row, i + sub);
                cp16(dst + (part * 32 + i + sub) * D + ch * 16, cache + (o >= 0 ? o : 0) + ch * 16, o >= 0);
              }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i)
            cp4(ring_sc + (st * kBlock + i * 32 + lane) * 4, scales + (at[i].scale >= 0 ? at[i].scale : 0), at[i].scale >= 0);
          cp_arrive(&full[st]);
          if (j == po.beg) {
            // the portion's queries, when the products of the one before have read theirs
            if (li > 0 && !(ok = warp_wait(q_empty, (li - 1) & 1, ctl))) break;
            const int t = is_v ? 1 : 0;
            if (p.q_box > 0) {
              // tiles of 128 / G tokens
              const int r0 = u.r0 + t * 128;
              if (lane < D / 64 && r0 < u.rows) {
                gemm::mbar_arrive_expect_tx(q_full, kHalfTile);
                tma_load_4d(smem_u32(sQ) + t * L::kTile + lane * kHalfTile, &tm_q, q_full, lane * 64, 0, po.kvh,
                            u.s.t0 + static_cast<int>(fdiv(static_cast<uint32_t>(r0), p.div_g)));
              } else {
                gemm::mbar_arrive(q_full);
              }
              __syncwarp();
            } else {
              constexpr int kQChunks = D / 8, kQRows = 32 / kQChunks;
              const int qc = lane % kQChunks, qsub = lane / kQChunks;
#pragma unroll 4
              for (int i = 0; i < 128 / kQRows; ++i) {
                const int in = i * kQRows + qsub;  // row of the tile
                const int r = u.r0 + t * 128 + in;
                const bool real = r < u.rows;
                const uint32_t tok = fdiv(static_cast<uint32_t>(real ? r : u.r0), p.div_g);
                const int hg = (real ? r : u.r0) - tok * p.G;
                const uint16_t* src = p.q + static_cast<int64_t>(u.s.t0 + tok) * p.q_t +
                                      static_cast<int64_t>(po.kvh * p.G + hg) * p.q_h + qc * 8;
                cp16(smem_u32(sQ) + t * L::kTile + (qc >> 3) * kHalfTile + in * 128 + (((qc & 7) ^ (in & 7)) << 4), src, real);
              }
              cp_arrive(q_full);
            }
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      // The last TMA boxes have landed when the converters are done with them;
      // after a timeout they are waited for here.
      if (!ok) {
        for (int k = max(0, c - R); k < c; ++k) gemm::wait_bar_drain(&full[k % R], (k / R) & 1, 100000000ull);
      }
      __syncwarp();
    }
  } else {
    // -------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int t = warp >> 2, quarter = warp & 3;
    const int in_unit = t * 128 + quarter * 32 + lane;
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t tS = t_lane + t * 128, tO = t_lane + kTmemO + t * D;
    int g = 0, c = 0;
    bool ok = true;
    for (int li = 0; ok && walk.next(p, po); ++li) {
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
      float row_mul = CAP == kNoCap ? p.mul : 1.0f;
      if (BF16) {
        if (!(ok = warp_wait(&rs_full[li & 1], (li >> 1) & 1, ctl))) break;
        if (real) row_mul *= rs[(li & 1) * kUnitRows + in_unit];
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&rs_empty[li & 1]);
      }
      float m = -INFINITY, l = 0.0f;
      const int jb = po.t_beg[t], je = po.t_end[t];
      for (int j = po.beg; j < po.end; ++j, ++c) {
        const int slot = c % kScaleSlots;
        if (!(ok = warp_wait(&sc_full[slot], (c / kScaleSlots) & 1, ctl))) break;
        if (j < jb || j >= je) {  // not a block of this tile
          if (lane == 0) gemm::mbar_arrive(&sc_empty[slot]);
          __syncwarp();
          continue;
        }
        const uint32_t buf = g & 1;
        if (!(ok = warp_wait(&s_full[t * 2 + buf], (g >> 1) & 1, ctl))) break;
        gemm::tc_fence_after();
        const float4* ks4 = reinterpret_cast<const float4*>(sc + slot * 3 * kBlock);
        const float4* lv4 = ks4 + kBlock / 4;
        const float4* iv4 = lv4 + kBlock / 4;
        float s[kBlock];
        {
          uint32_t raw[kBlock / 32][32];
#pragma unroll
          for (int c = 0; c < kBlock / 32; ++c) gemm::tmem_ld32(tS + buf * 64 + c * 32, raw[c]);
          gemm::tmem_wait_ld();
          const float2 mul2 = make_float2(row_mul, row_mul);
#pragma unroll
          for (int i = 0; i < kBlock; i += 4) {
            const float4 k = ks4[i / 4], v = lv4[i / 4];
            const float2 x0 = make_float2(__uint_as_float(raw[i / 32][i % 32]), __uint_as_float(raw[i / 32][i % 32 + 1]));
            const float2 x1 = make_float2(__uint_as_float(raw[i / 32][i % 32 + 2]), __uint_as_float(raw[i / 32][i % 32 + 3]));
            const float2 m0 = __fmul2_rn(make_float2(k.x, k.y), mul2), m1 = __fmul2_rn(make_float2(k.z, k.w), mul2);
            float2 y0, y1;
            if (CAP == kNoCap) {
              y0 = __ffma2_rn(x0, m0, make_float2(v.x, v.y));
              y1 = __ffma2_rn(x1, m1, make_float2(v.z, v.w));
            } else {
              y0 = make_float2(score<CAP>(p, x0.x * m0.x) + v.x, score<CAP>(p, x0.y * m0.y) + v.y);
              y1 = make_float2(score<CAP>(p, x1.x * m1.x) + v.z, score<CAP>(p, x1.y * m1.y) + v.w);
            }
            s[i] = y0.x;
            s[i + 1] = y0.y;
            s[i + 2] = y1.x;
            s[i + 3] = y1.y;
          }
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
        const float top = max2(max3(mx[0], mx[1], mx[2]), mx[3]);
        const float was = m;
        float alpha = 1.0f;
        bool moved = false;
        // A NaN score, and an infinite one (0 * top), makes the maximum NaN and
        // with it every weight and sum of the row from here on.
        if (!(top <= m + kLagF16)) {
          m = fmaf(0.0f, top, top);
          alpha = ex2(was - m);
          moved = j > jb;
        }
        // weights are rounded to f16, half a step each down to 2^-26 of the row's
        // largest (smaller ones by less than 2^-36 of it)
        const float ref = (m == -INFINITY ? 0.0f : m) - (kF16Reach - kLagF16);
        float2 sum2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 nm2 = make_float2(-ref, -ref);
        uint32_t pk[kBlock / 2];
#pragma unroll
        for (int c = 0; c < kBlock; c += 4) {
          const float4 iv = iv4[c / 4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = c + 2 * h;
            const float2 x = __fadd2_rn(make_float2(s[at], s[at + 1]), nm2);
            const float2 e = at % kFmaEvery == kFmaEvery - 2 ? ex2_fma<false>(x) : make_float2(ex2(x.x), ex2(x.y));
            sum2[h] = __ffma2_rn(e, h ? make_float2(iv.z, iv.w) : make_float2(iv.x, iv.y), sum2[h]);
            pk[at / 2] = pack16<false>(e.x, e.y);
          }
        }
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&sc_empty[slot]);
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
        ++g;
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

template <bool BF16, int D, int CAP>
int launch(Params p, cudaStream_t st) {
  auto kernel = tiles8_kernel<BF16, D, CAP>;
  static std::atomic<uint64_t> done{0};
  if (!attributes_set(done)) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess || fa.numRegs < kLaunchRegs ||  // setmaxnreg would wait
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout8<D>::kSmem) != cudaSuccess)
      return B200K_ERR_LAUNCH;
    attributes_done(done);
  }
  // Boxes of codes that lie together in a page and in a block, as in the 16-bit kernel.
  CUtensorMap tq, tk, tv;
  std::memset(&tq, 0, sizeof(tq));
  tk = tv = tq;
  p.box_rows = 0;
  const int rows = std::min(p.page_size & -p.page_size, kBlock);
  if (rows >= 8) {
    const int64_t sizes[4] = {D, p.page_size, p.Hkv, p.num_pages}, strides[3] = {p.c_slot, p.c_head, p.c_page};
    const cuuint32_t box[4] = {D, static_cast<cuuint32_t>(rows), 1, 1};
    if (make_map(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, CU_TENSOR_MAP_SWIZZLE_NONE, p.k8, sizes, strides, box) &&
        make_map(&tv, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, CU_TENSOR_MAP_SWIZZLE_NONE, p.v8, sizes, strides, box))
      p.box_rows = rows;
  }
  p.q_box = 0;
  if (p.G <= 128 && (p.G & (p.G - 1)) == 0) {  // a tile is whole tokens
    const int64_t sizes[4] = {D, p.G, p.Hkv, p.T}, strides[3] = {p.q_h, p.q_h * p.G, p.q_t};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(p.G), 1, static_cast<cuuint32_t>(128 / p.G)};
    if (make_map(&tq, gemm::tma_dtype(BF16 ? B200K_BF16 : B200K_F16), 2, CU_TENSOR_MAP_SWIZZLE_128B, p.q, sizes, strides, box))
      p.q_box = 1;
  }
  // launched under the row kernel's end, as the combine kernel is
  cudaLaunchConfig_t cfg;
  std::memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(static_cast<unsigned>(p.tile_ctas));
  cfg.blockDim = dim3(kThreads8);
  cfg.dynamicSmemBytes = Layout8<D>::kSmem;
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

int launch_tiles8(const Params& p, bool bf16, int dim, int cap, cudaStream_t st) {
  if (dim == 64) return bf16 ? launch_cap<true, 64>(p, cap, st) : launch_cap<false, 64>(p, cap, st);
  return bf16 ? launch_cap<true, 128>(p, cap, st) : launch_cap<false, 128>(p, cap, st);
}

}  // namespace paged
}  // namespace b200k
