// The tile kernel of b200k_paged_attention_quant: sequences with many query
// rows over e4m3 caches.  The plan, the portions, the products, the softmax and
// the parts are the 16-bit tile kernel's (paged_tiles.cuh); here
//   warps 12, 13 load codes (TMA boxes or 16-byte cp.async copies) and scales,
//   warps 16, 17 make a block's key codes 16-bit in shared memory, of q's type,
//   warps 18, 19 its value codes, f16: as they are (both types hold every code).
// Q K^T runs in q's type, P V in f16.  All scales stay out of the products: rounded
// into bf16 keys they would move every score, the output by 0.4 %; values of code *
// scale have to be divided by something that all rows share for f16 (the block's
// largest scale), and then a value that a row does not see, or gives no weight,
// takes bits from those that it does.  The softmax, which bounds the kernel, takes
// the scales in.  The registers are shared out by setmaxnreg: five warpgroups are
// launched with 96 a thread.  Measured: 5 chunks of 1024 behind up to 6000 keys, 32 /
// 8 heads of 128, 484-495 us = 535 TFLOP/s, with a cap in f16 680; 8 prompts of 2048, heads
// of 64, 515 us (values of code * scale / 2^E: 493, 652 and 490).  No unit is full (tensor
// pipe 25 %, issue 48 %, exponentials 20 %): the warps wait for one another.
#include "paged_tiles.cuh"

namespace b200k {
namespace paged {
namespace {

constexpr int kThreads8 = 640;
constexpr int kLaunchRegs = 96, kSoftmaxRegs = 160, kIssueRegs = 48, kConvertRegs = 64;
static_assert(2 * kSoftmaxRegs + 2 * kIssueRegs + kConvertRegs <= 5 * kLaunchRegs, "what the launch has");
template <int D>
struct Layout8 {
  static constexpr int kStages = D == 128 ? 3 : 4;         // of 16-bit keys and of values
  static constexpr int kRaw = D == 128 ? 3 : 4;            // of codes
  static constexpr uint32_t kTile = kHalfTile * (D / 64);  // a query tile
  static constexpr uint32_t kBlk = kHalfBlk * (D / 64);    // a 16-bit block
  static constexpr uint32_t kCodes = kBlock * D;           // a block of codes
  static constexpr uint32_t kOffK = 2 * kTile;
  static constexpr uint32_t kOffV = kOffK + kStages * kBlk;
  static constexpr uint32_t kOffRawK = kOffV + kStages * kBlk;
  static constexpr uint32_t kOffRawV = kOffRawK + kRaw * kCodes;
  static constexpr uint32_t kOffRawKs = kOffRawV + kRaw * kCodes;      // [kRaw][64] scales
  static constexpr uint32_t kOffRawVs = kOffRawKs + kRaw * kBlock * 4;
  static constexpr uint32_t kOffSc = kOffRawVs + kRaw * kBlock * 4;          // Shared::sc
  static constexpr uint32_t kOffBar = kOffSc + kScaleSlots * kScaleFloats * 4;
  static constexpr uint32_t kSmem = 1024 + kOffBar + 1024;
  static_assert(kSmem <= 232448 && kSmem > 116 * 1024, "one CTA per SM");
};
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
  uint64_t* q_full = reinterpret_cast<uint64_t*>(sbase + L::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* rk_full = q_empty + 1;   // codes
  uint64_t* rk_empty = rk_full + R;
  uint64_t* rv_full = rk_empty + R;
  uint64_t* rv_empty = rv_full + R;
  uint64_t* k_full = rv_empty + R;   // 16-bit
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
  float* sc = reinterpret_cast<float*>(sbase + L::kOffSc);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_empty + kScaleSlots);
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
  const Shared b{q_full, q_empty, k_full, k_empty, v_full, v_empty, s_full, p_full, o_done, o_free, drain, sQ, sK, sV, nullptr,
                 sc_full, sc_empty, sc};

  if (warp >= 8 && warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    issue_products<BF16, D, S, true>(p, walk, ctl, b, tmem_base, warp, lane);
  } else if (warp >= 16) {
    // ----------------------------------------------------------------- converters
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvertRegs));
    const bool is_v = warp >= 18;
    const int first = (warp & 1) * 32 + lane;  // of a block's 16-byte chunks, every 64th
    const uint8_t* raw = sbase + (is_v ? L::kOffRawV : L::kOffRawK);
    const float* raw_sc = reinterpret_cast<const float*>(sbase + (is_v ? L::kOffRawVs : L::kOffRawKs));
    uint8_t* dst0 = is_v ? sV : sK;
    uint64_t* r_full = is_v ? rv_full : rk_full;
    uint64_t* r_empty = is_v ? rv_empty : rk_empty;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    constexpr int kChunks = D / 16;  // 16-byte chunks of a row of codes
    const bool signs = (warp & 1) == 0;  // this warp leaves the block's scales
    Portion po;
    int c = 0;
    bool ok = true;
    while (ok && walk.next(p, po)) {
      for (int j = po.beg; j < po.end; ++j, ++c) {
        const int rst = c % R, st = c % S, slot = c % kScaleSlots;
        if (!(ok = warp_wait(&r_full[rst], (c / R) & 1, ctl))) break;
        if (signs) {
          if (!(ok = warp_wait(&sc_empty[slot], ((c / kScaleSlots) & 1) ^ 1, ctl))) break;
          float* to = sc + slot * kScaleFloats;
#pragma unroll
          for (int i = lane; i < kBlock; i += 32) {
            const float x = raw_sc[rst * kBlock + i];
            if (is_v) {
              const float v = value_scale(x);
              to[kBlock + i] = lg2(v);
              to[2 * kBlock + i] = 1.0f / v;
            } else {
              to[i] = CAP == kNoCap ? x * p.mul : x;
            }
          }
          __syncwarp();
          if (lane == 0) gemm::mbar_arrive(&sc_full[slot]);
        }
        if (!(ok = warp_wait(&empty[st], ((c / S) & 1) ^ 1, ctl))) break;
        const uint4* src = reinterpret_cast<const uint4*>(raw + rst * L::kCodes);
        uint8_t* dst = dst0 + st * L::kBlk;
#pragma unroll 2
        for (int i = 0; i < kBlock * kChunks / 64; ++i) {
          const int idx = i * 64 + first, row = idx / kChunks, ch = idx % kChunks;
          const uint4 x = src[idx];
          uint32_t y[8] = {codes_lo(x.x), codes_hi(x.x), codes_lo(x.y), codes_hi(x.y), codes_lo(x.z), codes_hi(x.z), codes_lo(x.w), codes_hi(x.w)};
          if (BF16 && !is_v) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&y[k]));
              y[k] = pack16<BF16>(a.x, a.y);
            }
          }
          // two 16-byte chunks; the upper half's lanes write theirs the other way
          // round, so that eight lanes cover all banks
          uint8_t* to = dst + (ch >> 2) * kHalfBlk + row * 128;
          const int c0 = (ch & 3) * 2, turn = (ch >> 2) & 1;
          const uint4 u = make_uint4(y[0], y[1], y[2], y[3]), v = make_uint4(y[4], y[5], y[6], y[7]);
          *reinterpret_cast<uint4*>(to + (((c0 + turn) ^ (row & 7)) << 4)) = turn ? v : u;
          *reinterpret_cast<uint4*>(to + (((c0 + 1 - turn) ^ (row & 7)) << 4)) = turn ? u : v;
        }
        gemm::fence_async_smem();  // the tile's writes, before the MMA's reads
        __syncwarp();
        if (lane == 0) {
          gemm::mbar_arrive(&full[st]);
          gemm::mbar_arrive(&r_empty[rst]);
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
      Portion po;
      int c = 0;
      int issued = 0, q_issued = 0;  // blocks and portions' queries whose copies have been issued
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
          issued = c + 1;
          if (j == po.beg) {
            // the portion's queries, when the products of the one before have read theirs
            if (li > 0 && !(ok = warp_wait(q_empty, (li - 1) & 1, ctl))) break;
            q_issued = li + 1;
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
      // No box is on its way when this warp leaves: the last ones have landed when
      // their readers are done with them, except after a timeout.  (Queries wait for
      // the other loader's arrivals too, which may not come then.)
      for (int k = max(0, issued - R); k < issued; ++k) gemm::wait_bar_drain(&full[k % R], (k / R) & 1, 100000000ull);
      if (q_issued > 0) gemm::wait_bar_drain(q_full, (q_issued - 1) & 1, 10000000ull);
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    softmax_rows<BF16, D, CAP, true>(p, walk, ctl, b, tmem_base, run, warp, lane);
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
