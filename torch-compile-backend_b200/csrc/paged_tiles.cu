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
#include "paged_tiles.cuh"

namespace b200k {
namespace paged {
namespace {

constexpr int kThreads = 448;
constexpr int kLoaders = 64;               // threads that arrive for a query tile; 32 for a key or value block
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
  const Shared b{q_full, q_empty, k_full, k_empty, v_full, v_empty, s_full, p_full, o_done, o_free, drain, sQ, sK, sV, copied,
                 nullptr, nullptr, nullptr};
  Portion po;

  if (warp >= 8 && warp < 12) {
    issue_products<BF16, D, S, false>(p, walk, ctl, b, tmem_base, warp, lane);
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
      int issued = 0, q_issued = 0;  // blocks and portions' queries whose copies have been issued
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
          issued = c + 1;
          if (j == po.beg) {
            // the portion's queries, when the products of the one before have read theirs
            if (li > 0 && !(ok = warp_wait(q_empty, (li - 1) & 1, ctl))) break;
            q_issued = li + 1;
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
      // No box is on its way when this warp leaves: the last ones have landed when
      // their readers are done with them, except after a timeout.  (Queries wait for
      // the other loader's arrivals too, which may not come then.)
      for (int k = max(0, issued - S); k < issued; ++k) gemm::wait_bar_drain(&full[k % S], (k / S) & 1, 100000000ull);
      if (q_issued > 0) gemm::wait_bar_drain(q_full, (q_issued - 1) & 1, 10000000ull);
      __syncwarp();
  } else {
    softmax_rows<BF16, D, CAP, false>(p, walk, ctl, b, tmem_base, run, warp, lane);
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
  auto kernel = tiles_kernel<BF16, D, CAP>;
  static std::atomic<uint64_t> done{0};
  if (!attributes_set(done)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::kSmem) != cudaSuccess)
      return B200K_ERR_LAUNCH;
    attributes_done(done);
  }
  // Boxes of the rows that lie together in a page and in a block: the largest
  // power of two, 8 to 64, that divides the page size.
  const CUtensorMapDataType type = gemm::tma_dtype(BF16 ? B200K_BF16 : B200K_F16);
  CUtensorMap tq, tk, tv;
  std::memset(&tq, 0, sizeof(tq));
  tk = tv = tq;
  p.box_rows = 0;
  const int both = p.page_size & -p.page_size;
  const int rows = std::min(both, kBlock);
  if (rows >= 8) {
    const int64_t sizes[4] = {D, p.page_size, p.Hkv, p.num_pages}, strides[3] = {p.c_slot, p.c_head, p.c_page};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1};
    if (make_map(&tk, type, 2, CU_TENSOR_MAP_SWIZZLE_128B, p.k, sizes, strides, box) &&
        make_map(&tv, type, 2, CU_TENSOR_MAP_SWIZZLE_128B, p.v, sizes, strides, box)) p.box_rows = rows;
  }
  p.q_box = 0;
  if (p.G <= 128 && (p.G & (p.G - 1)) == 0) {  // a tile is whole tokens
    const int64_t sizes[4] = {D, p.G, p.Hkv, p.T}, strides[3] = {p.q_h, p.q_h * p.G, p.q_t};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(p.G), 1, static_cast<cuuint32_t>(128 / p.G)};
    if (make_map(&tq, type, 2, CU_TENSOR_MAP_SWIZZLE_128B, p.q, sizes, strides, box)) p.q_box = 1;
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
