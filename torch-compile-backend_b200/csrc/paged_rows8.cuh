// The row kernel over e4m3 caches (b200k_paged_attention_quant), included by
// paged_attention.cu behind the row kernel over 16-bit ones, whose list of
// steps, parts and joins it shares; a step is 32 keys here, as many bytes.
//
// Half the bytes a key leave half the time for it, so the products are turned:
// S^T = K Q^T and O^T = V^T W^T with the keys and the columns as the MMAs' 16 rows
// and the query rows as their 8 columns, one or two times (ROWS 8 or 16): a single
// token of up to 8 heads a key head takes half the MMAs, scores and registers.
// Codes become f16 in registers, a conversion for two of them, and the order of
// the products' indexes is chosen for it: a lane's 16 neighbouring codes of a key
// (one 16-byte load) are four k-steps of K Q^T, the queries' fragments loaded in
// the same order; for V^T W^T a lane loads 16 (heads of 64: 8) neighbouring codes
// of four keys, byte permutes pair the keys of a column, and a lane ends with
// those columns of its rows.  Both rings are swizzled for these loads.  Scales:
// see paged.cuh.  Measured: one token of 64 sequences to 8192 keys, 32 / 8 heads of
// 128, 130-136 us = 5.2-5.4 TB/s (121 with the cache laid out head by head: rows of
// 128 bytes at 1 KB steps are what bounds it, the loads alone take 94 % of the
// time); of 3 sequences to 65536 keys 57-60 us.  Codes straight into e4m3 products,
// with queries as sums of two or three e4m3 numbers, were no faster (132 us) and in
// f16 slower (four proposed tokens in a window 17.9 us in place of 13.3).

// Of one warp.
template <int ROWS>
constexpr uint32_t kRing8Bytes = ROWS == 8 ? 18432 : 27648;

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ float2 lds_f2(uint32_t a) {
  float2 r;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(r.x), "=f"(r.y) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ float lds_f(uint32_t a) {
  float r;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void sts_f(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }

// Place of 16-byte chunk c of a row in a ring's tile.
template <int D>
__device__ __forceinline__ uint32_t k8_at(int row, int c) {
  return D == 128 ? row * 128 + ((c ^ ((row & 1) << 2)) << 4) : row * 64 + (c << 4);
}
template <int D>
__device__ __forceinline__ uint32_t v8_at(int row, int c) {
  const int turn = ((row >> 1) & 3) << 1;
  return D == 128 ? row * 128 + ((c ^ turn) << 4) : (row >> 1) * 128 + ((((row & 1) * 4 + c) ^ turn) << 4);
}

// An 8 x 8 matrix of 16-bit values, a row's pairs over four lanes, transposed.
__device__ __forceinline__ uint32_t turned8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// CTAs an SM: the registers of 8 rows leave room for more.
template <int D, int ROWS>
constexpr int kCtas8 = ROWS == 8 ? 3 : 2;
template <bool BF16, int D, int CAP, int ROWS>
__global__ void __launch_bounds__(kWarps * 32, kCtas8<D, ROWS>) rows8_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched early, ahead of its launch_dependents for the later ones' sake
  constexpr uint32_t kTile = kKeys8 * D, kStage = 2 * kTile + 512;  // codes of K and V, ks, vs, log2 vs, 1 / vs
  constexpr int S = kRing8Bytes<ROWS> / kStage;
  constexpr int NT = ROWS / 8;            // query rows, eight at a time
  constexpr int kChunks = D / 16;         // 16-byte chunks of a row
  constexpr int kRowsPerCp = 32 / kChunks;
  constexpr int E = D / 8;                // columns of a lane's V loads
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int worker = (static_cast<int>(blockIdx.x) - (p.tile_ctas > 0 ? 1 : 0)) * kWarps + warp;
  const uint32_t ring = smem_addr(smem) + warp * kRing8Bytes<ROWS>;
  if (worker < 0) {
    plan_tiles<kKeys8, ROWS>(p);
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // as in the 16-bit kernel

  // The whole list's length and, from it, this worker's run [w0, w1).
  const int limit = limit_of<kKeys8, ROWS>(p);
  int64_t total = 0, mine0 = 0, upto0 = 0;
  int longest = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int64_t mine = 0;
    if (b0 + lane < p.B) {
      const Work w = work_at<kKeys8, ROWS>(p, b0 + lane, limit);
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
  Cursor<kKeys8, ROWS> cur;
  cur.b = 0;
  int64_t seq0 = 0;  // the list's index of cur.b's first step
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int64_t mine = mine0, upto = upto0;
    if (p.B > 32) {
      mine = b0 + lane < p.B ? steps_of(p, work_at<kKeys8, ROWS>(p, b0 + lane, limit)) : 0;
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
  cur.w = work_at<kKeys8, ROWS>(p, cur.b, limit);
  const int unit = static_cast<int>(div64(w0 - seq0, cur.w.tiles));
  cur.tile = static_cast<int>((w0 - seq0) - static_cast<int64_t>(unit) * cur.w.tiles);
  cur.kvh = unit / cur.w.rts;
  cur.rt = unit - cur.kvh * cur.w.rts;

  Cursor<kKeys8, ROWS> ld = cur;
  int64_t ld_t = w0;
  // the page of this lane's key, fetched a step before its first use
  auto page_of = [&](const Cursor<kKeys8, ROWS>& c) {
    const int key = c.w.base + c.tile * kKeys8 + lane;
    if (key < c.w.s.lo || key >= c.w.s.n) return -1;
    return fetch<true>(p.table + c.b * p.table_stride + fdiv(static_cast<uint32_t>(key), p.div_page));
  };
  int page = page_of(ld);
  int ld_stage = 0;
  auto issue = [&] {
    if (ld_t < w1) {
      const uint32_t sk = ring + ld_stage * kStage, sv = sk + kTile, sc = sv + kTile;
      const int c = lane % kChunks;
      const int key = ld.w.base + ld.tile * kKeys8 + lane;
      if (!p.far_rows) {
        // Offsets in rows' 16 bytes and in scales, 32 bits each: one shuffle and
        // one multiply-add an address.
        uint32_t row16 = ~0u, scale = 0;
        if (page >= 0 && page < p.num_pages) {  // -1: no key
          const uint32_t in = static_cast<uint32_t>(key) - fdiv(static_cast<uint32_t>(key), p.div_page) * static_cast<uint32_t>(p.page_size);
          row16 = static_cast<uint32_t>(page) * p.c16_page + in * p.c16_slot + static_cast<uint32_t>(ld.kvh) * p.c16_head;
          scale = static_cast<uint32_t>(page) * static_cast<uint32_t>(p.s_page) + in * static_cast<uint32_t>(p.s_slot) +
                  static_cast<uint32_t>(ld.kvh) * static_cast<uint32_t>(p.s_head);
        } else if (key >= ld.w.s.lo && key < ld.w.s.n && p.status) {
          atomicCAS(p.status, 0, B200K_ERR_INDEX);
        }
        const uint8_t *kc = p.k8 + c * 16, *vc = p.v8 + c * 16;
#pragma unroll
        for (int i = 0; i < kKeys8 / kRowsPerCp; ++i) {
          const int row = i * kRowsPerCp + lane / kChunks;
          const uint32_t o = __shfl_sync(0xffffffffu, row16, row);
          const uint64_t e = static_cast<uint64_t>(o == ~0u ? 0u : o) * 16;
          cp16(sk + k8_at<D>(row, c), kc + e, o != ~0u);
          cp16(sv + v8_at<D>(row, c), vc + e, o != ~0u);
        }
        cp4(sc + lane * 4, p.ks + scale, row16 != ~0u);
        cp4(sc + 128 + lane * 4, p.vs + scale, row16 != ~0u);
      } else {
        const Place8 at = place8(p, page, key, ld.w.s.lo, ld.w.s.n, ld.kvh);
#pragma unroll 1
        for (int i = 0; i < kKeys8 / kRowsPerCp; ++i) {
          const int row = i * kRowsPerCp + lane / kChunks;
          const int64_t o = __shfl_sync(0xffffffffu, at.row, row);
          const int64_t e = (o >= 0 ? o : 0) + c * 16;
          cp16(sk + k8_at<D>(row, c), p.k8 + e, o >= 0);
          cp16(sv + v8_at<D>(row, c), p.v8 + e, o >= 0);
        }
        const bool real = at.scale >= 0;
        cp4(sc + lane * 4, p.ks + (real ? at.scale : 0), real);
        cp4(sc + 128 + lane * 4, p.vs + (real ? at.scale : 0), real);
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
  // rows of this lane: 8 t + 2 quad + i in the scores and sums, 8 t + g of the queries
  uint32_t qf[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2], rs[NT][2];
  int pos[NT][2], row_first = 0, row_last = 0;
  bool fresh = true;
  int stage = 0;
  int64_t unit0 = seq0 + static_cast<int64_t>(unit) * cur.w.tiles;  // the current unit's first step
  const int64_t c0 = run * (worker & ~(kWarps - 1)), c1 = c0 + run * kWarps;
  const bool joint = unit0 <= c0 && c1 <= unit0 + cur.w.tiles;  // all of this CTA's runs lie in one unit
#pragma unroll 1
  for (int64_t t = w0 - (S - 1); t < w1; ++t) {
    if (t >= w0) {
      cp_wait<S - 2>();
      __syncwarp();  // step t has landed, and all lanes are done with the stage of step t - 1
    }
    issue();
    if (t < w0) continue;
    if (fresh) {  // a new unit: its query rows as B fragments
      fresh = false;
      const int rows = cur.w.s.m * p.G, r0 = cur.rt * ROWS;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = r0 + n * 8 + g;
        const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
        const uint16_t* src = p.q + static_cast<int64_t>(cur.w.s.t0 + tok) * p.q_t +
                              static_cast<int64_t>(cur.kvh * p.G + (r - tok * p.G)) * p.q_h + quad * 16;
        uint4 q[D / 32];
#pragma unroll
        for (int k = 0; k < D / 32; ++k)  // 16 of every 64 columns
          q[k] = r < rows ? fetch<true>(reinterpret_cast<const uint4*>(src + (k >> 1) * 64 + (k & 1) * 8)) : make_uint4(0, 0, 0, 0);
        float mul = 1.0f;
        if (BF16) {
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
#pragma unroll
            for (uint32_t w : {q[k].x, q[k].y, q[k].z, q[k].w}) top = max(top, max((w << 16) & 0x7fffffffu, w & 0x7fff0000u));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const RowScale sc = row_scale(top);
          mul = sc.mul;
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            q[k] = make_uint4(bf16_to_f16(q[k].x, sc.div), bf16_to_f16(q[k].y, sc.div), bf16_to_f16(q[k].z, sc.div),
                              bf16_to_f16(q[k].w, sc.div));
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {  // a k-step is four columns a lane: two words
          qf[n][2 * k][0] = q[k].x;
          qf[n][2 * k][1] = q[k].y;
          qf[n][2 * k + 1][0] = q[k].z;
          qf[n][2 * k + 1][1] = q[k].w;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int in = quad * 2 + i;
          const float row_mul = BF16 ? __shfl_sync(0xffffffffu, mul, in * 4) : 1.0f;
          rs[n][i] = CAP == kNoCap ? row_mul * p.mul : row_mul;
          pos[n][i] = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(r0 + n * 8 + in), p.div_g));
          m[n][i] = -INFINITY;
          l[n][i] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < D / 16; ++k) o[n][k][0] = o[n][k][1] = o[n][k][2] = o[n][k][3] = 0.0f;
      }
      row_first = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(r0), p.div_g));
      row_last = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(min(r0 + ROWS, rows) - 1), p.div_g));
    }
    const uint32_t sk = ring + stage * kStage, sv = sk + kTile, sc = sv + kTile;
    {
      const float v = value_scale(lds_f(sc + 128 + lane * 4));
      sts_f(sc + 256 + lane * 4, lg2(v));
      sts_f(sc + 384 + lane * 4, 1.0f / v);
    }
    // scores of keys 16 h + g (elements 0, 1) and 16 h + 8 + g (2, 3)
    float s[2][NT][4] = {};
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 ka = lds16(sk + k8_at<D>(h * 16 + g, j * 4 + quad)), kb = lds16(sk + k8_at<D>(h * 16 + 8 + g, j * 4 + quad));
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a[4] = {codes_lo(wa[k]), codes_lo(wb[k]), codes_hi(wa[k]), codes_hi(wb[k])};
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<false>(s[h][n], a, qf[n][j * 4 + k][0], qf[n][j * 4 + k][1]);
        }
      }
    }
    __syncwarp();  // the scales' logarithms and reciprocals are there
    float iv[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t at = sc + (h * 16 + e * 8 + g) * 4;
        const float ks = lds_f(at), lv = lds_f(at + 256);
        iv[h][e] = lds_f(at + 384);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x = s[h][n][e * 2 + i] * ks;
            s[h][n][e * 2 + i] = CAP == kNoCap ? fmaf(x, rs[n][i], lv) : score<CAP>(p, x * rs[n][i]) + lv;
          }
      }
    const int key0 = cur.w.base + cur.tile * kKeys8;
    if (key0 + kKeys8 - 1 > row_first || (p.window > 0 && key0 <= row_last - p.window)) {  // warp-uniform
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + h * 16 + (e >> 1) * 8 + g, at = pos[n][e & 1];
            if (key > at || (p.window > 0 && key <= at - p.window)) s[h][n][e] = -INFINITY;
          }
    }
    bool moved = false;
    float alpha[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(fmaxf(s[0][n][i], s[0][n][2 + i]), fmaxf(s[1][n][i], s[1][n][2 + i]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        const float was = m[n][i];
        m[n][i] = fmaxf(was, x);
        const float top = m[n][i] == -INFINITY ? 0.0f : m[n][i], ref = top - kF16Reach;
        alpha[n][i] = ex2(was - top);
        moved |= m[n][i] != was;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s[h][n][i] = ex2(s[h][n][i] - ref);
          s[h][n][2 + i] = ex2(s[h][n][2 + i] - ref);
        }
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[n][i] *= alpha[n][i];
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            o[n][k][i] *= alpha[n][i];
            o[n][k][2 + i] *= alpha[n][i];
          }
        }
    }
    // weights rounded to f16 for the second product (the sum keeps fp32), half
    // a step each down to 2^-29 of the row's largest
    uint32_t pb[2][NT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float a = s[h][n][2 * e], b = s[h][n][2 * e + 1];
          l[n][0] = fmaf(a, iv[h][e], l[n][0]);
          l[n][1] = fmaf(b, iv[h][e], l[n][1]);
          pb[h][n][e] = turned8(pack16<false>(a, b));
        }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[4][E / 4];  // keys 16 h + 2 quad, + 1, and 8 behind
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = h * 16 + quad * 2 + (r & 1) + (r >> 1) * 8;
        if constexpr (D == 128) {
          const uint4 x = lds16(sv + v8_at<D>(row, g));
          v[r][0] = x.x;
          v[r][1] = x.y;
          v[r][2] = x.z;
          v[r][3] = x.w;
        } else {
          const uint2 x = lds8(sv + v8_at<D>(row, g >> 1) + (g & 1) * 8);
          v[r][0] = x.x;
          v[r][1] = x.y;
        }
      }
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        // columns 4 i and 4 i + 1, then the other two, of two keys side by side
        const uint32_t a0 = __byte_perm(v[0][i], v[1][i], 0x5140), a1 = __byte_perm(v[0][i], v[1][i], 0x7362);
        const uint32_t b0 = __byte_perm(v[2][i], v[3][i], 0x5140), b1 = __byte_perm(v[2][i], v[3][i], 0x7362);
        const uint32_t x[4] = {codes_lo(a0), codes_hi(a0), codes_lo(b0), codes_hi(b0)};
        const uint32_t y[4] = {codes_lo(a1), codes_hi(a1), codes_lo(b1), codes_hi(b1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma<false>(o[n][2 * i], x, pb[h][n][0], pb[h][n][1]);
          mma<false>(o[n][2 * i + 1], y, pb[h][n][0], pb[h][n][1]);
        }
      }
    }
    stage = stage + 1 == S ? 0 : stage + 1;

    const bool unit_ends = cur.tile + 1 == cur.w.tiles;
    if (unit_ends || t + 1 == w1) {
      const int rows = cur.w.s.m * p.G, r0 = cur.rt * ROWS;
      const bool whole = unit0 >= w0 && unit_ends;
      if (joint) {  // its last step: the rings are free
        cp_wait<0>();
        __syncwarp();
      }
      // this lane's columns are E g .. E g + E - 1: o[][k][i] has 2 k, o[][k][2 + i] the next
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float sum = l[n][i];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int in = n * 8 + quad * 2 + i, r = r0 + in;
          if (r >= rows) continue;
          if (whole && !joint) {
            const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
            uint16_t* dst = p.out + (static_cast<int64_t>(cur.w.s.t0 + tok) * p.H + cur.kvh * p.G + (r - tok * p.G)) * D + g * E;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int k = 0; k < E / 2; k += 4) {
              uint32_t w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) w[j] = pack16<BF16>(o[n][k + j][i] * inv, o[n][k + j][2 + i] * inv);
              reinterpret_cast<uint4*>(dst)[k / 4] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            const int64_t slot = static_cast<int64_t>(worker) * 2 + (unit0 < w0 ? 0 : 1);
            const int64_t at = slot * ROWS + in;
            float* dst = joint ? joint_rows<D, kRing8Bytes<ROWS>>(smem, warp) + in * kJointStride<D> : p.part_o + at * D;
            float* ml = joint ? dst + D : p.part_ml + at * 2;
            if (g == 0) *reinterpret_cast<float2*>(ml) = make_float2(m[n][i], sum);
#pragma unroll
            for (int k = 0; k < E / 2; k += 2)
              reinterpret_cast<float4*>(dst + g * E)[k / 2] =
                  make_float4(o[n][k][i], o[n][k][2 + i], o[n][k + 1][i], o[n][k + 1][2 + i]);
          }
        }
      if (joint) {
        __syncthreads();  // every warp of the CTA comes here once
        join_warps<BF16, D, kRing8Bytes<ROWS>, ROWS>(
            p, smem, warp, lane, min(ROWS, rows - r0), worker & ~(kWarps - 1), unit0 < c0 ? 0 : 1,
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
