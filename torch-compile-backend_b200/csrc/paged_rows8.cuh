// The row kernel over e4m3 caches (b200k_paged_attention_quant), included by
// paged_attention.cu behind the row kernel over 16-bit ones, whose list of
// steps, parts and joins it shares; a step is 32 keys here, as many bytes.
//
// Codes become f16 in registers, a conversion for two of them, and the order of
// the products' inner index is chosen for it: a lane's 16 neighbouring codes of
// a key (one 16-byte load) are four k-steps of Q K^T, the queries' fragments
// loaded in the same order; for P V a lane loads 16 (heads of 64: 8)
// neighbouring codes of four keys, byte permutes pair the keys of a column, and
// a lane ends with 32 (16) neighbouring columns of its rows.  Both rings are
// swizzled for these loads.  Scales: see paged.cuh.

constexpr uint32_t kRing8Bytes = 27648;  // of one warp

__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(real ? 4 : 0) : "memory");
}
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

template <bool BF16, int D, int CAP>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) rows8_kernel(const __grid_constant__ Params p) {
  constexpr uint32_t kTile = kKeys8 * D, kStage = 2 * kTile + 512;  // codes of K and V, ks, vs, log2 vs, 1 / vs
  constexpr int S = kRing8Bytes / kStage;
  constexpr int kChunks = D / 16;         // 16-byte chunks of a row
  constexpr int kRowsPerCp = 32 / kChunks;
  constexpr int E = D / 8;                // columns of a lane's V loads
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int worker = (static_cast<int>(blockIdx.x) - (p.tile_ctas > 0 ? 1 : 0)) * kWarps + warp;
  const uint32_t ring = smem_addr(smem) + warp * kRing8Bytes;
  if (worker < 0) {
    plan_tiles<kKeys8>(p);
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // as in the 16-bit kernel

  // The whole list's length and, from it, this worker's run [w0, w1).
  const int limit = limit_of<kKeys8>(p);
  int64_t total = 0, mine0 = 0, upto0 = 0;
  int longest = 0;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int64_t mine = 0;
    if (b0 + lane < p.B) {
      const Work w = work_at<kKeys8>(p, b0 + lane, limit);
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
  Cursor<kKeys8> cur;
  cur.b = 0;
  int64_t seq0 = 0;  // the list's index of cur.b's first step
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    int64_t mine = mine0, upto = upto0;
    if (p.B > 32) {
      mine = b0 + lane < p.B ? steps_of(p, work_at<kKeys8>(p, b0 + lane, limit)) : 0;
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
  cur.w = work_at<kKeys8>(p, cur.b, limit);
  const int unit = static_cast<int>(div64(w0 - seq0, cur.w.tiles));
  cur.tile = static_cast<int>((w0 - seq0) - static_cast<int64_t>(unit) * cur.w.tiles);
  cur.kvh = unit / cur.w.rts;
  cur.rt = unit - cur.kvh * cur.w.rts;

  Cursor<kKeys8> ld = cur;
  int64_t ld_t = w0;
  // the page of this lane's key, fetched a step before its first use
  auto page_of = [&](const Cursor<kKeys8>& c) {
    const int key = c.w.base + c.tile * kKeys8 + lane;
    if (key < c.w.s.lo || key >= c.w.s.n) return -1;
    return __ldg(p.table + c.b * p.table_stride + fdiv(static_cast<uint32_t>(key), p.div_page));
  };
  int page = page_of(ld);
  int ld_stage = 0;
  auto issue = [&] {
    if (ld_t < w1) {
      const uint32_t sk = ring + ld_stage * kStage, sv = sk + kTile, sc = sv + kTile;
      const int c = lane % kChunks;
      const Place8 at = place8(p, page, ld.w.base + ld.tile * kKeys8 + lane, ld.w.s.lo, ld.w.s.n, ld.kvh);
#pragma unroll
      for (int i = 0; i < kKeys8 / kRowsPerCp; ++i) {
        const int row = i * kRowsPerCp + lane / kChunks;
        const int64_t o = __shfl_sync(0xffffffffu, at.row, row);
        const bool real = o >= 0;
        const int64_t e = (real ? o : 0) + c * 16;
        cp16(sk + k8_at<D>(row, c), p.k8 + e, real);
        cp16(sv + v8_at<D>(row, c), p.v8 + e, real);
      }
      const bool real = at.scale >= 0;
      cp4(sc + lane * 4, p.ks + (real ? at.scale : 0), real);
      cp4(sc + 128 + lane * 4, p.vs + (real ? at.scale : 0), real);
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
  float m[2], l[2], rs[2];
  int pos[2], row_first = 0, row_last = 0;
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
    if (fresh) {  // a new unit: its query rows as A fragments
      fresh = false;
      const int rows = cur.w.s.m * p.G, r0 = cur.rt * kRows;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = r0 + g + 8 * i;
        const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
        const uint16_t* src = p.q + static_cast<int64_t>(cur.w.s.t0 + tok) * p.q_t +
                              static_cast<int64_t>(cur.kvh * p.G + (r - tok * p.G)) * p.q_h + quad * 16;
        pos[i] = cur.w.s.first + static_cast<int>(tok);
        m[i] = -INFINITY;
        l[i] = 0.0f;
        rs[i] = 1.0f;
        uint4 q[D / 32];
#pragma unroll
        for (int k = 0; k < D / 32; ++k)  // 16 of every 64 columns
          q[k] = r < rows ? __ldg(reinterpret_cast<const uint4*>(src + (k >> 1) * 64 + (k & 1) * 8)) : make_uint4(0, 0, 0, 0);
        if (BF16) {
          uint32_t top = 0;
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
#pragma unroll
            for (uint32_t w : {q[k].x, q[k].y, q[k].z, q[k].w}) top = max(top, max((w << 16) & 0x7fffffffu, w & 0x7fff0000u));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const RowScale sc = row_scale(top);
          rs[i] = sc.mul;
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            q[k] = make_uint4(bf16_to_f16(q[k].x, sc.div), bf16_to_f16(q[k].y, sc.div), bf16_to_f16(q[k].z, sc.div),
                              bf16_to_f16(q[k].w, sc.div));
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {  // a k-step is four columns a lane: two words
          qf[2 * k][i] = q[k].x;
          qf[2 * k][2 + i] = q[k].y;
          qf[2 * k + 1][i] = q[k].z;
          qf[2 * k + 1][2 + i] = q[k].w;
        }
      }
#pragma unroll
      for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
      row_first = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(r0), p.div_g));
      row_last = cur.w.s.first + static_cast<int>(fdiv(static_cast<uint32_t>(min(r0 + kRows, rows) - 1), p.div_g));
    }
    const uint32_t sk = ring + stage * kStage, sv = sk + kTile, sc = sv + kTile;
    {
      const float v = value_scale(lds_f(sc + 128 + lane * 4));
      sts_f(sc + 256 + lane * 4, lg2(v));
      sts_f(sc + 384 + lane * 4, 1.0f / v);
    }
    float s[4][4] = {};
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint4 kw = lds16(sk + k8_at<D>(n * 8 + g, j * 4 + quad));
        const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) mma<false>(s[n], qf[j * 4 + k], codes_lo(w[k]), codes_hi(w[k]));
      }
    }
    __syncwarp();  // the scales' logarithms and reciprocals are there
    float2 iv[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t at = sc + (n * 8 + quad * 2) * 4;
      const float2 ks = lds_f2(at), lv = lds_f2(at + 256);
      iv[n] = lds_f2(at + 384);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[n][i] = score<CAP>(p, s[n][i] * (i & 1 ? ks.y : ks.x) * rs[i >> 1]) + (i & 1 ? lv.y : lv.x);
    }
    const int key0 = cur.w.base + cur.tile * kKeys8;
    if (key0 + kKeys8 - 1 > row_first || (p.window > 0 && key0 <= row_last - p.window)) {  // warp-uniform
#pragma unroll
      for (int n = 0; n < 4; ++n)
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
      float x = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
      for (int n = 1; n < 4; ++n) x = fmaxf(x, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
      const float was = m[i];
      m[i] = fmaxf(was, x);
      const float top = m[i] == -INFINITY ? 0.0f : m[i], ref = top - kF16Reach;
      alpha[i] = ex2(was - top);
      moved |= m[i] != was;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
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
    // weights rounded to f16 for the second product (the sum keeps fp32), half
    // a step each down to 2^-29 of the row's largest
    uint32_t pa[2][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] = fmaf(s[n][2 * i], iv[n].x, fmaf(s[n][2 * i + 1], iv[n].y, l[i]));
        pa[n >> 1][(n & 1) * 2 + i] = pack16<false>(s[n][2 * i], s[n][2 * i + 1]);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[4][E / 4];  // keys 2 quad, 2 quad + 1, and 8 behind
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
        mma<false>(o[4 * i], pa[h], codes_lo(a0), codes_lo(b0));
        mma<false>(o[4 * i + 1], pa[h], codes_hi(a0), codes_hi(b0));
        mma<false>(o[4 * i + 2], pa[h], codes_lo(a1), codes_lo(b1));
        mma<false>(o[4 * i + 3], pa[h], codes_hi(a1), codes_hi(b1));
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
        // this lane's columns are 2 E quad .. + E - 1 in o[][2 i] and the E behind in o[][2 i + 1]
        if (whole && !joint) {
          const uint32_t tok = fdiv(static_cast<uint32_t>(r), p.div_g);
          uint16_t* dst = p.out + (static_cast<int64_t>(cur.w.s.t0 + tok) * p.H + cur.kvh * p.G + (r - tok * p.G)) * D + quad * 2 * E;
          const float inv = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < E; n += 8) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                w[k] = pack16<BF16>(o[n + 2 * k][2 * i + e] * inv, o[n + 2 * k + 1][2 * i + e] * inv);
              *reinterpret_cast<uint4*>(dst + e * E + n) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
          const int64_t slot = static_cast<int64_t>(worker) * 2 + (unit0 < w0 ? 0 : 1);
          const int64_t at = slot * kRows + in;
          float* dst = joint ? joint_rows<D, kRing8Bytes>(smem, warp) + in * kJointStride<D> : p.part_o + at * D;
          float* ml = joint ? dst + D : p.part_ml + at * 2;
          if (quad == 0) *reinterpret_cast<float2*>(ml) = make_float2(m[i], l[i]);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int n = 0; n < E; n += 4)
              *reinterpret_cast<float4*>(dst + quad * 2 * E + e * E + n) =
                  make_float4(o[n][2 * i + e], o[n + 1][2 * i + e], o[n + 2][2 * i + e], o[n + 3][2 * i + e]);
        }
      }
      if (joint) {
        __syncthreads();  // every warp of the CTA comes here once
        join_warps<BF16, D, kRing8Bytes>(
            p, smem, warp, lane, min(kRows, rows - r0), worker & ~(kWarps - 1), unit0 < c0 ? 0 : 1,
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
