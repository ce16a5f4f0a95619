// Residual addition + RMS norm in one pass over the rows (b200k_add_rms_norm,
// include/b200k.h), with a 16-bit / fp32 output or an e4m3 output with scales:
//
//   h = round(x + r)                        stored: the next residual
//   y = h * rsqrt(mean(h^2) + eps) * w      fp32
//   out = round(y), or q = e4m3(y * 448 / a) with scale a / 448,
//         a = max(max |y| over the scale's columns, 1e-12)
//
// No reference counterpart: the reference leaves the reduction to ATen and
// fuses only pointwise fragments (compiler/optimization/fusion_pointwise.py:12-30).
//
// What bounds it: HBM.  A row is read once (x and r) and written once (h and
// out); its sums live in registers between the two, so the bytes are the
// floor's.  16-bit rows are added as packed pairs (one rounding of an exact
// sum, as fp32 then round) and stay packed in registers.  h is normed as it is
// stored, rounded to x's type: the result is that of the addition followed by
// b200k_rownorm.  The sum of squares and y are fp32; out is rounded once (twice
// with B200K_ROWF_ROUND_NORMED, which reproduces models that round before the
// weight).  Measured: [16384, 8192] bf16 157 us = 6.83 TB/s (a copy: 6.52), with an
// e4m3 output and scales of 128 columns [8192, 4096] 38 us = 6.2 TB/s, one row
// of 2048 2.0 us.
#include <algorithm>
#include <cstring>

#include "e4m3.cuh"
#include "host_common.h"
#include "rowreduce.cuh"

namespace b200k {
namespace {

struct AddNormParams {
  int64_t rows;
  int32_t cols;
  int32_t group;  // columns of one scale (quantised output): cols or 128
  const void* x;
  const void* r;
  const void* w;
  void* h;
  void* out;
  float* scale;
  int64_t x_stride, r_stride;
  float eps;
  int32_t w_dt, flags;
};

template <int DT> struct Elem;
template <> struct Elem<B200K_F32> { using T = float; };
template <> struct Elem<B200K_F16> { using T = __half; };
template <> struct Elem<B200K_BF16> { using T = __nv_bfloat16; };

template <int DT>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (DT == B200K_BF16) return round_bf16(v);
  if constexpr (DT == B200K_F16) return round_f16(v);
  return v;
}

template <bool BF16>
__device__ __forceinline__ uint32_t add16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  if (BF16) asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Sum over the TPR threads of a row; each row group of a CTA has its own
// named barrier and slots.
template <int TPR, bool IS_MAX>
__device__ __forceinline__ uint32_t row_reduce(uint32_t v, uint32_t* slots, int grp) {
  if constexpr (IS_MAX) {
    v = __reduce_max_sync(0xffffffffu, v);
  } else {
    v = __float_as_uint(warp_sum(__uint_as_float(v)));
  }
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    uint32_t* s = slots + grp * W;
    const int t = threadIdx.x % TPR;
    if ((t & 31) == 0) s[t >> 5] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(TPR) : "memory");
    // every thread adds the W partials in the same order
    uint32_t a = s[0];
#pragma unroll
    for (int k = 1; k < W; ++k) {
      if constexpr (IS_MAX) a = max(a, s[k]);
      else a = __float_as_uint(__uint_as_float(a) + __uint_as_float(s[k]));
    }
    v = a;
  }
  return v;
}

// The row's statistics and output, from its sums in registers: a thread holds
// VPT vectors of 8 columns, vector t + i TPR, so 16 neighbouring lanes hold
// the 128 columns of a scale.  QUANT: 0 output of x's type, 1 e4m3 with one
// scale a row, 2 with one for 128 columns.  get(i, v) gives vector i.
template <int DT, int TPR, int VPT, int QUANT, typename Get>
__device__ __forceinline__ void finish_row(const AddNormParams& p, int64_t row, int grp, int t, int nvec, float ss,
                                           uint32_t (*slots)[32], Get get) {
  using T = typename Elem<DT>::T;
  ss = __uint_as_float(row_reduce<TPR, false>(__float_as_uint(ss), slots[0], grp));
  const float rstd = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  const bool round_n = p.flags & B200K_ROWF_ROUND_NORMED, plus1 = p.flags & B200K_ROWF_WEIGHT_PLUS_ONE;
  auto y_of = [&](int i, float (&v)[8]) {
    get(i, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= rstd;
    if (round_n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = round_to<DT>(v[j]);
    }
    if (p.w) {
      float w[8];
      if (p.w_dt == DT) load_vec8(p.w, min(t + i * TPR, nvec - 1) * 8, DT, w);  // the common case, without a switch
      else load_vec8(p.w, min(t + i * TPR, nvec - 1) * 8, p.w_dt, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= plus1 ? 1.0f + w[j] : w[j];
    }
  };
  if constexpr (QUANT == 1) {
    float v[VPT][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      y_of(i, v[i]);
      if (t + i * TPR < nvec) top = max(top, top8(v[i]));
    }
    top = row_reduce<TPR, true>(top, slots[1], grp);
    float inv;
    const float sc = scale_of(top, inv);
    if (t == 0) p.scale[row] = sc;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * TPR;
      if (c < nvec) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + row * p.cols + c * 8) = e4m3x8(v[i], inv);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t + i * TPR;
      float v[8];
      y_of(i, v);
      if constexpr (QUANT == 0) {
        if (c < nvec) store_vec8(static_cast<T*>(p.out) + row * p.cols, c * 8, DT, v);
      } else {
        uint32_t m = top8(v);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        float inv;
        const float sc = scale_of(m, inv);
        if (c < nvec) {
          if ((t & 15) == 0) p.scale[row * (p.cols >> 7) + (c >> 4)] = sc;
          *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + row * p.cols + c * 8) = e4m3x8(v, inv);
        }
      }
    }
  }
}

template <int DT, int TPR, int VPT, int QUANT, int THREADS>
__global__ void __launch_bounds__(THREADS) add_norm_kernel(const __grid_constant__ AddNormParams p) {
  constexpr int kGroups = THREADS / TPR;
  using T = typename Elem<DT>::T;
  __shared__ uint32_t slots[2][32];
  const int grp = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + grp;
  if (row >= p.rows) return;  // the whole group: its barrier is its own
  const int nvec = p.cols >> 3;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* r = static_cast<const T*>(p.r) + row * p.r_stride;
  T* h = static_cast<T*>(p.h) + row * p.cols;
  float ss = 0.0f;
  if constexpr (DT == B200K_F32) {
    float v[VPT][8], a[VPT][8];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {  // every load of the row before the first use
      const int c = min(t + i * TPR, nvec - 1) * 8;
      load_vec8(x, c, DT, v[i]);
      load_vec8(r, c, DT, a[i]);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += a[i][j];
      if (t + i * TPR < nvec) {
        store_vec8(h, (t + i * TPR) * 8, DT, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
      }
    }
    finish_row<DT, TPR, VPT, QUANT>(p, row, grp, t, nvec, ss, slots, [&](int i, float (&o)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[i][j];
    });
  } else {
    constexpr bool BF16 = DT == B200K_BF16;
    uint4 v[VPT];
    {
      uint4 a[VPT];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {  // every load of the row before the first use
        const int c = min(t + i * TPR, nvec - 1);
        v[i] = __ldg(reinterpret_cast<const uint4*>(x) + c);
        a[i] = __ldg(reinterpret_cast<const uint4*>(r) + c);
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        v[i].x = add16x2<BF16>(v[i].x, a[i].x);
        v[i].y = add16x2<BF16>(v[i].y, a[i].y);
        v[i].z = add16x2<BF16>(v[i].z, a[i].z);
        v[i].w = add16x2<BF16>(v[i].w, a[i].w);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (t + i * TPR < nvec) {
        reinterpret_cast<uint4*>(h)[t + i * TPR] = v[i];
        float f[8];
        unpack16<BF16>(v[i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(f[j], f[j], ss);
      }
    }
    finish_row<DT, TPR, VPT, QUANT>(p, row, grp, t, nvec, ss, slots, [&](int i, float (&o)[8]) { unpack16<BF16>(v[i], o); });
  }
}

// 16-bit rows of any width whose four tensors start on the same half of a
// 4-byte word in every row: TPR threads per row, PPT pairs of columns a thread
// in registers (odd widths shift the rows' alignment one by one; the
// columns at a row's ends are moved alone).  Bound by its 2-byte weight loads
// and ragged stores: 4096 rows of 5001 47.5 us (25 the bytes'; with
// add_norm_any_kernel 70), of 1001 11.5 (with 512 threads a row 19), 30000 of 99
// 10.2 (124).  Wider rows lose to add_norm_any_kernel: 4096 of 6501 86 and 84
// us, of 9001 131 and 118.
template <int DT, int QUANT, int PPT, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) add_norm_pair_kernel(const __grid_constant__ AddNormParams p) {
  constexpr bool BF16 = DT == B200K_BF16;
  __shared__ uint32_t slots[2][32];
  constexpr int kGroups = TPR < 256 ? 256 / TPR : 1;
  const int grp = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kGroups + grp;
  if (row >= p.rows) return;  // the whole group: its barrier is its own
  const uint16_t* x = static_cast<const uint16_t*>(p.x) + row * p.x_stride;
  const uint16_t* r = static_cast<const uint16_t*>(p.r) + row * p.r_stride;
  uint16_t* h = static_cast<uint16_t*>(p.h) + row * p.cols;
  const int odd = static_cast<int>((reinterpret_cast<uintptr_t>(x) >> 1) & 1);
  auto col = [&](int i) { return 2 * (t + i * TPR) - odd; };
  uint32_t v[PPT];
  {
    uint32_t a[PPT];
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      const int c = col(i);
      if (c >= 0 && c + 1 < p.cols) {
        v[i] = __ldg(reinterpret_cast<const uint32_t*>(x + c));
        a[i] = __ldg(reinterpret_cast<const uint32_t*>(r + c));
      } else {
        const bool lo = c >= 0 && c < p.cols, hi = c + 1 < p.cols;
        v[i] = (lo ? __ldg(x + c) : 0u) | (hi ? static_cast<uint32_t>(__ldg(x + c + 1)) << 16 : 0u);
        a[i] = (lo ? __ldg(r + c) : 0u) | (hi ? static_cast<uint32_t>(__ldg(r + c + 1)) << 16 : 0u);
      }
    }
#pragma unroll
    for (int i = 0; i < PPT; ++i) v[i] = add16x2<BF16>(v[i], a[i]);
  }
  auto store = [&](uint16_t* out, int c, uint32_t u) {
    if (c >= 0 && c + 1 < p.cols) {
      *reinterpret_cast<uint32_t*>(out + c) = u;
    } else {
      if (c >= 0 && c < p.cols) out[c] = static_cast<uint16_t>(u);
      if (c + 1 < p.cols) out[c + 1] = static_cast<uint16_t>(u >> 16);
    }
  };
  auto unpack = [](uint32_t u) {
    return BF16 ? make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u))
                : __half22float2(*reinterpret_cast<const __half2*>(&u));
  };
  // weights before the barrier; where they have x's type without a switch for each
  float2 wt[PPT];
  if (p.w && p.w_dt == DT) {
    const uint16_t* w = static_cast<const uint16_t*>(p.w);
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      const int c = col(i), last = p.cols - 1;
      wt[i] = unpack(__ldg(w + min(max(c, 0), last)) | static_cast<uint32_t>(__ldg(w + min(c + 1, last))) << 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      const int c = col(i), last = p.cols - 1;
      wt[i] = p.w ? make_float2(load_scalar(p.w, min(max(c, 0), last), p.w_dt), load_scalar(p.w, min(c + 1, last), p.w_dt))
                  : make_float2(1.0f, 1.0f);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < PPT; ++i) {  // columns outside the row hold zeros
    store(h, col(i), v[i]);
    const float2 f = unpack(v[i]);
    ss = fmaf(f.x, f.x, fmaf(f.y, f.y, ss));
  }
  ss = __uint_as_float(row_reduce<TPR, false>(__float_as_uint(ss), slots[0], grp));
  const float rstd = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  const bool round_n = p.flags & B200K_ROWF_ROUND_NORMED, plus1 = p.flags & B200K_ROWF_WEIGHT_PLUS_ONE;
  float2 y[PPT];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < PPT; ++i) {
    const int c = col(i);
    y[i] = unpack(v[i]);
    y[i].x *= rstd;
    y[i].y *= rstd;
    if (round_n) y[i] = make_float2(round_to<DT>(y[i].x), round_to<DT>(y[i].y));
    if (p.w) {
      y[i].x *= plus1 ? 1.0f + wt[i].x : wt[i].x;
      y[i].y *= plus1 ? 1.0f + wt[i].y : wt[i].y;
    }
    if (QUANT == 0) {
      store(static_cast<uint16_t*>(p.out) + row * p.cols, c,
            BF16 ? pack2<true>(y[i].x, y[i].y) : pack2<false>(y[i].x, y[i].y));
    } else {
      // (a row with an infinity has NaN outside itself too: 0 * inf; they do not count)
      if (c >= 0 && c < p.cols) top = max(top, mag(y[i].x));
      if (c + 1 < p.cols) top = max(top, mag(y[i].y));
    }
  }
  if (QUANT == 1) {
    top = row_reduce<TPR, true>(top, slots[1], grp);
    float inv;
    const float sc = scale_of(top, inv);
    if (t == 0) p.scale[row] = sc;
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.cols;
#pragma unroll
    for (int i = 0; i < PPT; ++i) {
      const int c = col(i);
      const uint16_t q = e4m3x2(y[i].x * inv, y[i].y * inv);
      if (c >= 0 && c < p.cols) out[c] = static_cast<uint8_t>(q);
      if (c + 1 < p.cols) out[c + 1] = static_cast<uint8_t>(q >> 8);
    }
  }
}

// Any width, stride and alignment: a CTA per row, one column a thread and
// step, x and r read again (from L2) for each pass.
template <int DT, int QUANT>
__global__ void __launch_bounds__(512) add_norm_any_kernel(const __grid_constant__ AddNormParams p) {
  using T = typename Elem<DT>::T;
  __shared__ uint32_t slots[2][32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* r = static_cast<const T*>(p.r) + row * p.r_stride;
  T* h = static_cast<T*>(p.h) + row * p.cols;
  auto sum_at = [&](int c) { return round_to<DT>(load_scalar(x, c, DT) + load_scalar(r, c, DT)); };
  float ss = 0.0f;
#pragma unroll 4
  for (int c = threadIdx.x; c < p.cols; c += 512) {
    const float v = sum_at(c);
    store_scalar(h, c, DT, v);
    ss = fmaf(v, v, ss);
  }
  ss = __uint_as_float(row_reduce<512, false>(__float_as_uint(ss), slots[0], 0));
  const float rstd = rsqrtf(ss / static_cast<float>(p.cols) + p.eps);
  const bool round_n = p.flags & B200K_ROWF_ROUND_NORMED, plus1 = p.flags & B200K_ROWF_WEIGHT_PLUS_ONE;
  auto y_at = [&](int c) {
    float n = sum_at(c) * rstd;
    if (round_n) n = round_to<DT>(n);
    if (p.w) {
      const float w = load_scalar(p.w, c, p.w_dt);
      n *= plus1 ? 1.0f + w : w;
    }
    return n;
  };
  if constexpr (QUANT == 0) {
#pragma unroll 4
    for (int c = threadIdx.x; c < p.cols; c += 512) store_scalar(static_cast<T*>(p.out) + row * p.cols, c, DT, y_at(c));
  } else {
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.cols;
    if constexpr (QUANT == 1) {
      uint32_t top = 0;
#pragma unroll 4
      for (int c = threadIdx.x; c < p.cols; c += 512) top = max(top, mag(y_at(c)));
      top = row_reduce<512, true>(top, slots[1], 0);
      float inv;
      const float sc = scale_of(top, inv);
      if (threadIdx.x == 0) p.scale[row] = sc;
#pragma unroll 4
      for (int c = threadIdx.x; c < p.cols; c += 512) out[c] = static_cast<uint8_t>(e4m3x2(y_at(c) * inv, 0.0f) & 0xff);
    } else {  // a warp per scale: 128 columns, 4 a lane
      const int lane = threadIdx.x & 31;
      for (int g = threadIdx.x >> 5; g < (p.cols >> 7); g += 16) {
        float y[4];
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[k] = y_at(g * 128 + k * 32 + lane);
          m = max(m, mag(y[k]));
        }
        m = __reduce_max_sync(0xffffffffu, m);
        float inv;
        const float sc = scale_of(m, inv);
        if (lane == 0) p.scale[row * (p.cols >> 7) + g] = sc;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          out[g * 128 + k * 32 + lane] = static_cast<uint8_t>(e4m3x2(y[k] * inv, 0.0f) & 0xff);
      }
    }
  }
}

template <int DT, int QUANT, int TPR, int VPT, int THREADS>
void launch_vec(const AddNormParams& p, cudaStream_t st) {
  constexpr int kGroups = THREADS / TPR;
  add_norm_kernel<DT, TPR, VPT, QUANT, THREADS>
      <<<static_cast<unsigned>((p.rows + kGroups - 1) / kGroups), THREADS, 0, st>>>(p);
}

template <int DT, int QUANT>
void launch(const AddNormParams& p, bool vec, cudaStream_t st) {
  const int nvec = p.cols >> 3;
  if (!vec || nvec > 4096) {
    const unsigned rows = static_cast<unsigned>(p.rows);
    if constexpr (DT != B200K_F32 && QUANT != 2) {
      // the same half of a word in every row, for all four tensors
      const auto half = [](const void* q, int64_t stride) {
        return ((reinterpret_cast<uintptr_t>(q) >> 1) & 1) | (static_cast<uintptr_t>(stride) & 1) << 1;
      };
      const auto want = half(p.x, p.rows > 1 ? p.x_stride : p.cols);
      const bool same = want == half(p.r, p.rows > 1 ? p.r_stride : p.cols) && want == half(p.h, p.cols) &&
                        (QUANT == 1 || want == half(p.out, p.cols));
      if (same && p.cols < 6 * 1024) {
        // 2 PPT TPR columns and more than cols
        if (p.cols < 128) add_norm_pair_kernel<DT, QUANT, 2, 32><<<(rows + 7) / 8, 256, 0, st>>>(p);
        else if (p.cols < 512) add_norm_pair_kernel<DT, QUANT, 8, 32><<<(rows + 7) / 8, 256, 0, st>>>(p);
        else if (p.cols < 1024) add_norm_pair_kernel<DT, QUANT, 4, 128><<<(rows + 1) / 2, 256, 0, st>>>(p);
        else if (p.cols < 2 * 1024) add_norm_pair_kernel<DT, QUANT, 4, 256><<<rows, 256, 0, st>>>(p);
        else if (p.cols < 4 * 1024) add_norm_pair_kernel<DT, QUANT, 8, 256><<<rows, 256, 0, st>>>(p);
        else add_norm_pair_kernel<DT, QUANT, 6, 512><<<rows, 512, 0, st>>>(p);
        return;
      }
    }
    add_norm_any_kernel<DT, QUANT><<<rows, 512, 0, st>>>(p);
  // Two vectors a thread, one at 2048 columns.  bf16 with two, one and four:
  // 4096 rows of 2048 13.4, 12.4 and 14.5 us, 2048 of 4096 13.3, 13.6 and 14.6,
  // 16384 of 8192 157, 188 and 159; with an e4m3 output 16384 of 1024 23, 28.
  } else if (nvec <= 64) {
    launch_vec<DT, QUANT, 32, 2, 256>(p, st);
  } else if (nvec <= 128) {
    launch_vec<DT, QUANT, 64, 2, 256>(p, st);
  } else if (nvec <= 256) {
    launch_vec<DT, QUANT, 256, 1, 256>(p, st);
  } else if (nvec <= 512) {
    launch_vec<DT, QUANT, 256, 2, 256>(p, st);
  } else if (nvec <= 1024) {
    launch_vec<DT, QUANT, 512, 2, 512>(p, st);
  } else if (nvec <= 2048) {
    launch_vec<DT, QUANT, 512, 4, 512>(p, st);
  } else {
    launch_vec<DT, QUANT, 1024, 4, 1024>(p, st);
  }
}

template <int DT>
void launch_quant(const AddNormParams& p, int quant, bool vec, cudaStream_t st) {
  if (quant == 0) launch<DT, 0>(p, vec, st);
  else if (quant == 1) launch<DT, 1>(p, vec, st);
  else launch<DT, 2>(p, vec, st);
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200k_add_rms_norm(const B200kAddNormArgs* a, void* stream_) {
  if (!a) return B200K_ERR_ARG;
  if (a->rows < 0 || a->cols < 0) return B200K_ERR_SHAPE;
  if (a->rows == 0 || a->cols == 0) return B200K_OK;
  if (!a->x || !a->residual || !a->sum || !a->out) return B200K_ERR_ARG;
  if (a->rows > 0x7fffffffLL || a->cols > 0x3fffffffLL) return B200K_ERR_SHAPE;
  if (a->dtype != B200K_F32 && a->dtype != B200K_F16 && a->dtype != B200K_BF16) return B200K_ERR_UNSUPPORTED;
  if (a->weight && a->w_dtype != B200K_F32 && a->w_dtype != B200K_F16 && a->w_dtype != B200K_BF16)
    return B200K_ERR_UNSUPPORTED;
  if (a->flags & ~(B200K_ROWF_ROUND_NORMED | B200K_ROWF_WEIGHT_PLUS_ONE)) return B200K_ERR_UNSUPPORTED;
  const int quant = a->out_dtype == B200K_E4M3 ? (a->group == 0 ? 1 : 2) : 0;
  if (quant == 0 && a->out_dtype != a->dtype) return B200K_ERR_UNSUPPORTED;
  if (quant != 0 && !a->scale) return B200K_ERR_ARG;
  if (quant == 2 && (a->group != 128 || a->cols % 128 != 0)) return B200K_ERR_SHAPE;
  AddNormParams p;
  std::memset(&p, 0, sizeof(p));
  p.rows = a->rows;
  p.cols = static_cast<int32_t>(a->cols);
  p.x = a->x;
  p.r = a->residual;
  p.w = a->weight;
  p.h = a->sum;
  p.out = a->out;
  p.scale = a->scale;
  p.x_stride = a->x_row_stride;
  p.r_stride = a->residual_row_stride;
  p.eps = a->eps;
  p.w_dt = a->w_dtype;
  p.flags = a->flags;
  // 8 columns a thread: 16-byte (fp32: two) loads of whole vectors
  const bool vec = a->cols % 8 == 0 && a->x_row_stride % 8 == 0 && a->residual_row_stride % 8 == 0 &&
                   aligned16(a->x) && aligned16(a->residual) && aligned16(a->sum) && aligned16(a->out) &&
                   (!a->weight || aligned16(a->weight));
  cudaStream_t st = static_cast<cudaStream_t>(stream_);
  if (a->dtype == B200K_BF16) launch_quant<B200K_BF16>(p, quant, vec, st);
  else if (a->dtype == B200K_F16) launch_quant<B200K_F16>(p, quant, vec, st);
  else launch_quant<B200K_F32>(p, quant, vec, st);
  return cudaGetLastError() == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
}
