// Activations to e4m3 with a scale for every 128 columns (b200k_quant_groups,
// include/b200k.h), the input of the block-scaled product:
//
//   y = x, or silu(x[:, :cols]) * x[:, cols:] (the gate in front),
//   scale = max(max |y|, 1e-12) / 448 of 128 columns,  out = e4m3(y / scale)
//
// No reference counterpart.  fp32 throughout, one rounding to e4m3; bound by
// HBM: x is read once, one or two bytes (four with a gate) for each byte
// written.  16 lanes hold the 128 columns of a scale, 8 each, so its maximum
// is four shuffles; with many rows each takes four groups, whose loads are issued
// together.  Measured: the SwiGLU of [16384, 2 x 8192] bf16 127-135 us = 5.0-5.3 TB/s
// (154 with every call's output in memory of its own), issue slots 76 % busy; 64 rows
// of 4096 2.0 us.
#include <algorithm>
#include <cstring>

#include "e4m3.cuh"
#include "host_common.h"

namespace b200k {
namespace {

struct QuantParams {
  int64_t units;       // rows * groups
  int32_t groups;      // of a row
  int32_t cols;
  int32_t swiglu;
  int32_t big;         // units past 2^31: 64-bit division
  FastDiv div_groups;
  const void* x;
  int64_t x_stride;
  uint8_t* out;
  float* scale;
};

// silu(g) u of two values, with h = e^(-|g| / 2):
//   g u / (1 + h^2) for g >= 0,  (g / (1 + h^2) h) (h u) below,
// so nothing overflows and no factor vanishes before the result does, whatever u is
// (g / (1 + e^-g) divides by more than 2^126 from g = -87.3 on, where fast division
// gives 0).  Packed but for the exponential, the reciprocal and the choice.
__device__ __forceinline__ float2 gated2(float2 g, float2 u) {
  constexpr float kHalfLog2e = 0.5f * 1.4426950408889634f;
  const float2 one = make_float2(1.0f, 1.0f), a = __fmul2_rn(g, make_float2(kHalfLog2e, kHalfLog2e));
  float2 h, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h.x) : "f"(-fabsf(a.x)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h.y) : "f"(-fabsf(a.y)));
  const float2 d = __ffma2_rn(h, h, one);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  const float2 m = make_float2(g.x < 0.0f ? h.x : 1.0f, g.y < 0.0f ? h.y : 1.0f);
  return __fmul2_rn(__fmul2_rn(__fmul2_rn(g, r), m), __fmul2_rn(m, u));
}
__device__ __forceinline__ float gated(float g, float u) { return gated2(make_float2(g, g), make_float2(u, u)).x; }

__device__ __forceinline__ void row_of(const QuantParams& p, int64_t unit, int64_t& row, int& group) {
  row = p.big ? unit / p.groups : fdiv(static_cast<uint32_t>(unit), p.div_groups);
  group = static_cast<int>(unit - row * p.groups);
}

constexpr int kThreads = 256;
constexpr int kPerCta = kThreads / 16;  // groups side by side

template <bool BF16, bool SWIGLU, int UNITS>
__global__ void __launch_bounds__(kThreads) quant16_kernel(const __grid_constant__ QuantParams p) {
  wait_for_earlier();
  const int c0 = (threadIdx.x & 15) * 8;
  const int64_t first = blockIdx.x * static_cast<int64_t>(kPerCta * UNITS) + threadIdx.x / 16;
  uint4 a[UNITS], b[UNITS];
  int64_t row[UNITS];
  int col[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    const int64_t unit = first + i * kPerCta;
    int g = 0;
    row[i] = 0;
    col[i] = p.cols;
    a[i] = b[i] = make_uint4(0, 0, 0, 0);
    if (unit < p.units) {
      row_of(p, unit, row[i], g);
      col[i] = g * 128 + c0;
    }
    if (col[i] < p.cols) {
      const uint16_t* x = static_cast<const uint16_t*>(p.x) + row[i] * p.x_stride + col[i];
      a[i] = fetch<true>(reinterpret_cast<const uint4*>(x));
      if (SWIGLU) b[i] = fetch<true>(reinterpret_cast<const uint4*>(x + p.cols));
    }
  }
#pragma unroll
  for (int i = 0; i < UNITS; ++i) {
    float y[8];
    unpack16<BF16>(a[i], y);
    if (SWIGLU) {
      float u[8];
      unpack16<BF16>(b[i], u);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 z = gated2(make_float2(y[j], y[j + 1]), make_float2(u[j], u[j + 1]));
        y[j] = z.x;
        y[j + 1] = z.y;
      }
    }
    uint32_t top = top8(y);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    float inv, rest;
    const float s = scale_of(top, inv, rest);
    if (col[i] >= p.cols) continue;
    *reinterpret_cast<uint2*>(p.out + row[i] * p.cols + col[i]) = e4m3x8(y, inv, rest);
    if (c0 == 0) p.scale[row[i] * p.groups + col[i] / 128] = s;
  }
}

// Any type, width, stride and alignment: a warp a group, four columns a lane.
template <int DT>
__global__ void __launch_bounds__(kThreads) quant_any_kernel(const __grid_constant__ QuantParams p) {
  wait_for_earlier();
  const int lane = threadIdx.x & 31;
  for (int64_t unit = (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x) / 32; unit < p.units;
       unit += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
    int64_t row;
    int g;
    row_of(p, unit, row, g);
    float y[4];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = g * 128 + j * 32 + lane;
      y[j] = 0.0f;
      if (c < p.cols) {
        y[j] = load_scalar<true>(p.x, row * p.x_stride + c, DT);
        if (p.swiglu) y[j] = gated(y[j], load_scalar<true>(p.x, row * p.x_stride + p.cols + c, DT));
      }
      top = max(top, mag(y[j]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    float inv, rest;
    const float s = scale_of(top, inv, rest);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = g * 128 + j * 32 + lane;
      if (c < p.cols) p.out[row * p.cols + c] = e4m3(y[j], inv, rest);
    }
    if (lane == 0) p.scale[unit] = s;
  }
}

template <bool BF16, bool SWIGLU>
int launch16(const QuantParams& p, int sms, cudaStream_t st) {
  const bool many = p.units >= static_cast<int64_t>(sms) * 2048;
  const int per = kPerCta * (many ? 4 : 1);
  const int64_t grid = (p.units + per - 1) / per;
  if (grid > 0x7fffffffLL) return B200K_ERR_SHAPE;
  return launch_early(many ? quant16_kernel<BF16, SWIGLU, 4> : quant16_kernel<BF16, SWIGLU, 1>, static_cast<unsigned>(grid), kThreads,
                      0, st, p);
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200k_quant_groups(const B200kQuantGroupsArgs* a, void* stream_) {
  if (!a) return B200K_ERR_ARG;
  if (a->rows < 0 || a->cols < 0 || a->cols > 0x3fffffffLL || a->x_row_stride < 0) return B200K_ERR_SHAPE;
  if (a->dtype != B200K_F32 && a->dtype != B200K_F16 && a->dtype != B200K_BF16) return B200K_ERR_UNSUPPORTED;
  if (a->rows == 0 || a->cols == 0) return B200K_OK;
  if (a->rows > (int64_t(1) << 62) / a->cols) return B200K_ERR_SHAPE;
  if (!a->x || !a->out || !a->scale) return B200K_ERR_ARG;
  const int sms = device_sm_count();
  if (sms <= 0) return B200K_ERR_DEVICE;
  QuantParams p;
  std::memset(&p, 0, sizeof(p));
  p.groups = static_cast<int32_t>((a->cols + 127) / 128);
  p.units = a->rows * p.groups;
  p.big = p.units > 0x7fffffffLL;
  p.cols = static_cast<int32_t>(a->cols);
  p.swiglu = a->swiglu ? 1 : 0;
  p.div_groups = make_fastdiv(static_cast<uint32_t>(p.groups));
  p.x = a->x;
  p.x_stride = a->x_row_stride;
  p.out = static_cast<uint8_t*>(a->out);
  p.scale = a->scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream_);
  const bool vec = a->dtype != B200K_F32 && a->cols % 8 == 0 && aligned16(a->x) && a->x_row_stride % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(a->out) % 8 == 0;
  if (vec) {
    if (a->dtype == B200K_BF16) return p.swiglu ? launch16<true, true>(p, sms, st) : launch16<true, false>(p, sms, st);
    return p.swiglu ? launch16<false, true>(p, sms, st) : launch16<false, false>(p, sms, st);
  }
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((p.units + 7) / 8, static_cast<int64_t>(sms) * 16));
  auto kernel = a->dtype == B200K_F32 ? quant_any_kernel<B200K_F32> : a->dtype == B200K_F16 ? quant_any_kernel<B200K_F16>
                                                                                            : quant_any_kernel<B200K_BF16>;
  return launch_early(kernel, grid, kThreads, 0, st, p);
}
