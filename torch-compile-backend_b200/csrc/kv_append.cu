// Rotary embedding of new queries and keys together with the append of the
// keys and values to a paged cache (b200k_rope_append, include/b200k.h):
//
//   rot(x)[j]       = x[j] cos[p, j] - x[j + R/2] sin[p, j]       j < R/2
//   rot(x)[j + R/2] = x[j + R/2] cos[p, j] + x[j] sin[p, j]
//   rot(x)[j]       = x[j]                                        j >= R
//   q_out[t] = rot(q[t]);  k_cache[slot[t]] = rot(k[t]);  v_cache[slot[t]] = v[t]
//
// No reference counterpart (its rotation is neg / cat / mul / add of ATen and
// generated kernels, and it has no cache).  One launch replaces the two
// rotations, the two scatters and the copies between them; what bounds it is
// HBM for prompts and latency for single tokens.  Products and sums are fp32
// (the tables' 32-bit values matter at far positions), each result is rounded
// once to the 16-bit type.
//
// A thread takes one pair of 8-element chunks, the two halves that a rotation
// mixes (or two chunks that are copied), of NH heads of one token: the table
// entries are read once for NH heads and NH x 32 bytes are in flight a thread.
#include <algorithm>
#include <cstring>

#include "common.cuh"
#include "host_common.h"

namespace b200k {
namespace {

struct AppendParams {
  FastDiv div_tok, div_unit;  // thread -> token; thread in token -> (head block, unit)
  int64_t tokens;
  int32_t heads, kv_heads, dim, rot;
  int32_t threads_per_token, units;  // units: pairs of chunks of a head
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_cache, *v_cache;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;      // element strides: token, head
  int64_t c_page, c_slot, c_head;            // cache strides (both caches)
  const void *cos, *sin;
  int64_t table_stride, table_rows;
  const void *positions, *slots;
  int32_t pos64, slot64;
  int32_t page_size;
  FastDiv div_page;
  int64_t total_slots;
  int32_t* status;
};

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? __ldg(static_cast<const long long*>(p) + i) : __ldg(static_cast<const int*>(p) + i);
}

// Where a token goes: its table row (clamped into the table) and its offset
// in the caches, -1 for a token that is not appended.  An index outside the
// table or the cache is reported and its token not appended.
struct Place {
  int64_t row, cache;
};
__device__ __forceinline__ Place place_of(const AppendParams& p, int64_t t) {
  int64_t pos = load_index(p.positions, t, p.pos64), slot = load_index(p.slots, t, p.slot64);
  const bool pos_ok = pos >= 0 && pos < p.table_rows;
  if (slot >= p.total_slots || (!pos_ok && slot >= 0)) {
    if (p.status) atomicCAS(p.status, 0, B200K_ERR_INDEX);
    slot = -1;
  }
  Place r;
  r.row = pos_ok ? pos : 0;
  r.cache = -1;
  if (slot >= 0) {
    const uint32_t page = fdiv(static_cast<uint32_t>(slot), p.div_page);
    const uint32_t off = static_cast<uint32_t>(slot) - page * static_cast<uint32_t>(p.page_size);
    r.cache = static_cast<int64_t>(page) * p.c_page + static_cast<int64_t>(off) * p.c_slot;
  }
  return r;
}

constexpr int kThreads = 128;  // 35.2 us for 16384 tokens of 48 heads of 64, 37.3 with CTAs of 256

template <bool BF16, int TAB_DT, int NH>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const __grid_constant__ AppendParams p) {
  const uint32_t gid = blockIdx.x * static_cast<uint32_t>(kThreads) + threadIdx.x;
  const uint32_t tok = fdiv(gid, p.div_tok);
  if (tok >= p.tokens) return;
  const uint32_t in_tok = gid - tok * p.div_tok.d;
  const uint32_t hb = fdiv(in_tok, p.div_unit);
  const int unit = static_cast<int>(in_tok - hb * p.div_unit.d);
  const int rot_units = p.rot >> 4;
  const bool turns = unit < rot_units;
  // the unit's two chunks: the halves of a rotation, or two neighbours behind it
  const int c0 = (turns ? unit : 2 * unit) * 8, c1 = turns ? c0 + (p.rot >> 1) : c0 + 8;
  const int head0 = static_cast<int>(hb) * NH, all = p.heads + 2 * p.kv_heads;
  uint4 a[NH], b[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const int h = min(head0 + i, all - 1);
    const uint16_t* src;
    if (h < p.heads) src = p.q + tok * p.q_t + h * p.q_h;
    else if (h < p.heads + p.kv_heads) src = p.k + tok * p.k_t + (h - p.heads) * p.k_h;
    else src = p.v + tok * p.v_t + (h - p.heads - p.kv_heads) * p.v_h;
    a[i] = __ldg(reinterpret_cast<const uint4*>(src + c0));
    b[i] = __ldg(reinterpret_cast<const uint4*>(src + c1));
  }
  const Place pl = place_of(p, tok);
  float cs[8], sn[8];
  if (turns) {
    load_vec8(p.cos, pl.row * p.table_stride + c0, TAB_DT, cs);
    load_vec8(p.sin, pl.row * p.table_stride + c0, TAB_DT, sn);
  }
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const int h = head0 + i;
    if (h >= all) break;
    uint16_t* dst;
    if (h < p.heads) {
      dst = p.q_out + (static_cast<int64_t>(tok) * p.heads + h) * p.dim;
    } else {
      if (pl.cache < 0) continue;
      dst = h < p.heads + p.kv_heads ? p.k_cache + pl.cache + (h - p.heads) * p.c_head
                                     : p.v_cache + pl.cache + (h - p.heads - p.kv_heads) * p.c_head;
    }
    uint4 oa = a[i], ob = b[i];
    if (turns && h < p.heads + p.kv_heads) {
      float x[8], y[8], u[8], w[8];
      unpack8<BF16>(a[i], x);
      unpack8<BF16>(b[i], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = x[j] * cs[j] - y[j] * sn[j];
        w[j] = y[j] * cs[j] + x[j] * sn[j];
      }
      oa = BF16 ? pack_bf16x8(u) : pack_f16x8(u);
      ob = BF16 ? pack_bf16x8(w) : pack_f16x8(w);
    }
    *reinterpret_cast<uint4*>(dst + c0) = oa;
    *reinterpret_cast<uint4*>(dst + c1) = ob;
  }
}

// Any even rotary width, head size and alignment: one element a thread.
template <bool BF16, int TAB_DT>
__global__ void __launch_bounds__(256) rope_append_any_kernel(const __grid_constant__ AppendParams p) {
  const int all = p.heads + 2 * p.kv_heads;
  const int64_t per_tok = static_cast<int64_t>(all) * p.dim, n = p.tokens * per_tok;
  constexpr int DT = BF16 ? B200K_BF16 : B200K_F16;
  for (int64_t e = blockIdx.x * 256ll + threadIdx.x; e < n; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t tok = e / per_tok;
    const int in_tok = static_cast<int>(e - tok * per_tok);
    const int h = in_tok / p.dim, j = in_tok - h * p.dim;
    const Place pl = place_of(p, tok);
    const uint16_t* src;
    if (h < p.heads) src = p.q + tok * p.q_t + h * p.q_h;
    else if (h < p.heads + p.kv_heads) src = p.k + tok * p.k_t + (h - p.heads) * p.k_h;
    else src = p.v + tok * p.v_t + (h - p.heads - p.kv_heads) * p.v_h;
    uint16_t* dst;
    if (h < p.heads) {
      dst = p.q_out + (tok * p.heads + h) * p.dim;
    } else {
      if (pl.cache < 0) continue;
      dst = h < p.heads + p.kv_heads ? p.k_cache + pl.cache + (h - p.heads) * p.c_head
                                     : p.v_cache + pl.cache + (h - p.heads - p.kv_heads) * p.c_head;
    }
    if (j < p.rot && h < p.heads + p.kv_heads) {
      const int half = p.rot >> 1, i = j < half ? j : j - half;
      const float c = load_scalar(p.cos, pl.row * p.table_stride + i, TAB_DT);
      const float s = load_scalar(p.sin, pl.row * p.table_stride + i, TAB_DT);
      const float x = load_scalar(src, i, DT), y = load_scalar(src, i + half, DT);
      store_scalar(dst, j, DT, j < half ? x * c - y * s : y * c + x * s);
    } else {
      dst[j] = src[j];
    }
  }
}

template <bool BF16, int TAB_DT>
int launch(AppendParams& p, bool vec, int sms, cudaStream_t st) {
  const int all = p.heads + 2 * p.kv_heads;
  if (vec) {
    p.units = p.dim / 16;
    p.div_unit = make_fastdiv(static_cast<uint32_t>(p.units));
    // Four heads a thread once one head a thread would fill half of the GPU's
    // threads; one below, where a launch is bound by the latency of its loads.
    // Of 48 heads of 128 with four and with one: 8192 tokens 33.7 and 37.7 us,
    // 1000 5.9 and 6.6, 500 3.5 and 3.7, 250 3.2 and 2.8, 100 2.8 and 2.3.
    const int64_t few = p.tokens * all * p.units;
    const int nh = few >= static_cast<int64_t>(sms) * 1024 ? 4 : 1;
    p.threads_per_token = p.units * ((all + nh - 1) / nh);
    const int64_t n = p.tokens * p.threads_per_token;
    if (n + kThreads <= 0x7fffffffLL) {
      p.div_tok = make_fastdiv(static_cast<uint32_t>(p.threads_per_token));
      const unsigned grid = static_cast<unsigned>((n + kThreads - 1) / kThreads);
      if (nh == 4) rope_append_kernel<BF16, TAB_DT, 4><<<grid, kThreads, 0, st>>>(p);
      else rope_append_kernel<BF16, TAB_DT, 1><<<grid, kThreads, 0, st>>>(p);
      return cudaGetLastError() == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
    }
  }
  const int64_t n = p.tokens * all * p.dim;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, static_cast<int64_t>(sms) * 8));
  rope_append_any_kernel<BF16, TAB_DT><<<grid, 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200K_OK : B200K_ERR_LAUNCH;
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200k_rope_append(const B200kRopeAppendArgs* a, void* stream_) {
  if (!a) return B200K_ERR_ARG;
  if (a->tokens < 0 || a->heads < 0 || a->kv_heads < 0 || a->head_dim < 0 || a->num_pages < 0 || a->page_size < 0)
    return B200K_ERR_SHAPE;
  if (a->tokens == 0 || a->head_dim == 0 || a->heads + a->kv_heads == 0) return B200K_OK;
  if (!a->positions || !a->slots || (a->heads && (!a->q || !a->q_out))) return B200K_ERR_ARG;
  if (a->kv_heads && (!a->k || !a->v)) return B200K_ERR_ARG;
  if (a->dtype != B200K_BF16 && a->dtype != B200K_F16) return B200K_ERR_UNSUPPORTED;
  if (a->table_dtype != B200K_F32 && a->table_dtype != a->dtype) return B200K_ERR_UNSUPPORTED;
  for (int dt : {a->positions_dtype, a->slots_dtype})
    if (dt != B200K_I32 && dt != B200K_I64) return B200K_ERR_UNSUPPORTED;
  if (a->rot_dim < 0 || a->rot_dim > a->head_dim || a->rot_dim % 2) return B200K_ERR_SHAPE;
  if (a->rot_dim && (!a->cos || !a->sin || a->table_rows <= 0)) return B200K_ERR_ARG;
  if (a->heads > 65536 || a->kv_heads > 65536 || a->head_dim > 65536 || a->tokens > 0x7fffffffLL ||
      a->page_size > 0x7fffffffLL || a->num_pages > 0x7fffffffLL || a->num_pages * a->page_size > 0x7fffffffLL)
    return B200K_ERR_SHAPE;
  const int64_t total = a->num_pages * a->page_size;
  if (a->kv_heads && total && (!a->k_cache || !a->v_cache)) return B200K_ERR_ARG;
  const int sms = device_sm_count();
  if (sms <= 0) return B200K_ERR_DEVICE;
  AppendParams p;
  std::memset(&p, 0, sizeof(p));
  p.tokens = a->tokens;
  p.heads = static_cast<int32_t>(a->heads);
  p.kv_heads = static_cast<int32_t>(a->kv_heads);
  p.dim = static_cast<int32_t>(a->head_dim);
  p.rot = static_cast<int32_t>(a->rot_dim);
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k);
  p.v = static_cast<const uint16_t*>(a->v);
  p.q_out = static_cast<uint16_t*>(a->q_out);
  p.k_cache = static_cast<uint16_t*>(a->k_cache);
  p.v_cache = static_cast<uint16_t*>(a->v_cache);
  p.q_t = a->q_strides[0]; p.q_h = a->q_strides[1];
  p.k_t = a->k_strides[0]; p.k_h = a->k_strides[1];
  p.v_t = a->v_strides[0]; p.v_h = a->v_strides[1];
  p.c_page = a->cache_strides[0]; p.c_slot = a->cache_strides[1]; p.c_head = a->cache_strides[2];
  p.cos = a->cos;
  p.sin = a->sin;
  p.table_stride = a->table_stride;
  p.table_rows = a->rot_dim ? a->table_rows : 0x7fffffffffffffffLL;
  p.positions = a->positions;
  p.slots = a->slots;
  p.pos64 = a->positions_dtype == B200K_I64;
  p.slot64 = a->slots_dtype == B200K_I64;
  p.page_size = static_cast<int32_t>(a->page_size);
  p.div_page = make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(1, a->page_size)));
  p.total_slots = total;
  p.status = a->status;
  bool vec = a->head_dim % 16 == 0 && a->rot_dim % 16 == 0 && a->table_stride % 8 == 0;
  for (const void* x : {a->q, a->k, a->v, static_cast<const void*>(a->q_out), static_cast<const void*>(a->k_cache),
                        static_cast<const void*>(a->v_cache), a->cos, a->sin})
    vec = vec && aligned16(x);
  for (int d = 0; d < 2; ++d) vec = vec && a->q_strides[d] % 8 == 0 && a->k_strides[d] % 8 == 0 && a->v_strides[d] % 8 == 0;
  for (int d = 0; d < 3; ++d) vec = vec && a->cache_strides[d] % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream_);
  const bool f32 = a->table_dtype == B200K_F32;
  if (a->dtype == B200K_BF16)
    return f32 ? launch<true, B200K_F32>(p, vec, sms, st) : launch<true, B200K_BF16>(p, vec, sms, st);
  return f32 ? launch<false, B200K_F32>(p, vec, sms, st) : launch<false, B200K_F16>(p, vec, sms, st);
}
