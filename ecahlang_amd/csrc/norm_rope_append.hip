// RMS norm of every query and key head, rotary embedding and K/V append in one launch:
//
//   pkv_append_paged_kv_cache_norm_rope  <- q_norm / k_norm and apply_rotary_pos_emb of models that normalise
//                                           their heads, then the hook's append (ecahlang/main.py:62-66)
//
// Per row x[0 .. D) of a query or key head with weight w, and the token's cos and sin:
//   y[d] = x[d] / sqrt(mean(x^2) + eps) * w[d]
//   out[d]       = y[d] cos[d]             - y[d + D/2] sin[d]            d < D/2
//   out[d + D/2] = y[d + D/2] cos[d + D/2] + y[d] sin[d + D/2]
// all in fp32 and rounded once, to the type of q_out or the cache, or to e4m3 with the row's scale
// (cache_fp8.h).  Without a weight the rows are not normalised.  Value rows are copied, or rounded to e4m3.
//
// A wave takes rows of one token: a group of D / 16 lanes (rounded up to a power of two) a row, each lane 8
// elements of either half, so the rotation's partners meet in one lane and the sum of squares takes a few
// lane exchanges.
#include "cache_fp8.h"
#include "../../include/pagedkv.h"

#include <type_traits>

using namespace pkv;
using namespace pkv::fp8;

namespace {

struct NormRopeArgs {
  const void* q;
  int64_t q_sn, q_sh;
  void* q_out;
  int64_t qo_sn, qo_sh;
  const void *k, *v;
  int64_t k_sn, k_sh, v_sn, v_sh;
  const void *qw, *kw;  // null: that kind of row is not normalised
  const void *cos, *sin;
  int64_t cs_sn;
  float eps;
  Table t;
  Dest o;
  int32_t nnz, hq, hkv, d, lanes, splits, w_f32, cs_f32;
  int32_t* err;
};

// 8 weights or angles, of the rows' type or fp32 (wave-uniform).
template <typename T, bool VEC>
__device__ __forceinline__ void load8f(const void* p, int64_t at, bool f32, float (&x)[8]) {
  if (f32) {
    Eight<float, VEC> r;
    r.load((const float*)p + at);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = r.e[j];
  } else {
    Eight<T, VEC> r;
    r.load((const T*)p + at);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = to_f32(r.e[j]);
  }
}

template <typename T, bool QUANT, bool VEC>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a) {
  const int lane = threadIdx.x & 63, sub = lane & (a.lanes - 1), per = 64 / a.lanes, half = a.d / 2;
  const bool act = 8 * sub < half;
  const int d0 = act ? 8 * sub : 0;
  const int rows = a.hq + 2 * a.hkv;
  const int gw = __builtin_amdgcn_readfirstlane(blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6));
  const int nt = gridDim.x * (blockDim.x >> 6) / a.splits;  // tokens at a time
  const int split = gw % a.splits;
  for (int64_t tok = gw / a.splits; tok < a.nnz && gw < nt * a.splits; tok += nt) {
    float c0[8], c1[8], s0[8], s1[8];
    load8f<T, VEC>(a.cos, tok * a.cs_sn + d0, a.cs_f32, c0);
    load8f<T, VEC>(a.cos, tok * a.cs_sn + d0 + half, a.cs_f32, c1);
    load8f<T, VEC>(a.sin, tok * a.cs_sn + d0, a.cs_f32, s0);
    load8f<T, VEC>(a.sin, tok * a.cs_sn + d0 + half, a.cs_f32, s1);
    int page = 0, slot = 0;
    const bool ok = resolve(a.t, tok, page, slot);
    if (!ok && split == 0 && lane == 0 && a.err) atomicAdd(a.err, 1);
    for (int r0 = split * per; r0 < rows; r0 += a.splits * per) {
      const int rr = r0 + lane / a.lanes, row = rr < rows ? rr : rows - 1;
      const bool isq = row < a.hq, isv = row >= a.hq + a.hkv;
      const int h = isq ? row : (isv ? row - a.hq - a.hkv : row - a.hq);
      const T* src = isq ? (const T*)a.q + tok * a.q_sn + h * a.q_sh
                         : (isv ? (const T*)a.v + tok * a.v_sn + h * a.v_sh : (const T*)a.k + tok * a.k_sn + h * a.k_sh);
      Eight<T, VEC> lo, hi;
      lo.load(src + d0);
      hi.load(src + d0 + half);
      float x[8], y[8];
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = to_f32(lo.e[j]), y[j] = to_f32(hi.e[j]);
        ss += x[j] * x[j] + y[j] * y[j];
      }
      ss = group_sum(act ? ss : 0.f, a.lanes);
      if (!isv) {
        const void* w = isq ? a.qw : a.kw;
        if (w) {
          const float rs = 1.f / sqrtf(ss / (float)a.d + a.eps);
          float w0[8], w1[8];
          load8f<T, VEC>(w, d0, a.w_f32, w0);
          load8f<T, VEC>(w, d0 + half, a.w_f32, w1);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = x[j] * rs * w0[j], y[j] = y[j] * rs * w1[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float u = x[j] * c0[j] - y[j] * s0[j], z = y[j] * c1[j] + x[j] * s1[j];
          x[j] = u, y[j] = z;
          lo.e[j] = from_f32<T>(u), hi.e[j] = from_f32<T>(z);
        }
      }
      const bool in = rr < rows && act;
      int e = 0;
      if constexpr (QUANT) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = amax_bits(amax_bits(m, x[j]), y[j]);
        e = scale_byte(group_max(act ? m : 0u, a.lanes));
      }
      if (isq) {
        if (in) {
          T* dst = (T*)a.q_out + tok * a.qo_sn + h * a.qo_sh + d0;
          lo.store(dst);
          hi.store(dst + half);
        }
      } else if (in && ok) {
        const int64_t at = page * a.o.page_stride + ((int64_t)slot * a.hkv + h) * a.d + d0;
        if constexpr (QUANT) {
          uint8_t* dst = (uint8_t*)(isv ? a.o.v : a.o.k) + at;
          const float inv = inv_scale(e);
          store8<VEC>(dst, x, inv);
          store8<VEC>(dst + half, y, inv);
          if (sub == 0) (isv ? a.o.vs : a.o.ks)[page * a.o.scale_stride + (int64_t)h * a.t.ps + slot] = (uint8_t)e;
        } else {
          T* dst = (T*)(isv ? a.o.v : a.o.k) + at;
          lo.store(dst);
          hi.store(dst + half);
        }
      }
    }
  }
}

}  // namespace

extern "C" int pkv_append_paged_kv_cache_norm_rope(
    const void* q, int64_t q_stride_n, int64_t q_stride_h, void* q_out, int64_t qo_stride_n, int64_t qo_stride_h,
    int32_t num_qo_heads, const void* append_key, int64_t k_stride_n, int64_t k_stride_h, const void* append_value,
    int64_t v_stride_n, int64_t v_stride_h, const void* q_weight, const void* k_weight, int32_t weight_dtype, float eps,
    const void* cos, const void* sin, int64_t cs_stride_n, int32_t cs_dtype, const int32_t* batch_indices,
    const int32_t* positions, int32_t nnz, void* k_cache, void* v_cache, int64_t page_stride, int64_t num_pages,
    void* k_scales, void* v_scales, int64_t scale_page_stride, const int32_t* kv_indices, int64_t num_indices,
    const int32_t* kv_indptr, int32_t batch, int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype,
    int32_t* err_count, void* stream) {
  const int es = dtype == kF32 ? 4 : (dtype == kF16 || dtype == kBF16) ? 2 : 0;
  if (!es || (weight_dtype != dtype && weight_dtype != kF32) || (cs_dtype != dtype && cs_dtype != kF32)) return kBadDType;
  if (nnz < 0 || num_qo_heads < 0 || num_kv_heads <= 0 || page_size <= 0 || batch < 0 || num_indices < 0) return kBadArg;
  if (!head_dim_ok(head_dim)) return kBadHeadDim;
  if (nnz == 0) return kOk;
  const bool quant = k_scales != nullptr;
  if (quant != (v_scales != nullptr) || !cos || !sin || !batch_indices || !positions || !kv_indptr) return kBadArg;
  const int lanes = lanes_of(head_dim), per = 64 / lanes, rows = num_qo_heads + 2 * num_kv_heads;
  // The waves a token's rows are shared by: all there is work for while tokens are few.
  const int most = (rows + per - 1) / per;
  const int64_t spread = (8192 + (int64_t)nnz - 1) / nnz;
  const int splits = spread < most ? (int)spread : most;
  const NormRopeArgs a{q, q_stride_n, q_stride_h, q_out, qo_stride_n, qo_stride_h, append_key, append_value, k_stride_n,
                       k_stride_h, v_stride_n, v_stride_h, q_weight, k_weight, cos, sin, cs_stride_n, eps,
                       {batch_indices, positions, nullptr, kv_indices, kv_indptr, num_indices, num_pages, batch, page_size},
                       {k_cache, v_cache, (uint8_t*)k_scales, (uint8_t*)v_scales, page_stride, scale_page_stride},
                       nnz, num_qo_heads, num_kv_heads, head_dim, lanes, splits,
                       weight_dtype == kF32, cs_dtype == kF32, err_count};
  const uintptr_t m = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)append_key | (uintptr_t)append_value;
  const uintptr_t cs = (uintptr_t)cos | (uintptr_t)sin, ws = (uintptr_t)q_weight | (uintptr_t)k_weight;
  const uintptr_t to = (uintptr_t)k_cache | (uintptr_t)v_cache;
  if ((m % es) || cs % (cs_dtype == kF32 ? 4 : es) || ws % (weight_dtype == kF32 ? 4 : es) || (!quant && to % es)) return kBadAlign;
  const int64_t st = q_stride_n | q_stride_h | qo_stride_n | qo_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h;
  const bool vec = (m | cs | ws) % 16 == 0 && st * es % 16 == 0 && cs_stride_n * (cs_dtype == kF32 ? 4 : es) % 16 == 0 &&
                   (quant ? to % 8 == 0 && page_stride % 8 == 0 : to % 16 == 0 && page_stride * es % 16 == 0);
  const int64_t waves = (int64_t)nnz * splits, want = (waves + 3) / 4;
  const dim3 grid((unsigned)(want < 16384 ? want : 16384));
  hipStream_t s = (hipStream_t)stream;
#define PKV_NORM_ROPE(T, Q, V) hipLaunchKernelGGL((norm_rope_kernel<T, Q, V>), grid, dim3(256), 0, s, a)
#define PKV_NORM_ROPE_T(T)                                                         \
  if (quant) { if (vec) PKV_NORM_ROPE(T, true, true); else PKV_NORM_ROPE(T, true, false); }    \
  else { if (vec) PKV_NORM_ROPE(T, false, true); else PKV_NORM_ROPE(T, false, false); }
  if (dtype == kF16) {
    PKV_NORM_ROPE_T(_Float16)
  } else if (dtype == kBF16) {
    PKV_NORM_ROPE_T(__hip_bfloat16)
  } else {
    PKV_NORM_ROPE_T(float)
  }
#undef PKV_NORM_ROPE_T
#undef PKV_NORM_ROPE
  return (int)hipGetLastError();
}
