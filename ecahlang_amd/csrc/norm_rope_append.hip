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
// A group of D / 16 lanes (rounded up to a power of two) takes a row, each lane 8 elements of either half, so
// the rotation's partners meet in one lane and the sum of squares takes a few lane exchanges.  The rows of all
// tokens are dealt out in one run, 8 of 128 dims to a wave, whatever the heads of a token are: a wave that kept
// to one token, its angles in registers, idled lanes wherever the heads do not divide by 8 and waited for each
// token's page by itself (4003 tokens, 32 / 8 heads of 128: 20 us for 30, a step of 4 tokens 3.0 for 4.8).
//
// What bounds it: the bytes, beside some 250 vector instructions a wave's 8 rows, about half the time at full
// rate: 16,003 tokens, 32 / 8 heads of 128, bf16 into 8 bits, 80 us for 369 MB (71 at the rate of a large copy).
#include "cache_fp8.h"
#include "../../include/pagedkv.h"

#include <type_traits>

using namespace pkv;
using namespace pkv::fp8;

namespace {

// Workgroups at most: more of them than the chip holds at once (1280), so that their phases mix (the bulk above: 88 us
// with 1024 or 2048, 83 with 4096, 79 with 8192, 81 with 16,384; a workgroup costs some 3.5 ns to start).
constexpr int kGrid = 8192;

struct NormRopeArgs {
  const void* q;
  void* q_out;
  const void *k, *v;
  Strides qs, os, ks, vs;
  const void *qw, *kw;  // null: that kind of row is not normalised
  const void *cos, *sin;
  Strides cs;
  float eps;
  Table t;
  Dest o;
  Div rows;
  int32_t nnz, hq, hkv, d, lanes, w_f32, cs_f32;
  int32_t* err;
};

// 8 weights or angles: of the rows' type, or (MIXED) of that or fp32 as the call says.
template <typename T, bool VEC, bool MIXED>
struct Coef {
  Eight<T, VEC> r;
  Eight<float, VEC> f;
  // 8 at element `at` of p
  __device__ __forceinline__ void load(const void* p, int at, bool f32) {
    if (MIXED && f32) f.load((const float*)p + at);
    else r.load((const T*)p + at);
  }
  __device__ __forceinline__ void get(float (&x)[8], bool f32) const {
    if (MIXED && f32) f.get(x);
    else r.get(x);
  }
};

// Rows of all tokens in one run (token, then query, key and value heads): a group of lanes takes one row at a
// time, wherever tokens end.  Everything a row needs is requested at once; only key and value rows look up
// their page.
template <typename T, bool QUANT, bool VEC, bool MIXED>
__global__ __launch_bounds__(256, 4) void norm_rope_kernel(NormRopeArgs a) {
  const int lane = threadIdx.x & 63, sub = lane & (a.lanes - 1), per = 64 / a.lanes, half = a.d / 2;
  const bool act = 8 * sub < half;
  const int d0 = act ? 8 * sub : 0;
  const uint32_t total = (uint32_t)a.nnz * a.rows.d;
  const uint32_t stride = gridDim.x * (blockDim.x >> 6) * per;
  const float inv_d = 1.f / (float)a.d;
  uint32_t base = __builtin_amdgcn_readfirstlane((blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6)) * per);
  for (; base < total; base += stride) {
    const uint32_t at = base + lane / a.lanes, idx = at < total ? at : total - 1;
    const uint32_t tok = a.rows.of(idx);
    const int row = idx - tok * a.rows.d;
    const bool isq = row < a.hq, isv = row >= a.hq + a.hkv, in = at < total && act;
    const int h = isq ? row : (isv ? row - a.hq - a.hkv : row - a.hq);
    const Strides st{isq ? a.qs.n : isv ? a.vs.n : a.ks.n, isq ? a.qs.h : isv ? a.vs.h : a.ks.h};
    const T* src = (const T*)row_at(isq ? a.q : isv ? a.v : a.k, st, tok, h) + d0;
    Eight<T, VEC> lo, hi;
    lo.load(src);
    hi.load(src + half);
    const void *cosr = row_at(a.cos, a.cs, tok, 0), *sinr = row_at(a.sin, a.cs, tok, 0);
    Coef<T, VEC, MIXED> c0, c1, s0, s1;
    c0.load(cosr, d0, a.cs_f32);
    c1.load(cosr, d0 + half, a.cs_f32);
    s0.load(sinr, d0, a.cs_f32);
    s1.load(sinr, d0 + half, a.cs_f32);
    asm volatile("" ::: "memory");
    int page = 0, slot = 0;
    bool ok = false;
    if (!isq) {
      ok = resolve(a.t, tok, page, slot);
      if (!ok && at < total && row == a.hq && sub == 0 && a.err) atomicAdd(a.err, 1);
    }
    float x[8], y[8];
    lo.get(x);
    hi.get(y);
    if (__ballot(!isv)) {
      // (four short sums and a Newton step on the hardware's 1 / sqrt: the factor is common to the row, so its error
      // moves every key next to a tie of e4m3 to the other side.  Some 20 of 16 million do so still, 28 with plain fp32
      // operations; none where keys are computed in 64 bits, which takes 143 us for 79 in the bulk above)
      float sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) sq[j & 3] = __builtin_fmaf(x[j], x[j], __builtin_fmaf(y[j], y[j], sq[j & 3]));
      float ss = (sq[0] + sq[1]) + (sq[2] + sq[3]);
      ss = group_sum(act ? ss : 0.f, a.lanes);
      if (!isv) {
        const void* w = isq ? a.qw : a.kw;
        if (w) {
          const float ms = __builtin_fmaf(ss, inv_d, a.eps), r0 = __builtin_amdgcn_rsqf(ms);
          const float off = __builtin_fmaf(-ms * r0, r0, 1.f), rs = off == off ? __builtin_fmaf(0.5f * r0, off, r0) : r0;
          Coef<T, VEC, MIXED> w0, w1;
          w0.load(w, d0, a.w_f32);
          w1.load(w, d0 + half, a.w_f32);
          float u[8];
          w0.get(u, a.w_f32);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= rs * u[j];
          w1.get(u, a.w_f32);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= rs * u[j];
        }
        float c[8], s[8], z[8];
        c0.get(c, a.cs_f32);
        s0.get(s, a.cs_f32);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = x[j] * c[j] - y[j] * s[j];
        c1.get(c, a.cs_f32);
        s1.get(s, a.cs_f32);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = y[j] * c[j] + x[j] * s[j], x[j] = z[j];
        if (!QUANT || isq) lo.set(x), hi.set(y);
      }
    }
    if (in && (isq || (!QUANT && ok))) {
      T* dst = (isq ? (T*)row_at(a.q_out, a.os, tok, h)
                    : (T*)(isv ? a.o.v : a.o.k) + page * a.o.page_stride + (uint32_t)((slot * a.hkv + h) * a.d)) + d0;
      lo.store(dst, !isq);
      hi.store(dst + half, !isq);
    }
    if (QUANT && __ballot(!isq)) {
      const int e = row_scale(x, y, act, a.lanes);
      if (in && ok) {
        uint8_t* dst = (uint8_t*)(isv ? a.o.v : a.o.k) + page * a.o.page_stride + (uint32_t)((slot * a.hkv + h) * a.d + d0);
        const float inv = inv_scale(e);
        store8<VEC>(dst, x, inv);
        store8<VEC>(dst + half, y, inv);
        if (sub == 0) (isv ? a.o.vs : a.o.ks)[page * a.o.scale_stride + (h * a.t.ps.d + slot)] = (uint8_t)e;
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
  if (!append_key || !append_value || (num_qo_heads > 0 && (!q || !q_out)) || (num_pages > 0 && (!k_cache || !v_cache)))
    return kBadArg;
  if (quant != (v_scales != nullptr) || !cos || !sin || !batch_indices || !positions || !kv_indptr) return kBadArg;
  const int lanes = lanes_of(head_dim), per = 64 / lanes, rows = num_qo_heads + 2 * num_kv_heads;
  const int64_t total = (int64_t)nnz * rows;
  if (total > INT32_MAX) return kBadArg;
  Strides qs, os, ks, vs, cs;
  if (!strides_of(q_stride_n, q_stride_h, es, &qs) || !strides_of(qo_stride_n, qo_stride_h, es, &os) ||
      !strides_of(k_stride_n, k_stride_h, es, &ks) || !strides_of(v_stride_n, v_stride_h, es, &vs) ||
      !strides_of(cs_stride_n, 0, cs_dtype == kF32 ? 4 : es, &cs) || !page_fits(page_size, num_kv_heads, head_dim))
    return kBadArg;
  const NormRopeArgs a{q, q_out, append_key, append_value, qs, os, ks, vs, q_weight, k_weight, cos, sin, cs, eps,
                       {batch_indices, positions, nullptr, kv_indices, kv_indptr, num_indices, num_pages, batch, Div(page_size)},
                       {k_cache, v_cache, (uint8_t*)k_scales, (uint8_t*)v_scales, page_stride, scale_page_stride},
                       Div(rows), nnz, num_qo_heads, num_kv_heads, head_dim, lanes, weight_dtype == kF32, cs_dtype == kF32,
                       err_count};
  const uintptr_t m = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)append_key | (uintptr_t)append_value;
  const uintptr_t an = (uintptr_t)cos | (uintptr_t)sin, ws = (uintptr_t)q_weight | (uintptr_t)k_weight;
  const uintptr_t to = (uintptr_t)k_cache | (uintptr_t)v_cache;
  if ((m % es) || an % (cs_dtype == kF32 ? 4 : es) || ws % (weight_dtype == kF32 ? 4 : es) || (!quant && to % es)) return kBadAlign;
  const int64_t st = q_stride_n | q_stride_h | qo_stride_n | qo_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h;
  const bool vec = (m | an | ws) % 16 == 0 && st * es % 16 == 0 && cs_stride_n * (cs_dtype == kF32 ? 4 : es) % 16 == 0 &&
                   (quant ? to % 8 == 0 && page_stride % 8 == 0 : to % 16 == 0 && page_stride * es % 16 == 0);
  const int64_t want = (total + 4 * per - 1) / (4 * per);
  const dim3 grid((unsigned)(want < kGrid ? want : kGrid));
  const bool mixed = weight_dtype != dtype || cs_dtype != dtype;
  hipStream_t s = (hipStream_t)stream;
#define PKV_NORM_ROPE(T, Q, V, M) hipLaunchKernelGGL((norm_rope_kernel<T, Q, V, M>), grid, dim3(256), 0, s, a)
#define PKV_NORM_ROPE_Q(T, Q)                                                              \
  if (vec) { if (mixed) PKV_NORM_ROPE(T, Q, true, true); else PKV_NORM_ROPE(T, Q, true, false); }   \
  else { if (mixed) PKV_NORM_ROPE(T, Q, false, true); else PKV_NORM_ROPE(T, Q, false, false); }
#define PKV_NORM_ROPE_T(T) \
  if (quant) { PKV_NORM_ROPE_Q(T, true) } else { PKV_NORM_ROPE_Q(T, false) }
  if (dtype == kF16) {
    PKV_NORM_ROPE_T(_Float16)
  } else if (dtype == kBF16) {
    PKV_NORM_ROPE_T(__hip_bfloat16)
  } else {
    PKV_NORM_ROPE_T(float)
  }
#undef PKV_NORM_ROPE_T
#undef PKV_NORM_ROPE_Q
#undef PKV_NORM_ROPE
  return (int)hipGetLastError();
}
