// RMS norm of every query and key head, rotary embedding and K/V append in one launch:
//
//   pkv_append_paged_kv_cache_norm_rope  <- q_norm / k_norm and apply_rotary_pos_emb of models that normalise
//                                           their heads, then the hook's append (ecahlang/main.py:62-66)
//
// Per row x[0 .. D) of a query or key head with weight w, and the token's cos and sin:
//   y[d] = x[d] / sqrt(mean(x^2) + eps) * w[d]
//   out[d]       = y[d] cos[d]             - y[d + D/2] sin[d]            d < D/2
//   out[d + D/2] = y[d + D/2] cos[d + D/2] + y[d] sin[d + D/2]
// all in fp32 and rounded once, to the type of q_out or the cache, or (exactly: see kErr) to e4m3 with the row's
// scale (cache_fp8.h).  Without a weight the rows are not normalised.  Value rows are copied, or rounded to e4m3.
//
// A group of D / 16 lanes (rounded up to a power of two) takes a row, each lane 8 elements of either half, so
// the rotation's partners meet in one lane and the sum of squares takes a few lane exchanges.  The rows of all
// tokens are dealt out in one run, 8 of 128 dims to a wave, whatever the heads of a token are: a wave that kept
// to one token, its angles in registers, idled lanes wherever the heads do not divide by 8 and waited for each
// token's page by itself (4003 tokens, 32 / 8 heads of 128: 20 us for 30, a step of 4 tokens 3.0 for 4.8).  All
// keys come first, then all values, then all queries, so that a wave has one kind to do (token by token, waves of
// several kinds do the work of each: 16,003 tokens into 8 bits, 14 / 2 heads of 64, 17.8 us for 23.3, 16 / 2 of 128, 40.7
// for 43.6; where 8 divides the heads it gains nothing, and the angles are read twice: 32 / 8 of 128 into bf16 80.4 for 78.6).
//
// What bounds it: the bytes, beside some 250 vector instructions a wave's 8 rows, about half the time at full
// rate: 16,003 tokens, 32 / 8 heads of 128, bf16 into 8 bits, 84.5 us for 369 MB (71 at the rate of a large
// copy), 2 us of them to look for undecided keys and 3 for the chain of latencies of those found; into bf16 80 us (77).
#include "cache_fp8.h"
#include "../../include/pagedkv.h"

#include <type_traits>

using namespace pkv;
using namespace pkv::fp8;

namespace {

// Workgroups at most: more of them than the chip holds at once (1280), so that their phases mix (the bulk above, before
// keys were looked at once more: 88 us with 1024 or 2048, 83 with 4096, 79 with 8192, 81 with 16,384; a workgroup costs
// some 3.5 ns to start).
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
  Div hqd, hkvd;
  int32_t nnz, hq, hkv, d, lanes;
  int32_t* err;
};

// Quantised keys are those of the exact y: an fp32 y decides a code unless it lies within its error of a tie of e4m3.
// With u = 2^-24: the sum of squares is off by at most 10 u (a chain of 4, 2 sums, up to 5 exchanges, less 1: the first
// product is the fused one's), the mean with eps by 2, so the root by 6, its reciprocal's step by 2; factor and weight
// 2; the rotation's product and sum 2: 12 u of |x| + |y|, a little more for cos and sin that a model scales.  The few
// rows that hold an undecided key (1 in some 50) are computed in 64 bits; doing so for all keys takes 143 us for 84 in
// the bulk above, and |x c| + |y s| for each key, which flags a third fewer, 91 (its registers leave 4 waves of 5).
constexpr float kErr = 14.f / (1 << 24);
constexpr uint32_t kUlps = 64;  // of the largest magnitude, that picks the scale: it is at least half of its |x| + |y|

__device__ __forceinline__ bool certain(const float (&x)[8], const float (&y)[8], const float (&mag)[8], float inv) {
  uint32_t differ = 0;
  const float f = inv * kErr;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float x0 = x[j] * inv, y0 = y[j] * inv, x1 = x[j + 1] * inv, y1 = y[j + 1] * inv, d0 = mag[j] * f, d1 = mag[j + 1] * f;
    differ |= pack4(x0 - d0, y0 - d0, x1 - d1, y1 - d1) ^ pack4(x0 + d0, y0 + d0, x1 + d1, y1 + d1);
  }
  return differ == 0;
}
// v as fp32, rounded to odd where it lies between two: rounding that to fewer bits is rounding v.
__device__ __forceinline__ float to_odd(double v) {
  const float f = (float)v;
  uint32_t b = __float_as_uint(f);
  if ((double)f != v && v == v) b = (b - (fabs((double)f) > fabs(v) ? 1u : 0u)) | 1u;
  return __uint_as_float(b);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  auto step = [&](auto fetch) __attribute__((always_inline)) {
    uint64_t b;
    __builtin_memcpy(&b, &v, 8);
    const uint64_t o = (uint64_t)fetch((uint32_t)(b >> 32)) << 32 | fetch((uint32_t)b);
    double x;
    __builtin_memcpy(&x, &o, 8);
    v += x;
  };
  step([](uint32_t x) { return wred::dpp<wred::kRor8>(x); });
  step([](uint32_t x) { return wred::dpp<wred::kRor4>(x); });
  step([](uint32_t x) { return wred::dpp<wred::kRor2>(x); });
  step([](uint32_t x) { return wred::dpp<wred::kRor1>(x); });
  const bool up16 = threadIdx.x & 16, up32 = threadIdx.x & 32;
  step([&](uint32_t x) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (uint32_t)(up16 ? r[0] : r[1]);
  });
  step([&](uint32_t x) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (uint32_t)(up32 ? r[0] : r[1]);
  });
  return v;
}
// A key row in 64 bits, by a whole wave: a lane has 1 to 4 of the pairs that the rotation mixes.
template <typename T, typename WT, typename CT>
__device__ __forceinline__ void exact_key(int tok, int h, int page, int slot) {
  // (the arguments read again: kept for this rare path they would take scalar registers of the usual one)
  typedef __attribute__((address_space(4))) const NormRopeArgs KernelArgs;
  KernelArgs* pa = (KernelArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(pa));
  const NormRopeArgs& a = *(const NormRopeArgs*)pa;
  const int lane = threadIdx.x & 63, half = a.d / 2;
  const T* src = (const T*)row_at(a.k, a.ks, tok, h);
  const CT *cos = (const CT*)row_at(a.cos, a.cs, tok, 0), *sin = (const CT*)row_at(a.sin, a.cs, tok, 0);
  const WT* w = (const WT*)a.kw;
  double ss = 0.0, rs = 1.0;
  float x[4], y[4];
  const int j0 = min(lane, half - 1);  // (the first pair's at once)
  const float wx = w ? to_f32(w[j0]) : 1.f, wy = w ? to_f32(w[half + j0]) : 1.f;
  const float c0 = to_f32(cos[j0]), c1 = to_f32(cos[half + j0]), s0 = to_f32(sin[j0]), s1 = to_f32(sin[half + j0]);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int j = min(64 * p + lane, half - 1);
    if (64 * p >= half) break;
    x[p] = to_f32(src[j]), y[p] = to_f32(src[half + j]);
  }
  if (w) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if (64 * p >= half) break;
      if (64 * p + lane < half) ss = __builtin_fma((double)x[p], (double)x[p], __builtin_fma((double)y[p], (double)y[p], ss));
    }
    const double ms = wave_sum_f64(ss) / a.d + (double)a.eps, r0 = __builtin_amdgcn_rsq(ms);  // (2^-26, and a Newton step)
    const double off = __builtin_fma(-ms * r0, r0, 1.0);
    rs = off == off ? __builtin_fma(0.5 * r0, off, r0) : r0;
  }
  uint32_t m = 0;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    if (64 * p >= half) break;
    const int j = min(64 * p + lane, half - 1);
    const double u = x[p] * rs * (p == 0 ? wx : w ? to_f32(w[j]) : 1.f), v = y[p] * rs * (p == 0 ? wy : w ? to_f32(w[half + j]) : 1.f);
    x[p] = to_odd(__builtin_fma(u, (double)(p == 0 ? c0 : to_f32(cos[j])), -v * (p == 0 ? s0 : to_f32(sin[j]))));
    y[p] = to_odd(__builtin_fma(v, (double)(p == 0 ? c1 : to_f32(cos[half + j])), u * (p == 0 ? s1 : to_f32(sin[half + j]))));
    const uint32_t bx = abs_bits(x[p]), by = abs_bits(y[p]);
    m = max(m, max(bx < kInfBits ? bx : 0u, by < kInfBits ? by : 0u));
  }
  const int e = scale_byte(wave_max_u32(m));
  const float inv = inv_scale(e);
  uint8_t* dst = (uint8_t*)a.o.k + page * a.o.page_stride + (uint32_t)((slot * a.hkv + h) * a.d);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    if (64 * p >= half) break;
    const int j = 64 * p + lane;
    const uint32_t c = pack4(x[p] * inv, y[p] * inv, 0.f, 0.f);
    if (j < half) dst[j] = (uint8_t)c, dst[half + j] = (uint8_t)(c >> 8);
  }
  if (lane == 0) a.o.ks[page * a.o.scale_stride + (h * a.t.ps.d + slot)] = (uint8_t)e;
}

// Rows of all tokens in one run (keys, values, queries; heads fastest): a group of lanes takes one row at a
// time, wherever tokens end.  Everything a row needs is requested at once; only key and value rows look up
// their page.
template <typename T, typename WT, typename CT, bool QUANT, bool VEC>
__global__ __launch_bounds__(256, 4) void norm_rope_kernel(NormRopeArgs a) {
  const int lane = threadIdx.x & 63, sub = lane & (a.lanes - 1), per = 64 / a.lanes, half = a.d / 2;
  const bool act = 8 * sub < half;
  const int d0 = act ? 8 * sub : 0;
  const uint32_t keys = (uint32_t)a.nnz * a.hkv, total = 2 * keys + (uint32_t)a.nnz * a.hq;
  const uint32_t stride = gridDim.x * (blockDim.x >> 6) * per;
  const float inv_d = 1.f / (float)a.d;
  uint32_t base = __builtin_amdgcn_readfirstlane((blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6)) * per);
  for (; base < total; base += stride) {
    const uint32_t at = base + lane / a.lanes, idx = at < total ? at : total - 1;
    const bool isq = idx >= 2 * keys, isv = !isq && idx >= keys, in = at < total && act;
    const uint32_t row = isq ? idx - 2 * keys : isv ? idx - keys : idx;
    const Div heads{isq ? a.hqd.m : a.hkvd.m, isq ? a.hqd.l : a.hkvd.l, isq ? a.hqd.d : a.hkvd.d};
    const uint32_t tok = heads.of(row);
    const int h = row - tok * heads.d;
    const Strides st{isq ? a.qs.n : isv ? a.vs.n : a.ks.n, isq ? a.qs.h : isv ? a.vs.h : a.ks.h};
    const T* src = (const T*)row_at(isq ? a.q : isv ? a.v : a.k, st, tok, h) + d0;
    Eight<T, VEC> lo, hi;
    lo.load(src);
    hi.load(src + half);
    const CT *cosr = (const CT*)row_at(a.cos, a.cs, tok, 0) + d0, *sinr = (const CT*)row_at(a.sin, a.cs, tok, 0) + d0;
    Eight<CT, VEC> c0, c1, s0, s1;
    if (__ballot(!isv)) {
      c0.load(cosr);
      c1.load(cosr + half);
      s0.load(sinr);
      s1.load(sinr + half);
    }
    asm volatile("" ::: "memory");
    int page = 0, slot = 0;
    bool ok = false;
    if (!isq) {
      ok = resolve(a.t, tok, page, slot);
      if (!ok && at < total && !isv && h == 0 && sub == 0 && a.err) atomicAdd(a.err, 1);
    }
    float x[8], y[8];
    lo.get(x);
    hi.get(y);
    const WT* w = (const WT*)(isq ? a.qw : a.kw) + d0;
    const bool normed = isq ? a.qw : a.kw;
    float mag[8];  // |x| + |y| of a pair that the rotation mixes
    if (__ballot(!isv)) {
      float sq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 8; ++j) sq[j & 3] = __builtin_fmaf(x[j], x[j], __builtin_fmaf(y[j], y[j], sq[j & 3]));
      float ss = (sq[0] + sq[1]) + (sq[2] + sq[3]);
      ss = group_sum(act ? ss : 0.f, a.lanes);
      if (!isv) {
        if (normed) {
          const float ms = __builtin_fmaf(ss, inv_d, a.eps), r0 = __builtin_amdgcn_rsqf(ms);
          const float off = __builtin_fmaf(-ms * r0, r0, 1.f), rs = off == off ? __builtin_fmaf(0.5f * r0, off, r0) : r0;
          Eight<WT, VEC> w0, w1;
          w0.load(w);
          w1.load(w + half);
          float u[8];
          w0.get(u);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= rs * u[j];
          w1.get(u);
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] *= rs * u[j];
        }
        if (QUANT) {
#pragma unroll
          for (int j = 0; j < 8; ++j) mag[j] = __builtin_fabsf(x[j]) + __builtin_fabsf(y[j]);
        }
        float c[8], s[8], z[8];
        c0.get(c);
        s0.get(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = x[j] * c[j] - y[j] * s[j];
        c1.get(c);
        s1.get(s);
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
      const uint32_t m = row_amax(x, y, act, a.lanes);
      const int e = scale_byte(m);
      const float inv = inv_scale(e);
      const bool key = in && ok && !isv;
      uint64_t todo = 0;
      if (__ballot(key)) {
        const bool sure = !key || (scale_byte(m - min(m, kUlps)) == scale_byte(m + kUlps) && certain(x, y, mag, inv));
        todo = __ballot(!sure);
      }
      const uint64_t group = (1ull << a.lanes) - 1;
      if (in && ok && !(todo >> (lane & ~(a.lanes - 1)) & group)) {
        uint8_t* dst = (uint8_t*)(isv ? a.o.v : a.o.k) + page * a.o.page_stride + (uint32_t)((slot * a.hkv + h) * a.d + d0);
        store8<VEC>(dst, x, inv);
        store8<VEC>(dst + half, y, inv);
        if (sub == 0) (isv ? a.o.vs : a.o.ks)[page * a.o.scale_stride + (h * a.t.ps.d + slot)] = (uint8_t)e;
      }
      while (todo) {
        const int l = __builtin_ctzll(todo) & ~(a.lanes - 1);
        todo &= ~(group << l);
        exact_key<T, WT, CT>(__builtin_amdgcn_readlane(tok, l), __builtin_amdgcn_readlane(h, l),
                             __builtin_amdgcn_readlane(page, l), __builtin_amdgcn_readlane(slot, l));
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
                       Div(num_qo_heads ? num_qo_heads : 1), Div(num_kv_heads), nnz, num_qo_heads, num_kv_heads, head_dim, lanes, err_count};
  const uintptr_t m = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)append_key | (uintptr_t)append_value;
  const uintptr_t an = (uintptr_t)cos | (uintptr_t)sin, ws = (uintptr_t)q_weight | (uintptr_t)k_weight;
  const uintptr_t to = (uintptr_t)k_cache | (uintptr_t)v_cache;
  if ((m % es) || an % (cs_dtype == kF32 ? 4 : es) || ws % (weight_dtype == kF32 ? 4 : es) || (!quant && to % es)) return kBadAlign;
  const int64_t st = q_stride_n | q_stride_h | qo_stride_n | qo_stride_h | k_stride_n | k_stride_h | v_stride_n | v_stride_h;
  const bool vec = (m | an | ws) % 16 == 0 && st * es % 16 == 0 && cs_stride_n * (cs_dtype == kF32 ? 4 : es) % 16 == 0 &&
                   (quant ? to % 8 == 0 && page_stride % 8 == 0 : to % 16 == 0 && page_stride * es % 16 == 0);
  const int64_t want = (total + 4 * per - 1) / (4 * per);
  const dim3 grid((unsigned)(want < kGrid ? want : kGrid));
  const bool wf = weight_dtype == kF32, cf = cs_dtype == kF32;
  hipStream_t s = (hipStream_t)stream;
#define PKV_NORM_ROPE(T, W, C)                                                                                    \
  if (quant) {                                                                                                    \
    if (vec) hipLaunchKernelGGL((norm_rope_kernel<T, W, C, true, true>), grid, dim3(256), 0, s, a);               \
    else hipLaunchKernelGGL((norm_rope_kernel<T, W, C, true, false>), grid, dim3(256), 0, s, a);                  \
  } else {                                                                                                        \
    if (vec) hipLaunchKernelGGL((norm_rope_kernel<T, W, C, false, true>), grid, dim3(256), 0, s, a);              \
    else hipLaunchKernelGGL((norm_rope_kernel<T, W, C, false, false>), grid, dim3(256), 0, s, a);                 \
  }
#define PKV_NORM_ROPE_T(T)                                                                             \
  if (wf) { if (cf) { PKV_NORM_ROPE(T, float, float) } else { PKV_NORM_ROPE(T, float, T) } }           \
  else { if (cf) { PKV_NORM_ROPE(T, T, float) } else { PKV_NORM_ROPE(T, T, T) } }
  if (dtype == kF16) {
    PKV_NORM_ROPE_T(_Float16)
  } else if (dtype == kBF16) {
    PKV_NORM_ROPE_T(__hip_bfloat16)
  } else {
    PKV_NORM_ROPE(float, float, float)
  }
#undef PKV_NORM_ROPE_T
#undef PKV_NORM_ROPE
  return (int)hipGetLastError();
}
