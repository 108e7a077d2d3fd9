// The 8-bit cache written and read back (format: cache_fp8.h).
//
//   pkv_append_paged_kv_cache_fp8  the append scatter (pkv_append_paged_kv_cache, ecahlang/manager.py:155-165,
//                                  175-185, 271-280) into an 8-bit cache: each row gets its scale and is rounded
//                                  to e4m3 on its way
//   pkv_read_paged_kv_cache_fp8    listed pages as 16-bit (or fp32) pages, for kernels that read those
#include "cache_fp8.h"
#include "../../include/pagedkv.h"

using namespace pkv;
using namespace pkv::fp8;

namespace {

// Workgroups of the append at most (65,536 tokens, 2 heads of 128: 22.7 us with 1024, 23.3 with 2048, 22.1 with 4096,
// 24.4 with 8192).
constexpr int kGrid = 4096;

struct AppendArgs {
  const void *k, *v;
  Strides ks, vs;
  Table t;
  Dest o;
  Div rows, hkv;
  int32_t nnz, d, lanes;
  int32_t* err;
};

// A group of `lanes` lanes takes one row (token, K or V, head; heads fastest, then K / V, then tokens):
// 8 elements of either half a lane.  The rows are requested before the page-table lookups.  65,536 fp16 tokens of
// 2 heads of 128 dims: 22 us for 101 MB, 19.5 at the rate of a large copy.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void append_fp8_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, sub = lane & (a.lanes - 1), per = 64 / a.lanes, half = a.d / 2;
  const bool act = 8 * sub < half;
  const int d0 = act ? 8 * sub : 0;
  const uint32_t hkv = a.hkv.d, total = (uint32_t)a.nnz * a.rows.d;
  const uint32_t wave = (blockIdx.x * (blockDim.x >> 6)) + (threadIdx.x >> 6), nw = gridDim.x * (blockDim.x >> 6);
  for (uint32_t base = wave * per; base < total; base += nw * per) {
    const uint32_t at = base + lane / a.lanes, idx = at < total ? at : total - 1;
    const uint32_t tok = a.rows.of(idx), r = idx - tok * a.rows.d;
    const bool isv = r >= hkv;
    const uint32_t h = isv ? r - hkv : r;
    const T* src = (const T*)(isv ? row_at(a.v, a.vs, tok, h) : row_at(a.k, a.ks, tok, h)) + d0;
    Eight<T, VEC> lo, hi;
    lo.load(src);
    hi.load(src + half);
    asm volatile("" ::: "memory");
    int page = 0, slot = 0;
    const bool ok = resolve(a.t, tok, page, slot) && at < total;
    float x[8], y[8];
    lo.get(x);
    hi.get(y);
    const int e = scale_byte(row_amax(x, y, act, a.lanes));
    const float inv = inv_scale(e);
    if (ok && act) {
      uint8_t* dst = (uint8_t*)(isv ? a.o.v : a.o.k) + page * a.o.page_stride + (uint32_t)((slot * hkv + h) * a.d + d0);
      store8<VEC>(dst, x, inv);
      store8<VEC>(dst + half, y, inv);
      if (sub == 0) (isv ? a.o.vs : a.o.ks)[page * a.o.scale_stride + (h * a.t.ps.d + slot)] = (uint8_t)e;
    }
    if (!ok && at < total && sub == 0 && a.err) atomicAdd(a.err, 1);
  }
}

struct ReadArgs {
  const uint8_t *k, *v, *ks, *vs;
  int64_t page_stride, scale_stride, num_pages;
  const int32_t *indices, *indptr;
  int64_t num_indices;
  Div rc, hkv;  // chunks of 8 a row, KV heads
  int32_t batch, d, ps;
  void* out;  // [pages][2][ps][hkv][d]
};

// Listed page i -> out page i, a workgroup a page: 8 codes a lane, so that both the loads and the stores
// of a wave are whole lines (8 sequences of 512 to 8704 tokens, 8 heads of 128 dims to bf16: 58 us for 316 MB over and
// over, 67 where each pass finds other pages; 61 at the rate of a large copy).  The stores go through the caches, since
// the attention reads the pages next: past them, the pass takes 64 us, and with the attention of 512 tokens over 60,000
// 542 for 529.
template <typename T>
__global__ __launch_bounds__(256) void read_fp8_kernel(ReadArgs a) {
  const int64_t listed = a.indptr[a.batch];
  const int64_t n = listed < a.num_indices ? listed : a.num_indices;
  const uint32_t rows = (uint32_t)a.ps * a.hkv.d, chunks = rows * a.rc.d;
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int page = a.indices[i];
    const bool ok = page >= 0 && page < a.num_pages;
    T* out = (T*)a.out + i * 2 * (int64_t)rows * a.d;
    for (uint32_t c = threadIdx.x; c < 2 * chunks; c += blockDim.x) {
      const bool isv = c >= chunks;
      const uint32_t w = isv ? c - chunks : c, row = a.rc.of(w), t = a.hkv.of(row), h = row - t * a.hkv.d;
      Eight<T, true> r;
      if (ok) {
        const uint2 x = *reinterpret_cast<const uint2*>((isv ? a.v : a.k) + page * a.page_stride + (int64_t)w * 8);
        const float s = scale_f32((isv ? a.vs : a.ks)[page * a.scale_stride + (h * a.ps + t)]);
        const auto p0 = __builtin_amdgcn_cvt_pk_f32_fp8(x.x, false), p1 = __builtin_amdgcn_cvt_pk_f32_fp8(x.x, true);
        const auto p2 = __builtin_amdgcn_cvt_pk_f32_fp8(x.y, false), p3 = __builtin_amdgcn_cvt_pk_f32_fp8(x.y, true);
        const float f[8] = {p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
        const float v[8] = {f[0] * s, f[1] * s, f[2] * s, f[3] * s, f[4] * s, f[5] * s, f[6] * s, f[7] * s};
        r.set(v);
      } else {
#pragma unroll
        for (int j = 0; j < r.N; ++j) r.w[j] = 0u;
      }
      r.store(out + (int64_t)c * 8);
    }
  }
}

}  // namespace

extern "C" int pkv_append_paged_kv_cache_fp8(
    const void* append_key, int64_t k_stride_n, int64_t k_stride_h, const void* append_value, int64_t v_stride_n,
    int64_t v_stride_h, const int32_t* batch_indices, const int32_t* positions, const int32_t* slots, int32_t nnz,
    void* k_cache, void* v_cache, int64_t page_stride, int64_t num_pages, void* k_scales, void* v_scales,
    int64_t scale_page_stride, const int32_t* kv_indices, int64_t num_indices, const int32_t* kv_indptr, int32_t batch,
    int32_t num_kv_heads, int32_t head_dim, int32_t page_size, int32_t dtype, int32_t* err_count, void* stream) {
  const int es = dtype == kF32 ? 4 : (dtype == kF16 || dtype == kBF16) ? 2 : 0;
  if (!es) return kBadDType;
  if (nnz < 0 || num_kv_heads <= 0 || page_size <= 0 || batch < 0 || num_indices < 0) return kBadArg;
  if (!head_dim_ok(head_dim)) return kBadHeadDim;
  if (nnz == 0) return kOk;
  if (!append_key || !append_value || !k_scales || !v_scales || (num_pages > 0 && (!k_cache || !v_cache)) || (!slots && (!batch_indices || !positions || !kv_indptr))) return kBadArg;
  const int lanes = lanes_of(head_dim);
  const int64_t total = (int64_t)nnz * 2 * num_kv_heads;
  if (total > INT32_MAX) return kBadArg;
  Strides ks, vs;
  if (!strides_of(k_stride_n, k_stride_h, es, &ks) || !strides_of(v_stride_n, v_stride_h, es, &vs)) return kBadArg;
  if (!page_fits(page_size, num_kv_heads, head_dim)) return kBadArg;
  const AppendArgs a{append_key, append_value, ks, vs,
                     {batch_indices, positions, slots, kv_indices, kv_indptr, num_indices, num_pages, batch, Div(page_size)},
                     {k_cache, v_cache, (uint8_t*)k_scales, (uint8_t*)v_scales, page_stride, scale_page_stride},
                     Div(2 * num_kv_heads), Div(num_kv_heads), nnz, head_dim, lanes, err_count};
  const uintptr_t in = (uintptr_t)append_key | (uintptr_t)append_value, to = (uintptr_t)k_cache | (uintptr_t)v_cache;
  if (in % es) return kBadAlign;
  const bool vec = in % 16 == 0 && (k_stride_n | k_stride_h | v_stride_n | v_stride_h) * es % 16 == 0 && to % 8 == 0 &&
                   page_stride % 8 == 0;
  const int per = 4 * (64 / lanes);  // rows a workgroup takes at a time
  const int64_t want = (total + per - 1) / per;
  const dim3 grid((unsigned)(want < kGrid ? want : kGrid));
  hipStream_t s = (hipStream_t)stream;
#define PKV_APPEND_FP8(T)                                                                        \
  if (vec) hipLaunchKernelGGL((append_fp8_kernel<T, true>), grid, dim3(256), 0, s, a);           \
  else hipLaunchKernelGGL((append_fp8_kernel<T, false>), grid, dim3(256), 0, s, a)
  if (dtype == kF16) {
    PKV_APPEND_FP8(_Float16);
  } else if (dtype == kBF16) {
    PKV_APPEND_FP8(__hip_bfloat16);
  } else {
    PKV_APPEND_FP8(float);
  }
#undef PKV_APPEND_FP8
  return (int)hipGetLastError();
}

extern "C" int pkv_read_paged_kv_cache_fp8(const void* k_cache, const void* v_cache, int64_t page_stride,
                                           int64_t num_pages, const void* k_scales, const void* v_scales,
                                           int64_t scale_page_stride, const int32_t* kv_indices, int64_t num_indices,
                                           const int32_t* kv_indptr, int32_t batch, int32_t num_kv_heads,
                                           int32_t head_dim, int32_t page_size, void* out, int32_t dtype,
                                           void* stream) {
  if (dtype != kF16 && dtype != kBF16 && dtype != kF32) return kBadDType;
  if (num_kv_heads <= 0 || page_size <= 0 || batch < 0 || num_indices < 0 || num_pages < 0) return kBadArg;
  if (!head_dim_ok(head_dim)) return kBadHeadDim;
  if (num_indices == 0 || batch == 0) return kOk;
  if (!kv_indptr || !kv_indices || !out || (num_pages > 0 && (!k_cache || !v_cache || !k_scales || !v_scales))) return kBadArg;
  if (!page_fits(page_size, num_kv_heads, head_dim)) return kBadArg;
  if ((((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)page_stride) % 8) || (uintptr_t)out % 16) return kBadAlign;
  const ReadArgs a{(const uint8_t*)k_cache, (const uint8_t*)v_cache, (const uint8_t*)k_scales, (const uint8_t*)v_scales,
                   page_stride, scale_page_stride, num_pages, kv_indices, kv_indptr, num_indices, Div(head_dim / 8),
                   Div(num_kv_heads), batch, head_dim, page_size, out};
  const dim3 grid((unsigned)(num_indices < 65536 ? num_indices : 65536));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == kF16) hipLaunchKernelGGL(read_fp8_kernel<_Float16>, grid, dim3(256), 0, s, a);
  else if (dtype == kBF16) hipLaunchKernelGGL(read_fp8_kernel<__hip_bfloat16>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(read_fp8_kernel<float>, grid, dim3(256), 0, s, a);
  return (int)hipGetLastError();
}
