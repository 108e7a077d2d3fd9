// The 8-bit cache format and its row arithmetic.
//
// A row x[0 .. D) of one token and KV head is kept as e4m3 codes (OCP: 4 exponent bits, bias 7, 3
// mantissa bits, largest value 448, 0x7F / 0xFF NaN) and one E8M0 scale byte e, the power of two
// 2^(e - 127): the smallest one >= 2^-126 with max|x| <= 448 * 2^(e - 127).  A power of two, and not
// max|x| / 448, because e4m3 rounds relative to the value, so a scale up to twice as large costs no
// precision (only values under max|x| / 2^13 come out coarser), and then x / scale is exact: the only
// rounding is the one to e4m3, a row read back and written again keeps its values, and every stored
// value is exact in bfloat16.  It also takes one byte a row where fp32 takes four.  Elements that are
// not finite are stored as NaN; the scale is that of the others.
//
// Scales lie beside the cache: scale of (page, slot, head) of K at
//   k_scales[page * scale_page_stride + head * page_size + slot]
// (V alike), one head's slots together, since attention takes one head's tokens at a time.
#pragma once
#include "common.h"

#include <type_traits>

namespace pkv {
namespace fp8 {

// Magnitudes as bits (the order of positive floats is that of their bits; what is not finite comes after all others).
constexpr uint32_t kInfBits = 0x7F800000u;
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
// Largest magnitude of 16 values; `finite`: of the finite ones among them.
__device__ __forceinline__ uint32_t amax_bits(const float (&x)[8], const float (&y)[8], bool finite = false) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t u = abs_bits(x[j]), v = abs_bits(y[j]);
    if (finite) u = u < kInfBits ? u : 0u, v = v < kInfBits ? v : 0u;
    m = max(m, max(u, v));
  }
  return m;
}
// The scale byte of a row: max|x| = a * 2^E with 1 <= a < 2 needs E - 8, or E - 7 if a > 1.75
// (448 = 1.75 * 2^8): adding 0x1FFFFF carries into the exponent exactly for mantissas over 0x600000.
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int e = (int)((amax + 0x1FFFFFu) >> 23) - 8;
  return e < 1 ? 1 : e;
}
// 1 / scale for a byte that scale_byte gave (1 .. 247): exact.
__device__ __forceinline__ float inv_scale(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }
// Any scale byte's value (0: 2^-127, 255: NaN).
__device__ __forceinline__ float scale_f32(uint32_t e) {
  const uint32_t b = e == 0 ? 0x00400000u : (e == 255 ? 0x7FC00000u : e << 23);
  return __uint_as_float(b);
}
// Four values, |x| <= 448 or not finite, as e4m3 (to nearest, ties to even; not finite: NaN).
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return (uint32_t)r;
}

// 8 consecutive elements of type T: 16-byte accesses when VEC (address a multiple of 16), else one by one.
template <typename T, bool VEC>
struct Eight {
  static constexpr int N = sizeof(T) * 2;  // words
  uint32_t w[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = p[j];
      __builtin_memcpy(w, e, sizeof(e));
    }
  }
  // nt: past the caches
  __device__ __forceinline__ void store(T* p, bool nt = false) const {
    if constexpr (VEC) {
      typedef uint32_t v4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int i = 0; i < N; i += 4)
        if (nt) __builtin_nontemporal_store((v4{w[i], w[i + 1], w[i + 2], w[i + 3]}), reinterpret_cast<v4*>(p) + i / 4);
        else *(reinterpret_cast<v4*>(p) + i / 4) = v4{w[i], w[i + 1], w[i + 2], w[i + 3]};
    } else {
      T e[8];
      __builtin_memcpy(e, w, sizeof(e));
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = e[j];
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (std::is_same<T, __hip_bfloat16>::value) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      T e[8];
      __builtin_memcpy(e, w, sizeof(e));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = to_f32(e[j]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {  // to nearest, ties to even; a conversion takes two
    typedef float f2 __attribute__((ext_vector_type(2)));
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(x[j]);
    } else {
      using E = typename std::conditional<std::is_same<T, __hip_bfloat16>::value, __bf16, _Float16>::type;
      typedef E e2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const e2 p = __builtin_convertvector((f2{x[2 * j], x[2 * j + 1]}), e2);
        __builtin_memcpy(&w[j], &p, 4);
      }
    }
  }
};

// Eight codes: x[0 .. 8) times inv, stored past the caches (nothing reads a large batch's rows back soon, and a
// store that allocates no line leaves the reads their room: 65,536 tokens of 2 heads of 128, 22.0 us for 26.1).
template <bool VEC>
__device__ __forceinline__ void store8(uint8_t* p, const float (&x)[8], float inv) {
  const uint32_t a = pack4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  const uint32_t b = pack4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
  if constexpr (VEC) {
    __builtin_nontemporal_store((uint64_t)b << 32 | a, reinterpret_cast<uint64_t*>(p));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = (uint8_t)(a >> (8 * j)), p[4 + j] = (uint8_t)(b >> (8 * j));
  }
}

// Reduction over groups of n lanes (n = 1, 2, 4, .. 32; wave-uniform), in registers: every lane of a
// group gets the result.  All 64 lanes must be active.
template <typename Op>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, int n, Op op) {
  if (n > 1) v = op(v, wred::dpp<0xB1>(v));   // quad_perm 1 0 3 2
  if (n > 2) v = op(v, wred::dpp<0x4E>(v));   // quad_perm 2 3 0 1
  if (n > 4) v = op(v, wred::dpp<0x141>(v));  // row_half_mirror (each quad holds one value)
  if (n > 8) v = op(v, wred::dpp<0x140>(v));  // row_mirror
  if (n > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op((uint32_t)r[0], (uint32_t)r[1]);
  }
  return v;
}
__device__ __forceinline__ uint32_t group_max(uint32_t v, int n) {
  return group_reduce(v, n, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ float group_sum(float v, int n) {
  return __uint_as_float(group_reduce(__float_as_uint(v), n, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// The largest finite magnitude of a row whose group of n lanes holds 16 values each (act: this lane does).
__device__ __forceinline__ uint32_t row_amax(const float (&x)[8], const float (&y)[8], bool act, int n) {
  uint32_t m = group_max(act ? amax_bits(x, y) : 0u, n);
  if (__ballot(m >= kInfBits)) m = group_max(act ? amax_bits(x, y, true) : 0u, n);
  return m;
}

// Lanes a row of d elements takes, 16 elements each (8 of either half), rounded up to a power of two:
// the row kernels take head_dim % 16 == 0 up to 512.
inline int lanes_of(int d) {
  int n = 1;
  while (n < d / 16) n *= 2;
  return n;
}
// Offsets within a page are 32-bit.
inline bool page_fits(int ps, int hkv, int d) { return (int64_t)2 * ps * hkv * d * 4 <= INT32_MAX; }
inline bool head_dim_ok(int d) { return d > 0 && d <= 512 && d % 16 == 0; }

// Division by a number that the launch fixes, for 0 <= n < 2^31: with 2^(l-1) < d <= 2^l and m = ceil(2^(31+l) / d),
// n / d = floor(n m / 2^(31+l)) (m is at most 2^32 - 1 but for d = 1, which keeps 2^31).
struct Div {
  uint32_t m, l, d;
  __host__ __device__ Div(uint32_t m_, uint32_t l_, uint32_t d_) : m(m_), l(l_), d(d_) {}
  explicit Div(uint32_t d_) : l(0), d(d_) {
    while ((1ull << l) < d) ++l;
    m = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return __umulhi(n << 1, m) >> l; }
};
// Strides in bytes below 2^32 (what the launch checks), so that an address is one 32 x 32 + 64 bit product each.
struct Strides {
  uint32_t n, h;
};
inline bool strides_of(int64_t sn, int64_t sh, int es, Strides* s) {
  if (sn < 0 || sh < 0 || sn * es > UINT32_MAX || sh * es > UINT32_MAX) return false;
  *s = Strides{(uint32_t)(sn * es), (uint32_t)(sh * es)};
  return true;
}
__device__ __forceinline__ const char* row_at(const void* p, Strides s, uint32_t tok, uint32_t h) {
  return (const char*)p + (uint64_t)tok * s.n + (uint64_t)h * s.h;
}

// Where a token goes.  `slots` null: page kv_indices[kv_indptr[b] + pos / ps], slot pos % ps; else
// slots[i] = page * ps + slot.  False for metadata outside the sequence's pages, the list or the pool.
struct Table {
  const int32_t *bidx, *pos, *slots, *indices, *indptr;
  int64_t num_indices, num_pages;
  int32_t batch;
  Div ps;
};
__device__ __forceinline__ bool resolve(const Table& t, uint32_t i, int& page, int& slot) {
  if (t.slots) {
    const int sl = t.slots[i];
    if (sl < 0) return false;
    page = t.ps.of(sl);
    slot = sl - page * (int)t.ps.d;
    return page < t.num_pages;
  }
  const int b = t.bidx[i], p = t.pos[i];
  if (b < 0 || b >= t.batch || p < 0) return false;
  const int base = t.indptr[b], np = t.indptr[b + 1] - base, pi = t.ps.of(p);
  if (base < 0 || pi >= np || (int64_t)base + pi >= t.num_indices) return false;
  page = t.indices[base + pi];
  slot = p - pi * (int)t.ps.d;
  return page >= 0 && page < t.num_pages;
}

// K or V of the destination cache, and (8 bits) its scales.
struct Dest {
  void *k, *v;
  uint8_t *ks, *vs;
  int64_t page_stride, scale_stride;
};

}  // namespace fp8
}  // namespace pkv
