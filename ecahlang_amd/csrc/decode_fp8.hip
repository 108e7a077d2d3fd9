// Paged decode over 8-bit caches (format: cache_fp8.h) on the matrix cores: fp16 / bf16 queries, head_dim
// 64, 128 or 256, any page size and any number of query heads a KV head.  Same contract as the other decode
// kernels (BatchDecodeWithPagedKVCacheWrapper.run, ecahlang/main.py:68).
//
//   o[h] = sum_t softmax_t(q[h] . k[t] ks[t] / sqrt D) v[t] vs[t]     k, v: the e4m3 values, ks, vs: the scales
//
// A token's scales are common to its row, so they stay out of the products: ks multiplies the score and vs
// the softmax weight.  The codes become operands of the query's type (K) and of bfloat16 (V) by v_cvt
// alone, exactly; the weights p vs, fp32, are split into a bfloat16 and the bfloat16 nearest to what is left,
// both in one product (its 32 reduction slots hold 16 tokens twice), so they lose 2^-17 and no reference
// exponent is needed for scales of any size.
//
// A workgroup (W = 4 waves) takes one KV head (16 of its query heads) of one part of one sequence; wave r takes
// the part's tiles of 16 tokens r, r + W, ...  With lane l = (lr = l % 16, lg = l / 16), a tile:
//   S[token][head]     = K . Q^T   A: K[token lr][dims 64 j + 16 lg + 0 .. 15], one 16-byte load for two steps
//   online softmax                 lane: head lr, tokens 4 lg + i
//   O^T[dim][head]    += V^T . P   A: V[token 4 lg + i][dims D/16 lr + 0 .. D/16), one load a token: its bytes
//                                  pair with the next token's by v_perm; B: the lane's own weights
// so K and V go from memory straight into registers (no LDS, no lane exchange), a wave's load covers whole rows,
// and each register set is refilled with the next tile's rows as soon as its products are issued.  The
// waves' states meet in LDS; a sequence of several parts is merged by the workgroup that arrives last.
#include <algorithm>
#include "attn_common.h"
#include "mfma_common.h"
#include "cache_fp8.h"
#include "../../include/pagedkv.h"

using namespace pkv;
using namespace pkv::mfma;

namespace {

constexpr int W = 4;               // waves per workgroup
constexpr int kMinTiles = 8;       // tiles per part of a cut sequence, about, at least
constexpr float kLazyMax = 8.f;    // a head's reference max moves only on jumps > 2^8
constexpr int kMergeParts = 8;     // parts whose rows the merge loads at a time

struct Fp8Cache {
  const uint8_t *ks, *vs;
  int64_t sstride;   // scale bytes between pages
  int32_t ncb;       // blocks of 16 query heads a KV head
};

template <typename T> struct Codes;
template <> struct Codes<_Float16> {
  static __device__ __forceinline__ uint32_t lo(uint32_t x) { return bitcast_<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false)); }
  static __device__ __forceinline__ uint32_t hi(uint32_t x) { return bitcast_<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true)); }
};
template <> struct Codes<__hip_bfloat16> {
  static __device__ __forceinline__ uint32_t lo(uint32_t x) { return bitcast_<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false)); }
  static __device__ __forceinline__ uint32_t hi(uint32_t x) { return bitcast_<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true)); }
};

__device__ __forceinline__ int parts_of(int tiles, int aim, int max_parts) {
  return max(min((tiles + aim - 1) / aim, max_parts), 1);
}

// N 4-byte words at p (aligned to them all, 16 bytes at most)
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    const u4v x = *reinterpret_cast<const u4v*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = x[i];
  }
}

// P16: page_size is a multiple of 16, so a tile lies in one page.
template <typename T, int D, bool P16>
__global__ __launch_bounds__(W * 64) void decode_fp8_kernel(DecodeParams P, Fp8Cache F, int nr, int max_parts) {
  constexpr int NK = D / 64;  // 16-byte pieces of a K row a lane holds
  constexpr int KS = D / 32;  // QK steps
  constexpr int VB = D / 16;  // bytes of a V row a lane holds
  constexpr int VW = VB / 4;
  constexpr int NT = D / 16;  // output tiles
  constexpr int NP = NT;      // 16-byte pieces of a lane's 4 NT output values
  __shared__ f4 s_o[W][NP][64];
  __shared__ float2 s_ml[W][16];
  __shared__ int s_last;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int B = P.batch, g = P.hq / P.hkv, H = P.hkv * F.ncb, ps = P.ps;
  const int hb = blockIdx.x % H, w = blockIdx.x / H;
  const int h = hb / F.ncb, c0 = (hb - h * F.ncb) * 16, gc = min(g - c0, 16);  // my query heads: h g + c0 + 0 .. gc

  // ---- workgroup w: the first part of sequence w, or (w >= B) the (w - B)-th of the further parts, which
  // follow each other in sequence order; those and cut sequences look for their place among the batch, 64
  // sequences a round.
  const int64_t cut = P.num_indices;
  // tokens of a sequence that the page list holds
  auto length_of = [&](int i0, int i1, int last) __attribute__((always_inline)) -> int {
    if (i0 < 0 || i1 <= i0) return 0;
    const int64_t np = i1 - i0, av = min((int64_t)i1, cut) - i0;
    const int64_t len = min((np - 1) * ps + min(max(last, 0), ps), max(av, (int64_t)0) * ps);
    return (int)min(len, (int64_t)(INT_MAX - 64));
  };
  int s0, len, b = min(w, B - 1), nparts, part = 0, more0 = 0;
  s0 = P.indptr[b];
  len = length_of(s0, P.indptr[b + 1], P.last[b]);
  const int64_t listed = max(min((int64_t)P.indptr[B], cut), (int64_t)0);
  const int total = (int)min((listed * ps + 15) / 16, (int64_t)(1 << 30));
  const int aim = max(kMinTiles, (total + nr - 1) / nr);
  nparts = parts_of((len + 15) / 16, aim, max_parts);
  if (w >= B || nparts > 1) {
    bool found = false;
    int base = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < B; b0 += 64) {
      const int bl = b0 + lane, i0 = P.indptr[min(bl, B)];
      const int ln = bl < B ? length_of(i0, P.indptr[min(bl + 1, B)], P.last[min(bl, B - 1)]) : 0;
      const int n = bl < B ? parts_of((ln + 15) / 16, aim, max_parts) - 1 : 0;
      int incl = n;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) {
        const int v = __shfl_up(incl, x, 64);
        incl += lane >= x ? v : 0;
      }
      const int all = __builtin_amdgcn_readlane(incl, 63);
      if (w < B ? w < b0 + 64 : w - B < base + all) {
        const int l = w < B ? w - b0 : __popcll(__ballot(base + incl <= w - B));
        more0 = base + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l);
        if (w >= B) {
          b = b0 + l;
          s0 = __builtin_amdgcn_readlane(i0, l);
          len = __builtin_amdgcn_readlane(ln, l);
          nparts = __builtin_amdgcn_readlane(n, l) + 1;
          part = 1 + w - B - more0;
        }
        found = true;
        break;
      }
      base += all;
    }
    if (!found) return;  // (the grid is sized for the most parts there can be)
    nparts = 1 + min(nparts - 1, max(nr - more0, 0));  // (a kv_indptr that runs backwards)
  }
  b = __builtin_amdgcn_readfirstlane(b);
  s0 = __builtin_amdgcn_readfirstlane(s0);
  len = __builtin_amdgcn_readfirstlane(len);
  // the part's tiles [p0, end)
  const int tiles = (len + 15) / 16, per = tiles / nparts, more = tiles - per * nparts;
  const int p0 = part * per + min(part, more), end = p0 + per + (part < more ? 1 : 0);
  const bool one = nparts == 1 && tiles <= 1;  // wave 0's alone
  if (one && wave > 0) return;

  const uint32_t rowb = P.hkv * D;  // bytes between token rows
  const uint8_t* kc = (const uint8_t*)P.k_cache + (int64_t)h * D;
  const uint8_t* vc = (const uint8_t*)P.v_cache + (int64_t)h * D;
  const uint8_t* ksc = F.ks + (int64_t)h * ps;
  const uint8_t* vsc = F.vs + (int64_t)h * ps;
  const int mt = P16 ? ps / 16 : 1;  // tiles a page
  // columns past the head block repeat its last head (never stored)
  const T* qc = (const T*)P.q + b * P.q_sn + (int64_t)(h * g + c0 + (lr < gc ? lr : gc - 1)) * P.q_sh;
  const uint8_t* dummy = (const uint8_t*)((const T*)P.q + b * P.q_sn + (int64_t)(h * g + c0) * P.q_sh);

  // The tile's rows, and the scales of tokens 4 lg + 0 .. 3 (a byte each).  Every load is unconditional, so
  // that all paths have the same ones in flight; where there is no page they read a query row instead.
  u4v kr[NK];
  uint32_t vr[4][VW], ke, ve;
  const uint32_t koff = lr * rowb + 16 * lg, voff = 4 * lg * rowb + VB * lr;
  // P16: a wave-uniform page id, -1 outside the pool or past the part
  auto page_of = [&](int tile) __attribute__((always_inline)) -> int {
    if (tile >= end) return -1;
    const int pid = P.indices[s0 + (mt == 1 ? tile : tile / mt)];
    return pid >= 0 && (int64_t)pid < P.num_pages ? pid : -1;
  };
  auto load_k = [&](int tile, int pid) __attribute__((always_inline)) {
    if constexpr (P16) {
      const bool ok = pid >= 0;
      const int sub = mt == 1 ? 0 : 16 * (tile % mt);
      const uint8_t* kp = ok ? kc + pid * P.page_stride + (int64_t)sub * rowb : dummy;
      const uint8_t* sp = ok ? ksc + pid * F.sstride + sub : dummy;
      const uint32_t o = ok ? koff : 0;
      ke = *reinterpret_cast<const uint32_t*>(sp + (ok ? 4 * lg : 0));
#pragma unroll
      for (int j = 0; j < NK; ++j) kr[j] = *reinterpret_cast<const u4v*>(kp + o + 64 * j);
    }
  };
  auto load_v = [&](int tile, int pid) __attribute__((always_inline)) {
    if constexpr (P16) {
      const bool ok = pid >= 0;
      const int sub = mt == 1 ? 0 : 16 * (tile % mt);
      const uint8_t* vp = ok ? vc + pid * P.page_stride + (int64_t)sub * rowb : dummy;
      const uint8_t* sp = ok ? vsc + pid * F.sstride + sub : dummy;
      const uint32_t o = ok ? voff : 0, rs = ok ? rowb : 0;
      ve = *reinterpret_cast<const uint32_t*>(sp + (ok ? 4 * lg : 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<VW>(vp + (o + i * rs), vr[i]);
    }
  };
  // Any page size: each lane looks up its own tokens' pages.  Returns which of tokens 4 lg + i exist.
  auto load_tokens = [&](int tile) __attribute__((always_inline)) -> int {
    auto find = [&](int t, int& slot) __attribute__((always_inline)) -> int {
      const int pi = t / ps;
      slot = t - pi * ps;
      const int pid = t < len ? P.indices[s0 + pi] : -1;
      return pid >= 0 && (int64_t)pid < P.num_pages ? pid : -1;
    };
    int slot;
    const int kp = find(16 * tile + lr, slot);
    const uint8_t* k = kp >= 0 ? kc + kp * P.page_stride + (int64_t)slot * rowb + 16 * lg : dummy;
#pragma unroll
    for (int j = 0; j < NK; ++j) kr[j] = *reinterpret_cast<const u4v*>(k + 64 * j);
    int in = 0;
    ke = ve = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int vp = find(16 * tile + 4 * lg + i, slot);
      const uint8_t* v = vp >= 0 ? vc + vp * P.page_stride + (int64_t)slot * rowb + VB * lr : dummy;
      load_words<VW>(v, vr[i]);
      ke |= (uint32_t)*(vp >= 0 ? ksc + vp * F.sstride + slot : dummy) << (8 * i);
      ve |= (uint32_t)*(vp >= 0 ? vsc + vp * F.sstride + slot : dummy) << (8 * i);
      in |= vp >= 0 ? 1 << i : 0;
    }
    return in;
  };

  int tile = p0 + wave, pid = -1;
  if constexpr (P16) {
    pid = page_of(tile);
    load_k(tile, pid);
    load_v(tile, pid);
  }
  uint4 qr[KS];
#pragma unroll
  for (int j = 0; j < NK; ++j) {
    qr[2 * j] = *reinterpret_cast<const uint4*>(qc + 64 * j + 16 * lg);
    qr[2 * j + 1] = *reinterpret_cast<const uint4*>(qc + 64 * j + 16 * lg + 8);
  }
  f4 o[NT];
#pragma unroll
  for (int e = 0; e < NT; ++e) o[e] = f4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, lsum = 0.f;

#pragma unroll 1
  for (; tile < end; tile += W) {
    int in = 15, npid = -1;  // in: which of my four tokens exist
    bool full = true;
    if constexpr (P16) {
      npid = page_of(tile + W);
      const int left = len - 16 * tile, nv = pid < 0 ? 0 : min(left, 16);
      full = nv == 16;
      const int mine = min(max(nv - 4 * lg, 0), 4);
      in = (1 << mine) - 1;
    } else {
      in = load_tokens(tile);
      full = false;
    }
    f4 sa = f4{0.f, 0.f, 0.f, 0.f}, sb = sa;  // (two chains: a product waits for the one two back)
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const uint4 a0 = make_uint4(Codes<T>::lo(kr[j][0]), Codes<T>::hi(kr[j][0]), Codes<T>::lo(kr[j][1]), Codes<T>::hi(kr[j][1]));
      const uint4 a1 = make_uint4(Codes<T>::lo(kr[j][2]), Codes<T>::hi(kr[j][2]), Codes<T>::lo(kr[j][3]), Codes<T>::hi(kr[j][3]));
      sa = Mma<T>::qk(a0, qr[2 * j], sa);
      sb = Mma<T>::qk(a1, qr[2 * j + 1], sb);
    }
    float sc[4], vsf[4];
    sa += sb;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i] = ldexpf(sa[i], (int)((ke >> (8 * i)) & 255) - 127) * P.scale_log2;
      vsf[i] = __uint_as_float(((ve >> (8 * i)) & 255) << 23);
    }
    if (P16) load_k(tile + W, npid);
    if (!full) {
      // tokens that do not exist: no score, no weight, and codes read as zeros (0 * NaN would poison P.V)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool x = in >> i & 1;
        sc[i] = x ? sc[i] : -INFINITY;
        vsf[i] = x ? vsf[i] : 0.f;
#pragma unroll
        for (int c = 0; c < VW; ++c) vr[i][c] = x ? vr[i][c] : 0u;
      }
    }
    const float cms = max_across_groups(max2f(max2f(sc[0], sc[1]), max2f(sc[2], sc[3])));
    const bool grow = cms > m + kLazyMax;  // (false while every score so far is -inf)
    if (__ballot(grow)) {
      const float mnew = grow ? cms : m;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m - mnew) : 1.f;
#pragma unroll
      for (int e = 0; e < NT; ++e) o[e] *= alpha;
      lsum *= alpha;
      m = mnew;
    }
    const float nm = m == -INFINITY ? 0.f : m;
    float wt[4], rest[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[i] = __builtin_amdgcn_exp2f(sc[i] - nm);
    lsum += (sc[0] + sc[1]) + (sc[2] + sc[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) wt[i] = sc[i] * vsf[i];
    using M16 = Mma<__hip_bfloat16>;
    const uint32_t h01 = M16::pack(wt[0], wt[1]), h23 = M16::pack(wt[2], wt[3]);
    rest[0] = wt[0] - __uint_as_float(h01 << 16), rest[1] = wt[1] - __uint_as_float(h01 & 0xFFFF0000u);
    rest[2] = wt[2] - __uint_as_float(h23 << 16), rest[3] = wt[3] - __uint_as_float(h23 & 0xFFFF0000u);
    const uint4 pb = make_uint4(h01, h23, M16::pack(rest[0], rest[1]), M16::pack(rest[2], rest[3]));
    using C16 = Codes<__hip_bfloat16>;
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      // bytes of tokens 0 / 1 (and 2 / 3) side by side, dims 4 c + 0, 1 and 2, 3
      const uint32_t t0 = __builtin_amdgcn_perm(vr[1][c], vr[0][c], 0x05010400u), t1 = __builtin_amdgcn_perm(vr[1][c], vr[0][c], 0x07030602u);
      const uint32_t u0 = __builtin_amdgcn_perm(vr[3][c], vr[2][c], 0x05010400u), u1 = __builtin_amdgcn_perm(vr[3][c], vr[2][c], 0x07030602u);
      const uint2 a[4] = {make_uint2(C16::lo(t0), C16::lo(u0)), make_uint2(C16::hi(t0), C16::hi(u0)),
                          make_uint2(C16::lo(t1), C16::lo(u1)), make_uint2(C16::hi(t1), C16::hi(u1))};
#pragma unroll
      for (int e = 0; e < 4; ++e) o[4 * c + e] = M16::qk(make_uint4(a[e].x, a[e].y, a[e].x, a[e].y), pb, o[4 * c + e]);
    }
    if (P16) load_v(tile + W, npid);
    pid = npid;
  }

  // ---- the waves' states in wave order (a wave without a tile: no mass)
  const float ltot = sum_across_groups(lsum);
  if (lg == 0) s_ml[wave][lr] = make_float2(m, ltot);
  lds_barrier();
  float2 v[W];
#pragma unroll
  for (int x = 0; x < W; ++x) v[x] = x == 0 || !one ? s_ml[x][lr] : make_float2(-INFINITY, 0.f);
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int x = 0; x < W; ++x) M = fmaxf(M, v[x].x);
  const float mu = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int x = 0; x < W; ++x) L += v[x].y * __builtin_amdgcn_exp2f(v[x].x - mu);
  const float cs = __builtin_amdgcn_exp2f(m - mu);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int c = 0; c < VW; ++c)  // dims VB (4 lg + i) + 4 c + (0 .. 3)
      s_o[wave][VW * i + c][lane] = f4{o[4 * c][i], o[4 * c + 1][i], o[4 * c + 2][i], o[4 * c + 3][i]} * cs;
  lds_barrier();
  typedef __attribute__((address_space(1))) T gT;
  gT* out = (gT*)P.out;
  auto store_row = [&](int64_t hq, int d, f4 x) __attribute__((always_inline)) {
    gT* dst = out + b * P.o_sn + hq * P.o_sh + d;
    if (P.o_vec) {
      *(__attribute__((address_space(1))) uint64_t*)dst = (uint64_t)Mma<T>::pack(x[2], x[3]) << 32 | Mma<T>::pack(x[0], x[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) ((__attribute__((address_space(1))) uint16_t*)dst)[e] = bitcast_<uint16_t>(from_f32<T>(x[e]));
    }
  };
  if (lr < gc) {
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const int64_t hq = h * g + c0 + lr;
#pragma unroll 1
    for (int pc = wave; pc < NP; pc += one ? 1 : W) {
      f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const f4 y = s_o[x][pc][lane];
        acc += x == 0 || !one ? y : f4{0.f, 0.f, 0.f, 0.f};
      }
      acc *= inv;
      const int d = VB * (4 * lg + pc / VW) + 4 * (pc % VW);
      if (nparts == 1) store_row(hq, d, acc);
      else st_dev4(P.part_o, (uint32_t)((((int64_t)w * P.hq + hq) * D + d) * sizeof(float)), acc);
    }
    if (nparts > 1 && wave == 0 && lg == 0) store_partial_ml(P, w, (int)hq, M, L);
  }
  if (nparts == 1) return;
  if (!arrive_last(P, b * H + hb, nparts, &s_last)) return;

  // ---- merge of the sequence's parts for these heads: four dims of one head a lane, the parts shared by nw
  // waves, the rows of kMergeParts parts requested at once and folded under a running max (a part without
  // mass holds zeros; repeats weigh nothing).  A line of (max, sum) pairs has a reader per head block, so
  // the pairs are loaded past the caches (ld_dev2); a head's partial rows are whole lines of its own.
  const int x0 = (h * g + c0) * (D / 4), nx = gc * (D / 4);
  const int groups = (nx + 63) / 64, nw = groups >= W ? 1 : W / groups;  // waves a group of 64 items
  const int share = (nparts + nw - 1) / nw;
  for (int gr = wave / nw; gr < (groups + W / nw - 1) / (W / nw) * (W / nw); gr += W / nw) {  // (the same rounds for every wave)
    const int x = x0 + min(gr * 64 + lane, nx - 1);
    const int hq = x / (D / 4), d = (x - hq * (D / 4)) * 4;
    const float2* ml = P.part_ml + hq;
    const float* po = P.part_o + (int64_t)hq * D + d;
    const int q1 = min(share * (wave % nw + 1), nparts);
    float M2 = -INFINITY, den = 0.f;
    f4 acc = f4{0.f, 0.f, 0.f, 0.f};
    for (int q0 = share * (wave % nw); q0 < q1; q0 += kMergeParts) {
      float2 y[kMergeParts];
      f4 row[kMergeParts];
#pragma unroll
      for (int q = 0; q < kMergeParts; ++q) {
        const int pq = min(q0 + q, q1 - 1);
        const int64_t sl = pq == 0 ? b : B + more0 + pq - 1;
        y[q] = ld_dev2(ml + sl * P.ml_stride);
        row[q] = *reinterpret_cast<const f4*>(po + sl * P.hq * D);
      }
      float Mn = M2;
#pragma unroll
      for (int q = 0; q < kMergeParts; ++q) Mn = fmaxf(Mn, y[q].x);
      const float mn = Mn == -INFINITY ? 0.f : Mn, f = __builtin_amdgcn_exp2f(M2 - mn);
      den *= f;
      acc *= f;
      M2 = Mn;
#pragma unroll
      for (int q = 0; q < kMergeParts; ++q)
        if (q0 + q < q1) {
          const float c = __builtin_amdgcn_exp2f(y[q].x - mn) * y[q].y;
          den += c;
          acc += c * row[q];
        }
    }
    if (nw > 1) {  // (then every group is a round of its own)
      __syncthreads();
      s_o[wave][0][lane] = acc;
      s_o[wave][1][lane] = f4{M2, den, 0.f, 0.f};
      __syncthreads();
      if (wave % nw != 0) continue;
      float Mn = -INFINITY;
      for (int y = 0; y < nw; ++y) Mn = fmaxf(Mn, s_o[wave + y][1][lane][0]);
      const float mn = Mn == -INFINITY ? 0.f : Mn;
      acc = f4{0.f, 0.f, 0.f, 0.f};
      den = 0.f;
      for (int y = 0; y < nw; ++y) {
        const f4 z = s_o[wave + y][1][lane];
        const float f = __builtin_amdgcn_exp2f(z[0] - mn);
        den += f * z[1];
        acc += f * s_o[wave + y][0][lane];
      }
    }
    if (gr * 64 + lane < nx) store_row(hq, d, acc * (den > 0.f ? 1.f / den : 0.f));
  }
}

}  // namespace

namespace {

inline int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Workspace: [counters: int32 a sequence and head block] [part_ml: S x ml_slot_stride(Hq) float2]
// [part_o: f32 S x Hq x D], S = nr + batch partial slots.
struct Fp8Layout {
  int64_t ml, o, total;
  int32_t blocks, nr;  // head blocks; further parts a launch has room for
};
bool fp8_layout(int32_t batch, int32_t hq, int32_t hkv, int32_t d, int32_t num_ctas, Fp8Layout* L) {
  if (batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv || num_ctas <= 0) return false;
  const int64_t blocks = (int64_t)hkv * ((hq / hkv + 15) / 16);
  const int64_t want = (int64_t)(d <= 128 ? 6 : 4) * num_ctas / (4 * blocks);
  const int64_t nr = std::max<int64_t>(std::min<int64_t>(num_ctas, want), 1), slots = nr + batch;
  if (blocks * slots > INT32_MAX) return false;
  // (partial rows are addressed with 31-bit byte offsets)
  if (slots * hq * d * (int64_t)sizeof(float) > INT32_MAX) return false;
  L->blocks = (int32_t)blocks;
  L->nr = (int32_t)nr;
  L->ml = align256(sizeof(int32_t) * batch * blocks);
  L->o = L->ml + align256((int64_t)sizeof(float2) * slots * ml_slot_stride(hq));
  L->total = L->o + align256((int64_t)sizeof(float) * slots * hq * d);
  return true;
}

}  // namespace

extern "C" int64_t pkv_decode_fp8_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t num_ctas) {
  Fp8Layout L;
  return fp8_layout(batch, num_qo_heads, num_kv_heads, head_dim, num_ctas, &L) ? L.total : (int64_t)kBadArg;
}

extern "C" int pkv_batch_decode_fp8(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k_cache,
                                    const void* v_cache, int64_t page_stride, int64_t num_pages, const void* k_scales,
                                    const void* v_scales, int64_t scale_page_stride, const int32_t* kv_indptr,
                                    const int32_t* kv_indices, int64_t num_indices, const int32_t* kv_last_page_len,
                                    int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t page_size, float sm_scale, int32_t num_ctas, void* workspace,
                                    int64_t workspace_bytes, void* out, int64_t o_stride_n, int64_t o_stride_h,
                                    int32_t dtype, void* stream) {
  if (dtype != kF16 && dtype != kBF16) return kBadDType;
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads) return kBadGroup;
  if (page_size <= 0) return kBadPageSize;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return kBadHeadDim;
  if (num_indices < 0 || num_pages < 0) return kBadArg;
  Fp8Layout L;
  if (!fp8_layout(batch, num_qo_heads, num_kv_heads, head_dim, num_ctas, &L)) return kBadArg;
  if (L.total > workspace_bytes) return kWorkspaceTooSmall;
  const bool p16 = page_size % 16 == 0;
  const int64_t st = (q_stride_n | q_stride_h) * 2;
  if (((uintptr_t)q | (uintptr_t)st) % 16 || ((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)page_stride) % 16)
    return kBadAlign;
  if (p16 && ((uintptr_t)k_scales | (uintptr_t)v_scales | (uintptr_t)scale_page_stride) % 4) return kBadAlign;
  DecodeParams P{};
  P.q = q; P.q_sn = q_stride_n; P.q_sh = q_stride_h;
  P.k_cache = k_cache; P.v_cache = v_cache; P.page_stride = page_stride;
  P.num_pages = num_pages; P.num_indices = num_indices;
  P.indptr = kv_indptr; P.indices = kv_indices; P.last = kv_last_page_len;
  P.batch = batch; P.hq = num_qo_heads; P.hkv = num_kv_heads; P.ps = page_size;
  P.scale_log2 = sm_scale * 1.4426950408889634f;
  P.out = out; P.o_sn = o_stride_n; P.o_sh = o_stride_h;
  char* ws = (char*)workspace;
  P.counters = (int32_t*)ws;
  P.part_ml = (float2*)(ws + L.ml);
  P.part_o = (float*)(ws + L.o);
  P.ml_stride = ml_slot_stride(num_qo_heads);
  P.o_vec = ((uintptr_t)out | (uintptr_t)(o_stride_n * 2) | (uintptr_t)(o_stride_h * 2)) % 8 == 0;
  const Fp8Cache F{(const uint8_t*)k_scales, (const uint8_t*)v_scales, scale_page_stride, L.blocks / num_kv_heads};
  const int max_parts = std::max(64, L.nr);
  const dim3 grid((unsigned)(((int64_t)L.nr + batch) * L.blocks));
  hipStream_t s = (hipStream_t)stream;
#define PKV_DECODE_FP8_P(T, D)                                                                                     \
  if (p16) hipLaunchKernelGGL((decode_fp8_kernel<T, D, true>), grid, dim3(W * 64), 0, s, P, F, L.nr, max_parts);   \
  else hipLaunchKernelGGL((decode_fp8_kernel<T, D, false>), grid, dim3(W * 64), 0, s, P, F, L.nr, max_parts)
#define PKV_DECODE_FP8(T)                               \
  if (head_dim == 64) { PKV_DECODE_FP8_P(T, 64); }      \
  else if (head_dim == 128) { PKV_DECODE_FP8_P(T, 128); } \
  else { PKV_DECODE_FP8_P(T, 256); }
  if (dtype == kF16) {
    PKV_DECODE_FP8(_Float16)
  } else {
    PKV_DECODE_FP8(__hip_bfloat16)
  }
#undef PKV_DECODE_FP8
#undef PKV_DECODE_FP8_P
  return (int)hipGetLastError();
}
