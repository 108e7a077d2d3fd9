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
// A workgroup (W = 4 or 8 waves) takes one KV head, or two neighbours (16 query heads at most), of one part of one
// sequence; wave r takes the part's tiles of 16 tokens r, r + W, ...  With lane l = (lr = l % 16, lg = l / 16),
// a tile of rows of RW bytes:
//   S[token][head]     = K . Q^T   A: K[token lr][dims 64 j + 16 lg + 0 .. 15], one 16-byte load for two steps
//   online softmax                 lane: head lr, tokens 4 lg + i
//   O^T[dim][head]    += V^T . P   A: V[token 4 lg + i][dims RW/16 lr + 0 .. RW/16), one load a token: its bytes
//                                  pair with the next token's by v_perm; B: the lane's own weights
// so K and V go from memory straight into registers (no LDS, no lane exchange), a wave's load covers whole rows,
// and each register set is refilled with the next tile's rows as soon as its products are issued.  Of two heads'
// rows each column takes its own head's scores, and the products of a column with the other head's dims are left
// aside: as many matrix instructions a head as with one, and half the softmax.
//
// What bounds it: the bytes.  A CU streams about 20 KB a us with 32 KB in flight, so the plan looks for parts that
// give each CU as many tiles as the others; then a batch runs at 5.3 to 5.5 TB/s (64 sequences of 9600 tokens, 28 / 4
// heads: 115 us for 635 MB).  A call has about 5 us besides (launch, page table, ids, rows, the waves' states), and
// where sequences are cut 2 to 5 us of partials, arrival and merge: 64 sequences of 512 to 4096 tokens, 16 / 2 heads,
// take 21.5 us for 79 MB, 15 at the rate of a large copy.
#include <algorithm>
#include "attn_common.h"
#include "mfma_common.h"
#include "cache_fp8.h"
#include "../../include/pagedkv.h"

using namespace pkv;
using namespace pkv::mfma;

namespace {

constexpr int kMinTiles = 8;       // tiles of a part, at least
constexpr int kWholeTiles = 24;    // longest sequence that is never cut
constexpr float kLazyMax = 8.f;    // a head's reference max moves only on jumps > 2^8
// Parts whose rows the merge loads at a time (64 sequences: 21.2 us, 21.7 with 16, 22.7 with 24, which spill).
constexpr int kMergeParts = 8;

struct Fp8Cache {
  const uint8_t *ks, *vs;
  int64_t sstride;   // scale bytes between pages
  int32_t ncb;       // blocks of 16 query heads a KV head
  const int32_t* plan;  // the planned `aim` and number of further parts, or null
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

// Parts whose weights the merge holds in the exchange buffer (16 columns of float2 each).
__host__ __device__ constexpr int max_parts_of(int row, int waves) { return waves * (row / 16 - 1) * 8; }

// Tokens of a sequence with pages [i0, i1) of a page list of `cut` entries.
__device__ __forceinline__ int length_of(int i0, int i1, int last, int ps, int64_t cut) {
  if (i0 < 0 || i1 <= i0) return 0;
  const int64_t np = i1 - i0, av = min((int64_t)i1, cut) - i0;
  return (int)min((np - 1) * ps + min(max(last, 0), ps), max(av, (int64_t)0) * ps);
}
__device__ __forceinline__ int tiles_of(int len) { return (len + 15) / 16; }
// Inclusive sum over the wave's lanes, in registers: within rows of 16 lanes by row shifts, then the rows' totals.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31 into rows 2 and 3
  return x;
}
// Parts of a sequence: of `aim` tiles at most, one if there are few.
__device__ __forceinline__ int parts_of(int tiles, int aim, int max_parts) {
  return tiles <= max(kWholeTiles, aim) ? 1 : min((tiles + aim - 1) / aim, max_parts);
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

// HB: KV heads a block takes (2: their rows are one run of memory, and the columns of both share a tile).
// P16: page_size is a multiple of 16, so a tile lies in one page.
template <typename T, int D, int HB, bool P16, int W>
__global__ __launch_bounds__(W * 64, HB * D == 256 ? 2 : 4) void decode_fp8_kernel(DecodeParams P, Fp8Cache F, int nr) {
  constexpr int RW = HB * D;   // bytes of a row
  constexpr int NK = RW / 64;  // 16-byte pieces of a K row a lane holds
  constexpr int KS = RW / 32;  // QK steps
  constexpr int VB = RW / 16;  // bytes of a V row a lane holds
  constexpr int VW = VB / 4;
  constexpr int NT = RW / 16;  // output tiles
  constexpr int NP = NT;      // 16-byte pieces of a lane's 4 NT output values
  constexpr int kMaxParts = max_parts_of(RW, W);
  static_assert(HB == 1 || (HB == 2 && RW <= 256 && P16), "two heads a block: 256 bytes at most, tiles in one page");
  __shared__ f4 s_o[W][NP][64];
  __shared__ float2 s_ml[W][16];
  __shared__ int s_last;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  const int B = P.batch, g = P.hq / P.hkv, H = P.hkv / HB * F.ncb, ps = P.ps;
  // (workgroups are dealt round-robin to the 8 XCDs: a part's heads, neighbours in memory, go to one)
  const int at = blockIdx.x / 8, hb = at % H, w = at / H * 8 + blockIdx.x % 8;
  if (w >= B + nr) return;
  // my KV heads h .. h + HB - 1 and query heads q0 .. q0 + gc - 1 (columns 0 .. gc - 1)
  const int h = HB * (hb / F.ncb), c0 = HB > 1 ? 0 : hb % F.ncb * 16, gc = HB > 1 ? HB * g : min(g - c0, 16);
  const int64_t q0 = (int64_t)h * g + c0;
  const int col = lr < gc ? lr : gc - 1;          // (columns past the block repeat its last one, and are never stored)
  const int hn = HB > 1 ? (col < g ? 0 : 1) : 0;  // my column's KV head in the block

  // ---- workgroup w: the first part of sequence w, or (w >= B) the (w - B)-th of the further parts, which
  // follow each other in sequence order; those and cut sequences look for their place among the batch, 64
  // sequences a round.
  typedef __attribute__((address_space(1))) uint16_t g16;  // (stores through a generic pointer would drain the loads in flight)
  int b = min(w, B - 1), nparts, part = 0, more0 = 0, aim;
  // (everything that may be needed is requested at once: my sequence's, and the first 64 sequences' for the search)
  int i0 = P.indptr[min(lane, B)], i1 = P.indptr[min(lane + 1, B)], lv = P.last[min(lane, B - 1)];
  int s0 = P.indptr[b];
  const int e0 = P.indptr[b + 1], l0 = P.last[b];
  if (F.plan) {  // (made for other lengths, it may hold too few parts: the last ones are longer then)
    aim = max(F.plan[0], 1);
    nr = min(max(F.plan[1], 0), nr);
    if (w >= B + nr) return;
  } else {
    const int64_t listed = max(min((int64_t)P.indptr[B], P.num_indices), (int64_t)0);
    aim = max(kMinTiles, (int)((listed * ps / 16 + nr) / nr));
  }
  int len = length_of(s0, e0, l0, ps, P.num_indices);
  nparts = parts_of(tiles_of(len), aim, kMaxParts);
  if (w >= B || nparts > 1) {
    bool found = false;
    int base = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < B; b0 += 64) {
      const int n0 = P.indptr[min(b0 + 64 + lane, B)], n1 = P.indptr[min(b0 + 65 + lane, B)];  // (the next round's)
      const int nl = P.last[min(b0 + 64 + lane, B - 1)];
      const int ln = b0 + lane < B ? length_of(i0, i1, lv, ps, P.num_indices) : 0;
      const int np = b0 + lane < B ? parts_of(tiles_of(ln), aim, kMaxParts) - 1 : 0;
      const int incl = wave_scan(np), all = __builtin_amdgcn_readlane(incl, 63);
      if (w < B ? w < b0 + 64 : w - B < base + all) {
        const int l = w < B ? w - b0 : __popcll(__ballot(base + incl <= w - B));
        more0 = base + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(np, l);
        if (w >= B) {
          b = b0 + l;
          s0 = __builtin_amdgcn_readlane(i0, l);
          len = __builtin_amdgcn_readlane(ln, l);
          nparts = __builtin_amdgcn_readlane(np, l) + 1;
          part = 1 + w - B - more0;
        }
        found = true;
        break;
      }
      base += all;
      i0 = n0, i1 = n1, lv = nl;
    }
    if (!found) return;  // (the grid is sized for the most parts there can be)
    nparts = 1 + min(nparts - 1, max(nr - more0, 0));  // (a kv_indptr that runs backwards)
  }
  b = __builtin_amdgcn_readfirstlane(b);
  s0 = __builtin_amdgcn_readfirstlane(s0);
  len = __builtin_amdgcn_readfirstlane(len);
  // the part's tiles [t0, t1)
  const int tiles = tiles_of(len), per = tiles / nparts, more = tiles - per * nparts;
  const int t0 = part * per + min(part, more), t1 = t0 + per + (part < more ? 1 : 0);
  const bool one = nparts == 1 && tiles <= 1;  // wave 0's alone
  if (one && wave > 0) return;

  const uint32_t rowb = P.hkv * D;  // bytes between token rows
  const uint8_t* kc = (const uint8_t*)P.k_cache + (int64_t)h * D;
  const uint8_t* vc = (const uint8_t*)P.v_cache + (int64_t)h * D;
  const uint8_t* ksc = F.ks + (int64_t)(h + hn) * ps;
  const uint8_t* vsc = F.vs + (int64_t)(h + hn) * ps;
  const int mt = P16 ? ps / 16 : 1;  // tiles a page
  const uint8_t* dummy = (const uint8_t*)((const T*)P.q + b * P.q_sn + q0 * P.q_sh);

  // The tile's rows, and the scales of tokens 4 lg + 0 .. 3 (a byte each).  Every load is unconditional, so
  // that all paths have the same ones in flight; where there is no page they read a query row instead.
  const uint32_t koff = lr * rowb + 16 * lg, voff = 4 * lg * rowb + VB * lr;
  u4v kr[NK];
  uint32_t vr[4][VW], ke = 0, ve = 0;
  // Pages.  P16: lane l has the id of this wave's tile k + l, for 64 tiles, -1 outside the pool or past the part.
  // Else: lane (lr, .) looks up token lr of the tile; `at` is its slot.
  int ids = -1, k = 0;
  auto valid = [&](int pid) __attribute__((always_inline)) -> int { return pid >= 0 && (int64_t)pid < P.num_pages ? pid : -1; };
  auto load_ids = [&](int first) __attribute__((always_inline)) {
    const int t = min(first + W * lane, t1 - 1);
    const int pid = t >= 0 ? P.indices[s0 + (mt == 1 ? t : t / mt)] : -1;
    ids = first + W * lane < t1 ? valid(pid) : -1;
  };
  struct Page {
    int id, at;
  };
  auto page_of = [&](int tile) __attribute__((always_inline)) -> Page {
    if constexpr (P16) {
      return Page{__builtin_amdgcn_readlane(ids, k & 63), mt == 1 ? 0 : 16 * (tile % mt)};
    } else {
      const int t = 16 * tile + lr, pi = t / ps;
      return Page{tile < t1 && t < len ? valid(P.indices[s0 + pi]) : -1, t - pi * ps};
    }
  };
  auto load_k = [&](Page pg) __attribute__((always_inline)) {
    const bool ok = pg.id >= 0;
    const uint8_t* kp = ok ? kc + pg.id * P.page_stride + (int64_t)pg.at * rowb : dummy;
    const uint32_t o = !ok ? 0 : P16 ? koff : 16 * lg;
#pragma unroll
    for (int j = 0; j < NK; ++j) kr[j] = *reinterpret_cast<const u4v*>(kp + o + 64 * j);
    const int64_t so = pg.id * F.sstride + pg.at;
    if constexpr (P16) {
      ke = *reinterpret_cast<const uint32_t*>(ok ? ksc + so + 4 * lg : dummy);
      ve = *reinterpret_cast<const uint32_t*>(ok ? vsc + so + 4 * lg : dummy);
    } else {  // (my token's, to be passed on)
      ke = *(ok ? ksc + so : dummy);
      ve = *(ok ? vsc + so : dummy);
    }
  };
  auto load_v = [&](Page pg) __attribute__((always_inline)) {
    if constexpr (P16) {
      const bool ok = pg.id >= 0;
      const uint8_t* vp = ok ? vc + pg.id * P.page_stride + (int64_t)pg.at * rowb : dummy;
      const uint32_t o = ok ? voff : 0, rs = ok ? rowb : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<VW>(vp + (o + i * rs), vr[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int id = __shfl(pg.id, 4 * lg + i, 64), at = __shfl(pg.at, 4 * lg + i, 64);
        load_words<VW>(id >= 0 ? vc + id * P.page_stride + (int64_t)at * rowb + VB * lr : dummy, vr[i]);
      }
    }
  };

  auto store_row = [&](int row, int64_t hq, int d, f4 x) __attribute__((always_inline)) {
    g16* dst = (g16*)P.out + row * P.o_sn + hq * P.o_sh + d;
    if (P.o_vec) {
      *(__attribute__((address_space(1))) uint64_t*)dst = (uint64_t)Mma<T>::pack(x[2], x[3]) << 32 | Mma<T>::pack(x[0], x[1]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[e] = bitcast_<uint16_t>(from_f32<T>(x[e]));
    }
  };

  int tile = t0 + wave;
  if constexpr (P16) load_ids(tile);
  Page pg = page_of(tile);
  load_k(pg);
  load_v(pg);
  const T* qc = (const T*)P.q + b * P.q_sn + (q0 + col) * P.q_sh;
  uint4 qr[KS / HB];
#pragma unroll
  for (int j = 0; j < NK / HB; ++j) {
    qr[2 * j] = *reinterpret_cast<const uint4*>(qc + 64 * j + 16 * lg);
    qr[2 * j + 1] = *reinterpret_cast<const uint4*>(qc + 64 * j + 16 * lg + 8);
  }
  f4 o[NT];
#pragma unroll
  for (int e = 0; e < NT; ++e) o[e] = f4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, lsum = 0.f;

#pragma unroll 1
  for (; tile < t1; tile += W) {
    int in = 15;  // which of my four tokens exist
    bool full = true;
    if constexpr (P16) {
      const int nv = pg.id < 0 ? 0 : min(len - 16 * tile, 16);
      full = nv == 16;
      in = (1 << min(max(nv - 4 * lg, 0), 4)) - 1;
    }
    ++k;
    if (P16 && (k & 63) == 0) {
      load_ids(tile + W);
      __builtin_amdgcn_s_waitcnt(0x0F70);  // (compiler-visible vmcnt(0): the usual path waits for nothing)
    }
    const Page next = page_of(tile + W);
    f4 sa = f4{0.f, 0.f, 0.f, 0.f}, sb = sa;  // (two chains: a product waits for the one two back)
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const uint4 a0 = make_uint4(Codes<T>::lo(kr[j][0]), Codes<T>::hi(kr[j][0]), Codes<T>::lo(kr[j][1]), Codes<T>::hi(kr[j][1]));
      const uint4 a1 = make_uint4(Codes<T>::lo(kr[j][2]), Codes<T>::hi(kr[j][2]), Codes<T>::lo(kr[j][3]), Codes<T>::hi(kr[j][3]));
      if constexpr (HB == 1) {
        sa = Mma<T>::qk(a0, qr[2 * j], sa);
        sb = Mma<T>::qk(a1, qr[2 * j + 1], sb);
      } else {  // (each head's scores by themselves: a column takes its own, so nothing of another head's key reaches it)
        f4& sj = j < NK / 2 ? sa : sb;
        sj = Mma<T>::qk(a0, qr[2 * (j % (NK / HB))], sj);
        sj = Mma<T>::qk(a1, qr[2 * (j % (NK / HB)) + 1], sj);
      }
    }
    float sc[4];
    int ev[4];
    if (HB == 1) sa += sb;
    else sa = hn == 0 ? sa : sb;
    if constexpr (!P16) {
      const uint32_t mine = ke | ve << 8 | (pg.id >= 0 ? 0x10000u : 0u);
      ke = ve = in = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = __shfl(mine, 4 * lg + i, 64);
        ke |= (x & 255) << (8 * i), ve |= ((x >> 8) & 255) << (8 * i);
        in |= (x >> 16) << i;
      }
      full = false;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i] = ldexpf(sa[i], (int)((ke >> (8 * i)) & 255) - 127) * P.scale_log2;
      ev[i] = (int)((ve >> (8 * i)) & 255) - 127;
    }
    const uint32_t both = ke | ve;
    if (__ballot((~both - 0x01010101u) & both & 0x80808080u)) {  // a byte of 255, perhaps: NaN
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (((ke >> (8 * i)) & 255) == 255 || ev[i] == 128) sc[i] = NAN;
    }
    load_k(next);
    if (!full) {
      // tokens that do not exist: no score, no weight, and codes read as zeros (0 * NaN would poison P.V)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool x = in >> i & 1;
        sc[i] = x ? sc[i] : -INFINITY;
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
    for (int i = 0; i < 4; ++i) wt[i] = ldexpf(sc[i], ev[i]);
    using M16 = Mma<__hip_bfloat16>;
    const uint32_t h01 = M16::pack(wt[0], wt[1]), h23 = M16::pack(wt[2], wt[3]);
    rest[0] = wt[0] - __uint_as_float(h01 << 16), rest[1] = wt[1] - __uint_as_float(h01 & 0xFFFF0000u);
    rest[2] = wt[2] - __uint_as_float(h23 << 16), rest[3] = wt[3] - __uint_as_float(h23 & 0xFFFF0000u);
    const uint4 pb = make_uint4(h01, h23, M16::pack(rest[0], rest[1]), M16::pack(rest[2], rest[3]));
    using C16 = Codes<__hip_bfloat16>;
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      // bytes of tokens 0 / 1 (and 2 / 3) side by side, dims 4 c + 0, 1 and 2, 3
      const uint32_t x0 = __builtin_amdgcn_perm(vr[1][c], vr[0][c], 0x05010400u), x1 = __builtin_amdgcn_perm(vr[1][c], vr[0][c], 0x07030602u);
      const uint32_t u0 = __builtin_amdgcn_perm(vr[3][c], vr[2][c], 0x05010400u), u1 = __builtin_amdgcn_perm(vr[3][c], vr[2][c], 0x07030602u);
      const uint2 a[4] = {make_uint2(C16::lo(x0), C16::lo(u0)), make_uint2(C16::hi(x0), C16::hi(u0)),
                          make_uint2(C16::lo(x1), C16::lo(u1)), make_uint2(C16::hi(x1), C16::hi(u1))};
#pragma unroll
      for (int e = 0; e < 4; ++e) o[4 * c + e] = M16::qk(make_uint4(a[e].x, a[e].y, a[e].x, a[e].y), pb, o[4 * c + e]);
    }
    load_v(next);
    pg = next;
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
  // (two heads a row: lanes lg / 2 hold the dims of head lg / 2)
  if (lr < gc && (HB == 1 || lg / 2 == hn)) {
    const float inv = L > 0.f ? 1.f / L : 0.f;
    const int64_t hq = q0 + lr;
#pragma unroll 1
    for (int pc = wave; pc < NP; pc += one ? 1 : W) {
      f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const f4 y = s_o[x][pc][lane];
        acc += x == 0 || !one ? y : f4{0.f, 0.f, 0.f, 0.f};
      }
      acc *= inv;
      const int d = VB * (4 * lg + pc / VW) + 4 * (pc % VW) - hn * D;
      if (nparts == 1) store_row(b, hq, d, acc);
      else st_dev4(P.part_o, (uint32_t)((((int64_t)w * P.hq + hq) * D + d) * sizeof(float)), acc);
    }
    if (nparts > 1 && wave == 0 && lg == 2 * hn) store_partial_ml(P, w, (int)hq, M, L);
  }
  if (nparts == 1) return;
  if (!arrive_last(P, b * H + hb, nparts, &s_last)) return;

  // ---- The merge of the sequence's parts for these heads.  First the weights: thread (part, column) takes a
  // (max, sum) pair; a line of pairs has a reader per head block, so they are loaded past the caches (ld_dev2).
  // Part x, column c weighs exp2(max - the column's) * sum, in s_w; a part without mass weighs nothing.
  float2* s_w = reinterpret_cast<float2*>(s_o);  // [part][16]
  f4* s_x = &s_o[0][0][0] + (W * NP - W) * 64;   // [W][64], behind them
  auto slot_of = [&](int x) __attribute__((always_inline)) -> int64_t { return x ? B + more0 + x - 1 : b; };
  {
    const int c = threadIdx.x & 15;
    const float2* ml = P.part_ml + q0 + (c < gc ? c : gc - 1);
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int x = threadIdx.x >> 4; x < nparts; x += W * 4) {
      const float2 y = ld_dev2(ml + slot_of(x) * P.ml_stride);
      s_w[x * 16 + c] = y;
      top = fmaxf(top, y.x);
    }
    top = max_across_groups(top);
    if (lg == 0) s_ml[wave][lr].x = top;
    lds_barrier();
#pragma unroll
    for (int x = 0; x < W; ++x) top = fmaxf(top, s_ml[x][c].x);
    const float mn = top == -INFINITY ? 0.f : top;
    for (int x = threadIdx.x >> 4; x < nparts; x += W * 4) {
      const float2 y = s_w[x * 16 + c];
      const float e = __builtin_amdgcn_exp2f(y.x - mn) * y.y;
      s_w[x * 16 + c].x = e;
      sum += e;
    }
    sum = sum_across_groups(sum);
    if (lg == 0) s_ml[wave][lr].y = sum;
    lds_barrier();
  }
  // Then the rows: four dims of one head a lane, the parts shared by nw waves; a head's partial rows are whole lines
  // of its own, so plain loads may bring them in, all of them in flight at once.
  const int nx = gc * (D / 4), groups = (nx + 63) / 64, nw = groups >= W ? 1 : W / groups;  // waves a group of 64 items
  const int rounds = (groups * nw + W - 1) / W, share = (nparts + nw - 1) / nw;
  for (int r = 0; r < rounds; ++r) {  // (the same rounds for every wave; one if waves share a group)
    const int gr = (r * W + wave) / nw, sub = (r * W + wave) % nw;
    const int it = min(gr * 64 + lane, nx - 1), c = it / (D / 4), d = (it - c * (D / 4)) * 4;
    const float* po = P.part_o + (q0 + c) * D + d;
    const int x1 = gr < groups ? min(share * (sub + 1), nparts) : 0;
    f4 acc = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int x0 = share * sub; x0 < x1; x0 += kMergeParts) {
      f4 row[kMergeParts];
#pragma unroll
      for (int x = 0; x < kMergeParts; ++x)
        row[x] = *reinterpret_cast<const f4*>(po + slot_of(min(x0 + x, x1 - 1)) * P.hq * D);
#pragma unroll
      for (int x = 0; x < kMergeParts; ++x) acc += row[x] * (x0 + x < x1 ? s_w[min(x0 + x, x1 - 1) * 16 + c].x : 0.f);
    }
    if (nw > 1) {
      s_x[wave * 64 + lane] = acc;
      lds_barrier();
      if (sub == 0)
        for (int x = 1; x < nw; ++x) acc += s_x[(wave + x) * 64 + lane];
    }
    float den = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) den += s_ml[x][c].y;
    if (sub == 0 && gr * 64 + lane < nx) store_row(b, q0 + c, d, acc * (den > 0.f ? 1.f / den : 0.f));
  }
}

// The plan: the longest part (`aim`, in tiles) with the least expected time, of a range of candidates that a wave
// each evaluates.  A CU streams about 20 KB a us however many workgroups it holds, so what counts is the most tiles
// a CU gets: with q workgroups a CU at most, q times the longest part, or with many, their average and one part more;
// each workgroup adds `start` tiles' time for its chain of latencies, cut sequences `join` and a little for each
// part.  One workgroup.
constexpr int kPlanSeqs = 4096;  // larger batches are not looked into: they fill the chip by their number
constexpr int kCandidates = 64;

__global__ __launch_bounds__(1024) void decode_fp8_plan_kernel(const int32_t* indptr, const int32_t* last, int B, int64_t cut,
                                                               int ps, int H, int nr, int cus, int max_parts, int start,
                                                               int join, int32_t* plan) {
  __shared__ int s_t[kPlanSeqs];
  __shared__ int s_sum[16], s_max[16];
  __shared__ float s_cost[kCandidates];
  __shared__ int s_aim[kCandidates], s_more[kCandidates];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int sum = 0, top = 0;
  for (int b = threadIdx.x; b < B; b += 1024) {
    const int t = tiles_of(length_of(indptr[b], indptr[b + 1], last[b], ps, cut));
    s_t[b] = t;
    sum += t;
    top = max(top, t);
  }
  sum = wave_sum_i32(sum);
  top = (int)wave_max_u32((uint32_t)top);
  if (lane == 0) s_sum[wave] = sum, s_max[wave] = top;
  __syncthreads();
  sum = wave_sum_i32(lane < 16 ? s_sum[lane] : 0);
  top = (int)wave_max_u32((uint32_t)(lane < 16 ? s_max[lane] : 0));
  const float lo = (float)max(kMinTiles, (sum + nr + B - 1) / (nr + B)), hi = fmaxf((float)top, lo);
  const float step = __log2f(hi / lo) / (kCandidates - 1);
  for (int i = wave; i < kCandidates; i += 16) {
    // (the longest first: it cuts nothing)
    const int aim = i == 0 ? (int)hi : (int)ceilf(lo * __builtin_amdgcn_exp2f(step * (float)(kCandidates - 1 - i)));
    int parts = 0, big = 0, most = 1;
    for (int b = lane; b < B; b += 64) {
      const int t = s_t[b], p = parts_of(t, aim, max_parts);
      parts += p;
      big = max(big, (t + p - 1) / p);
      most = max(most, p);
    }
    parts = wave_sum_i32(parts);
    big = (int)wave_max_u32((uint32_t)big);
    most = (int)wave_max_u32((uint32_t)most);
    const float wgs = (float)parts * H, c = (float)cus, q = ceilf(wgs / c);
    float cost = fminf(q * (float)(big + start) * (q > 1.f ? 1.08f : 1.f), ((float)sum * H + wgs * start) / c + (float)(big + start));
    if (most > 1) cost += (float)join * (1.f + (float)most * 0.03125f);
    if (lane == 0) s_cost[i] = parts - B <= nr ? cost : INFINITY, s_aim[i] = aim, s_more[i] = parts - B;
  }
  __syncthreads();
  if (wave == 0) {
    static_assert(kCandidates == 64, "a lane a candidate");
    const float mine = s_cost[lane];
    float best = mine;
#pragma unroll
    for (int x = 32; x; x >>= 1) best = fminf(best, __shfl_xor(best, x, 64));
    const uint64_t who = __ballot(mine == best);
    const int i = __builtin_ctzll(who);
    if (lane == 0) plan[0] = s_aim[i], plan[1] = min(s_more[i], nr);
  }
}

}  // namespace

namespace {

inline int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// Workspace: [counters: int32 a sequence and head block, kCounters of them at least, so that of wrappers that take
// turns on one workspace none lays its partials on another's] [the plan] [part_ml: S x ml_slot_stride(Hq) float2]
// [part_o: f32 S x Hq x D], S = nr + batch partial slots.
constexpr int64_t kCounters = 8192;
struct Fp8Layout {
  int64_t plan, ml, o, total;
  int32_t nr;             // further parts there is room for
  int32_t blocks, waves;  // of a launch: head blocks, waves a workgroup
  bool two;               // two KV heads a block
};
// The variant for a batch, by its sizes alone (num_indices: pages it may have).
//  * Two heads a block where their rows are one run of memory: a wave then reads 256 bytes a token instead of 128,
//    and its softmax serves both heads (32 sequences of 9600 tokens, 32 / 8 heads of 128: 116 us for 129; 123 of
//    1728, 28 / 4: 42.7 for 45.0).  With few workgroups its longer merge counts more: one sequence of 16,000
//    tokens 17.1 us for 15.9, of 2000 11.9 for 9.1, so heads of 128 dims take it from 128 sequences x KV heads on.
//    Rows of two heads of 64 dims are one line of 128 bytes: always (85 sequences, 16 / 16 heads: 23 us for 35).
//  * Eight waves a workgroup for long sequences and one-head blocks: fewer parts for as many loads in flight (one
//    sequence of 100,003 tokens, 28 / 4 heads: 27.3 us for 33; of 2000 tokens, 16 / 2: 10.3 for 9.1; pages that are not
//    whole tiles wait for more: 9 sequences of 100 to 9000 tokens, 32 / 8 heads, pages of 8: 16.5 for 20.4).  For
//    two-head blocks where a CU has few tiles: half as many turns a wave (64 sequences of 512 to 4096 tokens, 16 / 2 heads:
//    22.2 us for 23.2; of 9600, 28 / 4: 122 for 116).
bool fp8_layout(int32_t batch, int32_t hq, int32_t hkv, int32_t d, int32_t ps, int32_t num_ctas, int64_t num_indices, Fp8Layout* L) {
  if (batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv || num_ctas <= 0 || ps <= 0 || num_indices < 0) return false;
  if (num_indices > (INT32_MAX - 64) / ps) return false;  // (tokens in 32 bits)
  const int g = hq / hkv;
  const int64_t most = (int64_t)hkv * ((g + 15) / 16);
  L->two = ps % 16 == 0 && d <= 128 && hkv % 2 == 0 && g <= 8 && (d == 64 || (int64_t)batch * hkv >= 128);
  const int64_t blocks = L->two ? hkv / 2 : most;
  const int64_t cus = (num_ctas + 1) / 2, tiles = num_indices * ps / 16;
  const bool wide = L->two ? d == 128 && tiles * blocks < 48 * cus : d <= 128 && tiles >= (ps % 16 ? 48 : 128) * (int64_t)batch;
  L->waves = wide ? 8 : 4;
  const int64_t nr = std::max<int64_t>(2 * cus / blocks, 1), slots = nr + batch;
  if (most * (slots + 8) > INT32_MAX) return false;
  // (partial rows are addressed with 31-bit byte offsets)
  if (slots * hq * d * (int64_t)sizeof(float) > INT32_MAX) return false;
  L->nr = (int32_t)nr;
  L->blocks = (int32_t)blocks;
  L->plan = align256(sizeof(int32_t) * std::max(batch * most, kCounters));
  L->ml = L->plan + 256;
  L->o = L->ml + align256((int64_t)sizeof(float2) * slots * ml_slot_stride(hq));
  L->total = L->o + align256((int64_t)sizeof(float) * slots * hq * d);
  return true;
}

}  // namespace

extern "C" int64_t pkv_decode_fp8_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                                  int32_t head_dim, int32_t page_size, int32_t num_ctas,
                                                  int64_t num_indices) {
  Fp8Layout L;
  return fp8_layout(batch, num_qo_heads, num_kv_heads, head_dim, page_size, num_ctas, num_indices, &L) ? L.total
                                                                                                      : (int64_t)kBadArg;
}

extern "C" int pkv_decode_fp8_plan(const int32_t* kv_indptr, int64_t num_indices, const int32_t* kv_last_page_len,
                                   int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                   int32_t page_size, int32_t num_ctas, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  Fp8Layout L;
  if (!fp8_layout(batch, num_qo_heads, num_kv_heads, head_dim, page_size, num_ctas, num_indices, &L) || batch > kPlanSeqs ||
      !kv_indptr || !kv_last_page_len || !workspace)
    return kBadArg;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return kBadHeadDim;
  if (L.total > workspace_bytes) return kWorkspaceTooSmall;
  const int row = (L.two ? 2 : 1) * head_dim, unit = 256 / row;  // (a tile of a 256-byte row takes 0.4 us of a CU)
  hipLaunchKernelGGL(decode_fp8_plan_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, kv_indptr, kv_last_page_len, batch,
                     num_indices, page_size, L.blocks, L.nr, (num_ctas + 1) / 2, max_parts_of(row, L.waves), 6 * unit, 8 * unit,
                     (int32_t*)((char*)workspace + L.plan));
  return (int)hipGetLastError();
}

extern "C" int pkv_batch_decode_fp8(const void* q, int64_t q_stride_n, int64_t q_stride_h, const void* k_cache,
                                    const void* v_cache, int64_t page_stride, int64_t num_pages, const void* k_scales,
                                    const void* v_scales, int64_t scale_page_stride, const int32_t* kv_indptr,
                                    const int32_t* kv_indices, int64_t num_indices, const int32_t* kv_last_page_len,
                                    int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads, int32_t head_dim,
                                    int32_t page_size, float sm_scale, int32_t num_ctas, void* workspace,
                                    int64_t workspace_bytes, void* out, int64_t o_stride_n, int64_t o_stride_h,
                                    int32_t dtype, int32_t flags, void* stream) {
  if (dtype != kF16 && dtype != kBF16) return kBadDType;
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads) return kBadGroup;
  if (page_size <= 0) return kBadPageSize;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return kBadHeadDim;
  if (num_pages < 0 || (num_pages > 0 && (!k_cache || !v_cache || !k_scales || !v_scales))) return kBadArg;
  if (!q || !out || !kv_indptr || !kv_last_page_len || (num_indices > 0 && !kv_indices) || !workspace) return kBadArg;
  Fp8Layout L;
  if (!fp8_layout(batch, num_qo_heads, num_kv_heads, head_dim, page_size, num_ctas, num_indices, &L)) return kBadArg;
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
  const Fp8Cache F{(const uint8_t*)k_scales, (const uint8_t*)v_scales, scale_page_stride, L.two ? 1 : L.blocks / num_kv_heads,
                   flags & PKV_DECODE_PLANNED ? (const int32_t*)(ws + L.plan) : nullptr};
  const int nr = L.nr;
  const bool two = L.two, wide = L.waves == 8;
  const dim3 grid((unsigned)(((int64_t)nr + batch + 7) / 8 * 8 * L.blocks));
  hipStream_t s = (hipStream_t)stream;
#define PKV_DECODE_FP8_W(T, D, HB, P16, W) \
  hipLaunchKernelGGL((decode_fp8_kernel<T, D, HB, P16, W>), grid, dim3(W * 64), 0, s, P, F, nr)
#define PKV_DECODE_FP8_P(T, D, HB, P16)               \
  if (wide) { PKV_DECODE_FP8_W(T, D, HB, P16, 8); }   \
  else { PKV_DECODE_FP8_W(T, D, HB, P16, 4); }
#define PKV_DECODE_FP8(T)                                                                                     \
  if (head_dim == 64) {                                                                                       \
    if (two) { PKV_DECODE_FP8_W(T, 64, 2, true, 4); }                                                         \
    else if (p16) { PKV_DECODE_FP8_P(T, 64, 1, true); }                                                       \
    else { PKV_DECODE_FP8_P(T, 64, 1, false); }                                                               \
  } else if (head_dim == 128) {                                                                               \
    if (two) { PKV_DECODE_FP8_P(T, 128, 2, true); }                                                           \
    else if (p16) { PKV_DECODE_FP8_P(T, 128, 1, true); }                                                           \
    else { PKV_DECODE_FP8_P(T, 128, 1, false); }                                                              \
  } else {                                                                                                    \
    if (p16) { PKV_DECODE_FP8_W(T, 256, 1, true, 4); }                                                         \
    else { PKV_DECODE_FP8_W(T, 256, 1, false, 4); }                                                               \
  }
  if (dtype == kF16) {
    PKV_DECODE_FP8(_Float16)
  } else {
    PKV_DECODE_FP8(__hip_bfloat16)
  }
#undef PKV_DECODE_FP8
#undef PKV_DECODE_FP8_P
#undef PKV_DECODE_FP8_W
  return (int)hipGetLastError();
}
