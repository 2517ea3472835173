// Attention of up to 16 query rows of one key-value head by one wave, for the paged decode attention (paged.hip)
// and the prompt attention (prompt.hip).
//
//   S = K . Q^T (MFMA 16x16x32),  P = exp2(scale S - m),  O^T += V^T . P^T (MFMA 16x16x32)
//
// over tiles of 32 positions, with the running maximum m and sum l of a softmax.  Both products have the query row as
// their column, so m, l, P and O of a row live in the same lanes (l & 15) and nothing crosses lanes between the products:
//   * a lane's eight scores of a tile (two S tiles of four rows) are made those of positions 8 j .. 8 j + 7 (j = l >> 4) by
//     loading position 8 (m >> 2) + 4 t + (m & 3) as row m of S tile t; that is the second product's operand order;
//   * lane (i = l & 15, j) loads values D/16 i .. of the V rows 8 j .. 8 j + 7, whole rows by 16 lanes, and transposes
//     them in registers: operand c holds value D/16 i + c of the eight rows.
// K and V go from memory to registers and no LDS is used.
#pragma once
#include "wave_scan.h"

namespace {

typedef __bf16 abf8_t __attribute__((ext_vector_type(8)));
typedef __bf16 abf2_t __attribute__((ext_vector_type(2)));
typedef short as2_t __attribute__((ext_vector_type(2)));
typedef _Float16 ah2_t __attribute__((ext_vector_type(2)));
typedef unsigned short au2_t __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;
// The maximum that scores are taken against may lag behind by this much (in powers of two): weights up to 2^8 cost no
// precision in fp32 or bf16 and stay inside fp16, and the outputs are rescaled a few times per row instead of per tile.
constexpr float kMaxLag = 8.0f;

template <int DT>
__device__ __forceinline__ f4_t attn_mfma16(uint4 a, uint4 b, f4_t c) {
  if constexpr (DT == MP_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(abf8_t, a), __builtin_bit_cast(abf8_t, b), c, 0, 0,
                                                   0);
}

template <int DT>
__device__ __forceinline__ uint32_t attn_pack2(float a, float b) {
  if constexpr (DT == MP_F16) {
    const ah2_t v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    const abf2_t v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
  }
}

// sum + the two packed values: weights are summed as they are rounded for the second product, so that the rounding of a weight
// that dominates cancels in the quotient.
template <int DT>
__device__ __forceinline__ float attn_add2(uint32_t w, float sum) {
  if constexpr (DT == MP_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(ah2_t, w), ah2_t{1, 1}, sum, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(as2_t, w), as2_t{0x3F80, 0x3F80}, sum, false);
}

// What the packed values w leave of a and b, packed.
template <int DT>
__device__ __forceinline__ uint32_t attn_rest2(uint32_t w, float a, float b) {
  if constexpr (DT == MP_F16) {
    const ah2_t v = __builtin_bit_cast(ah2_t, w);
    return attn_pack2<DT>(a - static_cast<float>(v.x), b - static_cast<float>(v.y));
  } else {
    return attn_pack2<DT>(a - __uint_as_float(w << 16), b - __uint_as_float(w & 0xFFFF0000u));
  }
}

// The lowest fp16 magnitudes lose bits; weights are raised by 2^7 there, so that with the lag they end below 2^15 and keep
// their eleven bits down to 2^-21 of the largest.  The sum is raised alike.
template <int DT>
constexpr float kRaise = DT == MP_F16 ? 7.0f : 0.0f;

// 16-bit value not finite
template <int DT>
__device__ __forceinline__ bool attn_odd16(uint32_t v) {
  constexpr uint32_t e = DT == MP_F16 ? 0x7C00u : 0x7F80u;
  return (v & e) == e;
}

// Where the keys and values of a sequence lie, of one key-value head.  Strides in elements.
template <bool PAGED>
struct KvSource;

template <>
struct KvSource<true> {
  const uint16_t *k, *v;          // pool + head offset
  int64_t kpage, krow, vpage, vrow;
  const int32_t *table;           // the sequence's pages
  int shift, mask, pages, last;   // page size as a shift and a mask, pages in the pool, last entry that may be read

  // Page of position p (one past the end: the last page); ok: its number is one of the pool's.
  __device__ __forceinline__ int page(int p, bool &ok) const {
    const int id = table[min(p >> shift, last)];
    ok = id >= 0 && id < pages;
    return ok ? id : 0;
  }
  __device__ __forceinline__ const uint16_t *krow_at(int page, int p) const {
    return k + page * kpage + (p & mask) * krow;
  }
  __device__ __forceinline__ const uint16_t *vrow_at(int page, int p) const {
    return v + page * vpage + (p & mask) * vrow;
  }
};

template <>
struct KvSource<false> {
  const uint16_t *k, *v;  // the sequence's first row + head offset
  int64_t krow, vrow;
  int last;               // last position that may be read

  __device__ __forceinline__ int page(int, bool &ok) const {
    ok = true;
    return 0;
  }
  __device__ __forceinline__ const uint16_t *krow_at(int, int p) const { return k + min(p, last) * krow; }
  __device__ __forceinline__ const uint16_t *vrow_at(int, int p) const { return v + min(p, last) * vrow; }
};

template <int D>
struct KvTile {
  uint4 k[2][D / 32];
  uint32_t v[8][D / 32];
  bool ok;  // the page of this lane's eight positions exists
};

// Two 16-byte loads for D = 256, one for 128, an 8-byte one for 64.
template <int N>
__device__ __forceinline__ void attn_load_words(const uint16_t *p, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4 *>(p)[i];
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  }
}

// Pages of a tile's positions for this lane: those of its K rows and those of its V rows.
struct TilePages {
  int k, v;
  bool ok;
};
template <bool PAGED>
__device__ __forceinline__ TilePages attn_pages(const KvSource<PAGED> &src, int tile, int lane) {
  TilePages p;
  bool unused;
  p.k = src.page(tile + 8 * ((lane & 15) >> 2), unused);
  p.v = src.page(tile + 8 * (lane >> 4), p.ok);
  return p;
}

template <int D, bool PAGED>
__device__ __forceinline__ void attn_load_tile(const KvSource<PAGED> &src, const TilePages &pg, int tile, int lane,
                                               KvTile<D> &t) {
  const int i = lane & 15, j = lane >> 4;
  t.ok = pg.ok;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint16_t *row = src.krow_at(pg.k, tile + 8 * (i >> 2) + 4 * s + (i & 3)) + 8 * j;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) t.k[s][c] = *reinterpret_cast<const uint4 *>(row + 32 * c);
  }
#pragma unroll
  for (int r = 0; r < 8; ++r) attn_load_words(src.vrow_at(pg.v, tile + 8 * j + r) + (D / 16) * i, t.v[r]);
}

// State of 16 query rows in one wave: lane (l & 15) of the row, positions 8 j .. of every tile.
template <int D>
struct AttnRows {
  f4_t o[D / 16];  // o[c][r]: value D/16 (4 j + r) + c of the row, unnormalised
  float m, l;      // maximum (shared by a row's four lanes) and this lane's part of the sum, scores in powers of two
};

template <int D>
__device__ __forceinline__ void attn_clear(AttnRows<D> &a) {
#pragma unroll
  for (int c = 0; c < D / 16; ++c) a.o[c] = f4_t{0.f, 0.f, 0.f, 0.f};
  a.m = -INFINITY;
  a.l = 0.f;
}

// One tile into the rows' state.  `sees`: positions below it are visible to this lane's row; `end`: to any row of the wave;
// `full`: to all.  Rows that see nothing of the tile are left as they are, whatever its masked places hold: masked scores
// become -inf, V rows that no row sees are cleared, and a tile whose V has an infinity or NaN where only some rows see it
// is added position by position, to those rows alone (0 times an infinity is no zero).  CAUSAL: rows see different positions.
// Otherwise the second product takes the weights and then what their rounding leaves, so that they count with 16 (bf16) or 22
// bits.  That rest may be 0 or negative, which beside an infinity gives NaN: a tile whose V has one takes halves of the weights.
template <int D, int DT, bool CAUSAL>
__device__ __forceinline__ void attn_tile(AttnRows<D> &a, KvTile<D> &t, const uint4 (&q)[D / 32], int tile, int sees,
                                          int end, int full, float scale2, int lane) {
  const int j = lane >> 4, p0 = tile + 8 * j;
  f4_t s[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    s[h] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < D / 32; ++c) s[h] = attn_mfma16<DT>(t.k[h][c], q[c], s[h]);
  }
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3] * scale2;
  bool apart = false;
  if (tile + 32 > full || !__all(t.ok)) {
    const int to = t.ok ? sees : 0, any = t.ok ? end : 0;
    bool masked = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = p0 + i < to ? x[i] : -INFINITY;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        t.v[i][c] = p0 + i < any ? t.v[i][c] : 0u;
        if (CAUSAL) masked |= attn_odd16<DT>(t.v[i][c]) || attn_odd16<DT>(t.v[i][c] >> 16);
      }
    }
    if (CAUSAL) apart = tile + 32 > full && __any(masked);
  }
  float top = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
  if (__any(top > a.m + kMaxLag)) {  // also the first tile: -inf + lag
    float m = fmaxf(top, __shfl_xor(top, 16, 64));
    m = fmaxf(a.m, fmaxf(m, __shfl_xor(m, 32, 64)));
    const float f = a.m == m ? 1.0f : __builtin_amdgcn_exp2f(a.m - m);
    a.l *= f;
    a.m = m;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) a.o[c] *= f;
  }
  bool odd = false;  // an infinity or NaN in V
  if constexpr (!CAUSAL) {
    au2_t most = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        most = __builtin_elementwise_max(most, __builtin_bit_cast(au2_t, t.v[i][c] & 0x7FFF7FFFu));
    odd = __any(max(most.x, most.y) >= (DT == MP_F16 ? 0x7C00 : 0x7F80));
  }
  const float base = (a.m == -INFINITY ? 0.f : a.m - kRaise<DT>) + (odd ? 1.f : 0.f);
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(x[i] - base);
  // the weights in the values' type, for the matrix cores: off by up to 2^-11 (fp16) or 2^-8 (bf16) of themselves each
  uint4 w = make_uint4(attn_pack2<DT>(p[0], p[1]), attn_pack2<DT>(p[2], p[3]), attn_pack2<DT>(p[4], p[5]),
                       attn_pack2<DT>(p[6], p[7]));
  a.l = attn_add2<DT>(w.w, attn_add2<DT>(w.z, attn_add2<DT>(w.y, attn_add2<DT>(w.x, a.l))));
  const auto values = [&](int c) {
    const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
    return make_uint4(__builtin_amdgcn_perm(t.v[1][c / 2], t.v[0][c / 2], sel),
                      __builtin_amdgcn_perm(t.v[3][c / 2], t.v[2][c / 2], sel),
                      __builtin_amdgcn_perm(t.v[5][c / 2], t.v[4][c / 2], sel),
                      __builtin_amdgcn_perm(t.v[7][c / 2], t.v[6][c / 2], sel));
  };
  if constexpr (!CAUSAL) {
    uint4 rest = make_uint4(attn_rest2<DT>(w.x, p[0], p[1]), attn_rest2<DT>(w.y, p[2], p[3]), attn_rest2<DT>(w.z, p[4], p[5]),
                            attn_rest2<DT>(w.w, p[6], p[7]));
    if (odd) rest = w;
    a.l = attn_add2<DT>(rest.w, attn_add2<DT>(rest.z, attn_add2<DT>(rest.y, attn_add2<DT>(rest.x, a.l))));
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const uint4 vt = values(c);
      a.o[c] = attn_mfma16<DT>(vt, rest, attn_mfma16<DT>(vt, w, a.o[c]));
    }
    return;
  }
  if (!apart) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) a.o[c] = attn_mfma16<DT>(values(c), w, a.o[c]);
    return;
  }
  const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
  for (int pos = 0; pos < 32; ++pos) {  // one position at a time
    const bool mine = (pos >> 3) == j, row_sees = tile + pos < sees;
    uint4 one = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t half = (pos & 1) ? 0xFFFF0000u : 0x0000FFFFu;
      const uint32_t v = mine && ((pos & 7) >> 1) == i ? wd[i] & half : 0u;
      (i == 0 ? one.x : i == 1 ? one.y : i == 2 ? one.z : one.w) = v;
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      uint32_t vt[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = mine && (pos & 7) == 2 * i ? t.v[2 * i][c / 2] : 0u;
        const uint32_t hi = mine && (pos & 7) == 2 * i + 1 ? t.v[2 * i + 1][c / 2] : 0u;
        vt[i] = __builtin_amdgcn_perm(hi, lo, (c & 1) ? 0x07060302u : 0x05040100u);
      }
      const f4_t o = attn_mfma16<DT>(make_uint4(vt[0], vt[1], vt[2], vt[3]), one, f4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int r = 0; r < 4; ++r) a.o[c][r] += row_sees ? o[r] : 0.f;
    }
  }
}

// Tiles first, first + step, ... below `to` into the rows' state.  The next tile's rows and the table entries of the one
// after it are asked for before a tile is computed.
template <int D, int DT, bool CAUSAL, bool PAGED>
__device__ __forceinline__ void attn_walk(AttnRows<D> &a, const KvSource<PAGED> &src, const uint4 (&q)[D / 32], int first,
                                          int to, int step, int sees, int end, int full, float scale2, int lane) {
  if (first >= to) return;
  TilePages pg = attn_pages(src, first, lane);
  KvTile<D> cur;
  TilePages next = attn_pages(src, first + step, lane);
  attn_load_tile<D>(src, pg, first, lane, cur);
  for (int tile = first; tile < to; tile += step) {
    KvTile<D> ahead = cur;
    if (tile + step < to) {
      const TilePages after = attn_pages(src, tile + 2 * step, lane);
      attn_load_tile<D>(src, next, tile + step, lane, ahead);
      next = after;
    }
    attn_tile<D, DT, CAUSAL>(a, cur, q, tile, sees, end, full, scale2, lane);
    cur = ahead;
  }
}

// Sum of a row's weights over its four lanes, in the raise of the weights.
__device__ __forceinline__ float attn_row_sum(float l) {
  l += __shfl_xor(l, 16, 64);
  return l + __shfl_xor(l, 32, 64);
}

// ---- packed sequences
// Of the sequences' counts n(b), b < batch, in parts of `per`: which sequence the part `at` belongs to and which of its parts
// it is.  Called by whole waves with uniform arguments, each lane looks at one sequence.
template <class N>
__device__ __forceinline__ bool attn_find_part(N n, int batch, int per, int at, int &seq, int &part, int &count) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < batch; b0 += 64) {
    const int b = b0 + lane;
    const int parts = b < batch ? n(b, per) : 0;
    const int upto = static_cast<int>(wave_scan(static_cast<uint32_t>(parts)));
    const uint64_t past = __ballot(upto > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      seq = b0 + l;
      count = __builtin_amdgcn_readlane(parts, l);
      part = at - (__builtin_amdgcn_readlane(upto, l) - count);
      return true;
    }
    at -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

}  // namespace
