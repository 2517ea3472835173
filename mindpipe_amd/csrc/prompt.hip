// Causal attention of packed new tokens: whole prompts (keys and values packed alike) or chunks of new tokens behind what
// a paged cache holds of their sequences.
//
// The queries of the heads that share a key-value head are rows of one problem: row = token * group + head, and a row sees
// the positions up to its token's.  A workgroup takes kRows consecutive rows of a sequence and a key-value head, 32 to
// each wave, and walks over the positions in tiles:
//
//   S = K . Q^T,  P = exp2(scale S - m),  O^T += V^T . P^T   (MFMA 32x32x16)
//
// Both products have the query row as their column, so a row's maximum m, sum l, weights and outputs stay in its two lanes
// (l & 31) and the weights go from the first product's accumulators to the second's operand without crossing lanes.
// K and V tiles come by direct-to-LDS loads, a tile ahead; V is read transposed (ds_read_b64_tr_b16).  Rows of LDS are
// swizzled in 16-byte chunks so that neither reads a bank twice at a time.
//
// Bound by the matrix cores and the vector units in turn: three sequences of 1933 to 4096 tokens, 64 / 8 heads of 128 in bf16
// (420 GFLOP that are seen), 448 to 480 us by the card, 0.9 PFLOP/s, where a large matrix product reaches 1.37.  Matrix
// instructions are 47% of the time, the softmax's another 55%; the two waves of a SIMD cover part of it.  32 rows a wave, so
// that an operand from LDS serves 32 x 32 x 16 products (with 16, straight from memory, 2374 us).  Eight waves in two groups
// that take turns: 716 us; the next tile's scores ahead of a tile's weights in one wave, or wave priorities: no faster.
//
// Few rows leave most CUs without a workgroup: then the positions are split over `splits` workgroups, which leave their sums,
// maxima and outputs, unnormalised, in the workspace, and a second launch joins them.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "attn_common.h"

namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves;
constexpr int kTile = 64;  // positions

typedef short as4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) as4_t *lds_as4;

// Through buffer descriptors and integers, in non-template functions: the compiler makes LDS reads wait for the LDS loads that it
// recognises as such.  Offsets are below 2^31 (the launch sees to it) and rows inside the tensors.
__device__ __forceinline__ void prompt_lds_load16(const uint16_t *base, uint32_t offset, int8_t *lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      mp_rsrc(base, 0x80000000u), reinterpret_cast<__attribute__((address_space(3))) void *>(reinterpret_cast<uintptr_t>(lds)),
      16, offset, 0, 0, 0);
}
// The wave's loads have landed, and every wave is so far.
__device__ __forceinline__ void prompt_wait() { asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory"); }
// Four rows' values of one column: lane i of 16 gives 8 bytes of row i / 4 and gets column i of the four rows.
__device__ __forceinline__ as4_t prompt_read_tr(const __restrict__ lds_as4 p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }
__device__ __forceinline__ uint2 prompt_read_tr(const int8_t *lds) {
  return __builtin_bit_cast(uint2, prompt_read_tr((lds_as4) reinterpret_cast<uintptr_t>(lds)));
}

template <int DT>
__device__ __forceinline__ f16_t prompt_mfma(uint4 a, uint4 b, f16_t c) {
  if constexpr (DT == MP_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf8_t, a), __builtin_bit_cast(abf8_t, b), c, 0, 0,
                                                   0);
}

template <int D>
struct PromptTile {
  static constexpr int kChunks = D / 8;         // of 16 bytes in a row
  static constexpr int kBytes = kTile * D * 2;  // of K or of V
  static constexpr int kStage = 2 * kBytes;     // of both; two stages, 32 / 64 / 128 KB
  static constexpr int kLoads = kBytes / 1024 / kWaves;
  // LDS chunk of a row's chunk c (and back).  K is read by 16 rows at a time in one column of chunks, V by four rows at a time
  // in four columns; 256 bytes are all banks.
  static __device__ __forceinline__ int k_chunk(int row, int c) { return c ^ (D == 64 ? (row >> 1) & 7 : row & 15); }
  static __device__ __forceinline__ int v_chunk(int row, int c) {
    return c ^ (D == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3));
  }
};

struct PackedPlan {
  const int32_t *starts;
  int batch, rows, grp;
  // offsets of a sequence; sequence `batch` is what lies behind the last one, and batch + 1 what lies before the first
  __device__ __forceinline__ int first(int b) const { return b > batch ? 0 : min(max(starts[b], 0), rows); }
  __device__ __forceinline__ int end(int b) const { return b < batch ? max(first(b), first(b + 1)) : b == batch ? rows : first(0); }
  __device__ __forceinline__ int operator()(int b, int per) const {
    return static_cast<int>((static_cast<int64_t>(end(b) - first(b)) * grp + per - 1) / per);
  }
};

// Rows r0 .. r0 + 15 of a sequence and key-value head by the wave alone, K and V straight from memory.  A function of its own:
// inlined, its registers would be the kernel's.
template <bool PAGED>
struct PromptRows {
  KvSource<PAGED> src;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_row, q_head, out_row;
  int all, grp, before, room;  // rows, heads of a token, positions up to row 0's own, positions there are
  int from, to;                // positions that are looked at
  float scale2;
  float *part;           // [tokens, heads][dim + 2], row stride part_row; null: outputs are final
  int64_t part_row;
};
template <int D, int DT, bool PAGED>
__device__ __attribute__((noinline)) void prompt_rows16(const PromptRows<PAGED> &p, int r0) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, j = lane >> 4, at = min(r0 + i16, p.all - 1);
  const int token = at / p.grp, head = at - token * p.grp;
  const auto seen = [&](int r) { return max(min(p.before + min(r, p.all - 1) / p.grp, p.room), 0); };
  const int full = __builtin_amdgcn_readfirstlane(seen(r0)), end = __builtin_amdgcn_readfirstlane(seen(r0 + 15));
  uint4 qf[D / 32];
  const uint16_t *qp = p.q + token * p.q_row + head * p.q_head + 8 * j;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) qf[c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);
  AttnRows<D> a;
  attn_clear(a);
  attn_walk<D, DT, true>(a, p.src, qf, p.from, min(end, p.to), 32, seen(at), end, full, p.scale2, lane);
  const float l = attn_row_sum(a.l);
  if (r0 + i16 >= p.all) return;
  if (p.part) {
    float *z = p.part + token * p.part_row + head * (D + 2);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < D / 16; ++c) z[(D / 16) * (4 * j + r) + c] = a.o[c][r];
    if (j == 0) {
      z[D] = a.m;
      z[D + 1] = l;
    }
    return;
  }
  uint16_t *y = p.out + token * p.out_row + head * D + (D / 16) * 4 * j;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < D / 16; c += 2) {
      const float lo = l == 0.f ? 0.f : a.o[c][r] / l, hi = l == 0.f ? 0.f : a.o[c + 1][r] / l;
      *reinterpret_cast<uint32_t *>(y + (D / 16) * r + c) = attn_pack2<DT>(lo, hi);
    }
}

template <int D, int DT, bool PAGED>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void prompt_attention_kernel(
    const uint16_t *__restrict__ q, int64_t q_row, int64_t q_head, const uint16_t *__restrict__ k, int64_t kpage,
    int64_t khead, int64_t krow, const uint16_t *__restrict__ v, int64_t vpage, int64_t vhead, int64_t vrow, int pages,
    int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens,
    const int32_t *__restrict__ starts, int batch, int rows, int kvh, int grp, int tiles, float scale2,
    uint32_t flip, int splits, float *__restrict__ parts, uint16_t *__restrict__ out) {
  using T = PromptTile<D>;
  constexpr int kStage = T::kStage, kS = kTile / 32;
  extern __shared__ __attribute__((aligned(1024))) int8_t prompt_smem[];  // two stages of K and V
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i32 = lane & 31, h = lane >> 5;
  const int kh = blockIdx.x % kvh, unit = blockIdx.x / kvh, sp = unit % splits;
  const PackedPlan plan{starts, batch, rows, grp};
  int b, part, count;
  if (!attn_find_part(plan, batch + 2, kRows, tiles - 1 - unit / splits, b, part, count)) return;
  const int first = plan.first(b), n = plan.end(b) - first, all = n * grp;
  // positions of the sequence, the new tokens' included, and those that there is room for; none outside of the sequences.  A
  // row's own position goes by the length, as the append's does: a sequence longer than its table keeps the places of its rows.
  int len = 0, room = 0;
  if (b < batch) {
    len = PAGED ? max(lens[b], 0) : n;
    room = PAGED ? width << shift : n;
  }
  // positions seen by row r of the sequence, and by none of a wave's or workgroup's rows past their last
  const int before = len - n + 1;
  const auto seen = [&](int r) { return max(min(before + min(r, all - 1) / grp, room), 0); };
  const int r0 = part * kRows + wave * 32, at = r0 + i32;
  const bool row = at < all;
  const int token = row ? at / grp : 0, head = kh * grp + (row ? at - token * grp : 0);
  const int sees = row ? seen(at) : 0;
  // this workgroup's positions: `from` up to `end`, of them this wave's up to `wend`
  const int reach = seen(part * kRows + kRows - 1), share = (reach + kTile * splits - 1) / (kTile * splits) * kTile;
  const int from = __builtin_amdgcn_readfirstlane(min(sp * share, reach)), end = __builtin_amdgcn_readfirstlane(min(from + share, reach));
  const int full = r0 < all ? __builtin_amdgcn_readfirstlane(seen(r0)) : 0;
  const int wend = r0 < all ? min(__builtin_amdgcn_readfirstlane(seen(r0 + 31)), end) : 0;

  uint4 qf[D / 16];
  const uint16_t *qp = q + (first + token) * q_row + head * q_head + 8 * h;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const uint4 x = *reinterpret_cast<const uint4 *>(qp + 16 * c);
    qf[c] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
  }

  const uint16_t *kb = k + kh * khead + (PAGED ? 0 : first * krow), *vb = v + kh * vhead + (PAGED ? 0 : first * vrow);
  const int32_t *pg = PAGED ? table + static_cast<int64_t>(min(b, batch - 1)) * width : nullptr;
  // page of the tile's position `lane` (positions past the end: the last one's)
  const auto entry = [&](int tile) { return PAGED ? pg[min(tile + lane, end - 1) >> shift] : 0; };
  // Over pages, byte offsets of this lane's pieces in a whole tile are kept, from its first row or that of its page: they are
  // the same for all tiles, which start at multiples of kTile.  (1737 rows of 32 heads behind contexts 160 -> 151 us.  Packed
  // rows, whose offsets take less to work out, lose by the registers, 466 -> 472 us at 64 / 8 heads, and so do heads of 256,
  // 92 -> 102 us.)
  constexpr bool kKept = PAGED && D < 256;
  const int mask = PAGED ? (1 << shift) - 1 : 0;
  uint32_t koff[kKept ? T::kLoads : 1], voff[kKept ? T::kLoads : 1];
  if constexpr (kKept) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const int r = (wave * T::kLoads + i) * 64 / T::kChunks + lane / T::kChunks, c = lane % T::kChunks;
      koff[i] = 2 * ((r & mask) * static_cast<uint32_t>(krow) + 8 * T::k_chunk(r, c));
      voff[i] = 2 * ((r & mask) * static_cast<uint32_t>(vrow) + 8 * T::v_chunk(r, c));
    }
  }
  const auto load = [&](int tile, int id, int8_t *stage) {
    const bool whole = kKept && tile + kTile <= end;
    tile = min(tile, end - 1);  // past the last tile: rows that nothing reads
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const int slot = (wave * T::kLoads + i) * 64;
      // the rows of one load lie in one page
      const int64_t pid = PAGED ? __builtin_amdgcn_readlane(id, slot / T::kChunks) : 0;
      if (whole) {
        const int64_t at = tile & mask;
        prompt_lds_load16(kb + pid * kpage + at * krow, koff[kKept ? i : 0], stage + slot * 16);
        prompt_lds_load16(vb + pid * vpage + at * vrow, voff[kKept ? i : 0], stage + T::kBytes + slot * 16);
      } else {
        const int r = slot / T::kChunks + lane / T::kChunks, c = lane % T::kChunks, p = min(tile + r, end - 1);
        const uint32_t off = PAGED ? p & mask : p - tile;
        prompt_lds_load16(kb + (PAGED ? pid * kpage : tile * krow), 2 * (off * static_cast<uint32_t>(krow) + 8 * T::k_chunk(r, c)),
                          stage + slot * 16);
        prompt_lds_load16(vb + (PAGED ? pid * vpage : tile * vrow), 2 * (off * static_cast<uint32_t>(vrow) + 8 * T::v_chunk(r, c)),
                          stage + T::kBytes + slot * 16);
      }
    }
  };

  f16_t o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, l = 0.f;

  const auto fix = [&](int id, uint64_t &there) {  // page numbers outside the pool: page 0, unseen
    there = ~uint64_t(0);
    if constexpr (!PAGED) return 0;
    const bool ok = id >= 0 && id < pages;
    there = __ballot(ok);
    return ok ? id : 0;
  };
  uint64_t there = 0;  // which positions of the tile that is on its way exist
  int next_entry = 0, stage = 0;
  if (end > from) {
    load(from, fix(entry(from), there), prompt_smem);
    next_entry = entry(from + kTile);
  }
  uint32_t odd = 0;  // an infinity or NaN in V where only some of the wave's rows see it
  for (int tile = from; tile < end; tile += kTile) {
    // this tile's loads have landed, every wave's, and the stage of the last tile has been read
    prompt_wait();
    const uint64_t ok = there;
    load(tile + kTile, fix(next_entry, there), prompt_smem + (kStage - stage));
    next_entry = entry(tile + 2 * kTile);
    const int8_t *ks = prompt_smem + stage, *vs = ks + T::kBytes;
    stage = kStage - stage;
    if (tile >= wend) continue;  // rows that see nothing more load for the others
    f16_t s[kS];
#pragma unroll
    for (int t = 0; t < kS; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
    {
      constexpr int kC = D / 16, kAheadK = 1;  // pairs of operands that are read before they are used
      i4_t kf[kAheadK + 1][kS];
      const auto keys = [&](int c) {
#pragma unroll
        for (int t = 0; t < kS; ++t) {
          const int r = 32 * t + i32;
          kf[c % (kAheadK + 1)][t] = *reinterpret_cast<const i4_t *>(ks + r * (D * 2) + 16 * T::k_chunk(r, 2 * c + h));
        }
      };
#pragma unroll
      for (int c = 0; c < kAheadK; ++c) keys(c);
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        if (c + kAheadK < kC) keys(c + kAheadK);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < kS; ++t) s[t] = prompt_mfma<DT>(__builtin_bit_cast(uint4, kf[c % (kAheadK + 1)][t]), qf[c], s[t]);
      }
    }
    // s[t][r]: position 32 t + 8 (r >> 2) + 4 h + (r & 3) of the tile
    if (tile + kTile > full || ok != ~uint64_t(0)) {
      const uint64_t vis = ok >> (4 * h);
#pragma unroll
      for (int t = 0; t < kS; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int p = 32 * t + 8 * (r >> 2) + (r & 3);
          s[t][r] = tile + p + 4 * h < sees && ((vis >> p) & 1) ? s[t][r] : -INFINITY;
        }
      for (int e = lane; e < T::kBytes / 16; e += 64) {
        const i4_t x = *reinterpret_cast<const i4_t *>(vs + 16 * e);
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= attn_odd16<DT>(x[i]) || attn_odd16<DT>(static_cast<uint32_t>(x[i]) >> 16);
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < kS; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
    top *= scale2;
    if (__any(top > m + kMaxLag)) {
      const float new_m = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
      const float f = m == new_m ? 1.0f : __builtin_amdgcn_exp2f(m - new_m);
      l *= f;
      m = new_m;
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m - kRaise<DT>;
    // O^T: step c of 16 positions, whose weights are those of positions 16 c + 4 h + {0..3, 8..11}: s[c / 2][8 (c & 1) ..].  The
    // next step's weights are made between the matrix instructions of this one.
    constexpr int kSteps = kTile / 16, kD = D / 32;
    const int trow = 4 * h + ((lane & 15) >> 2), tcol = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    uint32_t w[2][4];
    constexpr int kAheadV = 2;  // operands of V that are read before they are used (1: 461 -> 470 us, 4: 463, heads of 256 92 -> 101 and 94)
    uint4 vf[kAheadV + 1];
    // Weights are rounded to the values' type, off by up to 2^-11 (fp16) or 2^-8 (bf16) of themselves each, and their sum takes
    // them as rounded: errors (rms) are 1.2 (fp16) to 1.3 times (bf16; heads of 256 1.4) those of 32-bit weights, 2.1e-3 for
    // 1.6e-3 of the packed prompts' outputs.  A second product with what the rounding leaves would take that away for 471 -> 611 us
    // there, 153 -> 209 for chunks of 32 heads and 91 -> 107 for heads of 256.
    const auto weight = [&](int c, int i) {
      const int r = 8 * (c & 1) + 2 * i;
      w[c & 1][i] = attn_pack2<DT>(__builtin_amdgcn_exp2f(fmaf(s[c / 2][r], scale2, -base)),
                                   __builtin_amdgcn_exp2f(fmaf(s[c / 2][r + 1], scale2, -base)));
      l = attn_add2<DT>(w[c & 1][i], l);
    };
    const auto values = [&](int j) {
      const int c = j / kD, d = j % kD;
      const int ra = 16 * c + trow, rb = ra + 8;
      const uint2 lo = prompt_read_tr(vs + ra * (D * 2) + 16 * T::v_chunk(ra, 4 * d + tcol) + 8 * (lane & 1));
      const uint2 hi = prompt_read_tr(vs + rb * (D * 2) + 16 * T::v_chunk(rb, 4 * d + tcol) + 8 * (lane & 1));
      vf[j % (kAheadV + 1)] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
#pragma unroll
    for (int j = 0; j < kAheadV; ++j) values(j);
#pragma unroll
    for (int i = 0; i < 4; ++i) weight(0, i);
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      const uint4 wf = make_uint4(w[c & 1][0], w[c & 1][1], w[c & 1][2], w[c & 1][3]);
#pragma unroll
      for (int d = 0; d < kD; ++d) {
        __builtin_amdgcn_sched_barrier(0);
        const int j = c * kD + d;
        o[d] = prompt_mfma<DT>(vf[j % (kAheadV + 1)], wf, o[d]);
        if (j + kAheadV < kSteps * kD) values(j + kAheadV);
        if (c + 1 < kSteps) {
#pragma unroll
          for (int i = 4 * d / kD; i < 4 * (d + 1) / kD; ++i) weight(c + 1, i);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing on its way to LDS when the workgroup ends
  if (__any(odd)) {
    // 0 times an infinity is no zero: these rows once more, with what they do not see left out one position at a time
    PromptRows<PAGED> p;
    if constexpr (PAGED) p.src = {kb, vb, kpage, krow, vpage, vrow, pg, shift, (1 << shift) - 1, pages, (end - 1) >> shift};
    else p.src = {kb, vb, krow, vrow, n - 1};
    p.q = q + first * q_row + kh * grp * q_head;
    p.q_row = q_row;
    p.q_head = q_head;
    p.out_row = static_cast<int64_t>(kvh) * grp * D;
    p.out = out + first * p.out_row + kh * grp * D;
    p.all = all;
    p.grp = grp;
    p.before = before;
    p.room = room;
    p.from = from;
    p.to = end;
    p.scale2 = flip ? -scale2 : scale2;
    p.part_row = static_cast<int64_t>(kvh) * grp * (D + 2);
    p.part = splits > 1 ? parts + sp * rows * p.part_row + first * p.part_row + kh * grp * (D + 2) : nullptr;
    for (int half = 0; half < 2; ++half)
      if (r0 + 16 * half < all) prompt_rows16<D, DT, PAGED>(p, r0 + 16 * half);
    return;
  }
  if (!row) return;
  l += __shfl_xor(l, 32, 64);
  if (splits > 1) {
    float *z = parts + ((static_cast<int64_t>(sp) * rows + first + token) * kvh * grp + head) * (D + 2);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 2) *reinterpret_cast<float2 *>(z + 32 * d + 8 * (r >> 2) + 4 * h + (r & 3)) = make_float2(o[d][r], o[d][r + 1]);
    if (h == 0) *reinterpret_cast<float2 *>(z + D) = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t *y = out + (static_cast<int64_t>(first + token) * kvh * grp + head) * D + 4 * h;
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = l == 0.f ? 0.f : o[d][r + i] * inv;
      *reinterpret_cast<uint2 *>(y + 32 * d + 2 * r) = make_uint2(attn_pack2<DT>(x[0], x[1]), attn_pack2<DT>(x[2], x[3]));
    }
}

// The splits of a row meet, one wave each.
template <int D, int DT>
__global__ __launch_bounds__(256) void prompt_join_kernel(const float *__restrict__ parts, int splits, int64_t rows,
                                                          uint16_t *__restrict__ out) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  const float *z = parts + row * (D + 2);
  const int64_t step = rows * (D + 2);
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 64) m = fmaxf(m, z[s * step + D]);
  m = mp_wave_max(m);
  float o[D / 64], l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float ms = z[s * step + D], f = ms == m ? 1.0f : __builtin_amdgcn_exp2f(ms - m);
    l += f * z[s * step + D + 1];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] += f * z[s * step + 64 * i + lane];
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const float v = l == 0.f ? 0.f : o[i] * inv;
    out[row * D + 64 * i + lane] = DT == MP_F16 ? mp_f2h(v) : mp_f2bf(v);
  }
}

// Row tiles of all sequences, at most: a part of one for each, and for the rows before the first and behind the last.
inline int64_t prompt_tiles(int64_t rows, int64_t grp, int64_t batch) { return rows * grp / kRows + batch + 2; }

// Splits of the positions (at most `reach`): so many that the workgroups come nearest to what the CUs hold at once (two each;
// one of heads of 256), with four tiles of positions each at least.  Workgroups are counted by the bound that the grid goes by.
// 16 rows behind 32768 positions (32 / 8 heads of 128): 666 us whole, 341 / 176 / 95 us in 2 / 4 / 8 splits, 40 us in the 32 that
// this gives; 1068 rows of 16 / 4 heads of 256 (148 workgroups, 136 with rows): 117 us whole, 91 in 2, 93 in 3; 1737 rows of 32
// heads of 128 (640 workgroups, 480 with rows): 149 whole, 168 in 2, the join reads and writes more than idle CUs cost.
inline int prompt_splits(int64_t rows, int64_t nh, int64_t kvh, int64_t dim, int64_t batch, int64_t reach) {
  const int64_t slots = (dim == 256 ? 1 : 2) * mp_cu_count(), blocks = prompt_tiles(rows, nh / kvh, batch) * kvh;
  const int64_t s = (slots + blocks / 2) / blocks, most = reach / 256;
  return static_cast<int>(s < 2 || most < 2 ? 1 : s < most ? s : most);
}

struct PromptCall {
  const void *q;
  int64_t q_row, q_head;
  const void *k, *v;
  int64_t kpage, khead, krow, vpage, vhead, vrow;
  int pages, shift, width;
  const int32_t *table, *lens, *starts;
  int64_t batch, rows;
  int nh, kvh, head_dim;
  float scale;
  void *out;
  int dtype;
  void *workspace;
  size_t workspace_bytes;
  hipStream_t stream;
};

template <bool PAGED>
int prompt_launch(const PromptCall &c) {
  if (c.dtype != MP_F16 && c.dtype != MP_BF16) return MP_ERR_DTYPE;
  if (!std::isfinite(c.scale * kLog2e)) return MP_ERR_ARG;
  if (c.rows < 0 || c.rows > INT32_MAX || c.batch < 1 || c.batch > INT32_MAX - 64) return MP_ERR_SHAPE;
  if (c.nh < 1 || c.kvh < 1 || c.nh > 65536 || c.nh % c.kvh) return MP_ERR_SHAPE;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return MP_ERR_SHAPE;
  for (int64_t s : {c.q_row, c.q_head, c.kpage, c.khead, c.krow, c.vpage, c.vhead, c.vrow})
    if (s < 0 || s % 8) return MP_ERR_SHAPE;
  for (const void *p : {c.q, c.k, c.v, static_cast<const void *>(c.out)})
    if (!mp_aligned(p, 16)) return MP_ERR_ALIGN;
  // byte offsets inside a page, or a tile, are 32 bits
  const int64_t span = PAGED ? int64_t(1) << c.shift : 64, reach = (int64_t(1) << 30) - 256;
  if (c.krow > reach / span || c.vrow > reach / span) return MP_ERR_SHAPE;
  if (c.rows == 0) return MP_OK;
  const int64_t grp = c.nh / c.kvh;
  const int64_t tiles = prompt_tiles(c.rows, grp, c.batch);
  if (c.rows * c.nh > INT32_MAX - kRows || tiles * c.kvh > INT32_MAX) return MP_ERR_SHAPE;
  if (mp_cu_count() <= 0) return MP_ERR_HIP;
  const int splits = prompt_splits(c.rows, c.nh, c.kvh, c.head_dim, c.batch, PAGED ? static_cast<int64_t>(c.width) << c.shift : c.rows);
  const int64_t blocks = tiles * c.kvh * splits;
  if (splits > 1) {
    if (!c.workspace) return MP_ERR_ARG;
    if (!mp_aligned(c.workspace, 16)) return MP_ERR_ALIGN;
    if (c.workspace_bytes < splits * c.rows * c.nh * (c.head_dim + 2) * sizeof(float)) return MP_ERR_WORKSPACE;
  }
  float *parts = static_cast<float *>(c.workspace);
  // the sign of the scale goes to the queries, so that the largest product gives the largest score; a scale of 0 becomes the
  // smallest normal number, which leaves every finite score 0 and a masked one -inf
  const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;
  const float scale2 = fmaxf(fabsf(c.scale) * kLog2e, FLT_MIN);
#define MP_PROMPT(D, DT)                                                                                                  \
  if (2 * PromptTile<D>::kStage > 64 * 1024 &&                                                                            \
      hipFuncSetAttribute(reinterpret_cast<const void *>(prompt_attention_kernel<D, DT, PAGED>),                          \
                          hipFuncAttributeMaxDynamicSharedMemorySize,                                                     \
                          2 * PromptTile<D>::kStage) != hipSuccess)                                                       \
    return MP_ERR_HIP;                                                                                                    \
  hipLaunchKernelGGL((prompt_attention_kernel<D, DT, PAGED>), dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves),     \
                     2 * PromptTile<D>::kStage, c.stream,                                                                 \
                     static_cast<const uint16_t *>(c.q), c.q_row, c.q_head, static_cast<const uint16_t *>(c.k), c.kpage,  \
                     c.khead, c.krow, static_cast<const uint16_t *>(c.v), c.vpage, c.vhead, c.vrow, c.pages, c.shift,     \
                     c.table, c.width, c.lens, c.starts, static_cast<int>(c.batch), static_cast<int>(c.rows), c.kvh,      \
                     static_cast<int>(grp), static_cast<int>(tiles), scale2, flip, splits, parts,                         \
                     static_cast<uint16_t *>(c.out));                                                                    \
  if (splits > 1) {                                                                                                       \
    MP_CHECK_LAUNCH();                                                                                                    \
    hipLaunchKernelGGL((prompt_join_kernel<D, DT>), dim3(static_cast<unsigned>(mp_cdiv(c.rows * c.nh, 4))), dim3(256), 0, \
                       c.stream, parts, splits, c.rows * c.nh, static_cast<uint16_t *>(c.out));                          \
  }
  if (c.dtype == MP_F16) {
    if (c.head_dim == 64) {
      MP_PROMPT(64, MP_F16)
    } else if (c.head_dim == 128) {
      MP_PROMPT(128, MP_F16)
    } else {
      MP_PROMPT(256, MP_F16)
    }
  } else {
    if (c.head_dim == 64) {
      MP_PROMPT(64, MP_BF16)
    } else if (c.head_dim == 128) {
      MP_PROMPT(128, MP_BF16)
    } else {
      MP_PROMPT(256, MP_BF16)
    }
  }
#undef MP_PROMPT
  MP_CHECK_LAUNCH();
  return MP_OK;
}

}  // namespace

extern "C" size_t mp_prompt_workspace_bytes(int64_t rows, int nh, int kvh, int head_dim, int64_t batch, int64_t reach) {
  if (rows <= 0 || rows > INT32_MAX || nh <= 0 || kvh <= 0 || nh % kvh || head_dim <= 0 || batch <= 0 || batch > INT32_MAX ||
      reach <= 0 || mp_cu_count() <= 0)
    return 0;
  const int splits = prompt_splits(rows, nh, kvh, head_dim, batch, reach);
  return splits > 1 ? static_cast<size_t>(splits) * rows * nh * (head_dim + 2) * sizeof(float) : 0;
}

extern "C" int mp_prompt_attention(const void *q, int64_t q_row, int64_t q_head, const void *k, int64_t k_row, int64_t k_head,
                                   const void *v, int64_t v_row, int64_t v_head, int64_t rows, int nh, int kvh, int head_dim,
                                   const int32_t *starts, int64_t batch, float scale, void *out, int dtype, void *workspace,
                                   size_t workspace_bytes, mp_stream_t stream) {
  if (!q || !k || !v || !starts || !out) return MP_ERR_ARG;
  return prompt_launch<false>({q, q_row, q_head, k, v, 0, k_head, k_row, 0, v_head, v_row, 0, 0, 0, nullptr, nullptr, starts,
                               batch, rows, nh, kvh, head_dim, scale, out, dtype, workspace, workspace_bytes,
                               reinterpret_cast<hipStream_t>(stream)});
}

extern "C" int mp_paged_prompt_attention(const void *q, int64_t q_row, int64_t q_head, int64_t rows, int nh, int kvh,
                                         int head_dim, const mp_pages *cache, const int32_t *lens, const int32_t *starts,
                                         int64_t batch, float scale, void *out, int dtype, void *workspace,
                                         size_t workspace_bytes, mp_stream_t stream) {
  if (!q || !cache || !cache->k || !cache->v || !cache->table || !lens || !starts || !out) return MP_ERR_ARG;
  int shift = -1;
  for (int s = 3; s < 16; ++s)
    if (cache->page_size == 1 << s) shift = s;
  if (shift < 0 || cache->pages < 1 || cache->pages > INT32_MAX || cache->width < 1 || cache->width > (1 << 30) >> shift)
    return MP_ERR_SHAPE;
  return prompt_launch<true>({q, q_row, q_head, cache->k, cache->v, cache->k_page, cache->k_head, cache->k_row, cache->v_page,
                              cache->v_head, cache->v_row, static_cast<int>(cache->pages), shift,
                              static_cast<int>(cache->width), cache->table, lens, starts, batch, rows, nh, kvh, head_dim,
                              scale, out, dtype, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream)});
}
