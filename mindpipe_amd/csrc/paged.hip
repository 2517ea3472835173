// A paged key-value cache: appending rotated keys and values, and attention of one new token per sequence.
//
// A layer's cache is two pools of pages, each page holding `page` positions of every key-value head (strides are free, the
// values of a position are contiguous).  A sequence's pages are listed in its row of a table; its positions are counted
// from zero, and everything goes by device memory (lengths, starts, table), so a step keeps its launches while the
// sequences grow and can be captured into a graph.  A page number outside the pool is an empty page: nothing is
// written to it, and its positions are not attended.
#include <climits>
#include <cmath>

#include "attn_common.h"

namespace {

// ---------------------------------------------------------------- rotation and append
// The sequence of packed row t (starts: batch + 1 ascending offsets), or -1 behind the last one.  Whole waves, t uniform.
__device__ __forceinline__ int seq_of_row(const int32_t *starts, int batch, int t, int &end) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 <= batch; b0 += 64) {
    const bool upto = b0 + lane <= batch && starts[min(b0 + lane, batch)] <= t;
    n += __popcll(__ballot(upto));
  }
  if (n < 1 || n > batch) return -1;
  end = starts[n];
  return n - 1;
}

template <int DT>
__device__ __forceinline__ float at16(uint32_t w, int half) {
  const uint16_t b = static_cast<uint16_t>(half ? w >> 16 : w);
  return DT == MP_F16 ? mp_h2f(b) : mp_bf2f(b);
}

// One workgroup per packed row and 256 of its 16-value pieces (a piece: eight pairs of a rotated head, or 16 values that
// are copied).  Pairs are (2 i, 2 i + 1), or (i, i + rotary / 2).  Rotated in fp32 and rounded once.
// Bound by its bytes: a row is read once and written once, the tables' rows come from the caches.  9219 rows of 64 / 8 heads of
// 128 in bf16, 382 MB: 70 us, 5.4 TB/s (a copy of 2 GiB: 4.9).  A row per workgroup keeps the look for its sequence uniform.
template <int DT, bool PAIRS>
__global__ __launch_bounds__(256) void paged_rope_append_kernel(
    const uint16_t *__restrict__ qkv, int64_t qkv_row, int nh, int kvh, int dim, const float *__restrict__ cos_t,
    const float *__restrict__ sin_t, int half, int64_t angles, uint16_t *__restrict__ q_out, uint16_t *__restrict__ k_pages,
    int64_t kpage, int64_t khead, int64_t krow, uint16_t *__restrict__ v_pages, int64_t vpage, int64_t vhead, int64_t vrow,
    int pages, int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens,
    const int32_t *__restrict__ starts, int batch) {
  const int t = blockIdx.x, per = dim / 16;
  int seq = t, end = t + 1;
  if (starts) seq = seq_of_row(starts, batch, t, end);
  const int piece = blockIdx.y * 256 + threadIdx.x, head = piece / per, at = piece % per * 16;
  if (head >= nh + 2 * kvh) return;
  const int64_t pos = seq < 0 ? -1 : static_cast<int64_t>(lens[seq]) - (end - t);
  const uint16_t *x = qkv + t * qkv_row + static_cast<int64_t>(head) * dim;
  // two 16-byte halves: consecutive ones, or those of a pair by halves
  const bool turn = head < nh + kvh && at < 2 * half;
  const int d0 = turn && !PAIRS ? at / 2 : at, d1 = turn && !PAIRS ? half + at / 2 : at + 8;
  uint4 lo = *reinterpret_cast<const uint4 *>(x + d0), hi = *reinterpret_cast<const uint4 *>(x + d1);
  const bool angle = pos >= 0 && pos < angles;
  if (turn && angle) {
    float c[8], s[8];
    const float4 *cp = reinterpret_cast<const float4 *>(cos_t + pos * half + at / 2);
    const float4 *sp = reinterpret_cast<const float4 *>(sin_t + pos * half + at / 2);
    const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
    s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (PAIRS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = at16<DT>(w[i], 0), b = at16<DT>(w[i], 1);
        w[i] = attn_pack2<DT>(a * c[i] - b * s[i], a * s[i] + b * c[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a0 = at16<DT>(w[i], 0), a1 = at16<DT>(w[i], 1), b0 = at16<DT>(w[4 + i], 0), b1 = at16<DT>(w[4 + i], 1);
        w[i] = attn_pack2<DT>(a0 * c[2 * i] - b0 * s[2 * i], a1 * c[2 * i + 1] - b1 * s[2 * i + 1]);
        w[4 + i] = attn_pack2<DT>(a0 * s[2 * i] + b0 * c[2 * i], a1 * s[2 * i + 1] + b1 * c[2 * i + 1]);
      }
    }
    lo = make_uint4(w[0], w[1], w[2], w[3]);
    hi = make_uint4(w[4], w[5], w[6], w[7]);
  }
  uint16_t *y;
  if (head < nh) {
    if (!angle) lo = hi = make_uint4(0, 0, 0, 0);  // a row of no sequence or without an angle
    y = q_out + (static_cast<int64_t>(t) * nh + head) * dim;
  } else {
    const int64_t entry = pos >> shift;
    if (!angle || entry >= width) return;
    const int page = table[static_cast<int64_t>(seq) * width + entry];
    if (page < 0 || page >= pages) return;
    const int64_t row = pos & ((1 << shift) - 1);
    y = head < nh + kvh ? k_pages + page * kpage + (head - nh) * khead + row * krow
                        : v_pages + page * vpage + (head - nh - kvh) * vhead + row * vrow;
  }
  *reinterpret_cast<uint4 *>(y + d0) = lo;
  *reinterpret_cast<uint4 *>(y + d1) = hi;
}

// ---------------------------------------------------------------- one new token per sequence
// The sequences' positions, in blocks of kBlock (an empty sequence has one, which writes its zeros), follow each other in one
// row of blocks for every key-value head, and the workgroups of a head (`share`, or one per block) take equal runs of it: run w
// is blocks w T / share .. (w + 1) T / share of T.  However ragged the lengths are, all have the same to read.  A sequence that lies
// in several runs is joined from its parts: a workgroup leaves at most two, that of the sequence its run begins inside of
// (slot 2 w) and that of the sequence its run ends inside of (slot 2 w + 1).
//
// The heads that share a key-value head are the columns of one matrix product, up to 16 in a wave, so K and V are read once for
// all of them:  S = K . Q^T,  P = exp2(scale S - m),  O^T += V^T . P^T  (MFMA 16x16x32; attn_tile).  The four waves take the 32
// positions of a block each, straight from memory to registers: nothing is read twice, so LDS would only delay it.  Bound by
// those reads: 64 sequences of up to 8192 positions, 64 / 8 heads of 128 in bf16 (945 MB), 171 us, 5.5 TB/s, and two of 131071
// (1.07 GB) 185 us, 5.8 TB/s, of the 6.4 TB/s that reads reach here; 200 short ones of 14 / 2 heads of 64 (75 MB), 21 us,
// where a workgroup's first loads wait for its look at the lengths, the table and a page in turn.  The matrix cores are 6% busy,
// with the weights' rest taken as well (4% without it, 1 us of 176 less).
constexpr int kWaves = 4;
constexpr int kBlock = 32 * kWaves;

struct DecodePlan {
  const int32_t *lens;
  int batch, capacity;  // capacity: positions that the table has room for
  __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), capacity); }
  __device__ __forceinline__ int operator()(int b, int) const { return max((len(b) + kBlock - 1) / kBlock, 1); }
  __device__ __forceinline__ uint32_t blocks() const {
    uint32_t n = 0;
    for (int b = threadIdx.x & 63; b < batch; b += 64) n += (*this)(b, 0);
    return wave_sum(n);
  }
};

// Workgroups of a head: as many as fit the card at once (decode_round of D per CU: their registers hold two tiles each), and not
// more.  64 sequences as above: each sequence cut into parts of its own 188 us, equal runs 176, joins included.
constexpr int decode_round(int dim) { return dim == 64 ? 4 : dim == 128 ? 2 : 1; }
inline int decode_share(int64_t heads, int dim) {
  const int64_t n = static_cast<int64_t>(decode_round(dim)) * mp_cu_count() / heads;
  return static_cast<int>(n > 1 ? n : 1);
}

template <int D, int DT>
__global__ __launch_bounds__(64 * kWaves, decode_round(D)) void paged_decode_kernel(
    const uint16_t *__restrict__ q, int64_t q_row, int64_t q_head, const uint16_t *__restrict__ k_pages, int64_t kpage,
    int64_t khead, int64_t krow, const uint16_t *__restrict__ v_pages, int64_t vpage, int64_t vhead, int64_t vrow, int pages,
    int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens, int batch, int kvh, int grp,
    int tiles, int share, float scale2, float *__restrict__ part_o, float *__restrict__ part_ml, int4 *__restrict__ joins,
    uint16_t *__restrict__ out) {
  extern __shared__ float sm[];  // [kWaves][rows][D] outputs, then [kWaves][rows][2] maxima and sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, j = lane >> 4;
  const int heads = kvh * tiles, h = blockIdx.x % heads, kh = h / tiles, run = blockIdx.x / heads;
  const DecodePlan plan{lens, batch, width << shift};
  const uint64_t all = plan.blocks();
  share = static_cast<int>(min(static_cast<uint64_t>(share), all));  // no run is empty
  const int from = static_cast<int>(run * all / share), to = static_cast<int>((run + 1) * all / share);
  int b, at, blocks;  // the sequence, and the block of it, that the run begins with
  if (run >= share || !attn_find_part(plan, batch, 0, from, b, at, blocks)) return;  // uniform over the workgroup
  const int g0 = h % tiles * 16, rows = min(16, grp - g0);  // query heads of this workgroup
  const int nh = kvh * grp;
  float *ml = sm + kWaves * rows * D;
  KvSource<true> src{k_pages + kh * khead, v_pages + kh * vhead, kpage, krow, vpage, vrow, nullptr, shift, (1 << shift) - 1, pages, 0};

  for (int left = to - from; left > 0; ++b, at = 0) {
    const int len = plan.len(b);
    blocks = plan(b, 0);
    const int end = min(at + left, blocks), t1 = min(end * kBlock, len);
    const bool whole = at == 0 && end == blocks;
    uint4 qf[D / 32];
    const uint16_t *qp = q + b * q_row + static_cast<int64_t>(kh * grp + g0 + min(i16, rows - 1)) * q_head + 8 * j;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) qf[c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);
    src.table = table + static_cast<int64_t>(b) * width;
    src.last = len > 0 ? (len - 1) >> shift : 0;
    AttnRows<D> a;
    attn_clear(a);
    attn_walk<D, DT, false>(a, src, qf, at * kBlock + 32 * wave, t1, kBlock, t1, t1, t1, scale2, lane);
    a.l = attn_row_sum(a.l);

    // the four waves' states meet
    if (i16 < rows) {
      float *o = sm + (wave * rows + i16) * D + (D / 16) * 4 * j;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[(D / 16) * r + c] = a.o[c][r];
      if (j == 0) {
        ml[(wave * rows + i16) * 2] = a.m;
        ml[(wave * rows + i16) * 2 + 1] = a.l;
      }
    }
    __syncthreads();
    const int64_t slot = (static_cast<int64_t>(2 * run + (left < to - from ? 1 : 0)) * heads + h) * min(grp, 16);
    if (at == 0 && threadIdx.x == 0) {
      const int last = static_cast<int>(((to - left + blocks) * static_cast<uint64_t>(share) - 1) / all);  // run of its last block
      joins[b * heads + h] = make_int4(run, last - run + 1, left < to - from ? 1 : 0, 0);
    }
    for (int e = threadIdx.x; e < rows * D; e += 64 * kWaves) {
      const int row = e / D, d = e % D;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = fmaxf(m, ml[(w * rows + row) * 2]);
      float o = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float mw = ml[(w * rows + row) * 2];
        const float f = mw == m ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
        o += f * sm[(w * rows + row) * D + d];
        l += f * ml[(w * rows + row) * 2 + 1];
      }
      if (whole) {
        const float v = l == 0.f ? 0.f : o / l;
        out[(static_cast<int64_t>(b) * nh + kh * grp + g0 + row) * D + d] = DT == MP_F16 ? mp_f2h(v) : mp_f2bf(v);
      } else {
        part_o[(slot + row) * D + d] = o;
        if (d == 0) {
          part_ml[(slot + row) * 2] = m;
          part_ml[(slot + row) * 2 + 1] = l;
        }
      }
    }
    left -= end - at;
    if (left > 0) __syncthreads();  // the next sequence's states go to the same place
  }
}

// The parts of a sequence's query head meet, in one workgroup: D / 4 threads take a part's output, 1024 / D parts at a time.
// joins, of (sequence, head tile): the first run, how many runs, and whether the first run begins before the sequence.  A launch
// of its own, 3 to 7 us: joined by the last of its workgroups, a sequence would need fences and counters over the XCDs' L2s.
template <int D, int DT>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(int heads, int kvh, int grp, const float *__restrict__ part_o,
                                                                const float *__restrict__ part_ml,
                                                                const int4 *__restrict__ joins, uint16_t *__restrict__ out) {
  constexpr int kCols = D / 4, kAt = 256 / kCols;
  __shared__ float4 acc[kAt][kCols];
  __shared__ float sums[kAt], tops[4];
  const int nh = kvh * grp, b = blockIdx.x / nh, qh = blockIdx.x % nh, per = min(grp, 16);
  const int kh = qh / grp, g = qh % grp, h = kh * (heads / kvh) + g / 16;
  const int4 of = joins[b * heads + h];
  if (of.y == 1) return;  // written already
  const auto at_part = [&](int p) {
    return (static_cast<int64_t>(2 * (of.x + p) + (p == 0 ? of.z : 0)) * heads + h) * per + g % 16;
  };
  float m = -INFINITY;
  for (int p = threadIdx.x; p < of.y; p += 256) m = fmaxf(m, part_ml[at_part(p) * 2]);
  m = mp_wave_max(m);
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const int col = threadIdx.x % kCols, at = threadIdx.x / kCols;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int p = at; p < of.y; p += kAt) {
    const float2 ml = reinterpret_cast<const float2 *>(part_ml)[at_part(p)];
    const float4 x = reinterpret_cast<const float4 *>(part_o)[at_part(p) * kCols + col];
    const float f = ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m);
    l += f * ml.y;
    o.x += f * x.x;
    o.y += f * x.y;
    o.z += f * x.z;
    o.w += f * x.w;
  }
  acc[at][col] = o;
  if (col == 0) sums[at] = l;
  __syncthreads();
  if (at != 0) return;
  for (int i = 1; i < kAt; ++i) {
    const float4 x = acc[i][col];
    l += sums[i];
    o.x += x.x;
    o.y += x.y;
    o.z += x.z;
    o.w += x.w;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const bool none = l == 0.f;
  reinterpret_cast<uint2 *>(out)[static_cast<int64_t>(blockIdx.x) * kCols + col] =
      make_uint2(attn_pack2<DT>(none ? 0.f : o.x * inv, none ? 0.f : o.y * inv),
                 attn_pack2<DT>(none ? 0.f : o.z * inv, none ? 0.f : o.w * inv));
}

inline bool strides8(int64_t a, int64_t b, int64_t c) { return a % 8 == 0 && b % 8 == 0 && c % 8 == 0 && a >= 0 && b >= 0 && c >= 0; }

// Page size as a shift: a power of two from 8 (a lane's eight positions lie in one page).
inline int page_shift(int page) {
  for (int s = 3; s < 16; ++s)
    if (page == 1 << s) return s;
  return -1;
}

}  // namespace

extern "C" int mp_paged_rope_append(const void *qkv, int64_t qkv_row, int64_t rows, int nh, int kvh, int head_dim,
                                    const float *cos_t, const float *sin_t, int rotary, int64_t angles, int pairs,
                                    void *q_out, const mp_pages *cache, const int32_t *lens, const int32_t *starts,
                                    int64_t batch, int dtype, mp_stream_t stream) {
  if (!qkv || !cos_t || !sin_t || !q_out || !cache || !cache->k || !cache->v || !cache->table || !lens) return MP_ERR_ARG;
  if (dtype != MP_F16 && dtype != MP_BF16) return MP_ERR_DTYPE;
  const int shift = page_shift(cache->page_size);
  if (rows < 0 || rows > INT32_MAX || batch < 1 || batch > INT32_MAX - 64 || (!starts && rows != batch)) return MP_ERR_SHAPE;
  if (nh < 1 || kvh < 1 || nh > 65536 || kvh > 65536 || head_dim < 16 || head_dim > 1024 || head_dim % 16) return MP_ERR_SHAPE;
  if (rotary < 16 || rotary > head_dim || rotary % 16 || angles < 1) return MP_ERR_SHAPE;
  if (shift < 0 || cache->pages < 1 || cache->pages > INT32_MAX || cache->width < 1 || cache->width > (1 << 30) >> shift) return MP_ERR_SHAPE;
  if (qkv_row < static_cast<int64_t>(nh + 2 * kvh) * head_dim || qkv_row % 8 ||
      !strides8(cache->k_page, cache->k_head, cache->k_row) || !strides8(cache->v_page, cache->v_head, cache->v_row))
    return MP_ERR_SHAPE;
  if (!mp_aligned(qkv, 16) || !mp_aligned(cos_t, 16) || !mp_aligned(sin_t, 16) || !mp_aligned(q_out, 16) ||
      !mp_aligned(cache->k, 16) || !mp_aligned(cache->v, 16))
    return MP_ERR_ALIGN;
  if (rows == 0) return MP_OK;
  const int64_t pieces = static_cast<int64_t>(nh + 2 * kvh) * (head_dim / 16);
  const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(mp_cdiv(pieces, 256)));
  if (grid.y > 65535) return MP_ERR_SHAPE;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define MP_APPEND(DT, P)                                                                                                 \
  hipLaunchKernelGGL((paged_rope_append_kernel<DT, P>), grid, dim3(256), 0, s, static_cast<const uint16_t *>(qkv),       \
                     qkv_row, nh, kvh, head_dim, cos_t, sin_t, rotary / 2, angles, static_cast<uint16_t *>(q_out),       \
                     static_cast<uint16_t *>(cache->k), cache->k_page, cache->k_head, cache->k_row,                      \
                     static_cast<uint16_t *>(cache->v), cache->v_page, cache->v_head, cache->v_row,                      \
                     static_cast<int>(cache->pages), shift, cache->table, static_cast<int>(cache->width), lens, starts,  \
                     static_cast<int>(batch))
  if (dtype == MP_F16) {
    if (pairs) MP_APPEND(MP_F16, true);
    else MP_APPEND(MP_F16, false);
  } else {
    if (pairs) MP_APPEND(MP_BF16, true);
    else MP_APPEND(MP_BF16, false);
  }
#undef MP_APPEND
  MP_CHECK_LAUNCH();
  return MP_OK;
}

extern "C" size_t mp_paged_decode_workspace_bytes(int64_t batch, int nh, int kvh, int head_dim) {
  const int cus = mp_cu_count();
  if (batch <= 0 || batch > INT32_MAX || nh <= 0 || kvh <= 0 || nh % kvh || head_dim <= 0 || cus <= 0) return 0;
  const int64_t grp = nh / kvh, heads = kvh * mp_cdiv(grp, 16), per = grp < 16 ? grp : 16;
  return static_cast<size_t>(2 * decode_share(heads, head_dim) * heads * per) * (head_dim + 2) * sizeof(float) +
         static_cast<size_t>(batch * heads) * sizeof(int4);
}

extern "C" int mp_paged_decode_attention(const void *q, int64_t q_row, int64_t q_head, int64_t batch, int nh, int kvh,
                                         int head_dim, const mp_pages *cache, const int32_t *lens, float scale, void *out,
                                         int dtype, void *workspace, size_t workspace_bytes, mp_stream_t stream) {
  if (!q || !cache || !cache->k || !cache->v || !cache->table || !lens || !out || !workspace) return MP_ERR_ARG;
  if (dtype != MP_F16 && dtype != MP_BF16) return MP_ERR_DTYPE;
  if (!std::isfinite(scale * kLog2e)) return MP_ERR_ARG;
  const int shift = page_shift(cache->page_size);
  if (batch < 0 || batch > INT32_MAX - 64 || nh < 1 || kvh < 1 || nh > 65536 || nh % kvh) return MP_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return MP_ERR_SHAPE;
  if (shift < 0 || cache->pages < 1 || cache->pages > INT32_MAX || cache->width < 1 || cache->width > (1 << 30) >> shift) return MP_ERR_SHAPE;
  if (q_row % 8 || q_head % 8 || q_row < 0 || q_head < 0 || !strides8(cache->k_page, cache->k_head, cache->k_row) ||
      !strides8(cache->v_page, cache->v_head, cache->v_row))
    return MP_ERR_SHAPE;
  if (!mp_aligned(q, 16) || !mp_aligned(out, 16) || !mp_aligned(cache->k, 16) || !mp_aligned(cache->v, 16) ||
      !mp_aligned(workspace, 16))
    return MP_ERR_ALIGN;
  if (batch == 0) return MP_OK;
  if (mp_cu_count() <= 0) return MP_ERR_HIP;
  if (workspace_bytes < mp_paged_decode_workspace_bytes(batch, nh, kvh, head_dim)) return MP_ERR_WORKSPACE;
  const int grp = nh / kvh, tiles = static_cast<int>(mp_cdiv(grp, 16)), per = grp < 16 ? grp : 16;
  const int64_t heads = static_cast<int64_t>(kvh) * tiles, share = decode_share(heads, head_dim), blocks = share * heads;
  float *part_o = static_cast<float *>(workspace), *part_ml = part_o + 2 * blocks * per * head_dim;
  int4 *joins = reinterpret_cast<int4 *>(part_ml + 2 * blocks * per * 2);
  const int64_t capacity = cache->width << shift;
  if (blocks > INT32_MAX || batch * nh > INT32_MAX || batch * mp_cdiv(capacity, kBlock) > INT32_MAX) return MP_ERR_SHAPE;
  const float scale2 = scale * kLog2e;
  const int lds = kWaves * per * (head_dim + 2) * static_cast<int>(sizeof(float));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define MP_DECODE(D, DT)                                                                                                  \
  do {                                                                                                                    \
    if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void *>(paged_decode_kernel<D, DT>),               \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)            \
      return MP_ERR_HIP;                                                                                                  \
    hipLaunchKernelGGL((paged_decode_kernel<D, DT>), dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves),              \
                       lds, s, static_cast<const uint16_t *>(q), q_row, q_head,        \
                       static_cast<const uint16_t *>(cache->k), cache->k_page, cache->k_head, cache->k_row,               \
                       static_cast<const uint16_t *>(cache->v), cache->v_page, cache->v_head, cache->v_row,               \
                       static_cast<int>(cache->pages), shift, cache->table, static_cast<int>(cache->width), lens,         \
                       static_cast<int>(batch), kvh, grp, tiles, static_cast<int>(share), scale2, part_o, part_ml, joins,                    \
                       static_cast<uint16_t *>(out));                                                                     \
    MP_CHECK_LAUNCH();                                                                                                    \
    if (capacity > kBlock) { /* else every sequence is one block */                                                       \
      hipLaunchKernelGGL((paged_decode_join_kernel<D, DT>), dim3(static_cast<unsigned>(batch * nh)), dim3(256), 0, s,     \
                         static_cast<int>(heads), kvh, grp, part_o, part_ml, joins, static_cast<uint16_t *>(out));        \
      MP_CHECK_LAUNCH();                                                                                                  \
    }                                                                                                                     \
  } while (0)
  if (dtype == MP_F16) {
    if (head_dim == 64) MP_DECODE(64, MP_F16);
    else if (head_dim == 128) MP_DECODE(128, MP_F16);
    else MP_DECODE(256, MP_F16);
  } else {
    if (head_dim == 64) MP_DECODE(64, MP_BF16);
    else if (head_dim == 128) MP_DECODE(128, MP_BF16);
    else MP_DECODE(256, MP_BF16);
  }
#undef MP_DECODE
  return MP_OK;
}
