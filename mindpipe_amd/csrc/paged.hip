// A paged key-value cache: appending rotated keys and values, and attention of one new token per sequence.
//
// A layer's cache is two pools of pages, each page holding `page` positions of every key-value head (strides are free, the
// values of a position are contiguous).  A sequence's pages are listed in its row of a table; its positions are counted
// from zero, and everything goes by device memory (lengths, starts, table), so a step keeps its launches while the
// sequences grow and can be captured into a graph.  A page number outside the pool is an empty page: nothing is
// written to it, and its positions are not attended.
#include <climits>

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
// Bound by its bytes: a row is read once and written once, the tables' rows come from the caches.
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
// Positions are split into chunks of one size for all sequences, the smallest multiple of kChunk that leaves about `goal`
// workgroups in all: a sequence has ceil(length / chunk) of them (an empty one has one, which writes its zeros).
constexpr int kWaves = 4;
constexpr int kChunk = 32 * kWaves;

struct DecodePlan {
  const int32_t *lens;
  int capacity;  // positions that the table has room for
  __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), capacity); }
  __device__ __forceinline__ int operator()(int b, int chunk) const {
    const int n = len(b);
    return n > 0 ? (n - 1) / chunk + 1 : 1;
  }
};

__device__ __forceinline__ int decode_chunk(const DecodePlan &plan, int batch, int heads, int goal) {
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  for (int b = lane; b < batch; b += 64) total += plan.len(b);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
  // a sequence is shorter than 2^30: a longer chunk says no more
  const int64_t chunk = min((total * heads / goal + kChunk) / kChunk * kChunk, static_cast<int64_t>(1) << 30);
  return __builtin_amdgcn_readfirstlane(static_cast<int>(chunk));
}

// Workgroups that a plan may need: the goal's and one more per sequence, of each head.
inline int64_t decode_parts(int64_t batch, int64_t heads, int64_t goal) { return goal / heads + 1 + batch; }

template <int D, int DT>
__global__ __launch_bounds__(64 * kWaves) void paged_decode_kernel(
    const uint16_t *__restrict__ q, int64_t q_row, int64_t q_head, const uint16_t *__restrict__ k_pages, int64_t kpage,
    int64_t khead, int64_t krow, const uint16_t *__restrict__ v_pages, int64_t vpage, int64_t vhead, int64_t vrow, int pages,
    int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens, int batch, int kvh, int grp,
    int tiles, int goal, float scale2, float *__restrict__ part_o, float *__restrict__ part_ml, uint16_t *__restrict__ out) {
  extern __shared__ float sm[];  // [kWaves][rows][D] outputs, then [kWaves][rows][2] maxima and sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, j = lane >> 4;
  const int heads = kvh * tiles, h = blockIdx.x % heads, kh = h / tiles;
  const DecodePlan plan{lens, width << shift};
  const int chunk = decode_chunk(plan, batch, heads, goal);
  int b, part, parts;
  if (!attn_find_part(plan, batch, chunk, blockIdx.x / heads, b, part, parts)) return;  // uniform over the workgroup
  const int len = plan.len(b), t0 = part * chunk, t1 = min(t0 + chunk, len);
  const int g0 = h % tiles * 16, rows = min(16, grp - g0);  // query heads of this workgroup
  const int nh = kvh * grp;

  uint4 qf[D / 32];
  const uint16_t *qp = q + b * q_row + static_cast<int64_t>(kh * grp + g0 + min(i16, rows - 1)) * q_head + 8 * j;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) qf[c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);

  KvSource<true> src{k_pages + kh * khead, v_pages + kh * vhead, kpage, krow, vpage, vrow,
                     table + static_cast<int64_t>(b) * width, shift, (1 << shift) - 1, pages,
                     len > 0 ? (len - 1) >> shift : 0};
  AttnRows<D> a;
  attn_clear(a);
  attn_walk<D, DT>(a, src, qf, t0 + 32 * wave, t1, kChunk, t1, t1, t1, scale2, lane);
  a.l = attn_row_sum(a.l);

  // the four waves' states meet
  float *ml = sm + kWaves * rows * D;
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
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * min(grp, 16);
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
    if (parts == 1) {
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
}

// The chunks of a sequence's query head meet: one wave each.
template <int D, int DT>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(const int32_t *__restrict__ lens, int capacity, int batch, int kvh,
                                                                int grp, int tiles, int goal, const float *__restrict__ part_o,
                                                                const float *__restrict__ part_ml,
                                                                uint16_t *__restrict__ out) {
  const int nh = kvh * grp, heads = kvh * tiles;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (unit >= static_cast<int64_t>(batch) * nh) return;  // uniform over the wave
  const int b = __builtin_amdgcn_readfirstlane(static_cast<int>(unit / nh)), qh = static_cast<int>(unit % nh);
  const DecodePlan plan{lens, capacity};
  const int chunk = decode_chunk(plan, batch, heads, goal);
  const int parts = plan(b, chunk);
  if (parts == 1) return;
  int before = 0;
  for (int s = lane; s < b; s += 64) before += plan(s, chunk);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
  const int kh = qh / grp, g = qh % grp, per = min(grp, 16);
  const auto slot = [&](int p) {
    return (static_cast<int64_t>(before + p) * heads + kh * tiles + g / 16) * per + g % 16;
  };
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 64) m = fmaxf(m, part_ml[slot(p) * 2]);
  m = mp_wave_max(m);
  float o[D / 64], l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
  for (int p = 0; p < parts; ++p) {
    const float mp = part_ml[slot(p) * 2];
    const float f = mp == m ? 1.0f : __builtin_amdgcn_exp2f(mp - m);
    l += f * part_ml[slot(p) * 2 + 1];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] += f * part_o[slot(p) * D + 64 * i + lane];
  }
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const float v = l == 0.f ? 0.f : o[i] / l;
    out[(static_cast<int64_t>(b) * nh + qh) * D + 64 * i + lane] = DT == MP_F16 ? mp_f2h(v) : mp_f2bf(v);
  }
}

inline bool strides8(int64_t a, int64_t b, int64_t c) { return a % 8 == 0 && b % 8 == 0 && c % 8 == 0 && a >= 0 && b >= 0 && c >= 0; }

// Page size as a shift: a power of two from 8 (a lane's eight positions lie in one page).
inline int page_shift(int page) {
  for (int s = 3; s < 16; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// Workgroups wanted for the decode attention: two of four waves on each CU.
inline int decode_goal() { return 2 * mp_cu_count(); }

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
  if (batch <= 0 || nh <= 0 || kvh <= 0 || nh % kvh || head_dim <= 0 || cus <= 0) return 0;
  const int64_t grp = nh / kvh, heads = kvh * mp_cdiv(grp, 16), per = grp < 16 ? grp : 16;
  return static_cast<size_t>(decode_parts(batch, heads, decode_goal()) * heads * per) * (head_dim + 2) * sizeof(float);
}

extern "C" int mp_paged_decode_attention(const void *q, int64_t q_row, int64_t q_head, int64_t batch, int nh, int kvh,
                                         int head_dim, const mp_pages *cache, const int32_t *lens, float scale, void *out,
                                         int dtype, void *workspace, size_t workspace_bytes, mp_stream_t stream) {
  if (!q || !cache || !cache->k || !cache->v || !cache->table || !lens || !out || !workspace) return MP_ERR_ARG;
  if (dtype != MP_F16 && dtype != MP_BF16) return MP_ERR_DTYPE;
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
  const int grp = nh / kvh, tiles = static_cast<int>(mp_cdiv(grp, 16)), per = grp < 16 ? grp : 16, goal = decode_goal();
  const int64_t heads = static_cast<int64_t>(kvh) * tiles, parts = decode_parts(batch, heads, goal), blocks = parts * heads;
  if (blocks > INT32_MAX || batch * nh > INT32_MAX) return MP_ERR_SHAPE;
  float *part_o = static_cast<float *>(workspace), *part_ml = part_o + blocks * per * head_dim;
  const int capacity = static_cast<int>(cache->width << shift);
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
                       static_cast<int>(batch), kvh, grp, tiles, goal, scale2, part_o, part_ml,                           \
                       static_cast<uint16_t *>(out));                                                                     \
    MP_CHECK_LAUNCH();                                                                                                    \
    if (capacity > kChunk) { /* else every sequence is one chunk */                                                       \
      hipLaunchKernelGGL((paged_decode_join_kernel<D, DT>), dim3(static_cast<unsigned>(mp_cdiv(batch * nh, 4))),          \
                         dim3(256), 0, s, lens, capacity, static_cast<int>(batch), kvh, grp, tiles, goal, part_o,         \
                         part_ml, static_cast<uint16_t *>(out));                                                          \
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
