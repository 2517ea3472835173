// Causal attention of packed new tokens: whole prompts (keys and values packed alike) or chunks of new tokens behind what
// a paged cache holds of their sequences.
//
// The queries of the heads that share a key-value head are rows of one problem: row = token * group + head.  A workgroup
// takes kRows consecutive rows of a sequence and a key-value head; row r sees the positions up to its token's.  The tiles of
// the last rows, which see most, are started first.
#include "attn_common.h"

namespace {

constexpr int kRows = 64;  // 16 for each of four waves

struct PackedPlan {
  const int32_t *starts;
  int batch, rows, grp;
  // offsets of a sequence; sequence `batch` is what lies behind the last one
  __device__ __forceinline__ int first(int b) const { return min(max(starts[b], 0), rows); }
  __device__ __forceinline__ int end(int b) const { return b < batch ? max(first(b), first(b + 1)) : rows; }
  __device__ __forceinline__ int operator()(int b, int per) const {
    return static_cast<int>((static_cast<int64_t>(end(b) - first(b)) * grp + per - 1) / per);
  }
};

template <int D, int DT, bool PAGED>
__global__ __launch_bounds__(256) void prompt_attention_kernel(
    const uint16_t *__restrict__ q, int64_t q_row, int64_t q_head, const uint16_t *__restrict__ k, int64_t kpage,
    int64_t khead, int64_t krow, const uint16_t *__restrict__ v, int64_t vpage, int64_t vhead, int64_t vrow, int pages,
    int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens,
    const int32_t *__restrict__ starts, int batch, int rows, int kvh, int grp, int tiles, float scale2,
    uint16_t *__restrict__ out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, j = lane >> 4;
  const int kh = blockIdx.x % kvh;
  const PackedPlan plan{starts, batch, rows, grp};
  int b, part, parts;
  if (!attn_find_part(plan, batch + 1, kRows, tiles - 1 - static_cast<int>(blockIdx.x / kvh), b, part, parts)) return;
  const int first = plan.first(b), n = plan.end(b) - first;
  int len = 0;  // positions of the sequence, the new tokens' included
  if (b < batch) len = PAGED ? min(max(lens[b], 0), width << shift) : n;
  const int at = part * kRows + wave * 16 + i16;  // row of this lane
  const bool row = at < n * grp;
  const int token = row ? at / grp : 0, head = kh * grp + (row ? at - token * grp : 0);
  // behind the last sequence (b == batch) nothing is seen, and zeros are written
  const int sees = row && b < batch ? max(len - n + token + 1, 0) : 0;
  int full = row ? sees : len, end = sees;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    full = min(full, __shfl_xor(full, o, 64));
    end = max(end, __shfl_xor(end, o, 64));
  }
  full = __builtin_amdgcn_readfirstlane(full);
  end = __builtin_amdgcn_readfirstlane(end);

  uint4 qf[D / 32];
  const uint16_t *qp = q + (first + token) * q_row + head * q_head + 8 * j;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) qf[c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);
  KvSource<PAGED> src;
  if constexpr (PAGED)
    src = {k + kh * khead, v + kh * vhead, kpage, krow, vpage, vrow, table + static_cast<int64_t>(min(b, batch - 1)) * width,
           shift, (1 << shift) - 1, pages, len > 0 ? (len - 1) >> shift : 0};
  else
    src = {k + first * krow + kh * khead, v + first * vrow + kh * vhead, krow, vrow, n - 1};
  AttnRows<D> a;
  attn_clear(a);
  attn_walk<D, DT>(a, src, qf, 0, end, 32, sees, end, full, scale2, lane);
  const float l = attn_row_sum(a.l);
  if (!row) return;
  uint16_t *y = out + (static_cast<int64_t>(first + token) * kvh * grp + head) * D + (D / 16) * 4 * j;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int c = 0; c < D / 16; c += 2) {
      const float lo = l == 0.f ? 0.f : a.o[c][r] / l, hi = l == 0.f ? 0.f : a.o[c + 1][r] / l;
      *reinterpret_cast<uint32_t *>(y + (D / 16) * r + c) = attn_pack2<DT>(lo, hi);
    }
  }
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
  hipStream_t stream;
};

template <bool PAGED>
int prompt_launch(const PromptCall &c) {
  if (c.dtype != MP_F16 && c.dtype != MP_BF16) return MP_ERR_DTYPE;
  if (c.rows < 0 || c.rows > INT32_MAX || c.batch < 1 || c.batch > INT32_MAX - 64) return MP_ERR_SHAPE;
  if (c.nh < 1 || c.kvh < 1 || c.nh > 65536 || c.nh % c.kvh) return MP_ERR_SHAPE;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return MP_ERR_SHAPE;
  for (int64_t s : {c.q_row, c.q_head, c.kpage, c.khead, c.krow, c.vpage, c.vhead, c.vrow})
    if (s < 0 || s % 8) return MP_ERR_SHAPE;
  for (const void *p : {c.q, c.k, c.v, static_cast<const void *>(c.out)})
    if (!mp_aligned(p, 16)) return MP_ERR_ALIGN;
  if (c.rows == 0) return MP_OK;
  const int64_t grp = c.nh / c.kvh;
  // a part of a tile for each sequence, and for the rows behind the last one
  const int64_t tiles = c.rows * grp / kRows + c.batch + 1, blocks = tiles * c.kvh;
  if (c.rows * grp > INT32_MAX - kRows || blocks > INT32_MAX) return MP_ERR_SHAPE;
#define MP_PROMPT(D, DT)                                                                                                  \
  hipLaunchKernelGGL((prompt_attention_kernel<D, DT, PAGED>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, c.stream, \
                     static_cast<const uint16_t *>(c.q), c.q_row, c.q_head, static_cast<const uint16_t *>(c.k), c.kpage,  \
                     c.khead, c.krow, static_cast<const uint16_t *>(c.v), c.vpage, c.vhead, c.vrow, c.pages, c.shift,     \
                     c.table, c.width, c.lens, c.starts, static_cast<int>(c.batch), static_cast<int>(c.rows), c.kvh,      \
                     static_cast<int>(grp), static_cast<int>(tiles), c.scale * kLog2e, static_cast<uint16_t *>(c.out))
  if (c.dtype == MP_F16) {
    if (c.head_dim == 64) MP_PROMPT(64, MP_F16);
    else if (c.head_dim == 128) MP_PROMPT(128, MP_F16);
    else MP_PROMPT(256, MP_F16);
  } else {
    if (c.head_dim == 64) MP_PROMPT(64, MP_BF16);
    else if (c.head_dim == 128) MP_PROMPT(128, MP_BF16);
    else MP_PROMPT(256, MP_BF16);
  }
#undef MP_PROMPT
  MP_CHECK_LAUNCH();
  return MP_OK;
}

}  // namespace

extern "C" int mp_prompt_attention(const void *q, int64_t q_row, int64_t q_head, const void *k, int64_t k_row, int64_t k_head,
                                   const void *v, int64_t v_row, int64_t v_head, int64_t rows, int nh, int kvh, int head_dim,
                                   const int32_t *starts, int64_t batch, float scale, void *out, int dtype,
                                   mp_stream_t stream) {
  if (!q || !k || !v || !starts || !out) return MP_ERR_ARG;
  return prompt_launch<false>({q, q_row, q_head, k, v, 0, k_head, k_row, 0, v_head, v_row, 0, 0, 0, nullptr, nullptr, starts,
                               batch, rows, nh, kvh, head_dim, scale, out, dtype, reinterpret_cast<hipStream_t>(stream)});
}

extern "C" int mp_paged_prompt_attention(const void *q, int64_t q_row, int64_t q_head, int64_t rows, int nh, int kvh,
                                         int head_dim, const mp_pages *cache, const int32_t *lens, const int32_t *starts,
                                         int64_t batch, float scale, void *out, int dtype, mp_stream_t stream) {
  if (!q || !cache || !cache->k || !cache->v || !cache->table || !lens || !starts || !out) return MP_ERR_ARG;
  int shift = -1;
  for (int s = 3; s < 16; ++s)
    if (cache->page_size == 1 << s) shift = s;
  if (shift < 0 || cache->pages < 1 || cache->pages > INT32_MAX || cache->width < 1 || cache->width > (1 << 30) >> shift)
    return MP_ERR_SHAPE;
  return prompt_launch<true>({q, q_row, q_head, cache->k, cache->v, cache->k_page, cache->k_head, cache->k_row, cache->v_page,
                              cache->v_head, cache->v_row, static_cast<int>(cache->pages), shift,
                              static_cast<int>(cache->width), cache->table, lens, starts, batch, rows, nh, kvh, head_dim,
                              scale, out, dtype, reinterpret_cast<hipStream_t>(stream)});
}
