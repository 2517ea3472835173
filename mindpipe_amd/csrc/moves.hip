// Moving what a paged cache holds: whole pages copied to other pages (a fork of sequences that go on apart), and positions of a
// sequence moved to its front (the accepted ones of a draft), of every layer's keys and values in one launch.
#include <climits>

#include "mp_common.h"

namespace {

struct MovePools {
  const uint16_t *k, *v;  // written as well
  int64_t k_layer, k_page, k_head, k_row, v_layer, v_page, v_head, v_row;
  int layers, pages, kvh, shift, chunks;  // chunks: of 16 bytes in a position of a head
  MpDivisor by_chunks, by_heads;
};

__device__ __forceinline__ uint16_t *move_at(const MovePools &p, bool values, int layer, int64_t page, int head, int64_t row) {
  uint16_t *base = const_cast<uint16_t *>(values ? p.v : p.k);
  return values ? base + layer * p.v_layer + page * p.v_page + head * p.v_head + row * p.v_row
                : base + layer * p.k_layer + page * p.k_page + head * p.k_head + row * p.k_row;
}

// A workgroup copies 256 16-byte pieces of one page, layer and pool, a piece a thread.  Bound by the memory: 40 whole pages of 131 KB
// in 32 layers, 671 MB read and written, 101 us, 6.6 TB/s, where a copy of as much in one piece takes 134; three partial pages of 16
// positions of 32 heads (22 MB) 7 us.  Two, four and eight pieces a thread: 118, 125 and 197 us, and 19, 19 and 10.
__global__ __launch_bounds__(256) void paged_copy_kernel(MovePools p, const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                                                         const int32_t *__restrict__ filled, int per) {
  const int pair = blockIdx.x / per, piece = (blockIdx.x - pair * per) * 256 + threadIdx.x, layer = blockIdx.y >> 1;
  const bool values = blockIdx.y & 1;
  const int from = src[pair], to = dst[pair], size = 1 << p.shift;
  if (from < 0 || from >= p.pages || to < 0 || to >= p.pages || from == to) return;
  const int rows = filled ? min(max(filled[pair], 0), size) : size;
  const int position = p.by_chunks(piece), row = position & (size - 1), head = position >> p.shift, c = piece - position * p.chunks;
  if (head >= p.kvh || row >= rows) return;
  *reinterpret_cast<uint4 *>(move_at(p, values, layer, to, head, row) + 8 * c) =
      *reinterpret_cast<const uint4 *>(move_at(p, values, layer, from, head, row) + 8 * c);
}

constexpr int kAhead = 8;  // positions that are read before the first of them is written

// A thread takes one 16-byte column (layer, pool, head, piece) of a sequence and moves its entries in their order.  They ascend
// and none lies before its new place, so what is read later has not been written.  Bound by its chain of loads, offsets, entries,
// pages and values: 40 sequences, up to seven of 64 positions, 8 heads of 128 in 32 layers (18 MB) 11 us, one sequence of 32 heads 3.8.
__global__ __launch_bounds__(256) void paged_keep_kernel(MovePools p, const int32_t *__restrict__ table, int width,
                                                         const int32_t *__restrict__ first, const int32_t *__restrict__ keep,
                                                         const int32_t *__restrict__ starts, int total, int per) {
  const int b = blockIdx.x / per, column = (blockIdx.x - b * per) * 256 + threadIdx.x;
  const int of = p.by_chunks(column), c = column - of * p.chunks, pool = p.by_heads(of), head = of - pool * p.kvh;
  if (pool >= 2 * p.layers) return;
  const int begin = min(max(starts[b], 0), total), end = min(max(starts[b + 1], begin), total);
  const int64_t base = first[b], room = static_cast<int64_t>(width) << p.shift;
  const int32_t *pages = table + static_cast<int64_t>(b) * width;
  const auto place = [&](int64_t pos) -> uint16_t * {
    if (pos < 0 || pos >= room) return nullptr;
    const int page = pages[pos >> p.shift];
    if (page < 0 || page >= p.pages) return nullptr;
    return move_at(p, pool & 1, pool >> 1, page, head, pos & ((1 << p.shift) - 1)) + 8 * c;
  };
  for (int i0 = begin; i0 < end; i0 += kAhead) {
    uint4 x[kAhead];
    uint16_t *y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      y[i] = nullptr;
      if (i0 + i >= end) continue;
      const int at = keep[i0 + i], to = i0 + i - begin;
      if (at == to) continue;  // it is there
      const uint16_t *z = place(base + at);
      uint16_t *w = place(base + to);
      if (!z || !w) continue;
      x[i] = *reinterpret_cast<const uint4 *>(z);
      y[i] = w;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (y[i]) *reinterpret_cast<uint4 *>(y[i]) = x[i];
  }
}

int move_pools(const mp_pages *c, int64_t layers, int64_t k_layer, int64_t v_layer, int kvh, int head_dim, bool table, MovePools &p) {
  if (!c || !c->k || !c->v || (table && !c->table)) return MP_ERR_ARG;
  int shift = -1;
  for (int s = 3; s < 16; ++s)
    if (c->page_size == 1 << s) shift = s;
  if (shift < 0 || c->pages < 1 || c->pages > INT32_MAX) return MP_ERR_SHAPE;
  if (table && (c->width < 1 || c->width > (1 << 30) >> shift)) return MP_ERR_SHAPE;
  if (layers < 1 || layers > 32767 || kvh < 1 || kvh > 65536 || head_dim < 8 || head_dim > 1024 || head_dim % 8) return MP_ERR_SHAPE;
  if ((static_cast<int64_t>(kvh) * head_dim / 8) << shift > INT32_MAX / 2) return MP_ERR_SHAPE;
  for (int64_t s : {k_layer, v_layer, c->k_page, c->k_head, c->k_row, c->v_page, c->v_head, c->v_row})
    if (s < 0 || s % 8) return MP_ERR_SHAPE;
  if (!mp_aligned(c->k, 16) || !mp_aligned(c->v, 16)) return MP_ERR_ALIGN;
  p = {static_cast<const uint16_t *>(c->k), static_cast<const uint16_t *>(c->v), k_layer, c->k_page, c->k_head, c->k_row, v_layer,
       c->v_page, c->v_head, c->v_row, static_cast<int>(layers), static_cast<int>(c->pages), kvh, shift, head_dim / 8,
       mp_divisor(head_dim / 8), mp_divisor(kvh)};
  return MP_OK;
}

}  // namespace

extern "C" int mp_paged_copy_pages(const mp_pages *cache, int64_t layers, int64_t k_layer, int64_t v_layer, int kvh, int head_dim,
                                   const int32_t *src, const int32_t *dst, const int32_t *filled, int64_t count, mp_stream_t stream) {
  if (!src || !dst) return MP_ERR_ARG;
  MovePools p;
  const int rc = move_pools(cache, layers, k_layer, v_layer, kvh, head_dim, false, p);
  if (rc != MP_OK) return rc;
  const int64_t per = mp_cdiv(static_cast<int64_t>(kvh) * p.chunks << p.shift, 256);
  if (count < 0 || count > kMpMaxGroups / per) return MP_ERR_SHAPE;
  if (count == 0) return MP_OK;
  hipLaunchKernelGGL(paged_copy_kernel, dim3(static_cast<unsigned>(count * per), static_cast<unsigned>(2 * layers)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), p, src, dst, filled, static_cast<int>(per));
  MP_CHECK_LAUNCH();
  return MP_OK;
}

extern "C" int mp_paged_keep_positions(const mp_pages *cache, int64_t layers, int64_t k_layer, int64_t v_layer, int kvh, int head_dim,
                                       int64_t batch, const int32_t *first, const int32_t *keep, int64_t total,
                                       const int32_t *starts, mp_stream_t stream) {
  if (!first || !keep || !starts) return MP_ERR_ARG;
  MovePools p;
  const int rc = move_pools(cache, layers, k_layer, v_layer, kvh, head_dim, true, p);
  if (rc != MP_OK) return rc;
  const int64_t columns = 2 * layers * kvh * p.chunks, per = mp_cdiv(columns, 256);
  if (columns > INT32_MAX - 256 || batch < 0 || batch > kMpMaxGroups / per || total < 0 || total > INT32_MAX / 2) return MP_ERR_SHAPE;
  if (batch == 0 || total == 0) return MP_OK;
  hipLaunchKernelGGL(paged_keep_kernel, dim3(static_cast<unsigned>(batch * per)), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                     p, cache->table, static_cast<int>(cache->width), first, keep, starts, static_cast<int>(total), static_cast<int>(per));
  MP_CHECK_LAUNCH();
  return MP_OK;
}
