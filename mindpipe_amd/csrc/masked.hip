// Attention of packed new tokens over a paged cache where a row sees other than all positions up to its own:
//
//   * trees of drafted tokens: a row sees what the cache holds before its sequence's new tokens, and of these the ones that its
//     mask names (a node's ancestors and itself);
//   * windows: a row sees the last `window` positions up to its own, and the first `sinks`.
//
// The queries of the heads that share a key-value head are rows of one problem: row = token * group + head.  Two forms:
//
//   * wide: the products of prompt.hip (prompt_tile.h), 128 rows to a workgroup, 32 to a wave, over tiles of 64 positions in LDS;
//   * narrow: those of the decode kernel (attn_common.h), 16 rows to a workgroup, whose four waves take 32 positions each of a
//     tile of 128, from memory to registers.
//
// The narrow form takes its weights and then what their rounding to 16 bits leaves, as decode does, whose tokens a draft's stand in
// for: the matrix cores idle there (26 nodes behind 1531 positions 17.9 -> 18.3 us, errors 2.6e-4 -> 2.1e-4).  The wide form takes
// them as rounded, like the prompts: with the rest 157 -> 204, 71 -> 86 and 305 -> 412 us for the batch of trees, short windows and the
// long chunk, errors (rms) 1.77e-3 -> 1.64e-3, 2.6e-4 -> 2.0e-4 and 2.3e-3 -> 1.7e-3.
//
// An item is up to 128 (16) rows of a sequence and key-value head.  It walks over the tiles that hold what its rows see, those that
// hold nothing seen left out.  Items that are much longer than an equal share of all tiles are cut into parts, which leave their
// outputs, unnormalised, maxima and sums in the workspace, and a second launch joins them, always in the same order.  A
// workgroup takes a part, and the longest come first, so that the short ones fill what the long ones leave.
//
// The wide form is bound as the prompts' attention is, by matrix and vector instructions in turn: 2.2 us for a tile of a
// workgroup, two to a CU.  2048 tokens behind 8192 positions with a window of 4096, 64 / 8 heads of 128 in bf16, 309 us, 0.9
// PFLOP/s of what is seen; 24 sequences of up to 8192 positions with trees of up to 64 nodes 147 us, 53 tiles an equal share and
// about 66 the longest path.  (Equal runs of tiles over all items, with a loop over items in the kernel, took 171 us there: the
// loop's state took the registers that hold the loads' offsets.)  The narrow form is bound by the chain from the lengths to a
// page and by the reads: 26 nodes behind 1531 positions, 32 / 32 heads, 13.5 us and a join of 4 to 5.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "prompt_tile.h"

namespace {

enum { kTree = 0, kWindow = 1 };

// The lowest n bits.
__device__ __forceinline__ uint64_t bits_below(int n) { return n <= 0 ? 0 : n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1; }

// What the rows see: plain arguments of a launch.
struct MaskedRule {
  const int64_t *masks;  // kTree: [rows, words]
  int words;
  int window, sinks;     // kWindow
  MpDivisor group;       // rows / group: tokens
};

// A sequence's rows and what they see, by the launch's rule.
template <int MODE>
struct MaskedSeq {
  int first, n;          // its packed rows
  int len, room;         // its positions, the new tokens' included, and those that there is room for; none outside of the sequences
  MaskedRule rule;

  __device__ __forceinline__ int context() const { return len - n; }  // position of its first row (negative: rows without a place)
  __device__ __forceinline__ int end() const { return min(len, room); }
  __device__ __forceinline__ int clamped(int64_t p) const {
    return static_cast<int>(max(min(p, static_cast<int64_t>(end())), int64_t(0)));
  }
  // Positions t .. t + 63 that token `token` of the sequence sees, as bits.  t is a multiple of 32.
  __device__ __forceinline__ uint64_t bits(int token, int t) const {
    if constexpr (MODE == kTree) {
      const int d = t - context();  // node of position t
      const int64_t *words = rule.masks + static_cast<int64_t>(first + token) * rule.words;
      uint64_t v = bits_below(-d);
      if (d > -64 && d < 64 * rule.words && token < n) {
        const int w = d >> 6, s = d & 63;  // bits of nodes d .. d + 63: from word w (-1: none) and the one after it
        if (w >= 0) v |= static_cast<uint64_t>(words[w]) >> s;
        if (s && w + 1 < rule.words) v |= static_cast<uint64_t>(words[w + 1]) << (64 - s);
      }
      return v & bits_below(end() - t);
    } else {
      const int64_t pos = static_cast<int64_t>(context()) + token;
      const int low = clamped(pos - rule.window + 1), upto = clamped(pos + 1);
      return bits_below(upto - t) & (bits_below(rule.sinks - t) | ~bits_below(low - t));
    }
  }
  // Rows of tokens a .. b: the tiles they look at lie below `to`, and of these none between `gap_from` and `gap_to` (multiples of
  // 64) is seen.
  __device__ __forceinline__ void span(int a, int b, int &to, int &gap_from, int &gap_to) const {
    gap_from = gap_to = 0;
    to = end();
    if constexpr (MODE == kWindow) {
      to = clamped(static_cast<int64_t>(context()) + b + 1);
      gap_to = min(clamped(static_cast<int64_t>(context()) + a - rule.window + 1), to) & ~63;
      gap_from = min((min(rule.sinks, to) + 63) & ~63, gap_to);
    }
  }
  // All of positions t .. upto - 1 are seen by tokens a .. b.
  __device__ __forceinline__ bool whole(int a, int b, int t, int upto) const {
    if (upto > end()) return false;
    if constexpr (MODE == kTree) return upto <= context();
    const int64_t pos = context();
    return upto <= pos + a + 1 && (upto <= rule.sinks || t >= pos + b - rule.window + 1);
  }
};

// The form of a kernel: rows of an item, positions of a tile, by how many tiles an item may pass an equal share and stay whole (half
// a share at most: joining costs what so many tiles do), and the share from which on items are cut finer, once one has to be.
struct Wide {
  static constexpr int kItem = kRows, kStep = kTile, kSlack = 8, kFiner = 12;
};
struct Narrow {
  static constexpr int kItem = 16, kStep = 128, kSlack = 2, kFiner = INT_MAX;
};
// How long a part may be, in tiles, with e tiles an equal share: as long as an item that stays whole, or finer.
template <class FORM>
constexpr int masked_keep(int e) { return e + (e / 2 < FORM::kSlack ? e / 2 : FORM::kSlack) + 1; }
constexpr int masked_finer(int e) { return e * 2 / 3 + 1; }
// Parts that have others, in shares at most: an item of T > limit tiles has up to 2 T / (limit + 1), all of them fewer than
// 2 (e + 1) / (limit + 1) of a share.
constexpr int kSlots = 3;
// How many more parts than items there are, at most: fewer than T / limit for an item that is cut, together (e + 1) / limit of a share,
// which is no more than 1 with a limit above e and at most 14 / 9 (e = 13, limit 9) with the finer one.
constexpr int64_t masked_more(int64_t share) { return share * 14 / 9 + 1; }
// The grid and the workspace rest on these two: checked for every e of 16 bits, from where on the finer limit's quotients are within
// 2e-5 of 3 / 2 and below 3.  (3 / 2 itself is too little for every e of 3 m + 1, and 14 / 9 for the 7 and 10 that are below kFiner.)
template <class FORM>
constexpr bool masked_bounds_hold() {
  for (int64_t e = 0; e < 1 << 16; ++e) {
    const int64_t keep = masked_keep<FORM>(static_cast<int>(e)), finer = e < FORM::kFiner ? keep : masked_finer(static_cast<int>(e));
    const int64_t limit = keep < finer ? keep : finer;
    if (2 * (e + 1) > kSlots * (limit + 1) || 9 * (e + 1) > 14 * limit) return false;
  }
  return true;
}
static_assert(masked_bounds_hold<Wide>() && masked_bounds_hold<Narrow>(), "a part without a workgroup, or without a place to join from");

constexpr int64_t kMaxBatch = 1 << 28;
constexpr int kPlanNear = 64;  // sequences, with the two that hold the other rows, which a wave sees at once

// What a workgroup takes: tiles of an item.
template <int MODE>
struct MaskedPart {
  MaskedSeq<MODE> seq;
  int b, item, part, parts;
  int slot;               // of the part, if there are others
  int to, gap_from, gap;  // positions looked at lie below `to`; virtual positions from gap_from on lie `gap` further
  int from, end;          // virtual positions of the part
};

template <int MODE, class FORM>
struct MaskedPlan {
  PackedPlan rows;
  const int32_t *lens;
  int capacity;  // positions that the table has room for
  MaskedRule rule;
  const int32_t *plan;  // of masked_plan_kernel

  __device__ __forceinline__ MaskedSeq<MODE> seq(int b) const {
    MaskedSeq<MODE> s;
    s.first = rows.first(b);
    s.n = rows.end(b) - s.first;
    s.len = b < rows.batch ? max(lens[b], 0) : 0;
    s.room = b < rows.batch ? capacity : 0;
    s.rule = rule;
    return s;
  }
  __device__ __forceinline__ int items(const MaskedSeq<MODE> &s) const {
    return (s.n * rows.grp + FORM::kItem - 1) / FORM::kItem;  // rows of all are below 2^31 - kItem
  }
  // Where an item looks.
  __device__ __forceinline__ void span(const MaskedSeq<MODE> &s, int item, int &to, int &gap_from, int &gap) const {
    int a = 0, b = 0;
    if constexpr (MODE == kWindow) {
      a = rule.group(item * FORM::kItem);
      b = min(rule.group(item * FORM::kItem + FORM::kItem - 1), s.n - 1);
    }
    int gap_to;
    s.span(a, b, to, gap_from, gap_to);
    gap = gap_to - gap_from;
  }
  static __device__ __forceinline__ int tiles(int to, int gap) { return (to - gap + FORM::kStep - 1) / FORM::kStep; }
  // Items of a sequence, and the tiles of its last one (one at least), which is the longest but for a tile where windows begin
  // inside of one.
  struct Row {
    int items, tiles;
  };
  __device__ __forceinline__ Row row(int b, uint64_t &held) const {
    Row r{0, 1};
    if (b < rows.batch + 2) {
      const MaskedSeq<MODE> s = seq(b);
      held += s.n;
      r.items = items(s);
      int to, from, gap;
      span(s, max(r.items - 1, 0), to, from, gap);
      r.tiles = max(tiles(to, gap), 1);
    }
    return r;
  }
  // How long parts may be, from all items' tiles.  each(f): f of every row; sum and most: over those who call it.  Items stay whole
  // where none is much longer than an equal share.  Otherwise parts are as long as such an item, or two thirds of a share, as the
  // longest part and the number of rounds have it (24 sequences of up to 8192 positions with trees of up to 64 nodes, 58 items of 1 to
  // 129 tiles for 64 workgroups: 186 us, 152 with the finer ones).
  template <class EACH, class SUM, class MOST>
  static __device__ __forceinline__ int limit_of(uint32_t all, int share, EACH each, SUM sum, MOST most) {
    const int equal = static_cast<int>(all / static_cast<uint32_t>(share)), keep = masked_keep<FORM>(equal);
    if (equal < FORM::kFiner) return keep;
    const int finer = masked_finer(equal);
    int took[2] = {0, 0};
    for (int i = 0; i < 2; ++i) {
      uint32_t count = 0;
      int longest = 0;
      each([&](const Row &r) {
        const int in = parts(r, i ? finer : keep);
        count += r.items * in;
        longest = max(longest, r.items ? (r.tiles + in - 1) / in : 0);
      });
      longest = most(longest);
      const int rounds = static_cast<int>((sum(count) + share - 1) / static_cast<uint32_t>(share));
      took[i] = min(rounds * longest, equal + longest) + 2 * rounds;  // two tiles to start a part
    }
    return took[1] && took[1] < took[0] ? finer : keep;
  }
  static __device__ __forceinline__ int parts(const Row &r, int limit) {
    return r.tiles > limit ? static_cast<int>(static_cast<uint32_t>(r.tiles + limit - 1) / static_cast<uint32_t>(limit)) : 1;
  }
  // Items in parts come first, then the whole ones, by halves.
  static __device__ __forceinline__ int order(const Row &r, int limit) {
    return r.tiles > limit ? 0 : 2 * r.tiles > limit ? 1 : 4 * r.tiles > limit ? 2 : 3;
  }
  // Part `at` of sequence b's items, whose number in all is `index`.  Uniform.
  __device__ __forceinline__ void take(MaskedPart<MODE> &p, int b, int in, int at, int index) const {
    p.b = b;
    p.parts = in;
    p.item = at;
    p.part = 0;
    p.slot = index;  // those in parts come first, below kSlots share
    p.seq = seq(b);
    p.seq.first = __builtin_amdgcn_readfirstlane(p.seq.first);
    p.seq.n = __builtin_amdgcn_readfirstlane(p.seq.n);
    p.seq.len = __builtin_amdgcn_readfirstlane(p.seq.len);
    if (in > 1) {
      p.item = at / in;
      p.part = at - p.item * in;
    }
    span(p.seq, p.item, p.to, p.gap_from, p.gap);
    p.from = 0;
    p.end = p.to - p.gap;
    if (in > 1) {  // the first ones take a tile more where they do not come out even
      const int t = tiles(p.to, p.gap), each = t / in, more = t - each * in;
      p.from = (p.part * each + min(p.part, more)) * FORM::kStep;
      p.end = min(((p.part + 1) * each + min(p.part + 1, more)) * FORM::kStep, p.end);
    }
  }
  // The part that this workgroup, number `at` of its head's, takes.  `share`: workgroups of a head that the card holds at once;
  // cut: how many of the parts have others.  Uniform; every wave looks at all sequences, one a lane, or where they are more at
  // what masked_plan_kernel left.
  __device__ __forceinline__ bool find(int at, int share, MaskedPart<MODE> &p, uint32_t &cut) const {
    const int lane = threadIdx.x & 63, n = rows.batch + 2;
    cut = 0;
    if (n > kPlanNear) {
      const int limit = plan[0];
      cut = plan[1];
      const int32_t *upto = plan + 2;  // running counts of parts, [order, sequence]
      int lo = 0, size = 4 * n;
      if (!limit || at >= upto[size - 1]) return false;
      while (size > 1) {  // the first above `at`
        const int step = (size + 63) / 64, i = min((lane + 1) * step, size) - 1;
        const int l = __builtin_ctzll(__ballot(upto[lo + i] > at));
        lo += l * step;
        size = min(step, size - l * step);
      }
      uint64_t unused = 0;
      const int b = lo % n, before = lo ? __builtin_amdgcn_readfirstlane(upto[lo - 1]) : 0;
      take(p, b, __builtin_amdgcn_readfirstlane(parts(row(b, unused), limit)), at - before, at);
      return true;
    }
    uint64_t held = 0;
    const Row near = row(lane, held);
    const uint32_t all = wave_sum(static_cast<uint32_t>(near.items * near.tiles));
    // offsets that do not ascend: the sequences' rows add up to more than there are
    if (wave_sum(held) != static_cast<uint64_t>(rows.rows)) return false;
    const auto most = [](int x) {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o, 64));
      return x;
    };
    const int limit = limit_of(all, share, [&](auto f) { f(near); }, [](uint32_t x) { return wave_sum(x); }, most);
    const int near_parts = parts(near, limit), mine = order(near, limit), index = at;
    if (at == 0) cut = wave_sum(static_cast<uint32_t>(near_parts > 1 ? near.items * near_parts : 0));
    for (int o = 0; o < 4; ++o) {
      const int count = mine == o ? near.items * near_parts : 0;
      const int upto = static_cast<int>(wave_scan(static_cast<uint32_t>(count)));
      const uint64_t past = __ballot(upto > at);
      if (past) {
        const int l = __builtin_ctzll(past);
        take(p, l, __builtin_amdgcn_readlane(near_parts, l),
             at - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(count, l)), index);
        return true;
      }
      at -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
  }
};

// Of more sequences than a wave has lanes: the limit of parts (0: offsets that do not ascend), how many parts have others, and the
// running counts of parts over orders and sequences.  One workgroup, before the others.  (Where each of them walked over all sequences
// itself, trees of 4 nodes behind 496 positions, 32 / 8 heads, took 1599 us for 1024 sequences, and 409 with this; 194 and 113 for 256.)
constexpr int kPlanThreads = 1024;
template <int MODE, class FORM>
__global__ __launch_bounds__(kPlanThreads) void masked_plan_kernel(const int32_t *__restrict__ starts, const int32_t *__restrict__ lens,
                                                                   int batch, int rows, int grp, int capacity, MaskedRule rule,
                                                                   int share, int32_t *__restrict__ out) {
  using Plan = MaskedPlan<MODE, FORM>;
  constexpr int kPlanWaves = kPlanThreads / 64;
  __shared__ uint64_t of_wave[kPlanWaves];
  const Plan plan{{starts, batch, rows, grp}, lens, capacity, rule, nullptr};
  const int n = batch + 2, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto gather = [&](uint64_t x, auto join) {  // of_wave[w] for every wave
    __syncthreads();  // what was there has been read
    if (lane == 0) of_wave[wave] = x;
    __syncthreads();
    uint64_t y = of_wave[0];
    for (int w = 1; w < kPlanWaves; ++w) y = join(y, of_wave[w]);
    return y;
  };
  const auto sum = [&](uint64_t x) { return gather(wave_sum(x), [](uint64_t p, uint64_t q) { return p + q; }); };
  const auto most = [&](int x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o, 64));
    return static_cast<int>(gather(static_cast<uint64_t>(x), [](uint64_t p, uint64_t q) { return max(p, q); }));
  };
  uint64_t held = 0, unused = 0;
  const typename Plan::Row near = plan.row(threadIdx.x, held);
  uint32_t own = near.items * near.tiles;
  for (int b = threadIdx.x + kPlanThreads; b < n; b += kPlanThreads) {
    const typename Plan::Row r = plan.row(b, held);
    own += r.items * r.tiles;
  }
  const uint32_t all = static_cast<uint32_t>(sum(own));
  if (sum(held) != static_cast<uint64_t>(rows)) {
    if (threadIdx.x == 0) out[0] = out[1] = 0;
    return;
  }
  const auto each = [&](auto f) {
    f(near);
    for (int b = threadIdx.x + kPlanThreads; b < n; b += kPlanThreads) f(plan.row(b, unused));
  };
  const int limit = Plan::limit_of(all, share, each, [&](uint32_t x) { return static_cast<uint32_t>(sum(x)); }, most);
  uint32_t before = 0, cut = 0;
  for (int o = 0; o < 4; ++o) {
    for (int b0 = 0; b0 < n; b0 += kPlanThreads) {
      const int b = b0 + threadIdx.x;
      const typename Plan::Row r = b0 ? plan.row(b, unused) : near;
      const uint32_t upto = wave_scan(static_cast<uint32_t>(Plan::order(r, limit) == o ? r.items * Plan::parts(r, limit) : 0));
      __syncthreads();  // what was there has been read
      if (lane == 63) of_wave[wave] = upto;
      __syncthreads();
      uint32_t ahead = 0, total = 0;
      for (int w = 0; w < kPlanWaves; ++w) {
        ahead += w < wave ? static_cast<uint32_t>(of_wave[w]) : 0;
        total += static_cast<uint32_t>(of_wave[w]);
      }
      if (b < n) out[2 + o * n + b] = static_cast<int32_t>(before + ahead + upto);
      before += total;
    }
    if (o == 0) cut = before;
  }
  if (threadIdx.x == 0) {
    out[0] = limit;
    out[1] = static_cast<int32_t>(cut);
  }
}
// Its words, if it runs.
constexpr int64_t masked_plan_words(int64_t batch) { return batch + 2 > kPlanNear ? 2 + 4 * (batch + 2) : 0; }

// Where an item's parts and its outputs go.
struct MaskedOut {
  uint16_t *out;    // the item's first token and head
  int64_t row;      // from token to token
  float *part;      // [rows of the item][D + 2]; null: outputs are final
};

// 16 rows of an item by the wave alone, K and V straight from memory (attn_tile), for tiles whose V has an infinity or NaN that only
// some rows see.  A function of its own: inlined, its registers would be the kernel's.
template <int MODE>
struct MaskedSeen {
  MaskedSeq<MODE> s;
  int token, a, b, gap_from, gap;  // this lane's token, and the wave's
  uint32_t mine;
  bool every;
  __device__ __forceinline__ int place(int v) const { return v < gap_from ? v : v + gap; }
  __device__ __forceinline__ void look(int tile) {
    every = s.whole(a, b, tile, tile + 32);
    mine = ~0u;
    if (!every) mine = static_cast<uint32_t>(s.bits(token, tile));
  }
  __device__ __forceinline__ bool sees(int p) const { return (mine >> (p & 31)) & 1; }
  __device__ __forceinline__ bool any(int) const { return true; }
  __device__ __forceinline__ bool whole(int) const { return every; }
};
template <int MODE>
struct MaskedRows {
  KvSource<true> src;
  MaskedSeen<MODE> seen;
  const uint16_t *q;  // the item's sequence's first row, its first head
  int64_t q_row, q_head;
  MaskedOut to;
  int all, grp, r0, from, end;  // rows of the sequence, heads of a token, the item's first row, virtual positions that are looked at
  float scale2;
};
template <int D, int DT, int MODE>
__device__ __attribute__((noinline)) void masked_rows16(const MaskedRows<MODE> &p, int at0) {
  const int lane = threadIdx.x & 63, i16 = lane & 15, j = lane >> 4, at = min(p.r0 + at0 + i16, p.all - 1);
  const int token = at / p.grp, head = at - token * p.grp;
  uint4 qf[D / 32];
  const uint16_t *qp = p.q + token * p.q_row + head * p.q_head + 8 * j;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) qf[c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);
  MaskedSeen<MODE> seen = p.seen;
  seen.token = token;
  AttnRows<D> a;
  attn_clear(a);
  attn_walk<D, DT, true, true>(a, p.src, qf, p.from, p.end, 32, seen, p.scale2, lane);
  const float l = attn_row_sum(a.l);
  if (p.r0 + at0 + i16 >= p.all) return;
  if (p.to.part) {
    float *z = p.to.part + (at0 + i16) * (D + 2);
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
  uint16_t *y = p.to.out + token * p.to.row + head * D + (D / 16) * 4 * j;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < D / 16; c += 2) {
      const float lo = l == 0.f ? 0.f : a.o[c][r] / l, hi = l == 0.f ? 0.f : a.o[c + 1][r] / l;
      *reinterpret_cast<uint32_t *>(y + (D / 16) * r + c) = attn_pack2<DT>(lo, hi);
    }
}

// Of an item's first part: its slot, how many there are, the item's first row counted from the sequence's, and the packed row that
// the sequence begins at.  Of the others: no parts.  And how many slots there are, from the first workgroup.
template <int MODE, class FORM>
__device__ __forceinline__ bool masked_find(const MaskedPlan<MODE, FORM> &plan, int kvh, int kh, int share, int4 *joins,
                                            MaskedPart<MODE> &p) {
  uint32_t cut;
  const int at = blockIdx.x / kvh;
  const bool found = plan.find(at, share, p, cut);
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) joins->x = cut;
    if (found && p.parts > 1)
      joins[1 + p.slot * kvh + kh] = make_int4(p.part == 0 ? p.parts : 0, min(p.seq.n * plan.rows.grp - p.item * FORM::kItem, FORM::kItem),
                                               p.item * FORM::kItem, p.seq.first);
  }
  return found;
}

template <int D, int DT, int MODE>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void masked_wide_kernel(
    const uint16_t *__restrict__ q, int64_t q_row, int64_t q_head, const uint16_t *__restrict__ k, int64_t kpage,
    int64_t khead, int64_t krow, const uint16_t *__restrict__ v, int64_t vpage, int64_t vhead, int64_t vrow, int pages,
    int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens,
    const int32_t *__restrict__ starts, int batch, int rows, int kvh, int grp, MaskedRule rule, int share, int slot_rows,
    float scale2, uint32_t flip, const int32_t *__restrict__ planned, float *__restrict__ parts, int4 *__restrict__ joins,
    uint16_t *__restrict__ out) {
  using T = PromptTile<D>;
  constexpr int kStage = T::kStage, kS = kTile / 32;
  extern __shared__ __attribute__((aligned(1024))) int8_t masked_smem[];  // two stages of K and V
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i32 = lane & 31, h = lane >> 5;
  const int kh = blockIdx.x % kvh;
  const MaskedPlan<MODE, Wide> plan{{starts, batch, rows, grp}, lens, width << shift, rule, planned};
  MaskedPart<MODE> p;
  if (!masked_find(plan, kvh, kh, share, joins, p)) return;
  const MaskedSeq<MODE> &seq = p.seq;
  const int from = __builtin_amdgcn_readfirstlane(p.from), end = __builtin_amdgcn_readfirstlane(p.end);
  const int mask = (1 << shift) - 1;
  // Of this lane's 16 bytes of a load: their chunk in LDS, and their bytes behind the load's first row.  The chunks of a wave's
  // loads differ by constants, for a wave's rows are 16.
  constexpr int kOf = 64 / T::kChunks;  // rows of a load
  static_assert(T::kLoads * kOf == 16, "a wave loads 16 rows");
  const uint32_t kx = T::k_chunk(lane / T::kChunks, lane % T::kChunks), kl = 2 * (lane / T::kChunks) * static_cast<uint32_t>(krow);
  const uint32_t vx = T::v_chunk(lane / T::kChunks, lane % T::kChunks), vl = 2 * (lane / T::kChunks) * static_cast<uint32_t>(vrow);

  const auto place = [&](int vp) { return vp < p.gap_from ? vp : vp + p.gap; };
  const int last = end > 0 ? (end <= p.gap_from ? end : end + p.gap) - 1 : 0;  // the part's last position

  const int n_rows = seq.n * grp, r0 = p.item * kRows + wave * 32, row_at = r0 + i32;
  const bool row = row_at < n_rows;
  const int token = row ? rule.group(row_at) : 0, head = kh * grp + (row ? row_at - token * grp : 0);
  const int wave_a = rule.group(r0), wave_b = min(rule.group(r0 + 31), seq.n - 1);
  uint4 qf[D / 16];
  const uint16_t *qp = q + (seq.first + token) * q_row + head * q_head + 8 * h;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    const uint4 x = *reinterpret_cast<const uint4 *>(qp + 16 * c);
    qf[c] = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
  }

  const uint16_t *kb = k + kh * khead, *vb = v + kh * vhead;
  const int32_t *pg = table + static_cast<int64_t>(min(p.b, batch - 1)) * width;
  const auto entry = [&](int vp) { return pg[min(place(vp) + lane, last) >> shift]; };
  const auto load = [&](int vp, int id, int8_t *stage) {
    const int tile = min(place(vp), last);  // past the last tile: rows that nothing reads
    if (tile + kTile <= last + 1) {
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        const int slot = (wave * T::kLoads + i) * 64;
        const int64_t pid = __builtin_amdgcn_readlane(id, slot / T::kChunks);  // the rows of one load lie in one page
        const int64_t in = (tile + slot / T::kChunks) & mask;
        prompt_lds_load16(kb + pid * kpage + in * krow, ((kx ^ T::k_chunk(i * kOf, 0)) << 4) + kl, stage + slot * 16);
        prompt_lds_load16(vb + pid * vpage + in * vrow, ((vx ^ T::v_chunk(i * kOf, 0)) << 4) + vl, stage + T::kBytes + slot * 16);
      }
      return;
    }
    // the last tile, with rows past the end in place of which it takes the last one.  (The lane is new to the compiler, which
    // would work these offsets out ahead of the loop and keep them.)
    int ln = lane;
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      const int slot = (wave * T::kLoads + i) * 64;
      const int64_t pid = __builtin_amdgcn_readlane(id, slot / T::kChunks);
      const int r = slot / T::kChunks + ln / T::kChunks, c = ln % T::kChunks, pos = min(tile + r, last) & mask;
      prompt_lds_load16(kb + pid * kpage, 2 * (pos * static_cast<uint32_t>(krow) + 8 * T::k_chunk(r, c)), stage + slot * 16);
      prompt_lds_load16(vb + pid * vpage, 2 * (pos * static_cast<uint32_t>(vrow) + 8 * T::v_chunk(r, c)), stage + T::kBytes + slot * 16);
    }
  };
  const auto fix = [&](int id, uint64_t &there) {  // page numbers outside the pool: page 0, unseen
    const bool ok = id >= 0 && id < pages;
    there = __ballot(ok);
    return ok ? id : 0;
  };

  f16_t o[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  uint64_t there = 0;  // which positions of the tile that is on its way exist
  int next_entry = 0, stage = 0;
  if (end > from) {
    load(from, fix(entry(from), there), masked_smem);
    next_entry = entry(from + kTile);
  }
  uint32_t odd = 0;  // an infinity or NaN in V where only some of the wave's rows see it
  for (int vp = from; vp < end; vp += kTile) {
    // this tile's loads have landed, every wave's, and the stage of the last tile has been read
    prompt_wait();
    const uint64_t ok = there;
    load(vp + kTile, fix(next_entry, there), masked_smem + (kStage - stage));
    next_entry = entry(vp + 2 * kTile);
    const int8_t *ks = masked_smem + stage, *vs = ks + T::kBytes;
    stage = kStage - stage;
    if (r0 >= n_rows) continue;  // no rows: it loads for the others
    const int tile = place(vp);
    uint64_t vis = ~uint64_t(0);
    const bool some = !seq.whole(wave_a, wave_b, tile, tile + kTile) || ok != ~uint64_t(0);
    if (some) {
      vis = row ? seq.bits(token, tile) & ok : 0;
      if (!__any(vis != 0)) continue;
    }
    f16_t s[kS];
    prompt_scores<D, DT>(ks, qf, s, i32, h);
    if (some) {
      vis >>= 4 * h;
#pragma unroll
      for (int t = 0; t < kS; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = (vis >> (32 * t + 8 * (r >> 2) + (r & 3))) & 1 ? s[t][r] : -INFINITY;
      prompt_odd_values<D, DT>(odd, vs, lane);
    }
#include "prompt_weigh.inc"
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing on its way to LDS when the workgroup ends
  if (r0 >= n_rows) return;
  const MaskedOut dst{out + (static_cast<int64_t>(seq.first) * kvh * grp + kh * grp) * D, static_cast<int64_t>(kvh) * grp * D,
                      p.parts > 1 ? parts + (static_cast<int64_t>(p.slot) * kvh + kh) * slot_rows * (D + 2) : nullptr};
  if (__any(odd)) {
    // 0 times an infinity is no zero: these rows once more, with what they do not see left out one position at a time
    MaskedRows<MODE> w;
    w.src = {kb, vb, kpage, krow, vpage, vrow, pg, shift, mask, pages, last >> shift};
    w.seen = {seq, 0, wave_a, wave_b, p.gap_from, p.gap, 0, false};
    w.q = q + seq.first * q_row + kh * grp * q_head;
    w.q_row = q_row;
    w.q_head = q_head;
    w.to = dst;
    w.all = n_rows;
    w.grp = grp;
    w.r0 = p.item * kRows;
    w.from = from;
    w.end = end;
    w.scale2 = flip ? -scale2 : scale2;
    for (int half = 0; half < 2; ++half)
      if (r0 + 16 * half < n_rows) masked_rows16<D, DT, MODE>(w, 32 * wave + 16 * half);
    return;
  }
  if (!row) return;
  l += __shfl_xor(l, 32, 64);
  if (p.parts > 1) {
    float *z = dst.part + (wave * 32 + i32) * (D + 2);
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        *reinterpret_cast<float2 *>(z + 32 * d + 8 * (r >> 2) + 4 * h + (r & 3)) = make_float2(o[d][r], o[d][r + 1]);
    if (h == 0) *reinterpret_cast<float2 *>(z + D) = make_float2(m, l);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  uint16_t *y = dst.out + token * dst.row + (head - kh * grp) * D + 4 * h;
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

// Workgroups of a CU whose registers hold two tiles each.
constexpr int masked_round(int dim) { return dim == 64 ? 4 : dim == 128 ? 2 : 1; }

template <int D, int DT, int MODE>
__global__ __launch_bounds__(64 * kWaves, masked_round(D)) void masked_narrow_kernel(
    const uint16_t *__restrict__ q, int64_t q_row, int64_t q_head, const uint16_t *__restrict__ k, int64_t kpage,
    int64_t khead, int64_t krow, const uint16_t *__restrict__ v, int64_t vpage, int64_t vhead, int64_t vrow, int pages,
    int shift, const int32_t *__restrict__ table, int width, const int32_t *__restrict__ lens,
    const int32_t *__restrict__ starts, int batch, int rows, int kvh, int grp, MaskedRule rule, int share, int slot_rows,
    float scale2, uint32_t flip, const int32_t *__restrict__ planned, float *__restrict__ parts, int4 *__restrict__ joins,
    uint16_t *__restrict__ out) {
  extern __shared__ __attribute__((aligned(16))) float narrow_smem[];  // the four waves' states (attn_meet)
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, j = lane >> 4;
  const int kh = blockIdx.x % kvh;
  const MaskedPlan<MODE, Narrow> plan{{starts, batch, rows, grp}, lens, width << shift, rule, planned};
  MaskedPart<MODE> p;
  if (!masked_find(plan, kvh, kh, share, joins, p)) return;
  const MaskedSeq<MODE> &seq = p.seq;
  const int n_rows = seq.n * grp, r0 = p.item * 16, held = min(n_rows - r0, 16), row_at = r0 + min(i16, held - 1);
  const int token = rule.group(row_at), head = kh * grp + row_at - token * grp;
  uint4 qf[D / 32];
  const uint16_t *qp = q + (seq.first + token) * q_row + head * q_head + 8 * j;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) qf[c] = *reinterpret_cast<const uint4 *>(qp + 32 * c);
  const KvSource<true> src{k + kh * khead, v + kh * vhead, kpage, krow, vpage, vrow,
                           table + static_cast<int64_t>(min(p.b, batch - 1)) * width, shift, (1 << shift) - 1, pages,
                           p.to > 0 ? (p.to - 1) >> shift : 0};
  const MaskedSeen<MODE> seen{seq, token, rule.group(r0), min(rule.group(r0 + 15), seq.n - 1), p.gap_from, p.gap, 0, false};
  AttnRows<D> a;
  attn_clear(a);
  attn_walk<D, DT, true, true>(a, src, qf, p.from + 32 * wave, p.end, Narrow::kStep, seen, flip ? -scale2 : scale2, lane);
  a.l = attn_row_sum(a.l);

  float *part = parts + (static_cast<int64_t>(p.slot) * kvh + kh) * slot_rows * (D + 2);
  attn_meet<D, kWaves>(a, narrow_smem, held, lane, wave, [&](int row, int d, float4 o, float m, float l) {
    if (p.parts == 1) {
      const int t = rule.group(r0 + row);
      *reinterpret_cast<uint2 *>(out + ((seq.first + static_cast<int64_t>(t)) * kvh * grp + kh * grp + r0 + row - t * grp) * D + d) =
          attn_outputs<DT>(o, l);
    } else {
      float2 *z = reinterpret_cast<float2 *>(part + row * (D + 2));  // rows are 8 bytes apart
      z[d / 2] = make_float2(o.x, o.y);
      z[d / 2 + 1] = make_float2(o.z, o.w);
      if (d == 0) z[D / 2] = make_float2(m, l);
    }
  });
}

// The parts of an item meet: 16 of its rows in a workgroup, four in a wave, 16 lanes to each.
template <int D, int DT, class FORM>
__global__ __launch_bounds__(256) void masked_join_kernel(int kvh, int grp, int slot_rows, MpDivisor group,
                                                          const float *__restrict__ parts, const int4 *__restrict__ joins,
                                                          uint16_t *__restrict__ out) {
  const int slot = blockIdx.x / kvh, kh = blockIdx.x - slot * kvh, i16 = threadIdx.x & 15;
  const int4 of = joins[1 + blockIdx.x];  // open past the last slot
  const int r = blockIdx.y * 16 + (threadIdx.x >> 4);
  if (slot >= joins->x || of.x < 2 || r >= of.y) return;
  const int64_t step = static_cast<int64_t>(kvh) * slot_rows * (D + 2) / 2;  // from part to part
  const float2 *z = reinterpret_cast<const float2 *>(parts + (static_cast<int64_t>(blockIdx.x) * slot_rows + r) * (D + 2));
  float m = -INFINITY, l = 0.f;
  float2 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) o[c] = make_float2(0.f, 0.f);
#pragma unroll 8
  for (int p = 0; p < of.x; ++p, z += step) {
    const float2 ml = z[D / 2];
    float2 x[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) x[c] = z[16 * c + i16];
    const float top = fmaxf(m, ml.x), f = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    const float g = ml.x == top ? 1.0f : __builtin_amdgcn_exp2f(ml.x - top);
    m = top;
    l = l * f + ml.y * g;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) o[c] = make_float2(o[c].x * f + x[c].x * g, o[c].y * f + x[c].y * g);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const bool none = l == 0.f;
  const int token = group(of.z + r), head = kh * grp + of.z + r - token * grp;
  uint32_t *y = reinterpret_cast<uint32_t *>(out + ((static_cast<int64_t>(of.w) + token) * kvh * grp + head) * D);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) y[16 * c + i16] = attn_pack2<DT>(none ? 0.f : o[c].x * inv, none ? 0.f : o[c].y * inv);
}

// Workgroups of a head: as many as fit the card at once.
template <class FORM>
int64_t masked_share(int64_t kvh, int dim) {
  const int64_t round = FORM::kItem == kRows ? (dim == 256 ? 1 : 2) : masked_round(dim);
  const int64_t n = round * mp_cu_count() / kvh;
  return n > 1 ? n : 1;
}
template <class FORM>
int64_t masked_slot_rows(int64_t rows, int64_t grp) {
  return rows * grp < FORM::kItem ? rows * grp : FORM::kItem;
}
template <class FORM>
int64_t masked_items(int64_t rows, int64_t grp, int64_t batch) {
  return rows * grp / FORM::kItem + batch + 4;
}
// The most positions that a row's tile looks at.
int64_t masked_reach(int64_t capacity, int64_t window, int64_t sinks) {
  return window ? std::min(capacity, window + sinks + 3 * 64) : capacity;
}
// Narrow: little work in all, counted in rounds of narrow tiles, which start sooner, though every 16 rows read an item's positions
// again; or few rows of a sequence and key-value head on the average, if it were little work with all rows in one of them, for the
// host does not know which sequences have new tokens.  Trees of bf16, us in the narrow and the wide form, by rows of a sequence and
// head:
//   one sequence of 1500, 32 / 8 heads of 128      64: 15, 22   256: 22, 35 (6 rounds)
//   one of 16000, 64 / 8                           64: 37, 44 (18)  128: 54, 56 (27)  192: 69, 47
//   16 of 3000, 64 / 8                             16: 39, 40   32: 41, 42         64: 66, 45 (39)
//   64 of 2000, 64 / 8                              8: 102, 113  16: 104, 113   32: 123, 114   64: 189, 119
//   4 of 2000, 16 / 4 heads of 256                128: 39, 45 (14)                192: 68, 42 (19)
//   32 of 3000, 8 / 8 heads of 256                 4: 147, 157  16: 150, 157   24: 191, 193      48: 258, 199
//   64 of 1000, 32 / 8 heads of 64                  4: 33, 41   16: 34, 41     32: 40, 41
//   16 of 2000, 28 / 4 heads of 64                 28: 15, 18                     56: 22, 20 (7)
// New tokens of one sequence among 64 that the call names, behind 8000 positions, 32 / 8 heads of 128:
//                                                128: 42, 65  256: 59, 48   512: 94, 54   2048: 317, 105
bool masked_narrow(int64_t rows, int64_t grp, int64_t kvh, int dim, int64_t batch, int64_t reach) {
  const int64_t slots = masked_round(dim) * mp_cu_count(), rounds = dim == 64 ? 4 : dim == 128 ? 18 : 12;
  const int64_t tiles = mp_cdiv(reach, Narrow::kStep) + 6;  // an item starts and ends in the time of six
  const int64_t items = rows * grp <= 32 * batch ? mp_cdiv(rows * grp, Narrow::kItem) : masked_items<Narrow>(rows, grp, batch);
  return items * tiles * kvh <= rounds * slots;
}

struct MaskedCall {
  const void *q;
  int64_t q_row, q_head, rows;
  int nh, kvh, head_dim;
  const mp_pages *cache;
  const int32_t *lens, *starts;
  int64_t batch;
  MaskedRule rule;
  float scale;
  void *out;
  int dtype;
  void *workspace;
  size_t workspace_bytes;
  hipStream_t stream;
  int64_t reach;
};

template <class FORM>
size_t masked_workspace(int64_t rows, int64_t nh, int64_t kvh, int dim, int64_t batch) {
  const int64_t grp = nh / kvh;
  const int64_t slots = kSlots * masked_share<FORM>(kvh, dim) * kvh;
  return static_cast<size_t>(1 + slots) * sizeof(int4) +
         static_cast<size_t>(slots * masked_slot_rows<FORM>(rows, grp)) * (dim + 2) * sizeof(float) +
         static_cast<size_t>(masked_plan_words(batch)) * sizeof(int32_t);
}
size_t masked_workspace(int64_t rows, int64_t nh, int64_t kvh, int dim, int64_t batch, int64_t reach) {
  return masked_narrow(rows, nh / kvh, kvh, dim, batch, reach) ? masked_workspace<Narrow>(rows, nh, kvh, dim, batch)
                                                               : masked_workspace<Wide>(rows, nh, kvh, dim, batch);
}

template <int D, int DT, int MODE, class FORM>
int masked_start(const MaskedCall &c, int shift) {
  constexpr bool kIsWide = FORM::kItem == kRows;
  const int grp = c.nh / c.kvh, share = static_cast<int>(masked_share<FORM>(c.kvh, D));
  const int slot_rows = static_cast<int>(masked_slot_rows<FORM>(c.rows, grp));
  int4 *joins = static_cast<int4 *>(c.workspace);
  float *parts = reinterpret_cast<float *>(joins + 1 + kSlots * static_cast<int64_t>(share) * c.kvh);
  int32_t *planned = reinterpret_cast<int32_t *>(parts + kSlots * static_cast<int64_t>(share) * c.kvh * slot_rows * (D + 2));
  // the sign of the scale goes to the queries, so that the largest product gives the largest score; a scale of 0 becomes the
  // smallest normal number, which leaves every finite score 0 and a masked one -inf
  const uint32_t flip = c.scale < 0.f ? 0x80008000u : 0u;
  const float scale2 = fmaxf(fabsf(c.scale) * kLog2e, FLT_MIN);
  constexpr int kLds = kIsWide ? 2 * PromptTile<D>::kStage : kWaves * 16 * (D + 6) * static_cast<int>(sizeof(float));
  constexpr auto kKernel = kIsWide ? &masked_wide_kernel<D, DT, MODE> : &masked_narrow_kernel<D, DT, MODE>;
  if (kLds > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void *>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess)
    return MP_ERR_HIP;
  const mp_pages &p = *c.cache;
  const int64_t blocks = (masked_items<FORM>(c.rows, grp, c.batch) + masked_more(share)) * c.kvh;
  if (blocks > kMpMaxGroups) return MP_ERR_SHAPE;
  if (masked_plan_words(c.batch)) {
    hipLaunchKernelGGL((masked_plan_kernel<MODE, FORM>), dim3(1), dim3(kPlanThreads), 0, c.stream, c.starts, c.lens,
                       static_cast<int>(c.batch), static_cast<int>(c.rows), grp, static_cast<int>(p.width << shift), c.rule, share,
                       planned);
    MP_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL(kKernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * kWaves), kLds, c.stream,
                     static_cast<const uint16_t *>(c.q), c.q_row, c.q_head, static_cast<const uint16_t *>(p.k), p.k_page,
                     p.k_head, p.k_row, static_cast<const uint16_t *>(p.v), p.v_page, p.v_head, p.v_row, static_cast<int>(p.pages),
                     shift, p.table, static_cast<int>(p.width), c.lens, c.starts, static_cast<int>(c.batch),
                     static_cast<int>(c.rows), c.kvh, grp, c.rule, share, slot_rows, scale2, flip, planned, parts, joins,
                     static_cast<uint16_t *>(c.out));
  MP_CHECK_LAUNCH();
  if (c.reach > FORM::kStep) {  // else items of one tile, which are never cut
    hipLaunchKernelGGL((masked_join_kernel<D, DT, FORM>), dim3(static_cast<unsigned>(kSlots * share * c.kvh), FORM::kItem / 16),
                       dim3(256), 0, c.stream, c.kvh, grp, slot_rows, c.rule.group, parts, joins, static_cast<uint16_t *>(c.out));
    MP_CHECK_LAUNCH();
  }
  return MP_OK;
}
template <int D, int DT, int MODE>
int masked_start(const MaskedCall &c, int shift) {
  return masked_narrow(c.rows, c.nh / c.kvh, c.kvh, D, c.batch, c.reach) ? masked_start<D, DT, MODE, Narrow>(c, shift)
                                                                         : masked_start<D, DT, MODE, Wide>(c, shift);
}

template <int MODE>
int masked_launch(MaskedCall c) {
  if (!c.q || !c.cache || !c.cache->k || !c.cache->v || !c.cache->table || !c.lens || !c.starts || !c.out || !c.workspace)
    return MP_ERR_ARG;
  if (c.dtype != MP_F16 && c.dtype != MP_BF16) return MP_ERR_DTYPE;
  if (!std::isfinite(c.scale * kLog2e)) return MP_ERR_ARG;
  const mp_pages &p = *c.cache;
  int shift = -1;
  for (int s = 3; s < 16; ++s)
    if (p.page_size == 1 << s) shift = s;
  if (shift < 0 || p.pages < 1 || p.pages > INT32_MAX || p.width < 1 || p.width > (1 << 30) >> shift) return MP_ERR_SHAPE;
  if (c.rows < 0 || c.rows > INT32_MAX || c.batch < 1 || c.batch > kMaxBatch) return MP_ERR_SHAPE;
  if (c.nh < 1 || c.kvh < 1 || c.nh > 65536 || c.nh % c.kvh) return MP_ERR_SHAPE;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return MP_ERR_SHAPE;
  for (int64_t s : {c.q_row, c.q_head, p.k_page, p.k_head, p.k_row, p.v_page, p.v_head, p.v_row})
    if (s < 0 || s % 8) return MP_ERR_SHAPE;
  for (const void *x : {c.q, static_cast<const void *>(p.k), static_cast<const void *>(p.v), static_cast<const void *>(c.out),
                        static_cast<const void *>(c.workspace)})
    if (!mp_aligned(x, 16)) return MP_ERR_ALIGN;
  // byte offsets inside a page are 32 bits, and so are a head's tiles
  const int64_t grp = c.nh / c.kvh, reach = (int64_t(1) << 30) - 256, span = int64_t(1) << shift;
  if (p.k_row > reach / span || p.v_row > reach / span) return MP_ERR_SHAPE;
  if (c.rows * c.nh > INT32_MAX - kRows) return MP_ERR_SHAPE;
  if (masked_items<Narrow>(c.rows, grp, c.batch) * mp_cdiv(p.width << shift, kTile) > INT32_MAX) return MP_ERR_SHAPE;
  if (c.rows == 0) return MP_OK;
  if (mp_cu_count() <= 0) return MP_ERR_HIP;
  c.reach = masked_reach(p.width << shift, c.rule.window, c.rule.sinks);
  if (c.workspace_bytes < masked_workspace(c.rows, c.nh, c.kvh, c.head_dim, c.batch, c.reach)) return MP_ERR_WORKSPACE;
  c.rule.group = mp_divisor(static_cast<int>(grp));
#define MP_MASKED(DT)                                                        \
  return c.head_dim == 64 ? masked_start<64, DT, MODE>(c, shift)             \
                          : c.head_dim == 128 ? masked_start<128, DT, MODE>(c, shift) : masked_start<256, DT, MODE>(c, shift)
  if (c.dtype == MP_F16) MP_MASKED(MP_F16);
  MP_MASKED(MP_BF16);
#undef MP_MASKED
}

}  // namespace

extern "C" size_t mp_masked_workspace_bytes(int64_t rows, int nh, int kvh, int head_dim, int64_t batch, int64_t capacity,
                                            int64_t window, int64_t sinks) {
  if (rows <= 0 || rows > INT32_MAX || nh <= 0 || kvh <= 0 || nh % kvh || head_dim <= 0 || batch <= 0 || batch > kMaxBatch ||
      capacity <= 0 || window < 0 || window > 1 << 30 || sinks < 0 || sinks > 1 << 30 || mp_cu_count() <= 0)
    return 0;
  return masked_workspace(rows, nh, kvh, head_dim, batch, masked_reach(capacity, window, sinks));
}

extern "C" int mp_masked_item_rows(int64_t rows, int nh, int kvh, int head_dim, int64_t batch, int64_t capacity, int64_t window,
                                   int64_t sinks) {
  if (!mp_masked_workspace_bytes(rows, nh, kvh, head_dim, batch, capacity, window, sinks)) return 0;
  return masked_narrow(rows, nh / kvh, kvh, head_dim, batch, masked_reach(capacity, window, sinks)) ? Narrow::kItem : Wide::kItem;
}

extern "C" int mp_paged_tree_attention(const void *q, int64_t q_row, int64_t q_head, int64_t rows, int nh, int kvh, int head_dim,
                                       const mp_pages *cache, const int32_t *lens, const int32_t *starts, int64_t batch,
                                       const int64_t *masks, int64_t words, float scale, void *out, int dtype, void *workspace,
                                       size_t workspace_bytes, mp_stream_t stream) {
  if (!masks) return MP_ERR_ARG;
  if (words < 1 || words > 1024) return MP_ERR_SHAPE;
  return masked_launch<kTree>({q, q_row, q_head, rows, nh, kvh, head_dim, cache, lens, starts, batch,
                               {masks, static_cast<int>(words), 0, 0, {}}, scale, out, dtype, workspace, workspace_bytes,
                               reinterpret_cast<hipStream_t>(stream), 0});
}

extern "C" int mp_paged_prompt_window_attention(const void *q, int64_t q_row, int64_t q_head, int64_t rows, int nh, int kvh,
                                                int head_dim, const mp_pages *cache, const int32_t *lens, const int32_t *starts,
                                                int64_t batch, int64_t window, int64_t sinks, float scale, void *out, int dtype,
                                                void *workspace, size_t workspace_bytes, mp_stream_t stream) {
  if (window < 1 || window > 1 << 30 || sinks < 0 || sinks > 1 << 30) return MP_ERR_SHAPE;
  return masked_launch<kWindow>({q, q_row, q_head, rows, nh, kvh, head_dim, cache, lens, starts, batch,
                                 {nullptr, 0, static_cast<int>(window), static_cast<int>(sinks), {}}, scale, out, dtype, workspace,
                                 workspace_bytes, reinterpret_cast<hipStream_t>(stream), 0});
}
