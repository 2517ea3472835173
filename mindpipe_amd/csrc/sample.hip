// Tokens from logits at given random numbers, each row with its own temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T),  1 where x_i is the maximum
//   kept: the k largest (equal values: the lowest indexes), of those the shortest run from the largest down whose weights
//         reach p of their sum, of those the ones with w_i >= min-p; the largest is always kept
//   token: the first index, in index order, at which the kept weights' running sum exceeds u times their sum
//
// A token is decided by which side of a border a sum over the vocabulary falls on, so weights are computed in 64 bits
// and summed as whole numbers of 2^-44: sums of up to 2^19 of them, 2^63 in a row of equal values, fit unsigned 64 bits,
// and no order of additions changes them.
//
// Nothing is sorted.  A workgroup takes a row.  It counts the values into 2048 bins of equal width below the maximum (counts for
// top-k, weights for top-p) and so finds the bin that the border of the kept is in.  The values down to that bin, few as a
// rule, are copied to LDS in index order, and the rest is done on them (on the whole row, where they are more than
// kListed): the bin's values are counted into bins of neighbouring values down to single ones, which gives the border, a
// value and how many of its ties; then weights are summed by spans of indexes and the token looked up.
//
// A row's bytes are read once where registers hold it (256 rows of 128256 bf16 are 66 MB, 10 us at the rate of a read), and the
// weights bound it: some 30 instructions each, twice over the row with top-p (once for the sum that p is a share of, once for
// the spans).  Those rows, by filter: none 57 us, top-k 33, min-p 30, top-k and top-p 38, top-p alone 105 (128256 values of
// which more than the list holds are kept).
#include "wave_scan.h"

namespace {

constexpr int kMaxWaves = 16;
constexpr int kMaxVocab = 1 << 19;
constexpr int kSpan = 512;                     // indexes of one step of a wave: eight neighbours per lane
constexpr int kMaxSpans = kMaxVocab / kSpan + kMaxWaves;  // the waves' counts are rounded up
constexpr int kBins = 2048;
constexpr int kTable = 1024;                   // 2^(44 + j / 1024)
constexpr double kOne = 17592186044416.0;      // 2^44
constexpr float kReach = 32.0f;                // e^-32 < 2^-46: past it a weight is no part of 2^-44

constexpr int kListed = kSpan;                 // values of a wave that LDS has room for

struct SampleShared {
  double table[kTable];
  uint64_t mass[kBins];
  uint64_t span_mass[kMaxSpans];
  uint64_t wave_mass[kMaxWaves];
  uint64_t before_mass;
  uint32_t count[kBins];
  uint32_t span_ties[kMaxSpans];
  uint32_t wave_count[kMaxWaves];
  float top[kMaxWaves];
  int at[kMaxWaves];
  int found;
  uint32_t before_count;
  float value[kMaxWaves][kListed];
  int index[kMaxWaves][kListed];
  int listed[kMaxWaves];
};

// Eight neighbouring values from index i on, past the end -inf.
template <int DT>
struct Eight {
  static constexpr int kWords = DT == MP_F32 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const uint8_t *row, int i, int vocab, bool vec) {
    if (vec && i + 8 <= vocab) {
      const uint4 *p = reinterpret_cast<const uint4 *>(row + static_cast<int64_t>(i) * (kWords / 2));
#pragma unroll
      for (int c = 0; c < kWords / 4; ++c) {
        const uint4 x = p[c];
        w[4 * c] = x.x;
        w[4 * c + 1] = x.y;
        w[4 * c + 2] = x.z;
        w[4 * c + 3] = x.w;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == MP_F32) {
        w[e] = i + e < vocab ? reinterpret_cast<const uint32_t *>(row)[i + e] : 0xFF800000u;
      } else {
        const uint32_t h = i + e < vocab ? reinterpret_cast<const uint16_t *>(row)[i + e] : (DT == MP_F16 ? 0xFC00u : 0xFF80u);
        w[e / 2] = e & 1 ? w[e / 2] | h << 16 : h;
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == MP_F32) v[e] = __uint_as_float(w[e]);
      else if constexpr (DT == MP_BF16) v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
      else v[e] = mp_h2f(static_cast<uint16_t>(e & 1 ? w[e / 2] >> 16 : w[e / 2]));
    }
  }
};

__device__ __forceinline__ void sample_renew(uint32_t &w) { asm volatile("" : "+v"(w)); }

// The row: in registers where it has up to CH chunks, or else (CH = 0) in memory, read anew in every pass (from the L2,
// past the first).
template <int DT, int CH>
struct SampleRow {
  const uint8_t *row;
  int vocab, chunks;  // a wave's steps of kSpan values: wave w has the spans w * chunks ..
  bool vec;
  bool infinite = false;  // the maximum is +inf: such values are 0, all others -inf
  Eight<DT> held[CH > 0 ? CH : 1];

  __device__ __forceinline__ int first(int c) const { return ((threadIdx.x >> 6) * chunks + c) * kSpan + 8 * (threadIdx.x & 63); }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c < chunks) held[c].load(row, first(c), vocab, vec);
  }
  template <bool RAW>
  __device__ __forceinline__ void values(const Eight<DT> &x, float (&v)[8]) const {
    x.get(v);
    if (!RAW) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaxf(v[e], -INFINITY);  // NaN
    }
    if (infinite) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] == INFINITY ? 0.f : -INFINITY;
    }
  }
  // f(chunk, its eight values); RAW: NaN as it is, for what compares with it or takes it for the last bin
  template <bool RAW = false, class F>
  __device__ __forceinline__ void each(F f) {
    if constexpr (CH > 0) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (c < chunks) {
          // the words are new to the compiler in every pass: it would keep what it unpacked in the last one, and spill it
#pragma unroll
          for (int i = 0; i < Eight<DT>::kWords; ++i) sample_renew(held[c].w[i]);
          float v[8];
          values<RAW>(held[c], v);
          f(c, v);
        }
      return;
    }
    constexpr int kAhead = DT == MP_F32 ? 2 : 4;  // steps that are asked for before they are looked at
    Eight<DT> x[kAhead];
#pragma unroll
    for (int c = 0; c < kAhead; ++c)
      if (c < chunks) x[c].load(row, first(c), vocab, vec);
    for (int c0 = 0; c0 < chunks; c0 += kAhead) {
#pragma unroll
      for (int c = 0; c < kAhead; ++c) {
        if (c0 + c >= chunks) break;
        const Eight<DT> now = x[c];
        if (c0 + c + kAhead < chunks) x[c].load(row, first(c0 + c + kAhead), vocab, vec);
        float v[8];
        values<RAW>(now, v);
        f(c0 + c, v);
      }
    }
  }
  template <class F>
  __device__ __forceinline__ void one(int c, F f) const {
    Eight<DT> x;
    x.load(row, first(c), vocab, vec);
    float v[8];
    values<false>(x, v);
    f(c, v);
  }
  __device__ __forceinline__ int index(int c, int e) const { return first(c) + e; }
  __device__ __forceinline__ int span(int c) const { return (threadIdx.x >> 6) * chunks + c; }
};

// What of it is in LDS, in the same order: one chunk, `per` neighbours to a thread.
template <int W>
struct SampleList {
  const SampleShared *s;
  static constexpr int chunks = 1;
  int per, all;
  float v[8];
  // wave and place of the list's entry i
  __device__ __forceinline__ void find(int i, int &wave, int &at) const {
    wave = 0;
    at = i;
#pragma unroll
    for (int w = 0; w < W - 1; ++w) {
      const bool on = wave == w && at >= s->listed[w];
      at -= on ? s->listed[w] : 0;
      wave += on ? 1 : 0;
    }
  }
  __device__ __forceinline__ void load() {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = -INFINITY;
      if (e < per && per * static_cast<int>(threadIdx.x) + e < all) {
        int wave, at;
        find(per * threadIdx.x + e, wave, at);
        v[e] = s->value[wave][at];
      }
    }
  }
  template <bool RAW = false, class F>
  __device__ __forceinline__ void each(F f) { f(0, v); }
  template <class F>
  __device__ __forceinline__ void one(int, F f) const { f(0, v); }
  __device__ __forceinline__ int index(int, int e) const {
    int wave, at;
    find(per * threadIdx.x + e, wave, at);
    return s->index[wave][at];
  }
  __device__ __forceinline__ int span(int) const { return threadIdx.x >> 6; }
};

// Order of the values as unsigned numbers, without the trailing bits that are alike in all values of the type.
template <int DT>
constexpr int kDrop = DT == MP_F32 ? 0 : DT == MP_F16 ? 13 : 16;
template <int DT>
__device__ __forceinline__ uint32_t sample_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 is 0
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> kDrop<DT>;
}
template <int DT>
__device__ __forceinline__ float sample_value(uint32_t key) {
  const uint32_t k = key << kDrop<DT>, low = (1u << kDrop<DT>) - 1;
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~(k | low));
}

struct Weight {
  const double *table;  // LDS: 2^(44 + j / 1024)
  double top, rate;     // the largest value, 1024 log2 e / T
  // exp((v - top) / T) in units of 2^-44: 2^(k / 1024) from the table, its whole powers added to the exponent, and the rest of
  // the exponent, up to 2^-11, by a cubic (off by less than 2^-50).  -inf and NaN weigh 0, as what is below 2^-45 does.
  __device__ __forceinline__ uint64_t operator()(float v) const {
    const double magic = 1.5 * 0x1p52;  // a sum with it is whole
    const double y = fmax((static_cast<double>(v) - top) * rate, -64.0 * kTable);
    const double t = y + magic, r = y - (t - magic);
    const int k = __double2loint(t);
    const double q = r * fma(r, fma(r, 5.169222938345892e-11, 2.290978498068816e-07), 0.0006769015435155716);
    const double e = table[k & (kTable - 1)];
    const double b = __hiloint2double(__double2hiint(e) + ((k & ~(kTable - 1)) << 10), __double2loint(e));
    const double w = fma(b, q, b) + 0x1p52;  // below 2^45: the sum's last bits are the number
    return static_cast<uint64_t>(__double_as_longlong(w)) & 0xFFFFFFFFFFFFFull;
  }
};

struct Border {  // the kept: keys above `key`, and the first `ties` indexes at it
  uint32_t key, ties;
};
template <int DT>
__device__ __forceinline__ float border_value(const Border &b) { return b.key ? sample_value<DT>(b.key) : -INFINITY; }

// What a border is looked for by: so many values, or so much weight.
struct Target {
  bool by_mass;
  uint32_t count;
  double mass;
};

template <int W>
__device__ __forceinline__ void clear_bins(SampleShared &s) {
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kBins; b += 64 * W) {
    s.mass[b + threadIdx.x] = 0;
    s.count[b + threadIdx.x] = 0;
  }
  __syncthreads();
}

// Sum of the waves' `v` before this wave; `all`: of all of them.  One barrier.
template <int W, class U>
__device__ __forceinline__ U waves_before(U *of_wave, U v, U &all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (lane == 0) of_wave[wave] = v;
  __syncthreads();
  const U upto = wave_scan(lane < W ? of_wave[lane] : U(0));
  all = last_lane(upto);
  return __shfl(upto, wave, 64) - v;
}

// The first bin, from bin 0 up, at which the running count or mass reaches the target, with what lies before it; the last
// bin where none does.  The thread whose bins the target is reached in says so.
template <int W>
__device__ __forceinline__ int find_bin(SampleShared &s, const Target &t, uint32_t &count, uint64_t &mass) {
  constexpr int kOwn = kBins / 64 / W;  // a thread's bins
  const int tid = threadIdx.x;
  if (t.by_mass) {
    uint64_t own[kOwn], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum += own[i] = s.mass[kOwn * tid + i];
    const uint64_t scan = wave_scan(sum);
    uint64_t at = scan - sum + waves_before<W>(s.wave_mass, last_lane(scan), all);
    bool open = tid == 0 || static_cast<double>(at) < t.mass;
    if (open && (static_cast<double>(at + sum) >= t.mass || tid == 64 * W - 1)) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (open && (static_cast<double>(at + own[i]) >= t.mass || i == kOwn - 1)) {
          s.found = kOwn * tid + i;
          s.before_mass = at;
          open = false;
        }
        at += own[i];
      }
    }
  } else {
    uint32_t own[kOwn], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) sum += own[i] = s.count[kOwn * tid + i];
    const uint32_t scan = wave_scan(sum);
    uint32_t at = scan - sum + waves_before<W>(s.wave_count, last_lane(scan), all);
    bool open = tid == 0 || at < t.count;
    if (open && (at + sum >= t.count || tid == 64 * W - 1)) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (open && (at + own[i] >= t.count || i == kOwn - 1)) {
          s.found = kOwn * tid + i;
          s.before_count = at;
          open = false;
        }
        at += own[i];
      }
    }
  }
  __syncthreads();
  if (t.by_mass) mass = s.before_mass;
  else count = s.before_count;
  return s.found;
}

struct RowCall {
  float t, top, half, per;  // half of the maximum, bins per unit of half the distance to it (distances may pass fp32's range)
  int k;                   // 0: all
  bool by_p;
  float p, floor_p, u;
  int64_t *token;
  float *logprob;
};

__device__ __forceinline__ int bin_of(float v, const RowCall &c) {
  return static_cast<int>(fminf(fmaf(-0.5f, v, c.half) * c.per, static_cast<float>(kBins - 1)));  // also of -inf
}

// The border inside a bin: `count` and `mass` lie before the bin, of it the values above from.key, and from.ties at it.
template <int DT, int W, class X>
__device__ __forceinline__ Border find_border(SampleShared &s, X &x, const RowCall &c, const Weight &weight, int bin,
                                              const Target &goal, uint32_t count, uint64_t mass, Border from) {
  const int tid = threadIdx.x;
  // keys that may fall into the bin: its edges, with a margin for the roundings of bin_of
  const float near = bin / c.per, far = (bin + 1) / c.per, margin = 0x1p-21f * fabsf(c.half);
  const float hi_v = 2.f * (c.half - near * (1.f - 0x1p-20f) + (margin + 0x1p-21f * near));
  const float lo_v = 2.f * (c.half - far * (1.f + 0x1p-20f) - (margin + 0x1p-21f * far));
  const uint32_t top_key = sample_key<DT>(c.top);
  uint32_t high = bin > 0 && hi_v < c.top ? min(top_key, sample_key<DT>(hi_v) + 1) : top_key;
  uint32_t low = lo_v == lo_v ? max(from.key, sample_key<DT>(lo_v)) : from.key;
  low = min(low, high);
  for (;;) {
    const int shift = max(0, 21 - __clz((high - low) | 1));  // 11 bits of the range
    clear_bins<W>(s);
    const float from_v = low ? sample_value<DT>(low) : -INFINITY, to_v = sample_value<DT>(high);
    x.template each<true>([&](int, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(v[e] >= from_v && v[e] <= to_v)) continue;
        const uint32_t key = sample_key<DT>(v[e]);
        if (key < low || key > high || key <= from.key || bin_of(v[e], c) != bin) continue;
        atomicAdd(&s.count[(high - key) >> shift], 1u);
        if (goal.by_mass && shift > 0)
          atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[(high - key) >> shift]),
                    static_cast<unsigned long long>(weight(v[e])));
      }
    });
    __syncthreads();
    if (from.ties && from.key >= low && from.key <= high) {
      const float v = sample_value<DT>(from.key);
      if (tid == 0 && bin_of(v, c) == bin) {
        s.count[(high - from.key) >> shift] += from.ties;
        s.mass[(high - from.key) >> shift] += from.ties * weight(v);
      }
      __syncthreads();
    }
    if (goal.by_mass && shift == 0) {  // one key a bin: its values weigh the same
#pragma unroll
      for (int b = tid; b < kBins; b += 64 * W)
        if (s.count[b]) s.mass[b] = s.count[b] * weight(sample_value<DT>(high - b));
      __syncthreads();
    }
    Target rest = goal;
    rest.count = goal.count - count;
    rest.mass = goal.mass - static_cast<double>(mass);
    uint32_t c2 = 0;
    uint64_t m2 = 0;
    const uint32_t bin2 = find_bin<W>(s, rest, c2, m2);
    const uint32_t n = s.count[bin2];
    const uint64_t in = s.mass[bin2];
    count += c2;
    mass += m2;
    if (shift == 0) {
      uint32_t ties = goal.count - count;
      if (goal.by_mass) {
        const double need = goal.mass - static_cast<double>(mass), w = n ? static_cast<double>(in / n) : 0.0;
        ties = w > 0.0 ? static_cast<uint32_t>(fmin(ceil(need / w), static_cast<double>(n))) : n;
      }
      ties = ties > n ? n : ties;
      return Border{high - bin2, ties < 1 ? 1 : ties};
    }
    const uint32_t up = high - (bin2 << shift), room = (1u << shift) - 1;
    low = up - low > room ? up - room : low;
    high = up;
  }
}

// Weights by bins, of the values above from.key and from.ties at it; returns their sum.
template <int DT, int W, class X>
__device__ __forceinline__ uint64_t bin_weights(SampleShared &s, X &x, const RowCall &c, const Weight &weight, Border from) {
  const int tid = threadIdx.x;
  clear_bins<W>(s);
  const float above = border_value<DT>(from);
  const auto add = [&](int, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int bin = bin_of(v[e], c);
      if (bin < kBins - 1 && v[e] > above)
        atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[bin]), static_cast<unsigned long long>(weight(v[e])));
    }
  };
  x.template each<true>(add);
  __syncthreads();
  if (from.ties) {
    const float v = sample_value<DT>(from.key);
    if (tid == 0) s.mass[bin_of(v, c)] += from.ties * weight(v);
    __syncthreads();
  }
  uint64_t own = 0, total;
#pragma unroll
  for (int b = tid; b < kBins; b += 64 * W) own += s.mass[b];
  waves_before<W>(s.wave_mass, wave_sum(own), total);
  __syncthreads();
  return total;
}

// The bin that the k-th largest value is in, and how many values are in those before it.
template <int DT, int W, class X>
__device__ __forceinline__ int find_bin_of_count(SampleShared &s, X &x, const RowCall &c, const Target &goal, uint32_t &count) {
  clear_bins<W>(s);
  x.each([&](int, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int bin = bin_of(v[e], c);
      if (bin < kBins - 1) atomicAdd(&s.count[bin], 1u);
    }
  });
  __syncthreads();
  uint64_t mass;
  return find_bin<W>(s, goal, count, mass);
}

// From the values of a row, or those of them that may be kept, to the token.  `bin`, with `count` or `mass` before it: where
// the border of `goal` is, if there is one.
template <int DT, int W, class X>
__device__ __forceinline__ void draw_token(SampleShared &s, X &x, const RowCall &c, const Weight &weight, bool filtered,
                                           const Target &goal, int bin, uint32_t count, uint64_t mass) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Border border{0, 0};
  if (filtered) {
    border = find_border<DT, W>(s, x, c, weight, bin, goal, count, mass, border);
    if (!goal.by_mass && c.by_p) {  // of the k largest, those down to p of their weight
      const uint64_t total = bin_weights<DT, W>(s, x, c, weight, border);
      const Target part{true, 0, static_cast<double>(c.p) * static_cast<double>(total)};
      const int at = find_bin<W>(s, part, count, mass);
      border = find_border<DT, W>(s, x, c, weight, at, part, 0, mass, border);
    }
  }

  // kept weight of each span, the ties at the border counted apart
  const uint64_t floor_w =
      c.floor_p > 0.f ? static_cast<uint64_t>(fmin(static_cast<double>(c.floor_p), 1.0) * kOne + 0.5) : 0;
  const float above = border_value<DT>(border);
  uint64_t tie_w = border.ties ? weight(sample_value<DT>(border.key)) : 0;
  if (tie_w < floor_w) tie_w = 0;
  x.template each<true>([&](int ch, const float (&v)[8]) {
    uint64_t m = 0;
    uint32_t ties = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint64_t w = weight(v[e]);
      m += v[e] > above && w >= floor_w ? w : 0;
      ties += v[e] == above ? 1 : 0;
    }
    if (__any(ties || m)) {
      m = wave_sum(m);
      ties = wave_sum(ties);
    }
    if (lane == 0) {
      s.span_mass[x.span(ch)] = m;
      s.span_ties[x.span(ch)] = ties;
    }
  });
  __syncthreads();

  // every wave: ties to weights, the sum, the span that the token is in; its wave finds the token
  const int spans = x.chunks * W;
  uint64_t total = 0;
  uint32_t taken = 0;
  for (int b = 0; b < spans; b += 64) {
    const bool in = b + lane < spans;
    const uint32_t ties = in ? s.span_ties[b + lane] : 0, upto = wave_scan(ties), before = taken + upto - ties;
    total += in ? s.span_mass[b + lane] + tie_w * min(ties, border.ties > before ? border.ties - before : 0) : 0;
    taken += last_lane(upto);
  }
  total = wave_sum(total);
  // u below 1 leaves the target below the sum; other u, and NaN, are held there
  const double target = fmin(fmax(static_cast<double>(c.u), 0.0) * static_cast<double>(total),
                             static_cast<double>(total) * (1.0 - 0x1p-52) - 1.0);
  uint64_t run = 0;
  uint32_t ties_before = 0;
  int span = spans - 1;
  taken = 0;
  for (int b = 0; b < spans; b += 64) {
    const bool in = b + lane < spans;
    const uint32_t ties = in ? s.span_ties[b + lane] : 0, tupto = wave_scan(ties), before = taken + tupto - ties;
    const uint64_t m = in ? s.span_mass[b + lane] + tie_w * min(ties, border.ties > before ? border.ties - before : 0) : 0;
    const uint64_t upto = run + wave_scan(m);
    const uint64_t past = __ballot(in && static_cast<double>(upto) > target);
    if (past) {
      const int l = __builtin_ctzll(past);
      span = b + l;
      run = __shfl(upto - m, l, 64);
      ties_before = __builtin_amdgcn_readlane(before, l);
      break;
    }
    run = last_lane(upto);
    taken += last_lane(tupto);
  }
  if (span / x.chunks != wave) return;
  x.one(span % x.chunks, [&](int ch, const float (&v)[8]) {
    uint64_t w[8], m = 0;
    uint32_t ties = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ties += v[e] == above ? 1 : 0;
    uint32_t before = ties_before + wave_scan(ties) - ties;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = v[e] > above ? weight(v[e]) : 0;
      if (w[e] < floor_w) w[e] = 0;
      if (v[e] == above) w[e] = before++ < border.ties ? tie_w : 0;
      m += w[e];
    }
    uint64_t upto = run + wave_scan(m) - m, own = 0;
    int found = INT32_MAX;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      upto += w[e];
      if (w[e] && static_cast<double>(upto) > target && found == INT32_MAX) {
        found = e;
        own = w[e];
      }
    }
    const uint64_t who = __ballot(found != INT32_MAX);
    if (who && lane == __builtin_ctzll(who)) {
      *c.token = x.index(ch, found);
      *c.logprob = static_cast<float>(log(static_cast<double>(own) / static_cast<double>(total)));
    }
  });
}

template <int DT, int W, int CH>
__global__ __launch_bounds__(64 * W) void sample_kernel(const uint8_t *__restrict__ logits, int64_t stride, int vocab,
                                                          const float *__restrict__ u, const float *__restrict__ temperature,
                                                          const int32_t *__restrict__ top_k, const float *__restrict__ top_p,
                                                          const float *__restrict__ min_p, int64_t *__restrict__ tokens,
                                                          float *__restrict__ logprobs) {
  extern __shared__ __attribute__((aligned(16))) uint8_t sample_smem[];
  SampleShared &s = *reinterpret_cast<SampleShared *>(sample_smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t r = blockIdx.x;
  SampleRow<DT, CH> x;
  x.row = logits + r * stride * (DT == MP_F32 ? 4 : 2);
  x.vocab = vocab;
  x.chunks = (vocab + W * kSpan - 1) / (W * kSpan);
  x.vec = reinterpret_cast<uintptr_t>(x.row) % 16 == 0;
  x.load();
  RowCall c;
  c.t = temperature ? temperature[r] : 1.0f;
  c.k = top_k ? top_k[r] : 0;
  c.k = c.k > 0 && c.k < vocab ? c.k : 0;
  c.p = top_p ? top_p[r] : 1.0f;
  c.by_p = c.p < 1.0f;
  c.floor_p = min_p ? min_p[r] : 0.f;
  c.u = u[r];
  c.token = tokens + r;
  c.logprob = logprobs + r;

  float top = -INFINITY;
  x.template each<true>([&](int, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, v[e]);
  });
  const float mine = top;  // this thread's
  top = mp_wave_max(top);
  if (lane == 0) s.top[wave] = top;
  for (int i = tid; i < kTable; i += 64 * W) s.table[i] = kOne * exp2(static_cast<double>(i) / kTable);  // for the weights
  __syncthreads();
#pragma unroll
  for (int w = 0; w < W; ++w) top = fmaxf(top, s.top[w]);
  if (top == -INFINITY) {  // nothing may be taken
    if (tid == 0) {
      *c.token = -1;
      *c.logprob = -INFINITY;
    }
    return;
  }
  if (!(c.t > 0.f)) {  // the largest is: its first index
    int at = INT32_MAX;
    x.each([&](int ch, const float (&v)[8]) {
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (v[e] == top) at = min(at, x.index(ch, e));
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    if (lane == 0) s.at[wave] = at;
    __syncthreads();
    for (int w = 0; w < W; ++w) at = min(at, s.at[w]);
    if (tid == 0) {
      *c.token = at;
      *c.logprob = 0.f;
    }
    return;
  }
  x.infinite = top == INFINITY;
  c.top = top = x.infinite ? 0.f : top;
  c.half = 0.5f * top;
  c.per = static_cast<float>(fmin(2 * (kBins - 1) / (kReach * static_cast<double>(c.t)), 0x1p127));
  const double rate = kTable * 1.4426950408889634 / static_cast<double>(c.t);
  const Weight weight{s.table, static_cast<double>(top), rate};

  // the bin that the border is in
  Target goal{!c.k, static_cast<uint32_t>(c.k), 0.0};
  int bin = kBins - 1;
  uint32_t count = 0;
  uint64_t mass = 0;
  // at least k values are in this bin or above: of the threads' maxima are
  bool bounded = c.k > 0 && c.k <= 64 * W && !x.infinite;
  if (bounded) {
    clear_bins<W>(s);
    const int b = bin_of(mine, c);
    if (b < kBins - 1) atomicAdd(&s.count[b], 1u);
    __syncthreads();
    bin = find_bin<W>(s, goal, count, mass);
    bounded = bin < kBins - 1;
  }
  if (c.k && !bounded) {
    bin = find_bin_of_count<DT, W>(s, x, c, goal, count);
    if (bin == kBins - 1) goal.by_mass = true;  // all that weighs anything is among the k largest
  }
  if (bin == kBins - 1 && c.by_p) {
    goal.mass = static_cast<double>(c.p) * static_cast<double>(bin_weights<DT, W>(s, x, c, weight, Border{0, 0}));
    bin = find_bin<W>(s, goal, count, mass);
  }
  const bool filtered = bin < kBins - 1;

  // to be listed: the values of that bin and above, or else those not below min-p's floor; a few more do no harm, which
  // leaves a margin for the roundings.  (Where top-p sums weights up, min-p has to wait for it.)
  const float reach = filtered ? 2.f * ((bin + 1) / c.per) : c.t * -logf(fminf(c.floor_p, 1.0f));
  const float least = top - reach * (1.f + 0x1p-10f) - 0x1p-10f * (c.t + 0x1p-10f * fabsf(top));
  bool list = (filtered || c.floor_p > 0.f) && least == least;
  if (list) {  // each wave its own, in index order
    uint32_t n = 0;
    x.template each<true>([&](int ch, const float (&v)[8]) {
      float most = v[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, v[e]);
      if (!__any(most >= least) || n > kListed) return;
      uint32_t own = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) own += v[e] >= least ? 1 : 0;
      const uint32_t upto = wave_scan(own);
      uint32_t at = n + upto - own;
      n += last_lane(upto);
      if (n > kListed) return;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v[e] >= least) {
          s.value[wave][at] = v[e];
          s.index[wave][at++] = x.index(ch, e);
        }
    });
    if (lane == 0) s.listed[wave] = n;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) list = list && s.listed[w] <= kListed;
  }
  if (list) {
    SampleList<W> l;
    l.s = &s;
    l.all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) l.all += s.listed[w];
    l.per = (l.all + 64 * W - 1) / (64 * W);
    l.load();
    if (bounded) bin = find_bin_of_count<DT, W>(s, l, c, goal, count);
    draw_token<DT, W>(s, l, c, weight, filtered, goal, bin, count, mass);
  } else {
    if (bounded) bin = find_bin_of_count<DT, W>(s, x, c, goal, count);
    draw_token<DT, W>(s, x, c, weight, filtered, goal, bin, count, mass);
  }
}

template <int DT, int W, int CH>
int sample_launch(const void *logits, int64_t stride, int64_t rows, int vocab, const float *u, const float *temperature,
                  const int32_t *top_k, const float *top_p, const float *min_p, int64_t *tokens, float *logprobs,
                  hipStream_t s) {
  if (hipFuncSetAttribute(reinterpret_cast<const void *>(sample_kernel<DT, W, CH>), hipFuncAttributeMaxDynamicSharedMemorySize,
                          sizeof(SampleShared)) != hipSuccess)
    return MP_ERR_HIP;
  hipLaunchKernelGGL((sample_kernel<DT, W, CH>), dim3(static_cast<unsigned>(rows)), dim3(64 * W), sizeof(SampleShared), s,
                     static_cast<const uint8_t *>(logits), stride, vocab, u, temperature, top_k, top_p, min_p, tokens, logprobs);
  MP_CHECK_LAUNCH();
  return MP_OK;
}

}  // namespace

extern "C" int mp_sample_tokens(const void *logits, int64_t stride, int64_t rows, int64_t vocab, int dtype, const float *u,
                                const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                                int64_t *tokens, float *logprobs, mp_stream_t stream) {
  if (!logits || !u || !tokens || !logprobs) return MP_ERR_ARG;
  if (dtype != MP_F16 && dtype != MP_BF16 && dtype != MP_F32) return MP_ERR_DTYPE;
  if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > kMaxVocab || stride < vocab) return MP_ERR_SHAPE;
  if (!mp_aligned(logits, dtype == MP_F32 ? 4 : 2)) return MP_ERR_ALIGN;
  if (rows == 0) return MP_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int n = static_cast<int>(vocab);
  // Waves of a row, and whether their registers hold it.  Eight hold up to 32768 values; sixteen 131072 of 16 bits, and past that
  // the row is read again in every pass.  256 rows of 128256 bf16, read again or held: no filter 57.9 / 56.1 us, top-k 36.6 /
  // 32.6, top-p 114.7 / 104.6.  Rows of 32000 in sixteen waves or eight: one row, top-k 17.0 / 14.9 us (the eight have fewer
  // counts to join); 256 rows 19.7 / 18.4, top-p 39.4 / 41.1.
#define MP_SAMPLE(DT, CH)                                                                                                     \
  (n <= 8 * 8 * kSpan                                                                                                         \
       ? sample_launch<DT, 8, 8>(logits, stride, rows, n, u, temperature, top_k, top_p, min_p, tokens, logprobs, s)           \
       : n <= 16 * CH * kSpan                                                                                                 \
             ? sample_launch<DT, 16, CH>(logits, stride, rows, n, u, temperature, top_k, top_p, min_p, tokens, logprobs, s)   \
             : sample_launch<DT, 16, 0>(logits, stride, rows, n, u, temperature, top_k, top_p, min_p, tokens, logprobs, s))
  if (dtype == MP_F16) return MP_SAMPLE(MP_F16, 16);
  if (dtype == MP_BF16) return MP_SAMPLE(MP_BF16, 16);
  return MP_SAMPLE(MP_F32, 0);
#undef MP_SAMPLE
}
