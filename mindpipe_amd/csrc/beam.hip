// The best continuations of each request over its beams and the vocabulary.
//
//   total(k, v) = score_k + x_kv - log sum_v exp x_kv      (an ended beam has one continuation, of its own score)
//   the `count` largest totals of a request, from the largest down; of equal ones those of the lowest beam, then token
//
// Which of two totals is larger decides a whole number, so they are made in 64 bits: the order inside of a row is that of its
// logits, and between rows the sums of exponentials decide, each off by less than 2^-39 of what its other values add to the largest
// one's 1, and by the roundings of some hundred additions, 2^-45.
//
// Two launches.  Of each row, workgroups take a part of the vocabulary each (a row is read once and stays in registers): they leave
// the part's maximum, its sum of exponentials and its `count` largest values in order.  No value can be among a request's best
// that is not among those.  Then a workgroup a request puts the best of its lists in order.
//
// Bound by vector instructions, 27 for a value, of which the exponential in 64 bits (as fast as 32 bits here) is 18: 48 requests of 8
// beams over 128256 bf16, 98 MB, 47 us, and the merge 10, where the reads alone would take 15.  One request of 4 over 32000: 6.2 and 8.4.
#include "logits.h"

namespace {

constexpr int kMaxBeams = 64, kMaxCount = 64;  // a lane to each
constexpr int kBeamWaves = 4, kBeamThreads = 64 * kBeamWaves;
constexpr int kBeamListed = 512;               // candidates of a part that LDS has room for
constexpr double kLog2eD = 1.4426950408889634;

// exp(d) for d from -690 to 0, in 64 bits (below -kBeamLost, 2^-865, no part of a sum): 2^n from the whole part of d log2 e and 2^r,
// r in [-1/2, 1/2], by the polynomial of degree eight that is 1 at 0 and otherwise off by the least share there, 2^-39.7.  A row's
// largest value so counts as 1: where nothing else has weight the logarithm of the sum is 0, and a certain token's total is its
// beam's score.  (Degree seven is off by 2^-34.5 where its constant term is free, and makes that token likelier than 1.)
constexpr float kBeamLost = 600.f;
__device__ __forceinline__ double beam_exp(double d) {
  const double magic = 1.5 * 0x1p52;  // a sum with it is whole
  const double t = fma(d, kLog2eD, magic), r = fma(d, kLog2eD, magic - t);
  double p = 1.3344183484134179e-06;
  p = fma(p, r, 1.5314209223349525e-05);
  p = fma(p, r, 0.0001540309828656179);
  p = fma(p, r, 0.0013333434157560176);
  p = fma(p, r, 0.009618129558838935);
  p = fma(p, r, 0.05550410959228811);
  p = fma(p, r, 0.2402265069474259);
  p = fma(p, r, 0.6931471805412327);
  p = fma(p, r, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));  // no underflow: n is above -1000
}
struct BeamPart {  // of a part of a row: its largest value and sum_v exp(x_v - top); top +inf: how many such values
  double sum;
  float top;
  int pad;
};
struct BeamValue {  // of a part's list, from the largest down; token -1: none
  float value;
  int token;
};

__device__ __forceinline__ uint32_t beam_order(float v) {  // of all types alike
  return sample_key<MP_F32>(v);
}

// Waves' counts, summed over the workgroup.
__device__ __forceinline__ uint32_t beam_total(uint32_t mine, uint32_t *of_wave) {
  const uint32_t n = wave_sum(mine);
  __syncthreads();  // what was there has been read
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = n;
  __syncthreads();
  uint32_t sum = 0;
#pragma unroll
  for (int w = 0; w < kBeamWaves; ++w) sum += of_wave[w];
  return sum;
}

// The lanes that want it put (key, index) on the list; one addition to the count for the wave.
__device__ __forceinline__ void beam_put(bool mine, uint32_t key, int i, uint64_t *list, uint32_t *listed) {
  const uint64_t in = __ballot(mine);
  if (!in) return;
  const int lane = threadIdx.x & 63, lead = __builtin_ctzll(in);
  uint32_t n = 0;
  if (lane == lead) n = atomicAdd(listed, static_cast<uint32_t>(__popcll(in)));
  n = __builtin_amdgcn_readlane(n, lead) + __popcll(in & ((uint64_t(1) << lane) - 1));
  if (mine && n < kBeamListed) list[n] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~i);
}

// The `count` largest of a part in which many values are equal, or ascend: more reach `key` than LDS has room for.  The least one
// that is wanted is that key, where few are above it, or else the `count`-th largest, by its bits; then come those above it, and
// of its ties the first in the order of their indexes, 512 in a wave's row, row by row.  Reads the part again, a row at a time.
template <int DT>
__device__ __attribute__((noinline)) int beam_many(const uint8_t *at, bool vec, int first, int rows, int vocab, int count, uint32_t key,
                                                   uint64_t *list, uint32_t *listed, uint32_t *of_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto row = [&](int g, float (&v)[8]) {
    Eight<DT> x;
    x.load(at, first + 8 * kBeamThreads * g, vocab, vec);
    x.get(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fmaxf(v[e], -INFINITY);
  };
  const auto reach = [&](uint32_t least) {  // how many values reach it
    uint32_t own = 0;
#pragma unroll 1
    for (int g = 0; g < rows; ++g) {
      float v[8];
      row(g, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) own += beam_order(v[e]) >= least ? 1 : 0;
    }
    return beam_total(own, of_wave);
  };
  uint32_t above = reach(key + 1);
  if (above >= static_cast<uint32_t>(count)) {
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
      const uint32_t trial = (key | bit) & ~(bit - 1);
      if (!(key & bit) && reach(trial) >= static_cast<uint32_t>(count)) key = trial;
    }
    above = reach(key + 1);
  }
  if (threadIdx.x == 0) *listed = 0;
  const float tie = sample_value<MP_F32>(key);
  int ties = count - static_cast<int>(above);
#pragma unroll 1
  for (int g = 0; g < rows; ++g) {
    float v[8];
    row(g, v);
    uint32_t own = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) own += v[e] == tie ? 1 : 0;
    const uint32_t upto = wave_scan(own);
    __syncthreads();  // the last row's counts have been read
    if (lane == 63) of_wave[wave] = upto;
    __syncthreads();
    int before = static_cast<int>(upto - own), all = 0;
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) {
      before += w < wave ? static_cast<int>(of_wave[w]) : 0;
      all += static_cast<int>(of_wave[w]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      beam_put(v[e] > tie || (v[e] == tie && before < ties), beam_order(v[e]), first + 8 * kBeamThreads * g + e, list, listed);
      before += v[e] == tie ? 1 : 0;
    }
    ties -= all;
  }
  __syncthreads();
  return min(static_cast<int>(*listed), kBeamListed);
}

template <int DT, int H>
__global__ __launch_bounds__(kBeamThreads) void beam_rows_kernel(const uint8_t *__restrict__ logits, int64_t stride, int vocab,
                                                                 const uint8_t *__restrict__ ended, int splits, int count,
                                                                 BeamPart *__restrict__ parts, BeamValue *__restrict__ lists) {
  __shared__ uint32_t tops[kBeamThreads], of_wave[kBeamWaves], listed;
  __shared__ double wave_sums[kBeamWaves];
  __shared__ float wave_top[kBeamWaves];
  __shared__ uint64_t list[kBeamListed];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / splits;
  if (ended && ended[row]) return;  // what it leaves is not looked at
  const int part = blockIdx.x % splits, first = part * (8 * H * kBeamThreads) + 8 * tid;  // index of this thread's first value
  const uint8_t *at = logits + row * stride * (DT == MP_F32 ? 4 : 2);
  const bool vec = reinterpret_cast<uintptr_t>(at) % 16 == 0;
  Eight<DT> held[H];
#pragma unroll
  for (int g = 0; g < H; ++g) held[g].load(at, first + 8 * kBeamThreads * g, vocab, vec);
  if (tid == 0) listed = 0;

  const auto each = [&](auto f, float least = -INFINITY) {  // f(index, its eight values), NaN and lower ones as `least`
#pragma unroll
    for (int g = 0; g < H; ++g) {
#pragma unroll
      for (int i = 0; i < Eight<DT>::kWords; ++i) sample_renew(held[g].w[i]);
      float v[8];
      held[g].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaxf(v[e], least);
      f(first + 8 * kBeamThreads * g, v);
    }
  };
  float top = -INFINITY, eight[H];  // the largest of each eight: only those that have a candidate are looked at again
#pragma unroll
  for (int g = 0; g < H; ++g) {
    float v[8];
    held[g].get(v);
    eight[g] = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    top = fmaxf(top, eight[g]);  // eight NaN are no part of it
  }
  tops[tid] = beam_order(fmaxf(top, -INFINITY));
  const float wtop = mp_wave_max(top);
  if (lane == 0) wave_top[wave] = wtop;
  __syncthreads();
  float most = wave_top[0];
#pragma unroll
  for (int w = 1; w < kBeamWaves; ++w) most = fmaxf(most, wave_top[w]);

  // the sum, against the part's largest value
  double sum = 0.0;
  if (most == INFINITY) {
    each([&](int, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += v[e] == INFINITY ? 1.0 : 0.0;
    });
  } else if (most > -INFINITY) {
    const double base = most;
    if (fabsf(most) < 0x1p29f) {  // fp32's steps are below 64: raised to `most` - kBeamLost, values count for nothing
      each([&](int, const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += beam_exp(static_cast<double>(v[e]) - base);
      }, most - kBeamLost);
    } else {
      each([&](int, const float (&v)[8]) {
        for (int e = 0; e < 8; ++e) sum += beam_exp(fmax(static_cast<double>(v[e]) - base, -kBeamLost));
      });
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) wave_sums[wave] = sum;

  // a value that `count` of the threads' largest reach, or none: so many are not below it.  (By fours of threads the search is
  // shorter, and as near for few: 16 of 64 leave some 18 candidates; 64 of 64 some 280, of 256 some 75.)
  const uint32_t none = beam_order(-INFINITY);
  uint32_t of[4], least = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) of[i] = tops[4 * lane + i];
  if (count <= 16) {
    of[0] = max(max(of[0], of[1]), max(of[2], of[3]));
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if (__popcll(__ballot(of[0] >= (least | bit))) >= count) least |= bit;
  } else {
#pragma unroll 1
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
      int reach = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) reach += __popcll(__ballot(of[i] >= (least | bit)));
      if (reach >= count) least |= bit;
    }
  }
  least = max(least, none + 1);
  const float limit = sample_value<MP_F32>(least);
#pragma unroll
  for (int g = 0; g < H; ++g) {
    if (!__any(eight[g] >= limit)) continue;
    float v[8];
    held[g].get(v);
#pragma unroll
    for (int e = 0; e < 8; ++e)  // (a branch for the wave: the lanes' own cost more than all the rest of the pass)
      beam_put(v[e] >= limit, beam_order(v[e]), first + 8 * kBeamThreads * g + e, list, &listed);
  }
  __syncthreads();
  int n = static_cast<int>(listed);
  if (tid == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) all += wave_sums[w];
    parts[blockIdx.x] = BeamPart{all, most, 0};
  }
  if (n > kBeamListed) n = beam_many<DT>(at, vec, first, H, vocab, count, least, list, &listed, of_wave);
  BeamValue *out = lists + static_cast<int64_t>(blockIdx.x) * count;
  for (int e = tid; e < n; e += kBeamThreads) {
    const uint64_t me = list[e];
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += list[i] > me ? 1 : 0;
    if (rank < count)
      out[rank] = BeamValue{sample_value<MP_F32>(static_cast<uint32_t>(me >> 32)), static_cast<int>(~static_cast<uint32_t>(me))};
  }
  for (int e = n + tid; e < count; e += kBeamThreads) out[e] = BeamValue{0.f, -1};
}

struct BeamBest {
  double total;
  int at;  // beam * vocab + token
  __device__ __forceinline__ bool before(double t, int i) const { return total > t || (total == t && at < i); }
};

constexpr int kBeamNear = 2048;  // continuations that LDS has room for

// One workgroup a request.  The largest total that `count` of 256 reach, the first ones of every list, is reached by `count`
// continuations; the few that reach it are put in order by counting, for each, those before it.
__global__ __launch_bounds__(256) void beam_merge_kernel(const BeamPart *__restrict__ parts, const BeamValue *__restrict__ lists,
                                                         const float *__restrict__ scores, const uint8_t *__restrict__ ended,
                                                         int beams, int splits, int count, int vocab, int pad, MpDivisor by_count,
                                                         MpDivisor by_splits, float *__restrict__ out_scores,
                                                         int64_t *__restrict__ out_beams, int64_t *__restrict__ out_tokens) {
  __shared__ double base[kMaxBeams], score[kMaxBeams], near_total[kBeamNear];  // base: log sum exp
  __shared__ int near_at[kBeamNear], listed;
  __shared__ uint32_t key[256];
  __shared__ double wave_total[4];
  __shared__ int wave_at[4];
  __shared__ uint8_t state[kMaxBeams];
  enum { kPlain, kInfinite, kEnded };
  const int64_t b = blockIdx.x;
  const int n_lists = beams * splits, values = n_lists * count, tid = threadIdx.x;
  const BeamValue *from = lists + b * values;
  if (tid < beams) {
    const BeamPart *p = parts + (b * beams + tid) * splits;
    score[tid] = scores[b * beams + tid];
    const bool done = ended && ended[b * beams + tid];
    float top = -INFINITY;
    double sum = 0.0;
    if (!done) {
      for (int s = 0; s < splits; ++s) {
        const BeamPart q = p[s];
        if (q.top > top) {
          sum = top > -INFINITY && q.top < INFINITY ? sum * beam_exp(fmax(static_cast<double>(top) - q.top, -kBeamLost)) : 0.0;
          top = q.top;
          sum += q.sum;
        } else if (q.top > -INFINITY) {
          sum += q.top == top ? q.sum : top < INFINITY ? q.sum * beam_exp(fmax(static_cast<double>(q.top) - top, -kBeamLost)) : 0.0;
        }
      }
    }
    // with infinite logits those alone count, as if they were 0, and all others are -inf
    state[tid] = done ? kEnded : top == INFINITY ? kInfinite : kPlain;
    base[tid] = (top == INFINITY ? 0.0 : static_cast<double>(top)) + log(sum);
  }
  if (tid == 0) listed = 0;
  __syncthreads();
  const double none = -INFINITY;
  // Entry `at` of a list; nothing there, or a total of -inf or NaN: -inf.
  const auto candidate = [&](int list, int at) {
    const int k = by_splits(list);
    BeamBest c{none, 0};
    if (state[k] == kEnded) {  // the row's first list has its one continuation
      if (list == k * splits && at == 0) c = BeamBest{score[k], k * vocab + pad};
    } else {
      const BeamValue v = from[list * count + at];
      if (v.token >= 0) {
        const double x = state[k] == kInfinite ? (v.value == INFINITY ? 0.0 : none) : static_cast<double>(v.value);
        c = BeamBest{score[k] + (x - base[k]), k * vocab + v.token};
      }
    }
    if (!(c.total > none)) c.total = none;
    return c;
  };
  // in 32 bits, rounded down, so that whatever reaches a total reaches it here
  const auto order = [&](double total) { return total > none ? beam_order(__double2float_rd(total)) : 0u; };
  // 256 of the totals, a thread each: the first ones of every list, or the best heads of several lists
  int deep = 0;
  while (n_lists << (deep + 1) <= 256) ++deep;
  uint32_t own = 0;
  if (n_lists <= 256) {
    const int list = tid >> deep, at = tid & ((1 << deep) - 1);
    if (list < n_lists && at < count) own = order(candidate(list, at).total);
  } else {
    for (int i = tid; i < n_lists; i += 256) own = max(own, order(candidate(i, 0).total));
  }
  key[tid] = own;
  __syncthreads();
  uint32_t of[4], least = 0;  // what `count` of them reach
#pragma unroll
  for (int i = 0; i < 4; ++i) of[i] = key[64 * i + (tid & 63)];
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
    int reach = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) reach += __popcll(__ballot(of[i] >= (least | bit)));
    if (reach >= count) least |= bit;
  }
  least = max(least, 1u);
  // totals descend in a list: a thread's entries are done with the first that is below
  const int stride = n_lists <= 256 ? 1 << deep : 1;
  for (int list = n_lists <= 256 ? tid >> deep : tid; list < n_lists; list += 256) {
    for (int at = n_lists <= 256 ? tid & (stride - 1) : 0; at < count; at += stride) {
      const BeamBest c = candidate(list, at);
      if (order(c.total) < least) break;
      const int n = atomicAdd(&listed, 1);
      if (n < kBeamNear) {
        near_total[n] = c.total;
        near_at[n] = c.at;
      }
    }
  }
  __syncthreads();
  const int n = listed;
  const auto put = [&](int i, BeamBest c) {
    const bool found = c.total > none;
    const int k = found ? c.at / vocab : -1;
    out_scores[b * count + i] = static_cast<float>(c.total);
    out_beams[b * count + i] = k;
    out_tokens[b * count + i] = found ? c.at - k * vocab : -1;
  };
  if (n <= 256) {
    const BeamBest me{tid < n ? near_total[tid] : none, tid < n ? near_at[tid] : INT32_MAX};
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += BeamBest{near_total[i], near_at[i]}.before(me.total, me.at) ? 1 : 0;
    if (tid < n && rank < count) put(rank, me);
    if (tid >= n && tid < count) put(tid, BeamBest{none, 0});
    return;
  }
  // Many are equal: one after the other, each the best of those behind the last, from LDS or, where it has no room, from the lists.
  const int all = n <= kBeamNear ? n : values;
  BeamBest last{INFINITY, -1};
  for (int i = 0; i < count; ++i) {
    BeamBest best{none, INT32_MAX};
    for (int e = tid; e < all; e += 256) {
      BeamBest c;
      if (n <= kBeamNear) {
        c = BeamBest{near_total[e], near_at[e]};
      } else {
        const int list = by_count(e);
        c = candidate(list, e - list * count);
      }
      if (last.before(c.total, c.at) && c.before(best.total, best.at)) best = c;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const BeamBest c{__shfl_xor(best.total, o, 64), __shfl_xor(best.at, o, 64)};
      if (c.before(best.total, best.at)) best = c;
    }
    __syncthreads();  // the last round's have been read
    if ((tid & 63) == 0) {
      wave_total[tid >> 6] = best.total;
      wave_at[tid >> 6] = best.at;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const BeamBest c{wave_total[w], wave_at[w]};
      if (c.before(best.total, best.at)) best = c;
    }
    if (tid == 0) put(i, best);
    last = best;
  }
}

// Eights of a thread: eight, of which 116 registers leave four workgroups to a CU, but as few as keep 512 workgroups or more in the
// launch.  48 requests as above: sixteen 57 us, eight 50, four 50 with a merge of 14 in place of 10 us (before the looks for candidates
// were cut down to 45).
inline int beam_eights(int64_t rows, int64_t vocab) {
  int h = 8;
  while (h > 2 && rows * mp_cdiv(vocab, 8 * h * kBeamThreads) < 512) h /= 2;
  return h;
}
inline int64_t beam_splits(int64_t rows, int64_t vocab) { return mp_cdiv(vocab, 8 * beam_eights(rows, vocab) * kBeamThreads); }

template <int DT, int H>
void beam_rows_launch(const void *logits, int64_t stride, int64_t rows, int vocab, const uint8_t *ended, int splits, int count,
                      BeamPart *parts, BeamValue *lists, hipStream_t s) {
  hipLaunchKernelGGL((beam_rows_kernel<DT, H>), dim3(static_cast<unsigned>(rows * splits)), dim3(kBeamThreads), 0, s,
                     static_cast<const uint8_t *>(logits), stride, vocab, ended, splits, count, parts, lists);
}

}  // namespace

extern "C" size_t mp_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t count) {
  if (batch <= 0 || batch > INT32_MAX || beams < 1 || beams > kMaxBeams || vocab < 1 || vocab > kMaxVocab || count < 1 ||
      count > kMaxCount)
    return 0;
  const int64_t parts = batch * beams * beam_splits(batch * beams, vocab);
  return static_cast<size_t>(parts) * (sizeof(BeamPart) + count * sizeof(BeamValue));
}

extern "C" int mp_beam_select(const void *logits, int64_t stride, int64_t batch, int64_t beams, int64_t vocab, int dtype,
                              const float *scores, const uint8_t *ended, int64_t pad, int64_t count, float *out_scores,
                              int64_t *out_beams, int64_t *out_tokens, void *workspace, size_t workspace_bytes, mp_stream_t stream) {
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens || !workspace) return MP_ERR_ARG;
  if (dtype != MP_F16 && dtype != MP_BF16 && dtype != MP_F32) return MP_ERR_DTYPE;
  if (batch < 0 || beams < 1 || beams > kMaxBeams || vocab < 1 || vocab > kMaxVocab || count < 1 || count > kMaxCount ||
      stride < vocab || pad < 0 || pad >= vocab)
    return MP_ERR_SHAPE;
  if (batch > INT32_MAX / beams / 256) return MP_ERR_SHAPE;  // a row has 256 parts at most
  if (!mp_aligned(logits, dtype == MP_F32 ? 4 : 2) || !mp_aligned(workspace, 16)) return MP_ERR_ALIGN;
  if (batch == 0) return MP_OK;
  if (workspace_bytes < mp_beam_select_workspace_bytes(batch, beams, vocab, count)) return MP_ERR_WORKSPACE;
  const int64_t rows = batch * beams;
  const int h = beam_eights(rows, vocab), n = static_cast<int>(vocab), k = static_cast<int>(count);
  const int splits = static_cast<int>(beam_splits(rows, vocab));
  if (rows * splits > kMpMaxGroups) return MP_ERR_SHAPE;
  BeamPart *parts = static_cast<BeamPart *>(workspace);
  BeamValue *lists = reinterpret_cast<BeamValue *>(parts + rows * splits);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define MP_BEAM(DT)                                                                                                        \
  do {                                                                                                                     \
    if (h == 8) beam_rows_launch<DT, 8>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                       \
    else if (h == 4) beam_rows_launch<DT, 4>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                  \
    else beam_rows_launch<DT, 2>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                              \
  } while (0)
  if (dtype == MP_F16) MP_BEAM(MP_F16);
  else if (dtype == MP_BF16) MP_BEAM(MP_BF16);
  else MP_BEAM(MP_F32);
#undef MP_BEAM
  MP_CHECK_LAUNCH();
  hipLaunchKernelGGL(beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(256), 0, s, parts, lists, scores, ended,
                     static_cast<int>(beams), splits, k, n, static_cast<int>(pad), mp_divisor(k), mp_divisor(splits), out_scores,
                     out_beams, out_tokens);
  MP_CHECK_LAUNCH();
  return MP_OK;
}
