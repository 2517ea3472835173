// The best continuations of each request over its beams and the vocabulary.
//
//   total(k, v) = score_k + x_kv - log sum_v exp x_kv      (an ended beam has one continuation, of its own score)
//   the `count` largest totals of a request, from the largest down; of equal ones those of the lowest beam, then token
//
// Which of two totals is larger decides a whole number, so they are made in 64 bits: the order inside of a row is that of its
// logits, and between rows the sums of exponentials decide, each off by less than 2^-34 of itself.
//
// Two launches.  Of each row, workgroups take a part of the vocabulary each (a row is read once and stays in registers): they leave
// the part's maximum, its sum of exponentials and its `count` largest values in order.  No value can be among a request's best
// that is not among those.  Then a workgroup a request puts the best of its lists in order.
//
// Bound by vector instructions, 26 for a value, of which the exponential in 64 bits (as fast as 32 bits here) is 17: 48 requests of 8
// beams over 128256 bf16, 98 MB, 45 us, and the merge 10, where the reads alone would take 15.  One request of 4 over 32000: 6.4 and 7.2.
#include "logits.h"

namespace {

constexpr int kMaxBeams = 64, kMaxCount = 64;  // a lane to each
constexpr int kBeamWaves = 4, kBeamThreads = 64 * kBeamWaves;
constexpr int kBeamListed = 512;               // candidates of a part that LDS has room for
constexpr int kQuads = kBeamThreads / 4;       // a lane of a wave to each
constexpr double kLog2eD = 1.4426950408889634;

// exp(d) for d from -690 to 0, in 64 bits (below -kBeamLost, 2^-865, no part of a sum): 2^n from the whole part of d log2 e and 2^r, r in [-1/2, 1/2], by the polynomial of
// degree seven that is off by the least share there, 2^-34.5.
constexpr float kBeamLost = 600.f;
__device__ __forceinline__ double beam_exp(double d) {
  const double magic = 1.5 * 0x1p52;  // a sum with it is whole
  const double t = fma(d, kLog2eD, magic), r = fma(d, kLog2eD, magic - t);
  double p = 1.5201921594169677e-05;
  p = fma(p, r, 0.00015469291141683767);
  p = fma(p, r, 0.001333392256354045);
  p = fma(p, r, 0.00961802725366847);
  p = fma(p, r, 0.05550410353447978);
  p = fma(p, r, 0.24022651198157585);
  p = fma(p, r, 0.693147180728447);
  p = fma(p, r, 0.9999999999616819);
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

template <int DT, int H>
__global__ __launch_bounds__(kBeamThreads) void beam_rows_kernel(const uint8_t *__restrict__ logits, int64_t stride, int vocab,
                                                                 const uint8_t *__restrict__ ended, int splits, int count,
                                                                 BeamPart *__restrict__ parts, BeamValue *__restrict__ lists) {
  __shared__ uint32_t quad[kQuads], of_wave[kBeamWaves], listed;
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
  const float four = fmaxf(fmaxf(top, __shfl_xor(top, 1, 64)), fmaxf(__shfl_xor(top, 2, 64), __shfl_xor(top, 3, 64)));
  if ((tid & 3) == 0) quad[tid >> 2] = beam_order(four);
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

  // a value that `count` quads of threads reach, or none: so many are not below it
  const uint32_t mine = quad[lane], none = beam_order(-INFINITY);
  uint32_t least = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
    if (__popcll(__ballot(mine >= (least | bit))) >= count) least |= bit;
  least = max(least, none + 1);
  const auto want = [&](uint32_t key, int i) {
    const uint32_t n = atomicAdd(&listed, 1u);
    if (n < kBeamListed) list[n] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~i);
  };
  const float limit = sample_value<MP_F32>(least);
#pragma unroll
  for (int g = 0; g < H; ++g) {
    if (!__any(eight[g] >= limit)) continue;
    float v[8];
    held[g].get(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // (a branch for the wave: the lanes' own cost more than all the rest of the pass)
      if (__any(v[e] >= limit)) {
        if (v[e] >= limit) want(beam_order(v[e]), first + 8 * kBeamThreads * g + e);
      }
    }
  }
  __syncthreads();
  int n = static_cast<int>(listed);
  if (tid == 0) {
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) all += wave_sums[w];
    parts[blockIdx.x] = BeamPart{all, most, 0};
  }
  if (n > kBeamListed) {
    // Many equal or ascending values: the value of the `count`-th largest, by bits, and then the index up to which its ties
    // are wanted.
    uint32_t key = least;  // reached by `count` values
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
      if (key & bit) continue;
      const uint32_t trial = (key | bit) & ~(bit - 1);
      uint32_t own = 0;
      each([&](int, const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) own += beam_order(v[e]) >= trial ? 1 : 0;
      });
      if (beam_total(own, of_wave) >= static_cast<uint32_t>(count)) key = trial;
    }
    uint32_t own = 0;
    each([&](int, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) own += beam_order(v[e]) > key ? 1 : 0;
    });
    const uint32_t above = beam_total(own, of_wave), ties = static_cast<uint32_t>(count) - above;
    int upto = 0;  // fewer than `ties` of the ties lie below it, and with it itself no more than those
    for (int bit = kMaxVocab / 2; bit; bit >>= 1) {
      own = 0;
      each([&](int i, const float (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) own += beam_order(v[e]) == key && i + e < (upto | bit) ? 1 : 0;
      });
      if (beam_total(own, of_wave) < ties) upto |= bit;
    }
    __syncthreads();
    if (tid == 0) listed = 0;
    __syncthreads();
    each([&](int i, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t k = beam_order(v[e]);
        if (k > key || (k == key && i + e <= upto)) want(k, i + e);
      }
    });
    __syncthreads();
    n = min(static_cast<int>(listed), kBeamListed);
  }
  BeamValue *out = lists + static_cast<int64_t>(blockIdx.x) * count;
  for (int e = tid; e < n; e += kBeamThreads) {
    const uint64_t me = list[e];
    int rank = 0;
    for (int i = 0; i < n; ++i) rank += list[i] > me ? 1 : 0;
    if (rank < count) out[rank] = BeamValue{sample_value<MP_F32>(static_cast<uint32_t>(me >> 32)), static_cast<int>(~static_cast<uint32_t>(me))};
  }
  for (int e = n + tid; e < count; e += kBeamThreads) out[e] = BeamValue{0.f, -1};
}

struct BeamBest {
  double total;
  int at;  // beam * vocab + token
  __device__ __forceinline__ bool before(double t, int i) const { return total > t || (total == t && at < i); }
};

constexpr int kBeamNear = 2048;  // continuations that LDS has room for

// One workgroup a request.  The best of the lists' heads, one a lane, that `count` of them reach is reached by `count`
// continuations; the few that reach it are put in order by counting, for each, those before it.
__global__ __launch_bounds__(256) void beam_merge_kernel(const BeamPart *__restrict__ parts, const BeamValue *__restrict__ lists,
                                                         const float *__restrict__ scores, const uint8_t *__restrict__ ended,
                                                         int beams, int splits, int count, int vocab, int pad, MpDivisor by_count,
                                                         MpDivisor by_splits, float *__restrict__ out_scores,
                                                         int64_t *__restrict__ out_beams, int64_t *__restrict__ out_tokens) {
  __shared__ double base[kMaxBeams], score[kMaxBeams], near_total[kBeamNear];  // base: log sum exp
  __shared__ int near_at[kBeamNear], listed;
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
  // in 32 bits, rounded down, so that whatever reaches a head reaches it here
  const auto order = [&](double total) { return total > none ? beam_order(__double2float_rd(total)) : 0u; };
  uint32_t head = 0;
  for (int i = tid & 63; i < n_lists; i += 64) head = max(head, order(candidate(i, 0).total));
  uint32_t least = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
    if (__popcll(__ballot(head >= (least | bit))) >= count) least |= bit;
  least = max(least, 1u);
  for (int i = tid; i < values; i += 256) {
    const int list = by_count(i);
    const BeamBest c = candidate(list, i - list * count);
    if (order(c.total) >= least) {
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
  if (n <= kBeamNear) {
    for (int e = tid; e < n; e += 256) {
      const BeamBest me{near_total[e], near_at[e]};
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += BeamBest{near_total[i], near_at[i]}.before(me.total, me.at) ? 1 : 0;
      if (rank < count) put(rank, me);
    }
    for (int e = n + tid; e < count; e += 256) put(e, BeamBest{none, 0});
    return;
  }
  // More are equal than LDS has room for: one after the other, each the best of those behind the last.
  BeamBest last{INFINITY, -1};
  for (int i = 0; i < count; ++i) {
    BeamBest best{none, INT32_MAX};
    for (int e = tid; e < values; e += 256) {
      const int list = by_count(e);
      const BeamBest c = candidate(list, e - list * count);
      if (last.before(c.total, c.at) && c.before(best.total, best.at)) best = c;
    }
    __syncthreads();  // the last round's have been read
    near_total[tid] = best.total;
    near_at[tid] = best.at;
    __syncthreads();
    for (int e = 0; e < 256; ++e) {
      const BeamBest c{near_total[e], near_at[e]};
      if (c.before(best.total, best.at)) best = c;
    }
    if (tid == 0) put(i, best);
    last = best;
  }
}

// Eights of a thread: eight, of which 116 registers leave four workgroups to a CU, but as few as keep 512 workgroups or more in the
// launch.  48 requests as above: sixteen 57 us, eight 50, four 50 with a merge of 14 in place of 10 us (before the looks for candidates
// were cut down to 45).
inline int beam_eights(int64_t rows, int64_t vocab, int dtype) {
  int h = 8;
  while (h > 2 && rows * mp_cdiv(vocab, 8 * h * kBeamThreads) < 512) h /= 2;
  return h;
}
inline int64_t beam_splits(int64_t rows, int64_t vocab, int dtype) { return mp_cdiv(vocab, 8 * beam_eights(rows, vocab, dtype) * kBeamThreads); }

template <int DT, int H>
void beam_rows_launch(const void *logits, int64_t stride, int64_t rows, int vocab, const uint8_t *ended, int splits, int count,
                      BeamPart *parts, BeamValue *lists, hipStream_t s) {
  hipLaunchKernelGGL((beam_rows_kernel<DT, H>), dim3(static_cast<unsigned>(rows * splits)), dim3(kBeamThreads), 0, s,
                     static_cast<const uint8_t *>(logits), stride, vocab, ended, splits, count, parts, lists);
}

}  // namespace

extern "C" size_t mp_beam_select_workspace_bytes(int64_t batch, int64_t beams, int64_t vocab, int64_t count, int dtype) {
  if (batch <= 0 || batch > INT32_MAX || beams < 1 || beams > kMaxBeams || vocab < 1 || vocab > kMaxVocab || count < 1 ||
      count > kMaxCount)
    return 0;
  const int64_t parts = batch * beams * beam_splits(batch * beams, vocab, dtype);
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
  if (workspace_bytes < mp_beam_select_workspace_bytes(batch, beams, vocab, count, dtype)) return MP_ERR_WORKSPACE;
  const int64_t rows = batch * beams;
  const int h = beam_eights(rows, vocab, dtype), n = static_cast<int>(vocab), k = static_cast<int>(count);
  const int splits = static_cast<int>(beam_splits(rows, vocab, dtype));
  BeamPart *parts = static_cast<BeamPart *>(workspace);
  BeamValue *lists = reinterpret_cast<BeamValue *>(parts + rows * splits);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define MP_BEAM(DT)                                                                                                        \
  do {                                                                                                                     \
    if (h == 8) beam_rows_launch<DT, 8>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                  \
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
