// The best continuations of each request over its beams and the vocabulary.
//
//   total(k, v) = score_k + x_kv - log sum_v exp x_kv      (an ended beam has one continuation, of its own score)
//   the `count` largest totals of a request, from the largest down; of equal ones those of the lowest beam, then token
//
// Which of two totals is larger decides a whole number, so they are made in 64 bits: the order inside of a row is that of its
// logits, and between rows the sums of exponentials decide, each off by less than 2^-36 of itself.
//
// Two launches.  Of each row, workgroups take a part of the vocabulary each (a row is read once and stays in registers): they leave
// the part's maximum, its sum of exponentials and its `count` largest values in order.  No value can be among a request's best
// that is not among those.  Then one wave a request merges the parts' lists, taking the best of their heads each time.
#include "logits.h"

namespace {

constexpr int kMaxBeams = 64, kMaxCount = 64;  // a lane to each
constexpr int kBeamWaves = 4, kBeamThreads = 64 * kBeamWaves;
constexpr int kBeamListed = 512;               // candidates of a part that LDS has room for
constexpr int kQuads = kBeamThreads / 4;       // a lane of a wave to each
constexpr double kLog2eD = 1.4426950408889634;

// exp(d) for d <= 0, in 64 bits: 2^n from the whole part of d log2 e and 2^r, r in [-1/2, 1/2], by the series of exp(r ln 2) up to
// its ninth power, which leaves less than 2^-37.  Below e^-800: 0.
__device__ __forceinline__ double beam_exp(double d) {
  const double magic = 1.5 * 0x1p52;  // a sum with it is whole
  d = fmax(d, -800.0);
  const double t = fma(d, kLog2eD, magic), r = fma(d, kLog2eD, magic - t);
  double p = 1.017808600923970e-7;                         // (ln 2)^9 / 9!
  p = fma(p, r, 1.321548679014431e-6);
  p = fma(p, r, 1.525273380405984e-5);
  p = fma(p, r, 1.540353039338161e-4);
  p = fma(p, r, 1.333355814642844e-3);
  p = fma(p, r, 9.618129107628477e-3);
  p = fma(p, r, 5.550410866482158e-2);
  p = fma(p, r, 2.402265069591007e-1);
  p = fma(p, r, 6.931471805599453e-1);
  p = fma(p, r, 1.0);
  return ldexp(p, __double2loint(t));
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

  const auto each = [&](auto f) {  // f(index, its eight values), NaN as -inf
#pragma unroll
    for (int g = 0; g < H; ++g) {
#pragma unroll
      for (int i = 0; i < Eight<DT>::kWords; ++i) sample_renew(held[g].w[i]);
      float v[8];
      held[g].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fmaxf(v[e], -INFINITY);
      f(first + 8 * kBeamThreads * g, v);
    }
  };
  float top = -INFINITY;
  each([&](int, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, v[e]);
  });
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
    each([&](int, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += beam_exp(static_cast<double>(v[e]) - base);
    });
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
  each([&](int i, const float (&v)[8]) {
    float eight = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) eight = fmaxf(eight, v[e]);
    if (eight < limit) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v[e] >= limit) want(beam_order(v[e]), i + e);
  });
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
  int beam, token;
  __device__ __forceinline__ bool before(const BeamBest &o) const {
    return total > o.total || (total == o.total && (beam < o.beam || (beam == o.beam && token < o.token)));
  }
};

constexpr int kBeamLists = 8192;  // values of the lists that LDS has room for

__global__ __launch_bounds__(256) void beam_merge_kernel(const BeamPart *__restrict__ parts, const BeamValue *__restrict__ lists,
                                                         const float *__restrict__ scores, const uint8_t *__restrict__ ended,
                                                         int beams, int splits, int count, int pad, float *__restrict__ out_scores,
                                                         int64_t *__restrict__ out_beams, int64_t *__restrict__ out_tokens) {
  extern __shared__ __attribute__((aligned(16))) uint8_t beam_smem[];
  __shared__ double base[kMaxBeams];  // log sum exp
  __shared__ bool infinite[kMaxBeams];
  const int64_t b = blockIdx.x;
  const int n_lists = beams * splits, values = n_lists * count;
  const BeamValue *from = lists + b * values;
  if (values <= kBeamLists) {
    BeamValue *near = reinterpret_cast<BeamValue *>(beam_smem);
    for (int i = threadIdx.x; i < values; i += 256) near[i] = from[i];
    from = near;
  }
  if (threadIdx.x < beams) {
    const BeamPart *p = parts + (b * beams + threadIdx.x) * splits;
    float top = -INFINITY;
    for (int s = 0; s < splits; ++s) top = fmaxf(top, p[s].top);
    double sum = 0.0;
    if (top == INFINITY) {
      for (int s = 0; s < splits; ++s) sum += p[s].top == INFINITY ? p[s].sum : 0.0;
    } else if (top > -INFINITY) {
      for (int s = 0; s < splits; ++s)
        if (p[s].top > -INFINITY) sum += p[s].sum * beam_exp(static_cast<double>(p[s].top) - static_cast<double>(top));
    }
    // with infinite logits those alone count, as if they were 0, and all others are -inf
    infinite[threadIdx.x] = top == INFINITY;
    base[threadIdx.x] = (top == INFINITY ? 0.0 : static_cast<double>(top)) + log(sum);
  }
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  const double none = -INFINITY;

  // entry `at` of a list as a candidate; nothing there: -inf
  const auto candidate = [&](int list, int at) {
    BeamBest c{none, INT32_MAX, INT32_MAX};
    const int k = list / splits;
    const double score = scores[b * beams + k];
    if (ended && ended[b * beams + k]) {  // the row's first list has its one continuation
      if (list % splits == 0 && at == 0) c = BeamBest{score, k, pad};
    } else if (at < count) {
      const BeamValue v = from[list * count + at];
      if (v.token >= 0) {
        const double x = infinite[k] ? (v.value == INFINITY ? 0.0 : none) : static_cast<double>(v.value);
        c = BeamBest{score + (x - base[k]), k, v.token};
      }
    }
    if (!(c.total > none)) c = BeamBest{none, INT32_MAX, INT32_MAX};  // -inf and NaN
    return c;
  };
  // a lane's lists are lane, lane + 64, ..; taken[i] of each are gone, the best of their heads is `mine`
  uint8_t *taken = beam_smem + (values <= kBeamLists ? values * sizeof(BeamValue) : 0);
  for (int i = lane; i < n_lists; i += 64) taken[i] = 0;
  int of = 0;
  const auto best_own = [&]() {
    BeamBest m{none, INT32_MAX, INT32_MAX};
    for (int i = lane; i < n_lists; i += 64) {
      const BeamBest c = candidate(i, taken[i]);
      if (c.before(m)) {
        m = c;
        of = i;
      }
    }
    return m;
  };
  BeamBest mine = best_own();
  for (int i = 0; i < count; ++i) {
    BeamBest best = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const BeamBest other{__shfl_xor(best.total, o, 64), __shfl_xor(best.beam, o, 64), __shfl_xor(best.token, o, 64)};
      if (other.before(best)) best = other;
    }
    if (lane == 0) {
      const bool found = best.total > none;
      out_scores[b * count + i] = static_cast<float>(best.total);
      out_beams[b * count + i] = found ? best.beam : -1;
      out_tokens[b * count + i] = found ? best.token : -1;
    }
    if (best.total > none && mine.beam == best.beam && mine.token == best.token) {
      ++taken[of];
      mine = best_own();
    }
  }
}

// Eights of a thread: as many as hold a row in few parts, but as few as keep 512 workgroups or more in the launch.
inline int beam_eights(int64_t rows, int64_t vocab, int dtype) {
  int h = dtype == MP_F32 ? 8 : 16;
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
    if (h == 16) beam_rows_launch<DT, DT == MP_F32 ? 8 : 16>(logits, stride, rows, n, ended, splits, k, parts, lists, s);  \
    else if (h == 8) beam_rows_launch<DT, 8>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                  \
    else if (h == 4) beam_rows_launch<DT, 4>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                  \
    else beam_rows_launch<DT, 2>(logits, stride, rows, n, ended, splits, k, parts, lists, s);                              \
  } while (0)
  if (dtype == MP_F16) MP_BEAM(MP_F16);
  else if (dtype == MP_BF16) MP_BEAM(MP_BF16);
  else MP_BEAM(MP_F32);
#undef MP_BEAM
  MP_CHECK_LAUNCH();
  const int64_t values = beams * splits * count;
  const size_t lds = (values <= kBeamLists ? values * sizeof(BeamValue) : 0) + beams * splits;
  if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void *>(beam_merge_kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)) != hipSuccess)
    return MP_ERR_HIP;
  hipLaunchKernelGGL(beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(256), lds, s, parts, lists, scores, ended,
                     static_cast<int>(beams), splits, k, static_cast<int>(pad), out_scores, out_beams, out_tokens);
  MP_CHECK_LAUNCH();
  return MP_OK;
}
