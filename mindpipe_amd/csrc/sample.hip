// Tokens from logits at given random numbers, each row with its own temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T),  1 where x_i is the maximum
//   kept: the k largest (equal values: the lowest indexes), of those the shortest run from the largest down whose weights
//         reach p of their sum, of those the ones with w_i >= min-p; the largest is always kept
//   token: the first index, in index order, at which the kept weights' running sum exceeds u times their sum
//
// A token is decided by which side of a border a sum over the vocabulary falls on, so weights are computed in 64 bits
// and summed as whole numbers of 2^-44: sums of up to 2^19 of them fit 63 bits, and no order of additions changes them.
#include "mp_common.h"

namespace {

constexpr int kThreads = 1024, kWavesPerRow = kThreads / 64;
constexpr int kMaxVocab = 1 << 19;
constexpr int kSpan = 512;                     // indexes of one wave step: eight per lane
constexpr int kMaxSpans = kMaxVocab / kSpan;
constexpr int kBins = 2048;
constexpr double kOne = 17592186044416.0;      // 2^44
constexpr float kReach = 32.0f;                // e^-32 < 2^-46: past it a weight is no part of 2^-44

__device__ __forceinline__ float sample_value(const void *x, int64_t i, int dt) {
  const float v = mp_load_as_f32(x, i, dt);
  return v != v ? -INFINITY : v + 0.0f;  // NaN is never taken; -0 is 0
}

// Eight values from index i on, past the end -inf.
template <int DT>
__device__ __forceinline__ void sample_load8(const uint8_t *row, int i, int vocab, bool vec, float (&v)[8]) {
  if (vec && i + 8 <= vocab) {
    constexpr int N = MpChunk16<DT>::N;
    const uint4 *p = reinterpret_cast<const uint4 *>(row + static_cast<int64_t>(i) * (16 / N));
#pragma unroll
    for (int c = 0; c < 8 / N; ++c) {
      float f[N];
      mp_chunk_to_f32<DT>(p[c], f);
#pragma unroll
      for (int e = 0; e < N; ++e) v[c * N + e] = f[e] != f[e] ? -INFINITY : f[e] + 0.0f;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = i + e < vocab ? sample_value(row, i + e, DT) : -INFINITY;
}

// Order of the values as unsigned numbers, without the trailing bits that are alike in all values of the type.
template <int DT>
__device__ __forceinline__ uint32_t sample_key(float v) {
  constexpr int kDrop = DT == MP_F32 ? 0 : DT == MP_F16 ? 13 : 16;
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u ? ~b : b | 0x80000000u) >> kDrop;
}

__device__ __forceinline__ uint64_t sample_weight(float v, float top, double inv_t) {
  if (v == top) return static_cast<uint64_t>(kOne);
  const double d = (static_cast<double>(v) - static_cast<double>(top)) * inv_t;
  return d > -kReach ? static_cast<uint64_t>(exp(d) * kOne + 0.5) : 0;  // also -inf
}

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t u = __shfl_up(v, o, 64);
    v += lane >= o ? u : 0;
  }
  return v;
}

struct Border {       // the kept: keys above `key`, and the first `ties` indexes at it
  uint32_t key;
  uint32_t ties;
  uint64_t mass;      // weight of the kept
};

// What a border is looked for by: so many values, or so much weight.
struct Target {
  bool by_mass;
  uint32_t count;
  double mass;
};

struct SampleShared {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t span_mass[kMaxSpans];
  uint32_t span_ties[kMaxSpans];
  float top[kWavesPerRow];
  int at[kWavesPerRow];
  uint64_t wave_mass[kWavesPerRow];
  uint32_t wave_count[kWavesPerRow];
  int found;
  uint64_t before_mass;
  uint32_t before_count;
};

// The first bin, from bin 0 up, at which the running count or mass reaches the target, with what lies before it.  The last
// bin where none does.  All threads; kThreads = kBins / 2.
__device__ __forceinline__ int find_bin(SampleShared &s, const Target &t, uint32_t &count, uint64_t &mass) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
  const uint64_t m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
  uint64_t upto = wave_scan64(m0 + m1, lane);
  uint32_t cupto = static_cast<uint32_t>(wave_scan64(c0 + c1, lane));
  if (lane == 63) {
    s.wave_mass[wave] = upto;
    s.wave_count[wave] = cupto;
  }
  if (tid == 0) s.found = kBins - 1;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    upto += s.wave_mass[w];
    cupto += s.wave_count[w];
  }
  const auto there = [&](uint32_t c, uint64_t m) {
    return t.by_mass ? static_cast<double>(m) >= t.mass : c >= t.count;
  };
  if (there(cupto - c1, upto - m1)) atomicMin(&s.found, 2 * tid);
  else if (there(cupto, upto)) atomicMin(&s.found, 2 * tid + 1);
  __syncthreads();
  const int bin = s.found;
  if (bin >> 1 == tid) {
    const bool odd = bin & 1;
    s.before_count = cupto - c1 - (odd ? 0 : c0);
    s.before_mass = upto - m1 - (odd ? 0 : m0);
  }
  __syncthreads();
  count = s.before_count;
  mass = s.before_mass;
  return bin;
}

// The border inside the values of [low, high] (keys; those above `high` are `count` with weight `mass`): bins of keys,
// refined until a bin is one key.
template <int DT>
__device__ __forceinline__ Border find_border(SampleShared &s, const uint8_t *row, int vocab, bool vec, float top, double inv_t,
                                              uint32_t low, uint32_t high, Target t, uint32_t count, uint64_t mass) {
  const int tid = threadIdx.x;
  for (;;) {
    const int shift = max(0, 21 - __clz((high - low) | 1));  // 11 bits of the range
    __syncthreads();
    for (int b = tid; b < kBins; b += kThreads) {
      s.mass[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
    for (int i = tid * 8; i < vocab; i += kThreads * 8) {
      float v[8];
      sample_load8<DT>(row, i, vocab, vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t key = sample_key<DT>(v[e]);
        if (key >= low && key <= high && i + e < vocab) {
          const uint32_t bin = (high - key) >> shift;
          atomicAdd(&s.count[bin], 1u);
          atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[bin]),
                    static_cast<unsigned long long>(sample_weight(v[e], top, inv_t)));
        }
      }
    }
    __syncthreads();
    Target rest = t;
    rest.count = t.count - count;
    rest.mass = t.mass - static_cast<double>(mass);
    uint32_t c;
    uint64_t m;
    const uint32_t bin = find_bin(s, rest, c, m);
    const uint32_t n = s.count[bin];
    const uint64_t in = s.mass[bin];
    count += c;
    mass += m;
    if (shift == 0) {
      // one key: all of its values weigh the same
      const uint32_t key = high - bin;
      uint32_t ties = t.count - count;
      if (t.by_mass) {
        const uint64_t w = n ? in / n : 0;
        const double need = t.mass - static_cast<double>(mass);
        ties = w ? static_cast<uint32_t>(fmin(ceil(need / static_cast<double>(w)), static_cast<double>(n))) : n;
      }
      ties = min(max(ties, 1u), n);
      return {key, ties, mass + (n ? in / n * ties : 0)};
    }
    const uint32_t up = high - (bin << shift);
    const uint32_t down = up - low > (1u << shift) - 1 ? up - ((1u << shift) - 1) : low;
    high = up;
    low = down;
  }
}

// One workgroup per row.
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(const uint8_t *__restrict__ logits, int64_t stride, int vocab,
                                                          const float *__restrict__ u, const float *__restrict__ temperature,
                                                          const int32_t *__restrict__ top_k, const float *__restrict__ top_p,
                                                          const float *__restrict__ min_p, int64_t *__restrict__ tokens,
                                                          float *__restrict__ logprobs) {
  extern __shared__ uint8_t sample_smem[];
  SampleShared &s = *reinterpret_cast<SampleShared *>(sample_smem);
  constexpr int kSize = DT == MP_F32 ? 4 : 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const uint8_t *row = logits + r * stride * kSize;
  const bool vec = reinterpret_cast<uintptr_t>(row) % 16 == 0;

  // the maximum and its first index
  float top = -INFINITY;
  int at = INT32_MAX;
  for (int i = tid * 8; i < vocab; i += kThreads * 8) {
    float v[8];
    sample_load8<DT>(row, i, vocab, vec, v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v[e] > top) {
        top = v[e];
        at = i + e;
      }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float v = __shfl_xor(top, o, 64);
    const int a = __shfl_xor(at, o, 64);
    if (v > top || (v == top && a < at)) {
      top = v;
      at = a;
    }
  }
  if (lane == 0) {
    s.top[wave] = top;
    s.at[wave] = at;
  }
  __syncthreads();
  for (int w = 0; w < kWavesPerRow; ++w)
    if (s.top[w] > top || (s.top[w] == top && s.at[w] < at)) {
      top = s.top[w];
      at = s.at[w];
    }
  const float t = temperature ? temperature[r] : 1.0f;
  if (top == -INFINITY || !(t > 0.f)) {  // nothing may be taken, or the largest is
    if (tid == 0) {
      tokens[r] = top == -INFINITY ? -1 : at;
      logprobs[r] = top == -INFINITY ? -INFINITY : 0.f;
    }
    return;
  }
  const double inv_t = 1.0 / static_cast<double>(t);
  const int k = top_k ? top_k[r] : 0;
  const float p = top_p ? top_p[r] : 1.0f;
  const bool by_k = k > 0 && k < vocab, by_p = p < 1.0f;

  Border border{0, 0xFFFFFFFFu, 0};
  if (by_k || by_p) {
    // bins of equal width below the maximum, down to where weights end
    const float per = static_cast<float>((kBins - 1) / (kReach * static_cast<double>(t)));
    const auto bin_of = [&](float v) {
      const float d = (top - v) * per;  // NaN for two infinities
      return v == top ? 0 : static_cast<int>(fminf(d, static_cast<float>(kBins - 1)));
    };
    for (int b = tid; b < kBins; b += kThreads) {
      s.mass[b] = 0;
      s.count[b] = 0;
    }
    __syncthreads();
    uint32_t rest = 0;
    for (int i = tid * 8; i < vocab; i += kThreads * 8) {
      float v[8];
      sample_load8<DT>(row, i, vocab, vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (i + e >= vocab) continue;
        const int bin = bin_of(v[e]);
        if (bin == kBins - 1) {
          ++rest;
        } else {
          atomicAdd(&s.count[bin], 1u);
          atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[bin]),
                    static_cast<unsigned long long>(sample_weight(v[e], top, inv_t)));
        }
      }
    }
    // the last bin's weights are below 2^-45 each
    rest = static_cast<uint32_t>(wave_sum64(rest));
    if (lane == 0 && rest) atomicAdd(&s.count[kBins - 1], rest);
    __syncthreads();
    uint64_t total = 0;
    // keys of a bin: the values of the row that fall into it, found by its edges with a step of slack
    const auto border_of = [&](const Target &target) {
      uint32_t count;
      uint64_t mass;
      const int bin = find_bin(s, target, count, mass);
      if (bin == kBins - 1) return Border{0, 0xFFFFFFFFu, mass};  // what weighs nothing is never taken
      // smallest and largest key of the bin
      if (tid == 0) {
        s.count[0] = 0xFFFFFFFFu;
        s.count[1] = 0;
      }
      __syncthreads();
      uint32_t low = 0xFFFFFFFFu, high = 0;
      for (int i = tid * 8; i < vocab; i += kThreads * 8) {
        float v[8];
        sample_load8<DT>(row, i, vocab, vec, v);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < vocab && bin_of(v[e]) == bin) {
            low = min(low, sample_key<DT>(v[e]));
            high = max(high, sample_key<DT>(v[e]));
          }
      }
      atomicMin(&s.count[0], low);
      atomicMax(&s.count[1], high);
      __syncthreads();
      low = s.count[0];
      high = s.count[1];
      return find_border<DT>(s, row, vocab, vec, top, inv_t, low, high, target, count, mass);
    };
    if (by_p && !by_k) {
      uint64_t mine = s.mass[2 * tid] + s.mass[2 * tid + 1];
      mine = wave_sum64(mine);
      if (lane == 0) s.wave_mass[wave] = mine;
      __syncthreads();
      for (int w = 0; w < kWavesPerRow; ++w) total += s.wave_mass[w];
      __syncthreads();
      border = border_of({true, 0, static_cast<double>(p) * static_cast<double>(total)});
    } else {
      border = border_of({false, static_cast<uint32_t>(k), 0.0});
      if (by_p) {
        // the same search over the kept alone
        const uint32_t key = border.key, ties = border.ties;
        const double need = static_cast<double>(p) * static_cast<double>(border.mass);
        const Border q = find_border<DT>(s, row, vocab, vec, top, inv_t, key, sample_key<DT>(top), {true, 0, need}, 0, 0);
        border = q.key > key ? q : Border{key, min(q.ties, ties), 0};
      }
    }
  }

  // kept weight of each span of the row, with the ties at the border counted apart
  const uint64_t floor_w = min_p && min_p[r] > 0.f
                               ? static_cast<uint64_t>(fmin(static_cast<double>(min_p[r]), 1.0) * kOne + 0.5)
                               : 0;
  const int spans = (vocab + kSpan - 1) / kSpan;
  __shared__ uint64_t tie_w;
  if (tid == 0) tie_w = 0;
  __syncthreads();
  for (int sp = wave; sp < spans; sp += kWavesPerRow) {
    const int i = sp * kSpan + lane * 8;
    float v[8];
    sample_load8<DT>(row, i, vocab, vec, v);
    uint64_t mass = 0;
    uint32_t ties = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t key = sample_key<DT>(v[e]);
      if (key < border.key || i + e >= vocab) continue;
      const uint64_t w = sample_weight(v[e], top, inv_t);
      if (w < floor_w) continue;
      if (key > border.key) {
        mass += w;
      } else {
        ++ties;
        tie_w = w;  // the same for all
      }
    }
    mass = wave_sum64(mass);
    ties = static_cast<uint32_t>(wave_sum64(ties));
    if (lane == 0) {
      s.span_mass[sp] = mass;
      s.span_ties[sp] = ties;
    }
  }
  __syncthreads();
  if (wave != 0) return;

  // one wave: ties to weights, the sum, the span that the token is in, the token
  uint64_t total = 0;
  uint32_t taken = 0;
  for (int b = 0; b < spans; b += 64) {
    const bool in = b + lane < spans;
    const uint32_t ties = in ? s.span_ties[b + lane] : 0;
    const uint32_t upto = static_cast<uint32_t>(wave_scan64(ties, lane));
    const uint32_t before = taken + upto - ties;
    const uint32_t room = border.ties > before ? border.ties - before : 0;
    const uint32_t mine = min(ties, room);
    uint64_t m = in ? s.span_mass[b + lane] + tie_w * mine : 0;
    if (in) {
      s.span_mass[b + lane] = m;
      s.span_ties[b + lane] = before;  // ties before the span
    }
    taken += __builtin_amdgcn_readlane(upto, 63);
    total += wave_sum64(m);
  }
  // u below 1 leaves the target below the sum; rounding and other u are held there
  const double target = fmin(fmax(static_cast<double>(u[r]), 0.0) * static_cast<double>(total),
                             static_cast<double>(total) * (1.0 - 0x1p-52) - 1.0);
  uint64_t run = 0;
  int span = spans - 1;
  for (int b = 0; b < spans; b += 64) {
    const uint64_t m = b + lane < spans ? s.span_mass[b + lane] : 0;
    const uint64_t upto = run + wave_scan64(m, lane);
    const uint64_t past = __ballot(b + lane < spans && static_cast<double>(upto) > target);
    if (past) {
      const int l = __builtin_ctzll(past);
      span = b + l;
      run = __shfl(upto - m, l, 64);
      break;
    }
    run = __shfl(upto, 63, 64);
  }
  const int i = span * kSpan + lane * 8;
  float v[8];
  sample_load8<DT>(row, i, vocab, vec, v);
  uint64_t w[8], mass = 0;
  uint32_t ties = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t key = sample_key<DT>(v[e]);
    w[e] = key >= border.key && i + e < vocab ? sample_weight(v[e], top, inv_t) : 0;
    if (w[e] < floor_w) w[e] = 0;
    ties += key == border.key && w[e] ? 1 : 0;
  }
  uint32_t before = s.span_ties[span] + static_cast<uint32_t>(wave_scan64(ties, lane)) - ties;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (sample_key<DT>(v[e]) == border.key && w[e]) w[e] = before++ < border.ties ? w[e] : 0;
    mass += w[e];
  }
  uint64_t upto = run + wave_scan64(mass, lane) - mass;
  int found = INT32_MAX;
  uint64_t weight = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    upto += w[e];
    if (w[e] && static_cast<double>(upto) > target && found == INT32_MAX) {
      found = i + e;
      weight = w[e];
    }
  }
  const uint64_t who = __ballot(found != INT32_MAX);
  if (who && lane == __builtin_ctzll(who)) {
    tokens[r] = found;
    logprobs[r] = static_cast<float>(log(static_cast<double>(weight) / static_cast<double>(total)));
  }
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
  const dim3 grid(static_cast<unsigned>(rows));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const auto *x = static_cast<const uint8_t *>(logits);
  const int n = static_cast<int>(vocab);
#define MP_SAMPLE(DT)                                                                                                       \
  hipLaunchKernelGGL(sample_kernel<DT>, grid, dim3(kThreads), sizeof(SampleShared), s, x, stride, n, u, temperature, top_k, \
                     top_p, min_p, tokens, logprobs)
  if (dtype == MP_F16) MP_SAMPLE(MP_F16);
  else if (dtype == MP_BF16) MP_SAMPLE(MP_BF16);
  else MP_SAMPLE(MP_F32);
#undef MP_SAMPLE
  MP_CHECK_LAUNCH();
  return MP_OK;
}
