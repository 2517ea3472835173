// Tiles of 64 positions of keys and values in LDS, and their products with the 32 query rows of a wave, for the attention of packed
// rows (prompt.hip, masked.hip).
#pragma once
#include "attn_common.h"

namespace {

constexpr int kWaves = 4, kRows = 32 * kWaves;
constexpr int kTile = 64;  // positions

typedef short as4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) as4_t *lds_as4;

// Through buffer descriptors and integers, in non-template functions: the compiler makes LDS reads wait for the LDS loads that it
// recognises as such.  Offsets are below 2^31 (the launch sees to it) and rows inside the tensors.
__device__ __forceinline__ void prompt_lds_load16(const uint16_t *base, uint32_t offset, int8_t *lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      mp_rsrc(base, 0x80000000u), reinterpret_cast<__attribute__((address_space(3))) void *>(reinterpret_cast<uintptr_t>(lds)),
      16, offset, 0, 0, 0);
}
// The wave's loads have landed, and every wave is so far.
__device__ __forceinline__ void prompt_wait() { asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory"); }
// Four rows' values of one column: lane i of 16 gives 8 bytes of row i / 4 and gets column i of the four rows.
__device__ __forceinline__ as4_t prompt_read_tr(const __restrict__ lds_as4 p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }
__device__ __forceinline__ uint2 prompt_read_tr(const int8_t *lds) {
  return __builtin_bit_cast(uint2, prompt_read_tr((lds_as4) reinterpret_cast<uintptr_t>(lds)));
}

template <int DT>
__device__ __forceinline__ f16_t prompt_mfma(uint4 a, uint4 b, f16_t c) {
  if constexpr (DT == MP_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(abf8_t, a), __builtin_bit_cast(abf8_t, b), c, 0, 0,
                                                   0);
}

template <int D>
struct PromptTile {
  static constexpr int kChunks = D / 8;         // of 16 bytes in a row
  static constexpr int kBytes = kTile * D * 2;  // of K or of V
  static constexpr int kStage = 2 * kBytes;     // of both; two stages, 32 / 64 / 128 KB
  static constexpr int kLoads = kBytes / 1024 / kWaves;
  // LDS chunk of a row's chunk c (and back).  K is read by 16 rows at a time in one column of chunks, V by four rows at a time
  // in four columns; 256 bytes are all banks.
  static __device__ __forceinline__ int k_chunk(int row, int c) { return c ^ (D == 64 ? (row >> 1) & 7 : row & 15); }
  static __device__ __forceinline__ int v_chunk(int row, int c) {
    return c ^ (D == 64 ? ((row & 2) << 1) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3));
  }
};

struct PackedPlan {
  const int32_t *starts;
  int batch, rows, grp;
  // offsets of a sequence; sequence `batch` is what lies behind the last one, and batch + 1 what lies before the first
  __device__ __forceinline__ int first(int b) const { return b > batch ? 0 : min(max(starts[b], 0), rows); }
  __device__ __forceinline__ int end(int b) const { return b < batch ? max(first(b), first(b + 1)) : b == batch ? rows : first(0); }
  __device__ __forceinline__ int operator()(int b, int per) const {
    return static_cast<int>((static_cast<int64_t>(end(b) - first(b)) * grp + per - 1) / per);
  }
};

// Scores of the tile's positions, unscaled: s[t][r] is position 32 t + 8 (r >> 2) + 4 h + (r & 3) for the row of this lane.
template <int D, int DT>
__device__ __forceinline__ void prompt_scores(const int8_t *ks, const uint4 (&qf)[D / 16], f16_t (&s)[kTile / 32], int i32, int h) {
  using T = PromptTile<D>;
  constexpr int kS = kTile / 32;
#pragma unroll
  for (int t = 0; t < kS; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
  constexpr int kC = D / 16, kAheadK = 1;  // pairs of operands that are read before they are used
  i4_t kf[kAheadK + 1][kS];
  const auto keys = [&](int c) {
#pragma unroll
    for (int t = 0; t < kS; ++t) {
      const int r = 32 * t + i32;
      kf[c % (kAheadK + 1)][t] = *reinterpret_cast<const i4_t *>(ks + r * (D * 2) + 16 * T::k_chunk(r, 2 * c + h));
    }
  };
#pragma unroll
  for (int c = 0; c < kAheadK; ++c) keys(c);
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    if (c + kAheadK < kC) keys(c + kAheadK);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < kS; ++t) s[t] = prompt_mfma<DT>(__builtin_bit_cast(uint4, kf[c % (kAheadK + 1)][t]), qf[c], s[t]);
  }
}

// 16 bytes of the values' tile hold an infinity or NaN.
template <int D, int DT>
__device__ __forceinline__ uint32_t prompt_odd_values(const int8_t *vs, int lane) {
  uint32_t odd = 0;
  for (int e = lane; e < PromptTile<D>::kBytes / 16; e += 64) {
    const i4_t x = *reinterpret_cast<const i4_t *>(vs + 16 * e);
#pragma unroll
    for (int i = 0; i < 4; ++i) odd |= attn_odd16<DT>(x[i]) || attn_odd16<DT>(static_cast<uint32_t>(x[i]) >> 16);
  }
  return odd;
}

// The tile's scores (-inf where masked) into the row's maximum m, sum l and outputs o.
template <int D, int DT>
__device__ __forceinline__ void prompt_weigh(const f16_t (&s)[kTile / 32], const int8_t *vs, f16_t (&o)[D / 32], float &m, float &l,
                                             float scale2, int lane) {
  using T = PromptTile<D>;
  constexpr int kS = kTile / 32;
  const int h = lane >> 5;
  float top = s[0][0];
#pragma unroll
  for (int t = 0; t < kS; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[t][r]);
  top *= scale2;
  if (__any(top > m + kMaxLag)) {
    const float new_m = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, 64)));
    const float f = m == new_m ? 1.0f : __builtin_amdgcn_exp2f(m - new_m);
    l *= f;
    m = new_m;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= f;
  }
  const float base = m == -INFINITY ? 0.f : m - kRaise<DT>;
  // O^T: step c of 16 positions, whose weights are those of positions 16 c + 4 h + {0..3, 8..11}: s[c / 2][8 (c & 1) ..].  The
  // next step's weights are made between the matrix instructions of this one.
  constexpr int kSteps = kTile / 16, kD = D / 32;
  const int trow = 4 * h + ((lane & 15) >> 2), tcol = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  uint32_t w[2][4];
  constexpr int kAheadV = 2;  // operands of V that are read before they are used (1: 461 -> 470 us, 4: 463, heads of 256 92 -> 101 and 94)
  uint4 vf[kAheadV + 1];
  // Weights are rounded to the values' type, off by up to 2^-11 (fp16) or 2^-8 (bf16) of themselves each, and their sum takes
  // them as rounded: errors (rms) are 1.2 (fp16) to 1.3 times (bf16; heads of 256 1.4) those of 32-bit weights, 2.1e-3 for
  // 1.6e-3 of the packed prompts' outputs.  A second product with what the rounding leaves would take that away for 471 -> 611 us
  // there, 153 -> 209 for chunks of 32 heads and 91 -> 107 for heads of 256.
  const auto weight = [&](int c, int i) {
    const int r = 8 * (c & 1) + 2 * i;
    w[c & 1][i] = attn_pack2<DT>(__builtin_amdgcn_exp2f(fmaf(s[c / 2][r], scale2, -base)),
                                 __builtin_amdgcn_exp2f(fmaf(s[c / 2][r + 1], scale2, -base)));
    l = attn_add2<DT>(w[c & 1][i], l);
  };
  const auto values = [&](int j) {
    const int c = j / kD, d = j % kD;
    const int ra = 16 * c + trow, rb = ra + 8;
    const uint2 lo = prompt_read_tr(vs + ra * (D * 2) + 16 * T::v_chunk(ra, 4 * d + tcol) + 8 * (lane & 1));
    const uint2 hi = prompt_read_tr(vs + rb * (D * 2) + 16 * T::v_chunk(rb, 4 * d + tcol) + 8 * (lane & 1));
    vf[j % (kAheadV + 1)] = make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
#pragma unroll
  for (int j = 0; j < kAheadV; ++j) values(j);
#pragma unroll
  for (int i = 0; i < 4; ++i) weight(0, i);
#pragma unroll
  for (int c = 0; c < kSteps; ++c) {
    const uint4 wf = make_uint4(w[c & 1][0], w[c & 1][1], w[c & 1][2], w[c & 1][3]);
#pragma unroll
    for (int d = 0; d < kD; ++d) {
      __builtin_amdgcn_sched_barrier(0);
      const int j = c * kD + d;
      o[d] = prompt_mfma<DT>(vf[j % (kAheadV + 1)], wf, o[d]);
      if (j + kAheadV < kSteps * kD) values(j + kAheadV);
      if (c + 1 < kSteps) {
#pragma unroll
        for (int i = 4 * d / kD; i < 4 * (d + 1) / kD; ++i) weight(c + 1, i);
      }
    }
  }
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace
