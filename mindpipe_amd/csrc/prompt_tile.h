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

// odd: whether the values' tile holds an infinity or NaN.
template <int D, int DT>
__device__ __forceinline__ void prompt_odd_values(uint32_t &odd, const int8_t *vs, int lane) {
  for (int e = lane; e < PromptTile<D>::kBytes / 16; e += 64) {
    const i4_t x = *reinterpret_cast<const i4_t *>(vs + 16 * e);
#pragma unroll
    for (int i = 0; i < 4; ++i) odd |= attn_odd16<DT>(x[i]) || attn_odd16<DT>(static_cast<uint32_t>(x[i]) >> 16);
  }
}

}  // namespace
