// Rows of logits: eight neighbouring values at a time, and the order of values as unsigned numbers.
#pragma once
#include "wave_scan.h"

namespace {

constexpr int kMaxVocab = 1 << 19;

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

// The word is new to the compiler from here on: it would keep what it unpacked from many held words, and spill it.
__device__ __forceinline__ void sample_renew(uint32_t &w) { asm volatile("" : "+v"(w)); }

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

}  // namespace
