// Sums over the lanes of a wave, 32 and 64 bits, by DPP (cross-lane moves of the VALU; __shfl goes through the LDS).
#pragma once
#include "mp_common.h"

namespace {

// One step of a scan over the wave: lanes whose row or bank is masked, or whose source is none, add 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_from(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_from(uint64_t v) {
  const uint32_t lo = dpp_from<CTRL, ROWS>(static_cast<uint32_t>(v)), hi = dpp_from<CTRL, ROWS>(static_cast<uint32_t>(v >> 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}
// Sums up to and with each lane: within rows of 16 (row_shr 1, 2, 4, 8), then row 0 into 1 and 2 into 3, then 1 into 2 and 3.
template <class U>
__device__ __forceinline__ U wave_scan(U v) {
  v += dpp_from<0x111, 0xF>(v);
  v += dpp_from<0x112, 0xF>(v);
  v += dpp_from<0x114, 0xF>(v);
  v += dpp_from<0x118, 0xF>(v);
  v += dpp_from<0x142, 0xA>(v);  // row_bcast 15
  v += dpp_from<0x143, 0xC>(v);  // row_bcast 31
  return v;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  return static_cast<uint64_t>(last_lane(static_cast<uint32_t>(v >> 32))) << 32 | last_lane(static_cast<uint32_t>(v));
}
template <class U>
__device__ __forceinline__ U wave_sum(U v) {
  return last_lane(wave_scan(v));
}

}  // namespace
