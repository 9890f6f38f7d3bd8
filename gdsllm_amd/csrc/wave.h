// Sums over a wave by lane, in VALU data movement (no LDS round trips).
#pragma once

#include "common.h"

namespace gdsllm {

// Inclusive sums over a wave, in 16-lane rows (DPP shifts) and then across them
// (DPP broadcasts of lanes 15 and 31).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_shift(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_shift(uint64_t v) {
    const uint32_t lo = dpp_shift<CTRL, ROWS>(static_cast<int>(v)), hi = dpp_shift<CTRL, ROWS>(static_cast<int>(v >> 32));
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_shift(double v) {
    return __builtin_bit_cast(double, dpp_shift<CTRL, ROWS>(__builtin_bit_cast(uint64_t, v)));
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp_shift<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v += dpp_shift<0x112, 0xF>(v);
    v += dpp_shift<0x114, 0xF>(v);
    v += dpp_shift<0x118, 0xF>(v);
    v += dpp_shift<0x142, 0xA>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
    v += dpp_shift<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
    return v;
}
// Lane 63's value, in every lane.
__device__ __forceinline__ int last_lane(int v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ double lane_double(double v, int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), l));
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), l));
    return __builtin_bit_cast(double, (hi << 32) | lo);
}
__device__ __forceinline__ int wave_sum(int v) { return last_lane(wave_scan(v)); }
// The largest of the wave's values, none of them negative, in every lane.
__device__ __forceinline__ int wave_max(int v) {
    v = max(v, dpp_shift<0x111, 0xF>(v));
    v = max(v, dpp_shift<0x112, 0xF>(v));
    v = max(v, dpp_shift<0x114, 0xF>(v));
    v = max(v, dpp_shift<0x118, 0xF>(v));
    v = max(v, dpp_shift<0x142, 0xA>(v));
    v = max(v, dpp_shift<0x143, 0xC>(v));
    return last_lane(v);
}

}  // namespace gdsllm
