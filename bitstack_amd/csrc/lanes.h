// Values from other lanes by the VALU's own lane shifts (no LDS): sums over the lanes of a wave.
#pragma once

#include "common.h"

// the value of another lane by CTRL (0 where there is none, and in the rows of 16 that ROWS leaves out)
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t bs_lane(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double bs_lane(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)bs_lane<CTRL, ROWS>((uint32_t)u) | (uint64_t)bs_lane<CTRL, ROWS>((uint32_t)(u >> 32)) << 32);
}
__device__ __forceinline__ uint32_t bs_read(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ double bs_read(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)bs_read((uint32_t)u, lane) | (uint64_t)bs_read((uint32_t)(u >> 32), lane) << 32);
}
// F's sum over the lanes up to this one (0 is its neutral value): within rows of 16 by shifts, then over the rows.  (By shuffles through LDS one of these takes 0.3 us.)
template <typename T, typename F>
__device__ __forceinline__ T bs_row_scan(T v, F f) {
    v = f(v, bs_lane<0x111>(v));
    v = f(v, bs_lane<0x112>(v));
    v = f(v, bs_lane<0x114>(v));
    return f(v, bs_lane<0x118>(v));
}
template <typename T, typename F>
__device__ __forceinline__ T bs_scan(T v, F f) {
    v = bs_row_scan(v, f);
    v = f(v, bs_lane<0x142, 0xa>(v));            // the last of rows 0 and 2 to rows 1 and 3
    return f(v, bs_lane<0x143, 0xc>(v));         // the last of row 1 to rows 2 and 3
}
// the value of the lane before this one, 0 in the first
template <typename T>
__device__ __forceinline__ T bs_lane_before(T v) { return bs_lane<0x138>(v); }
