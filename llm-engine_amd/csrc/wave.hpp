// Scans over a wave's lanes by register moves.
#pragma once

#include "common.hpp"

namespace em {

// v of the lane that a DPP control names, `none` where there is none or the row
// is masked out: a register move, where a shuffle goes through LDS.
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp_move(T v, T none) {
    static_assert(sizeof(T) == 4 || sizeof(T) == 8);
    int o[sizeof(T) / 4], x[sizeof(T) / 4];
    __builtin_memcpy(o, &none, sizeof(T));
    __builtin_memcpy(x, &v, sizeof(T));
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 4; ++i)
        x[i] = __builtin_amdgcn_update_dpp(o[i], x[i], CTRL, ROWS, 0xf, false);
    __builtin_memcpy(&v, x, sizeof(T));
    return v;
}
// Inclusive scan over a wave's lanes: within rows of 16 by shifts of 1, 2, 4
// and 8, then each odd row takes the last of the row before, then the upper two
// that of the lower two.
template <class T, class Op>
__device__ __forceinline__ T wave_scan(T v, T none, Op op) {
    v = op(v, dpp_move<0x111, 0xf>(v, none));
    v = op(v, dpp_move<0x112, 0xf>(v, none));
    v = op(v, dpp_move<0x114, 0xf>(v, none));
    v = op(v, dpp_move<0x118, 0xf>(v, none));
    v = op(v, dpp_move<0x142, 0xa>(v, none));
    v = op(v, dpp_move<0x143, 0xc>(v, none));
    return v;
}
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    return wave_scan(v, T(0), [](T a, T b) { return a + b; });
}
// The last lane's value, in every lane.
template <class T>
__device__ __forceinline__ T last_lane(T v) {
    int x[sizeof(T) / 4];
    __builtin_memcpy(x, &v, sizeof(T));
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 4; ++i) x[i] = __builtin_amdgcn_readlane(x[i], kWave - 1);
    __builtin_memcpy(&v, x, sizeof(T));
    return v;
}

}  // namespace em
