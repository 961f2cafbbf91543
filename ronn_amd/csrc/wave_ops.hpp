// Reductions and prefix sums over a wave on the DPP path (a few cycles per step where a shuffle goes through LDS); all lanes
// must be active.
#pragma once

#include <hip/hip_runtime.h>

template <int CTRL, int ROWMASK>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWMASK, 0xf, false);
}
// Inclusive prefix sum.
__device__ __forceinline__ int wave_scan_i(int v) {
    v = dpp_add<0x111, 0xf>(v);  // row_shr:1
    v = dpp_add<0x112, 0xf>(v);  // row_shr:2
    v = dpp_add<0x114, 0xf>(v);  // row_shr:4
    v = dpp_add<0x118, 0xf>(v);  // row_shr:8
    v = dpp_add<0x142, 0xa>(v);  // row_bcast15
    return dpp_add<0x143, 0xc>(v);  // row_bcast31
}
__device__ __forceinline__ int wave_sum_i(int v) { return __builtin_amdgcn_readlane(wave_scan_i(v), 63); }

template <int CTRL, int ROWMASK, typename F>
__device__ __forceinline__ float dpp_with(float v, float none, F f) {
    return f(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWMASK, 0xf, false)));
}
// The wave's values brought together by f, in an order that is always the same; `none` leaves a value as it is.
template <typename F>
__device__ __forceinline__ float wave_all(float v, float none, F f) {
    v = dpp_with<0x111, 0xf>(v, none, f);
    v = dpp_with<0x112, 0xf>(v, none, f);
    v = dpp_with<0x114, 0xf>(v, none, f);
    v = dpp_with<0x118, 0xf>(v, none, f);
    v = dpp_with<0x142, 0xa>(v, none, f);
    v = dpp_with<0x143, 0xc>(v, none, f);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_all(v, -INFINITY, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float wave_min(float v) {
    return wave_all(v, INFINITY, [](float x, float y) { return fminf(x, y); });
}
__device__ __forceinline__ float wave_sum(float v) {
    return wave_all(v, 0.0f, [](float x, float y) { return x + y; });
}
