// kd_waves.h - sums and maxima over a wave's lanes by data parallel primitives, without LDS.
#pragma once

#include "kd_internal.h"

namespace kd {

// The value of the lane that `Control` names, `otherwise` where there is none.
template <int Control, int Rows, typename T> __device__ __forceinline__ T dpp_from(T v, T otherwise) {
    constexpr int kWords = sizeof(T) / 4;
    int in[kWords], rest[kWords];
    __builtin_memcpy(in, &v, sizeof v);
    __builtin_memcpy(rest, &otherwise, sizeof v);
#pragma unroll
    for (int i = 0; i < kWords; ++i) in[i] = __builtin_amdgcn_update_dpp(rest[i], in[i], Control, Rows, 0xf, false);
    __builtin_memcpy(&v, in, sizeof v);
    return v;
}
// v + that value, or + 0; within rows of lanes the hardware's own 0 stands in for it.
template <int Control, int Rows = 0xf> __device__ __forceinline__ double dpp_add(double v) {
    if constexpr (Rows != 0xf) return v + dpp_from<Control, Rows>(v, 0.0);
    int2 in;
    __builtin_memcpy(&in, &v, 8);
    in.x = __builtin_amdgcn_mov_dpp(in.x, Control, 0xf, 0xf, true);
    in.y = __builtin_amdgcn_mov_dpp(in.y, Control, 0xf, 0xf, true);
    double other;
    __builtin_memcpy(&other, &in, 8);
    return v + other;
}
template <int Control, int Rows = 0xf, typename T> __device__ __forceinline__ T dpp_max(T v) {
    return fmax(v, dpp_from<Control, Rows>(v, v));
}
template <typename T> __device__ __forceinline__ T from_lane(T v, int lane) {
    int in[sizeof(T) / 4];
    __builtin_memcpy(in, &v, sizeof v);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 4); ++i) in[i] = __builtin_amdgcn_readlane(in[i], lane);
    __builtin_memcpy(&v, in, sizeof v);
    return v;
}
// Running sums in each row of 16 lanes, then the rows' last ones handed on: the whole stays in the vector registers.
__device__ __forceinline__ double sum_of_16(double v) {
    v = dpp_add<0x111>(v);  // row_shr by 1, 2, 4, 8
    v = dpp_add<0x112>(v);
    v = dpp_add<0x114>(v);
    return dpp_add<0x118>(v);
}
__device__ __forceinline__ double wave_total(double v) {
    v = sum_of_16(v);
    v = dpp_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v = dpp_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return from_lane(v, 63);
}

// The largest that is no NaN.
template <typename T> __device__ __forceinline__ T most_of_16(T v) {
    v = dpp_max<0x111>(v);
    v = dpp_max<0x112>(v);
    v = dpp_max<0x114>(v);
    return dpp_max<0x118>(v);
}
template <typename T> __device__ __forceinline__ T wave_most(T v) {
    v = most_of_16(v);
    v = dpp_max<0x142, 0xa>(v);
    v = dpp_max<0x143, 0xc>(v);
    return from_lane(v, 63);
}

} // namespace kd
