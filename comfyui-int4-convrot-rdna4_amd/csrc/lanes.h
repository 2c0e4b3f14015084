// Reductions over the first lanes of a wave's power-of-two parts, every lane
// getting the result, in an order that depends on nothing but L: the same
// values give the same bits.
#pragma once

#include "mxfp4.h"

namespace convrot {

constexpr int DPP_HALF_MIRROR = 0x141;

template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xf, 0xf, true);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// op(v, v of the lanes that share this lane's part of L lanes)
template <int L, typename T, typename Op>
__device__ __forceinline__ T all_lanes(T v, Op op) {
    static_assert(L >= 1 && L <= 64 && (L & (L - 1)) == 0, "parts of a wave");
    if constexpr (L >= 2) v = op(v, dpp<DPP_XOR1>(v));
    if constexpr (L >= 4) v = op(v, dpp<DPP_XOR2>(v));
    if constexpr (L >= 8) v = op(v, dpp<DPP_HALF_MIRROR>(v));    // quads are uniform: the other quad of eight
    if constexpr (L >= 16) v = op(v, dpp<DPP_ROR8>(v));          // the other eight of sixteen
    if constexpr (L >= 32) v = op(v, __shfl_xor(v, 16));
    if constexpr (L >= 64) v = op(v, __shfl_xor(v, 32));
    return v;
}

template <int L, typename T>
__device__ __forceinline__ T sum_lanes(T v) {
    return all_lanes<L>(v, [](T a, T b) { return a + b; });
}
template <int L>
__device__ __forceinline__ float max_lanes(float v) {
    return all_lanes<L>(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace convrot
