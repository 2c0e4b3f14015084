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

// v of the lanes 0 .. 15 and 16 .. 31 of each half of a wave (HALF 16), or of a wave's first and second half (HALF 32),
// the first's in both and the second's in both
template <int HALF>
__device__ __forceinline__ void halves(uint32_t v, uint32_t& first, uint32_t& second) {
    static_assert(HALF == 16 || HALF == 32, "rows or halves of a wave");
    const auto r = HALF == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    first = r[0];
    second = r[1];
}
template <int HALF>
__device__ __forceinline__ void halves(float v, float& first, float& second) {
    uint32_t a, b;
    halves<HALF>(__float_as_uint(v), a, b);
    first = __uint_as_float(a);
    second = __uint_as_float(b);
}
template <int HALF>
__device__ __forceinline__ void halves(double v, double& first, double& second) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    uint32_t al, ah, bl, bh;
    halves<HALF>((uint32_t)u, al, bl);
    halves<HALF>((uint32_t)(u >> 32), ah, bh);
    first = __longlong_as_double((long long)((uint64_t)ah << 32 | al));
    second = __longlong_as_double((long long)((uint64_t)bh << 32 | bl));
}

// v of this lane's part of D lanes and of the part beside it, where each part's lanes share one value: `a` and `b` are
// the same two values in both parts, in either order.
template <int D, typename T>
__device__ __forceinline__ void neighbours(T v, T& a, T& b) {
    static_assert(D == 1 || D == 2 || D == 4 || D == 8 || D == 16 || D == 32, "parts of a wave");
    a = v;
    if constexpr (D == 1) b = dpp<DPP_XOR1>(v);
    else if constexpr (D == 2) b = dpp<DPP_XOR2>(v);
    else if constexpr (D == 4) b = dpp<DPP_HALF_MIRROR>(v);          // the other quad of eight
    else if constexpr (D == 8) b = dpp<DPP_ROR8>(v);                 // the other eight of sixteen
    else halves<D>(v, a, b);
}

// op over the L lanes of this lane's part; op is symmetric
template <int L, int D = 1, typename T, typename Op>
__device__ __forceinline__ T all_lanes(T v, Op op) {
    if constexpr (D >= L) return v;
    else {
        T a, b;
        neighbours<D>(v, a, b);
        return all_lanes<L, 2 * D>(op(a, b), op);
    }
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
