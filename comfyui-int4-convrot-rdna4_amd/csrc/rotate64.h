// The exact block-Hadamard ("ConvRot") rotation in fp64 that the quantizers
// share (rotquant.hip, rmsnorm.hip): a lane holds 16 consecutive elements, a
// wave 1024; how far it is exact is said in rotquant.hip.
#pragma once

#include "common.h"

namespace convrot {

constexpr int kChunk = 16;       // elements per lane per pass
constexpr int kPad = 17;         // fp64 words per lane slot in the transpose buffer

// radix-4 stage of the regular Hadamard H4 on four values:
// H4 v = (sum v) 1 - 2 reverse(v)   (H4 as in _int4/eager.py:32-36)
// (every value is exact: sums of inputs times powers of two; fma keeps one op)
__device__ __forceinline__ void h4_stage(double& a, double& b, double& c, double& d, double scale) {
    const double S = (scale == 1.0) ? ((a + b) + (c + d)) : ((a + b) + (c + d)) * scale;
    double t = -2.0 * scale;
    // -2 is an inline constant of the 3-operand fma; any other factor would be
    // a literal, which only the 2-operand fmac takes (plus a copy of S per
    // output): hold it in an SGPR pair instead
    if (scale != 1.0) asm("" : "+s"(t));
    const double na = __builtin_fma(t, d, S), nb = __builtin_fma(t, c, S);
    const double nc = __builtin_fma(t, b, S), nd = __builtin_fma(t, a, S);
    a = na; b = nb; c = nc; d = nd;
}

// stage over one base-4 digit of the 16-entry register array (stride 1 or 4)
template <int STRIDE>
__device__ __forceinline__ void stage16(double (&v)[16], double scale) {
#pragma unroll
    for (int base = 0; base < 16; ++base) {
        if ((base / STRIDE) % 4 != 0) continue;
        h4_stage(v[base], v[base + STRIDE], v[base + 2 * STRIDE], v[base + 3 * STRIDE], scale);
    }
}

// group-local element index held in register slot i after the last stage,
// for lane position gl within the group (see the transpose below)
template <int G>
__device__ __forceinline__ int final_elem(int gl, int i) {
    if constexpr (G == 256) return gl + 16 * i;
    else if constexpr (G == 64) return 16 * (i >> 2) + 4 * gl + (i & 3);
    else return i;
}

// all butterfly stages of one chunk (16 values of the lane in v); tbuf is the
// wave's transpose buffer
template <int G>
__device__ __forceinline__ void rotate_chunk(double (&v)[16], double* tbuf, int lane, int gl, int gfirst) {
    if constexpr (G == 16) {
        stage16<1>(v, 1.0);
        stage16<4>(v, 0.25);
    } else {
        stage16<1>(v, 1.0);
        stage16<4>(v, 1.0);
#pragma unroll
        for (int i = 0; i < 16; ++i) tbuf[lane * kPad + i] = v[i];
        wave_sync();
        if constexpr (G == 256) {
#pragma unroll
            for (int m = 0; m < 16; ++m) v[m] = tbuf[(gfirst + m) * kPad + gl];
            stage16<1>(v, 1.0);
            stage16<4>(v, 1.0 / 16.0);
        } else {
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int a = 0; a < 4; ++a) v[a + 4 * b] = tbuf[(gfirst + b) * kPad + 4 * gl + a];
            stage16<4>(v, 1.0 / 8.0);
        }
        wave_sync();
    }
}

}  // namespace convrot
