// Microscaled 4-bit floats (MXFP4): what the quantizer, the products and the
// expert routing share.
//
// A row of K values (K % 32 == 0) is K/2 bytes of E2M1 codes (sign, two
// exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6; value 2j in the
// low half of byte j) and K/32 scale bytes.  Scale byte s stands for 2^(s-127);
// 255 stands for NaN, and with it every value of its 32.
#pragma once

#include "common.h"

namespace convrot {

constexpr int MX_BLOCK = 32;         // values that share a scale
constexpr int MX_MAX_N = 0x7fffff00; // columns of a product: a tile's past them stay below 2^31

typedef unsigned v4u_mx __attribute__((ext_vector_type(4)));
typedef unsigned v2u_mx __attribute__((ext_vector_type(2)));

// v of another lane: dpp_ctrl as in the ISA (quad_perm 0x00.., row_ror 0x120 + n, row_mirror 0x140)
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_XOR3 = 0x1B, DPP_ROR4 = 0x124, DPP_ROR8 = 0x128,
              DPP_MIRROR = 0x140;

// One base-4 digit of the rotation: y_a = (x_0 + x_1 + x_2 + x_3) / 2 - x_{3-a}
// is row a of [[1,1,1,-1],[1,1,-1,1],[1,-1,1,1],[-1,1,1,1]] / 2, which is
// orthogonal and its own inverse.  The sums are fp32.
__device__ __forceinline__ void digit4(float& a, float& b, float& c, float& d) {
    const float h = 0.5f * ((a + b) + (c + d));
    const float a1 = h - d, b1 = h - c, c1 = h - b, d1 = h - a;
    a = a1; b = b1; c = c1; d = d1;
}

// The rotation in groups of G (0: none, 16, 64, 256) of values held 16
// consecutive ones a lane, groups starting at a lane that is a multiple of
// G/16: the low two digits are in the lane, the third is the lane's place in
// its quad, the fourth the quad's place in its row of 16 lanes.  Every digit
// at most doubles a value, so no partial sum is more than 2 sqrt(G) <= 32 times
// the group's largest value: below 2^122 none overflows.
template <int G>
__device__ __forceinline__ void rotate_digits(float (&v)[16]) {
    if constexpr (G >= 16) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) digit4(v[i], v[i + 1], v[i + 2], v[i + 3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) digit4(v[i], v[i + 4], v[i + 8], v[i + 12]);
    }
    if constexpr (G >= 64) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float s = v[i] + dpp<DPP_XOR1>(v[i]);
            v[i] = 0.5f * (s + dpp<DPP_XOR2>(s)) - dpp<DPP_XOR3>(v[i]);
        }
    }
    if constexpr (G >= 256) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float s = v[i] + dpp<DPP_ROR8>(v[i]);
            v[i] = 0.5f * (s + dpp<DPP_ROR4>(s)) - dpp<DPP_XOR3>(dpp<DPP_MIRROR>(v[i]));   // mirror, xor 3: lane ^ 12
        }
    }
}

// Whether `p` holds in a lane of this lane's rotation group; `some`: of the wave.
template <int G>
__device__ __forceinline__ bool group_any(bool p, bool& some) {
    const unsigned long long b = __ballot(p);
    some = b != 0;
    if constexpr (G <= 16) return p;
    constexpr int L = G / 16;
    return (b >> (threadIdx.x & 63 & ~(L - 1)) & ((1ull << L) - 1)) != 0;
}

// The rotation of any values: finite wherever the exact result is.  A group with
// a value of 2^122 or more is rotated 2^-6 times as large, which is exact but for
// bits below 2^-143.
template <int G>
__device__ __forceinline__ void rotate16(float (&v)[16]) {
    if constexpr (G > 0) {
        float m = __builtin_fabsf(v[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) m = fmaxf(m, __builtin_fabsf(v[i]));
        bool some;
        const bool large = group_any<G>(m >= 0x1p122f, some);
        if (some) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= large ? 0x1p-6f : 1.0f;
        }
        rotate_digits<G>(v);
        if (some) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= large ? 0x1p6f : 1.0f;
        }
    }
}

// 16 consecutive values of element type DT at `p` (32-byte or 64-byte aligned to 16)
template <int DT>
__device__ __forceinline__ void load16(const void* p, float (&v)[16]) {
    const v4u_mx* q = reinterpret_cast<const v4u_mx*>(p);
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v4u_mx w = q[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * i + j] = __uint_as_float(w[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const v4u_mx w = q[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[8 * i + 2 * j] = DT == DT_BF16 ? bf16lo_to_f32(w[j]) : f16bits_to_f32(w[j]);
                v[8 * i + 2 * j + 1] = DT == DT_BF16 ? bf16hi_to_f32(w[j]) : f16bits_to_f32(w[j] >> 16);
            }
        }
    }
}

// The scale byte of a block whose largest magnitude is `amax`: 2^(floor(log2
// amax) - 2), the largest value's exponent less that of E2M1's largest (6 = 1.5
// 2^2), down to 2^-127; 255 where the block holds a NaN or an infinity.
__device__ __forceinline__ uint32_t mx_scale_byte(float amax) {
    const uint32_t e = __float_as_uint(amax) >> 23;         // amax >= 0: the biased exponent, 0 for subnormal values
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// Two values / 2^(scale byte - 127) -> byte BYTE of `old`: codes rounded to
// nearest, ties to even, magnitudes past 6 to 6.
template <int BYTE>
__device__ __forceinline__ uint32_t mx_pack2(uint32_t old, float a, float b, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, scale, BYTE);
}

// The 16 values of a lane, one half of a block that it shares with its
// neighbour (lane ^ 1) -> 8 code bytes and the block's scale byte.  Scales
// below 2^-63 take the values times 2^64 (exact) to a scale that is a normal
// number; a block with a NaN or an infinity gets codes 0.
__device__ __forceinline__ v2u_mx mx_encode16(const float (&v)[16], uint32_t& scale_byte) {
    float m = __builtin_fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) m = __builtin_elementwise_maximum(m, __builtin_fabsf(v[i]));   // a NaN stays
    m = __builtin_elementwise_maximum(m, dpp<DPP_XOR1>(m));
    scale_byte = mx_scale_byte(m);
    const bool small = scale_byte < 64u;
    const float up = small ? 0x1p64f : 1.0f;
    const float scale = __uint_as_float((scale_byte + (small ? 64u : 0u)) << 23);
    v2u_mx c = {0u, 0u};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w = 0;
        w = mx_pack2<0>(w, v[8 * h] * up, v[8 * h + 1] * up, scale);
        w = mx_pack2<1>(w, v[8 * h + 2] * up, v[8 * h + 3] * up, scale);
        w = mx_pack2<2>(w, v[8 * h + 4] * up, v[8 * h + 5] * up, scale);
        w = mx_pack2<3>(w, v[8 * h + 6] * up, v[8 * h + 7] * up, scale);
        c[h] = scale_byte == 255u ? 0u : w;
    }
    return c;
}

}  // namespace convrot
