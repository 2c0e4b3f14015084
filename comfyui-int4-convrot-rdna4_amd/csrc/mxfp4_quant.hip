// Quantization of rows to microscaled 4-bit floats, with the block-Hadamard
// rotation on the way, and back.
//
// Per 32 values: s = 2^(floor(log2 max|y|) - 2), code = E2M1 nearest to y / s
// (ties to even, past 6 to 6), y = x or x rotated in groups of 16, 64 or 256.
// Bound by memory: a value is read once (2 or 4 bytes) and leaves 17/32 bytes.
// A lane holds 16 consecutive values, so a block is two neighbouring lanes, a
// rotation group 1, 4 or 16 of them, and every exchange is a DPP operand of the
// instruction that uses it: no LDS, no barrier.  Blocks and groups lie whole in
// a row, so the matrix is walked as one array and rows do not matter, except
// where the codes' rows are padded.
//
// Measured on MI355X, kernel trace: 16384 x 5120 bf16 42.8 us (5.0 TB/s of values
// in and codes out, the rate of a device copy; 28.7 with the values in the last
// cache, 34.9 rotated in groups of 256 on top); back to bf16 32 us (6.6 TB/s, the codes from cache); one row
// 1.5 us each way, a launch's latency.

#include "mxfp4_gemm.h"

#include <type_traits>

namespace convrot {

template <int DT, int G>
__global__ __launch_bounds__(256) void mxfp4_quant_kernel(const uint8_t* __restrict__ x, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, long long units, long long first) {
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const long long u = (first + blockIdx.x) * 256 + threadIdx.x;        // 16 values of the matrix
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    if (u < units) load16<DT>(x + (size_t)u * 16 * ES, v);
    rotate16<G>(v);
    uint32_t sb;
    const v2u_mx c = mx_encode16(v, sb);
    if (u < units) {
        *reinterpret_cast<v2u_mx*>(codes + (size_t)u * 8) = c;
        if ((threadIdx.x & 1) == 0) scales[u >> 1] = (uint8_t)sb;
    }
}

// 16 scale bytes of weight row n of expert e (piece i: 512 k number i / N % (Ks/16)) into the order of staged tiles:
// [E, N, nb] -> [E, Ks/16, N, 16].
struct MxTileScales { const uint8_t* src; uint8_t* dst; long long pieces; int N, nb; };

__device__ __forceinline__ void tile_scales(const MxTileScales& w, long long i, int Ks) {
    if (i >= w.pieces) return;
    const long long run = i / w.N;                         // e Ks/16 + 512 k number
    const int n = (int)(i - run * w.N), per = Ks / 16;
    const long long e = run / per;
    const int b0 = (int)(run - e * per) * 16;
    const uint8_t* s = w.src + (size_t)(e * w.N + n) * w.nb + b0;
    v4u_mx o = {0u, 0u, 0u, 0u};
    if (w.nb % 16 == 0) {
        const v4u_mx r = *reinterpret_cast<const v4u_mx*>(s);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[mx_scale_place(j) >> 2] |= (r[j >> 2] >> (8 * (j & 3)) & 255u) << (8 * (mx_scale_place(j) & 3));
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (b0 + j < w.nb) o[mx_scale_place(j) >> 2] |= (uint32_t)s[j] << (8 * (mx_scale_place(j) & 3));
    }
    reinterpret_cast<v4u_mx*>(w.dst)[i] = o;
}

// The activation of a product: rows of codes padded to Kp values (a multiple of 256) with codes 0, scales in rows of
// Ks bytes or (TILES) in the order of staged tiles (mxfp4_gemm.h), 16 bytes of 512 k a row either way.  A workgroup
// takes 512 k of 8 rows, so that its scales leave as one run of 128 bytes.  The grid's last workgroups lay out the
// weight's scales for staged tiles: a launch of its own for them took 3.5 us more.
template <int DT, int G, bool TILES>
__global__ __launch_bounds__(256) void mxfp4_quant_rows_kernel(const uint8_t* __restrict__ x, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, int M, int K, int Kp, int Ks,
                                                               unsigned blocks, MxTileScales w, unsigned first) {
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) uint8_t sc[8][16];
    const unsigned b = first + blockIdx.x;
    if constexpr (TILES) {
        if (b >= blocks) return tile_scales(w, (long long)(b - blocks) * 256 + threadIdx.x, Ks);
    }
    const int per = Ks / 16;
    const int ss = b % per, row0 = (int)(b / per) * 8;
    const int r = threadIdx.x >> 5, l = threadIdx.x & 31;
    const unsigned row = (unsigned)row0 + r;
    const int k = ss * 512 + l * 16;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    if (row < (unsigned)M && k < K) load16<DT>(x + ((size_t)row * K + k) * ES, v);
    rotate16<G>(v);
    uint32_t sb;
    const v2u_mx c = mx_encode16(v, sb);
    if (row < (unsigned)M && k < Kp) *reinterpret_cast<v2u_mx*>(codes + (size_t)row * (Kp / 2) + k / 2) = c;
    if ((l & 1) == 0) sc[r][TILES ? mx_scale_place(l >> 1) : l >> 1] = (uint8_t)sb;
    __syncthreads();
    const unsigned m = row0 + threadIdx.x;
    if (threadIdx.x < 8 && m < (unsigned)M)
        *reinterpret_cast<v4u_mx*>(scales + (TILES ? ((size_t)ss * M + m) * 16 : (size_t)m * Ks + ss * 16)) =
                *reinterpret_cast<const v4u_mx*>(sc[threadIdx.x]);
}

// Values of the codes, rotated back (the rotation is its own inverse), rounded once to the output type.
template <int DT, int G>
__global__ __launch_bounds__(256) void mxfp4_dequant_kernel(const uint8_t* __restrict__ codes,
                                                            const uint8_t* __restrict__ scales, uint8_t* __restrict__ out,
                                                            long long units, long long first) {
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const long long u = (first + blockIdx.x) * 256 + threadIdx.x;
    v2u_mx c = {0u, 0u};
    uint32_t sb = 127u;
    if (u < units) {
        c = *reinterpret_cast<const v2u_mx*>(codes + (size_t)u * 8);
        sb = scales[u >> 1];
    }
    // code -> value / 2: sign, exponent and mantissa bits moved to their places in a float whose
    // exponent 0 is a half unit (0 and 1 are 0 and .5: the mantissa bit counts 2^-2 there), times
    // 2^126, which makes subnormal numbers of the moved bits normal ones.
    float scale = sb == 255u ? __builtin_nanf("") : sb == 0u ? 0x1p-127f : __uint_as_float(sb << 23);
    // as rotate16; by the scale, since 2^126 times a code's value can be past fp32 where the rotated values are not
    bool some = false;
    const bool large = G > 0 && group_any<G>(sb >= 240u, some);
    if (some) scale *= large ? 0x1p-8f : 1.0f;
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t n = (c[i >> 3] >> (4 * (i & 7))) & 15u;
        const float m = __uint_as_float(((n & 8u) << 28) | ((n & 7u) << 22));
        v[i] = (m * 0x1p126f) * scale;
    }
    rotate_digits<G>(v);
    if (some) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] *= large ? 0x1p8f : 1.0f;
    }
    if (u >= units) return;
    uint8_t* o = out + (size_t)u * 16 * ES;
    if constexpr (DT == DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4*>(o)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v4u_mx w;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = v[8 * i + 2 * j], b = v[8 * i + 2 * j + 1];
                w[j] = DT == DT_BF16 ? pack_bf16x2(a, b) : pack_f16x2(a, b);
            }
            reinterpret_cast<v4u_mx*>(o)[i] = w;
        }
    }
}

template <int DT, int G>
static hipError_t quant_go(const void* x, void* codes, void* scales, int M, int K, hipStream_t st) {
    const long long units = (long long)M * (K / 16);
    return launch_parts((units + 255) / 256, 256, [&](long long first, dim3 grid) {
        hipLaunchKernelGGL((mxfp4_quant_kernel<DT, G>), grid, dim3(256), 0, st, reinterpret_cast<const uint8_t*>(x),
                           reinterpret_cast<uint8_t*>(codes), reinterpret_cast<uint8_t*>(scales), units, first);
    });
}

// f(type code, group) as compile-time constants
template <typename F>
static auto by_type_and_group(int dt, int G, F f) {
    using std::integral_constant;
    auto group = [&](auto d) {
        switch (G) {
            case 0: return f(d, integral_constant<int, 0>{});
            case 16: return f(d, integral_constant<int, 16>{});
            case 64: return f(d, integral_constant<int, 64>{});
            default: return f(d, integral_constant<int, 256>{});
        }
    };
    switch (dt) {
        case DT_F32: return group(integral_constant<int, DT_F32>{});
        case DT_BF16: return group(integral_constant<int, DT_BF16>{});
        default: return group(integral_constant<int, DT_F16>{});
    }
}

// x [M, K] -> codes [M, K/2], scales [M, K/32]
hipError_t mxfp4_quant_launch(const void* x, int dt, void* codes, void* scales, int M, int K, int G, hipStream_t st) {
    return by_type_and_group(dt, G, [&](auto d, auto g) {
        return quant_go<decltype(d)::value, decltype(g)::value>(x, codes, scales, M, K, st);
    });
}

// x [rows, K] as the operand p.a, p.as of a product; with `tiles` in the order of staged tiles, and p.ws as p.wp
hipError_t mxfp4_operands_launch(const void* x, int G, const MxProblem& p, bool tiles, hipStream_t st) {
    const long long blocks = (p.as_rows + 7LL) / 8 * (p.Ks / 16);
    MxTileScales w{p.ws, const_cast<uint8_t*>(p.wp), (long long)p.E * p.N * (p.Ks / 16), p.N, p.K / 32};
    const long long all = tiles ? blocks + (w.pieces + 255) / 256 : blocks;
    if (all > 0xffffffffLL) return hipErrorInvalidValue;
    return by_type_and_group(p.dt, G, [&](auto d, auto g) {
        constexpr int DT = decltype(d)::value, GG = decltype(g)::value;
        const auto xb = reinterpret_cast<const uint8_t*>(x);
        const auto cb = const_cast<uint8_t*>(p.a), sb = const_cast<uint8_t*>(p.as);
        return launch_parts(all, 256, [&](long long first, dim3 grid) {
            if (tiles)
                hipLaunchKernelGGL((mxfp4_quant_rows_kernel<DT, GG, true>), grid, dim3(256), 0, st, xb, cb, sb, p.as_rows, p.K,
                                   p.Kp, p.Ks, (unsigned)blocks, w, (unsigned)first);
            else
                hipLaunchKernelGGL((mxfp4_quant_rows_kernel<DT, GG, false>), grid, dim3(256), 0, st, xb, cb, sb, p.as_rows, p.K,
                                   p.Kp, p.Ks, (unsigned)blocks, w, (unsigned)first);
        });
    });
}

// codes [M, K/2], scales [M, K/32] -> out [M, K]
hipError_t mxfp4_dequant_launch(const void* codes, const void* scales, void* out, int dt, int M, int K, int G,
                                hipStream_t st) {
    const long long units = (long long)M * (K / 16);
    return by_type_and_group(dt, G, [&](auto d, auto g) {
        return launch_parts((units + 255) / 256, 256, [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((mxfp4_dequant_kernel<decltype(d)::value, decltype(g)::value>), grid, dim3(256), 0, st,
                               reinterpret_cast<const uint8_t*>(codes), reinterpret_cast<const uint8_t*>(scales),
                               reinterpret_cast<uint8_t*>(out), units, first);
        });
    });
}

}  // namespace convrot
