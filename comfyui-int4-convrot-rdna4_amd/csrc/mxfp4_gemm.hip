// The product of MXFP4 rows with MXFP4 weights, for one weight matrix or one per expert.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 multiplies 4-bit floats and applies both
// operands' block scales itself: lane l supplies row l % 32, the 32 values of
// block l / 32 of the 64 (16 bytes) and that block's scale byte.

#include "mxfp4_gemm.h"

namespace convrot {

typedef int v8i_mx __attribute__((ext_vector_type(8)));
typedef float v16f_mx __attribute__((ext_vector_type(16)));

constexpr int MX_FP4 = 4;                  // operand format code of E2M1

__device__ __forceinline__ v8i_mx mx_operand(v4u_mx c) {
    return (v8i_mx){(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
}

// 64 x 64 outputs by four waves of 32 x 32, operands from memory to registers.
__global__ __launch_bounds__(256) void mxfp4_gemm_direct_kernel(MxProblem p, int tiles_n) {
    constexpr int BM = 64, BN = 64;
    if ((int)(blockIdx.x / tiles_n) >= mx_tile_count<BM>(p)) return;
    const MxTile t = mx_tile<BM>(p, blockIdx.x / tiles_n);
    const int n0 = (blockIdx.x % tiles_n) * BN;
    if (t.e == p.E && p.offsets != nullptr) return mx_zero(p, t.m0, t.m1, n0, min(n0 + BN, p.N));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = t.m0 + (wave >> 1) * 32 + (lane & 31), half = lane >> 5;
    const int n = n0 + (wave & 1) * 32 + (lane & 31);
    // rows and columns past the edge repeat the last one; they are not stored
    const size_t ar = (size_t)(p.order != nullptr ? mx_source_row(p, min(r, t.m1 - 1)) : min(r, t.m1 - 1));
    const size_t wr = (size_t)t.e * p.N + min(n, p.N - 1);
    const uint8_t* a = p.a + ar * (p.Kp / 2);
    const uint8_t* as = p.as + ar * p.Ks;
    const uint8_t* w = p.w + wr * (p.K / 2);
    const uint8_t* ws = p.ws + wr * (p.K / 32);
    v16f_mx acc = {0};
    for (int k = 0; k < p.K; k += 64) {
        const int b = k / 32 + half;                      // past K: the activation's padding (zero) against block b - 1
        const int bw = min(b, p.K / 32 - 1);
        const v4u_mx ca = *reinterpret_cast<const v4u_mx*>(a + (size_t)b * 16);
        const v4u_mx cw = *reinterpret_cast<const v4u_mx*>(w + (size_t)bw * 16);
        const int sw = b == bw ? ws[bw] : 127;
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(cw), mx_operand(ca), acc, MX_FP4, MX_FP4, 0, sw, 0,
                                                              (int)as[b]);
    }
    // lane: output row m = lane % 32, columns 8 (i / 4) + 4 half + i % 4
    if (r >= t.m1) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int c = n0 + (wave & 1) * 32 + 8 * g + 4 * half;
        if (c >= p.N) continue;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = acc[4 * g + j];
            if (p.bias != nullptr && c + j < p.N) v[j] += mx_read(p.bias, p.bias_dt, (size_t)t.e * p.N + c + j);
        }
        mx_store4(p.out, p.dt, (size_t)r * p.N + c, v, min(4, p.N - c), p.N % 4 == 0);
    }
}

bool mxfp4_gemm_staged(const MxProblem& p);
hipError_t mxfp4_gemm_staged_launch(const MxProblem& p, hipStream_t st);

hipError_t mxfp4_gemm_launch(const MxProblem& p, hipStream_t st) {
    if (p.R == 0 || p.N == 0) return hipSuccess;
    if (mxfp4_gemm_staged(p)) return mxfp4_gemm_staged_launch(p, st);
    const int tiles_n = (p.N + 63) / 64;
    const long long grid = mx_row_tiles(p.R, p.E, p.offsets != nullptr, 64) * tiles_n;
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL(mxfp4_gemm_direct_kernel, dim3((unsigned)grid), dim3(256), 0, st, p, tiles_n);
    return hipGetLastError();
}

}  // namespace convrot
