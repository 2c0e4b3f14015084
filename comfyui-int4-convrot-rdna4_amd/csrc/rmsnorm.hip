// Root-mean-square norm of rows, with the residual's addition in front, its gradient, and its rotated 8-bit form.
//
//   h = T(x + residual)          (T: the rows' type; without a residual h = x)
//   y = T(h rstd w),  rstd = 1 / sqrt(mean(h^2) + eps)
// The norm is of the sum as it is kept, so norm and residual stream agree, and the gradient needs h alone.
//
// Squares are added in fp64 (full rate here): they cannot overflow, and no order of the sum shows in the result.  y is
// made in fp32 as ((h 2^n) a) w with rstd = a 2^n: no step leaves the range where the result does not.

#include "b6t_layout.h"
#include "lanes.h"
#include "rmsnorm.h"
#include "rotate64.h"

namespace convrot {

// 16 bytes of a row as floats.  Rows of a width that is no whole number of pieces lie at any multiple of their
// element's size: loads and stores of 16 bytes may, and the last piece goes one element at a time.
typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(2)));

template <int DT>
struct NormPiece {
    static constexpr int N = DT == DT_F32 ? 4 : 8, ES = DT == DT_F32 ? 4 : 2;
    static __device__ __forceinline__ float one(const void* row, int e) {
        if constexpr (DT == DT_F32) return reinterpret_cast<const float*>(row)[e];
        const uint32_t h = reinterpret_cast<const uint16_t*>(row)[e];
        return DT == DT_BF16 ? __uint_as_float(h << 16) : f16bits_to_f32(h);
    }
    static __device__ __forceinline__ void unpack(v4u_mx w, float (&v)[N]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == DT_F32) v[j] = __uint_as_float(w[j]);
            else {
                v[2 * j] = DT == DT_BF16 ? bf16lo_to_f32(w[j]) : f16bits_to_f32(w[j]);
                v[2 * j + 1] = DT == DT_BF16 ? bf16hi_to_f32(w[j]) : f16bits_to_f32(w[j] >> 16);
            }
        }
    }
    static __device__ __forceinline__ v4u_mx pack(const float (&v)[N]) {
        v4u_mx w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == DT_F32) w[j] = __float_as_uint(v[j]);
            else w[j] = DT == DT_BF16 ? pack_bf16x2(v[2 * j], v[2 * j + 1]) : pack_f16x2(v[2 * j], v[2 * j + 1]);
        }
        return w;
    }
    // piece i of a row of D, zeros past its end
    static __device__ __forceinline__ void load(const void* row, int i, int D, float (&v)[N]) {
        if ((i + 1) * N <= D) unpack(*reinterpret_cast<const v4u_any*>(reinterpret_cast<const uint8_t*>(row) + (size_t)i * 16), v);
        else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = i * N + j < D ? one(row, i * N + j) : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(void* row, int i, int D, const float (&v)[N]) {
        if ((i + 1) * N <= D) *reinterpret_cast<v4u_any*>(reinterpret_cast<uint8_t*>(row) + (size_t)i * 16) = pack(v);
        else {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (i * N + j >= D) break;
                if constexpr (DT == DT_F32) reinterpret_cast<float*>(row)[i * N + j] = v[j];
                else reinterpret_cast<uint16_t*>(row)[i * N + j] =
                             (uint16_t)(DT == DT_BF16 ? pack_bf16x2(v[j], 0.0f) : pack_f16x2(v[j], 0.0f));
            }
        }
    }
};

// N values of the weight from element e on; 1 without one, 0 past the end
template <int N>
__device__ __forceinline__ void load_weight(const void* w, int dt, int e, int D, float (&v)[N]) {
    if (w == nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 1.0f;
        return;
    }
    static_assert(N % 4 == 0, "whole pieces");
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        float f[4];
        if (e + j + 4 <= D) {
            if (dt == DT_F32) {
                const float4 q = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + e + j);
                f[0] = q.x; f[1] = q.y; f[2] = q.z; f[3] = q.w;
            } else {
                const uint2 q = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(w) + e + j);
                f[0] = dt == DT_BF16 ? bf16lo_to_f32(q.x) : f16bits_to_f32(q.x);
                f[1] = dt == DT_BF16 ? bf16hi_to_f32(q.x) : f16bits_to_f32(q.x >> 16);
                f[2] = dt == DT_BF16 ? bf16lo_to_f32(q.y) : f16bits_to_f32(q.y);
                f[3] = dt == DT_BF16 ? bf16hi_to_f32(q.y) : f16bits_to_f32(q.y >> 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[i] = 0.0f;
                if (e + j + i < D) f[i] = dt == DT_F32 ? NormPiece<DT_F32>::one(w, e + j + i) : dt == DT_BF16 ? NormPiece<DT_BF16>::one(w, e + j + i)
                                                                                                       : NormPiece<DT_F16>::one(w, e + j + i);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j + i] = f[i];
    }
}

// The sum over a workgroup's waves of a value that each wave's lanes share, in wave order; `slot`: 16 doubles in LDS that
// no wave reads any more.
__device__ __forceinline__ double sum_waves(double v, double* slot) {
    const int W = blockDim.x >> 6;
    if (W == 1) return v;
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < W; ++i) s += slot[i];
    return s;
}

// rstd = a 2^n, a in [1/2, 1); infinity and NaN as they are, n = 0
struct Rstd { float a; int n; };
__device__ __forceinline__ Rstd split_rstd(double rstd) {
    if (!(rstd < __builtin_inf())) return {(float)rstd, 0};
    return {(float)__builtin_amdgcn_frexp_mant(rstd), __builtin_amdgcn_frexp_exp(rstd)};
}

template <int DT, int P>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a, unsigned first) {
    using V = NormPiece<DT>;
    constexpr int N = V::N;
    __shared__ double slot[16];
    const size_t at = (size_t)(first + blockIdx.x) * a.D * V::ES;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x) + at;
    float h[P][N];
    double ss = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = p * blockDim.x + threadIdx.x;
        V::load(x, i, a.D, h[p]);
        if (a.residual != nullptr) {
            float r[N];
            V::load(reinterpret_cast<const uint8_t*>(a.residual) + at, i, a.D, r);
#pragma unroll
            for (int j = 0; j < N; ++j) h[p][j] = round_to_dt<DT>(h[p][j] + r[j]);
            V::store(reinterpret_cast<uint8_t*>(a.h) + at, i, a.D, h[p]);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) ss = __builtin_fma((double)h[p][j], (double)h[p][j], ss);
    }
    ss = sum_waves(sum_lanes<64>(ss), slot);
    const Rstd s = split_rstd(1.0 / sqrt(ss / a.D + a.eps));
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = p * blockDim.x + threadIdx.x;
        float w[N];
        load_weight<N>(a.weight, a.weight_dt, i * N, a.D, w);
#pragma unroll
        for (int j = 0; j < N; ++j) h[p][j] = __builtin_amdgcn_ldexpf(h[p][j], s.n) * s.a * w[j];
        V::store(reinterpret_cast<uint8_t*>(a.y) + at, i, a.D, h[p]);
    }
}

// The gradient: with n = h rstd and g = w d_y,  d_x = rstd (g - n mean(g n)) + d_h,  d_weight = sum over rows of d_y n.
// A workgroup walks rows and keeps its part of d_weight in registers; the parts are added by a second launch, in order.
template <int DT, int P>
__global__ __launch_bounds__(1024) void norm_grad_kernel(NormGradArgs a) {
    using V = NormPiece<DT>;
    constexpr int N = V::N;
    __shared__ double slots[2][2][16];
    float w[P][N], dw[P][N] = {};
#pragma unroll
    for (int p = 0; p < P; ++p) load_weight<N>(a.weight, a.weight_dt, (p * blockDim.x + threadIdx.x) * N, a.D, w[p]);
    int turn = 0;
    for (long long row = blockIdx.x; row < a.M; row += gridDim.x, turn ^= 1) {
        const size_t at = (size_t)row * a.D * V::ES;
        float h[P][N], g[P][N];
        double ss = 0.0, gh = 0.0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = p * blockDim.x + threadIdx.x;
            V::load(reinterpret_cast<const uint8_t*>(a.h) + at, i, a.D, h[p]);
            V::load(reinterpret_cast<const uint8_t*>(a.d_y) + at, i, a.D, g[p]);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                ss = __builtin_fma((double)h[p][j], (double)h[p][j], ss);
                gh = __builtin_fma((double)(g[p][j] * w[p][j]), (double)h[p][j], gh);
            }
        }
        ss = sum_lanes<64>(ss);
        gh = sum_lanes<64>(gh);
        const int W = blockDim.x >> 6;
        if (W > 1) {
            double (&s)[2][16] = slots[turn];
            if ((threadIdx.x & 63) == 0) {
                s[0][threadIdx.x >> 6] = ss;
                s[1][threadIdx.x >> 6] = gh;
            }
            __syncthreads();
            ss = gh = 0.0;
            for (int i = 0; i < W; ++i) {
                ss += s[0][i];
                gh += s[1][i];
            }
        }
        const double rstd = 1.0 / sqrt(ss / a.D + a.eps);
        const Rstd s = split_rstd(rstd);
        const float mean = (float)(gh * rstd / a.D);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = p * blockDim.x + threadIdx.x;
            float dx[N], dh[N] = {};
            if (a.d_h != nullptr) V::load(reinterpret_cast<const uint8_t*>(a.d_h) + at, i, a.D, dh);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float n = __builtin_amdgcn_ldexpf(h[p][j], s.n) * s.a;
                dx[j] = __builtin_amdgcn_ldexpf((g[p][j] * w[p][j] - n * mean) * s.a, s.n) + dh[j];
                dw[p][j] = __builtin_fmaf(g[p][j], n, dw[p][j]);
            }
            if (a.d_x != nullptr) V::store(reinterpret_cast<uint8_t*>(a.d_x) + at, i, a.D, dx);
        }
    }
    if (a.partial == nullptr) return;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int e = (p * blockDim.x + threadIdx.x) * N;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (e + j < a.D) a.partial[(size_t)blockIdx.x * a.D + e + j] = dw[p][j];
    }
}

// d_weight[e] = the sum of `parts` rows of partial sums, a lane a column, sixteen waves a sixteenth of the rows each
__global__ __launch_bounds__(1024) void norm_weight_grad_kernel(const float* __restrict__ partial, void* __restrict__ d_weight,
                                                                int dt, int D, int parts) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
    const int b0 = (int)((long long)parts * wave / 16), b1 = (int)((long long)parts * (wave + 1) / 16);
    float s = 0.0f;
    if (e < D) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) s += partial[(size_t)b * D + e];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || e >= D) return;
    for (int v = 1; v < 16; ++v) s += part[v][lane];
    if (dt == DT_F32) reinterpret_cast<float*>(d_weight)[e] = s;
    else reinterpret_cast<uint16_t*>(d_weight)[e] = (uint16_t)(dt == DT_BF16 ? pack_bf16x2(s, 0.0f) : pack_f16x2(s, 0.0f));
}

// ---------------------------------------------------------------------------
// The 8-bit form:
//   z = H_G(h w) rstd,  s = fl32(max(max |z|, 1e-10) / 127),  q = rint_even(z / s)
// A lane holds 16 consecutive values.  Everything up to the code is fp64 (full rate here), so a code is the formula's
// nearest one and not a matter of the order of sums; rstd commutes with the rotation, so it is not waited for.  A row
// with a value that is not finite (or zeros over eps = 0) gets scale NaN and codes 0.
// ---------------------------------------------------------------------------
template <int DT, int G, int P, bool TILED>
__global__ __launch_bounds__(1024) void norm_int8_kernel(NormArgs a, unsigned first) {
    using V = NormPiece<DT>;
    constexpr int N = V::N, LPG = G / kChunk, PIECES = kChunk / N;
    extern __shared__ __attribute__((aligned(16))) double norm_lds[];
    const int W = blockDim.x >> 6, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    double* tbuf = norm_lds + wv * (64 * kPad);
    double* slot = norm_lds + W * (64 * kPad);                // [2][16]
    uint8_t* cb = reinterpret_cast<uint8_t*>(tbuf);
    const int nchunks = a.D / kChunk, gl = lane % LPG, gfirst = lane - gl;
    const long long row = (long long)first + blockIdx.x;
    int8_t* q = reinterpret_cast<int8_t*>(a.y);
    const auto code_at = [&](int c) {
        if constexpr (TILED)
            return reinterpret_cast<uint4*>(q + ((size_t)(row >> 8) * (a.D >> 6) + (c >> 2)) * I8T_CHUNK + i8t_off((int)(row & 255), c & 3));
        else return reinterpret_cast<uint4*>(q + (size_t)row * a.D + (size_t)c * kChunk);
    };
    if (TILED && row >= a.M) {                                // padding rows hold zeros
        for (int c = threadIdx.x; c < nchunks; c += blockDim.x) *code_at(c) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const size_t at = (size_t)row * a.D * V::ES;
    double z[P][kChunk], ss = 0.0, most = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = (p * W + wv) * 64 + lane;
        const bool ok = c < nchunks;
        float h[PIECES][N], w[kChunk] = {};
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) h[i][j] = 0.0f;
            if (ok) {
                V::load(reinterpret_cast<const uint8_t*>(a.x) + at, c * PIECES + i, a.D, h[i]);
                if (a.residual != nullptr) {
                    float r[N];
                    V::load(reinterpret_cast<const uint8_t*>(a.residual) + at, c * PIECES + i, a.D, r);
#pragma unroll
                    for (int j = 0; j < N; ++j) h[i][j] = round_to_dt<DT>(h[i][j] + r[j]);
                    V::store(reinterpret_cast<uint8_t*>(a.h) + at, c * PIECES + i, a.D, h[i]);
                }
            }
        }
        if (ok) load_weight<kChunk>(a.weight, a.weight_dt, c * kChunk, a.D, w);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            const double v = (double)h[i / N][i % N];
            z[p][i] = v * (double)w[i];
            ss = __builtin_fma(v, v, ss);
            ss = __builtin_fma(z[p][i], 0.0, ss);             // a NaN where the product is not finite
        }
        rotate_chunk<G>(z[p], tbuf, lane, gl, gfirst);
#pragma unroll
        for (int i = 0; i < kChunk; ++i) most = fmax(most, fabs(z[p][i]));
    }
    ss = sum_lanes<64>(ss);
    most = all_lanes<64>(most, [](double u, double v) { return fmax(u, v); });
    if (W > 1) {
        if (lane == 0) {
            slot[wv] = ss;
            slot[16 + wv] = most;
        }
        __syncthreads();
        ss = 0.0;
        for (int i = 0; i < W; ++i) {
            ss += slot[i];
            most = fmax(most, slot[16 + i]);
        }
    }
    const double rstd = 1.0 / sqrt(ss / a.D + a.eps);
    const bool finite = ss < __builtin_inf() && rstd < __builtin_inf();
    const float s = finite ? (float)(fmax(most * rstd, 1e-10) / 127.0) : __builtin_nanf("");
    const double steps = rstd / (double)s;
    if (threadIdx.x == 0) a.scales[row] = s;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = (p * W + wv) * 64 + lane;
        wave_sync();
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            // low byte of the sum with 1.5 2^52: rint_even; |z steps| <= 127 (1 + 2^-23)
            const uint32_t code = (uint32_t)__double_as_longlong(__builtin_fma(z[p][i], steps, 0x1.8p52));
            const int e = final_elem<G>(gl, i);
            cb[(gfirst + e / kChunk) * kChunk + e % kChunk] = finite ? (uint8_t)code : (uint8_t)0;
        }
        wave_sync();
        if (c < nchunks) *code_at(c) = reinterpret_cast<const uint4*>(cb)[lane];
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Waves and pieces a lane of a row of `pieces`
struct NormShape { int W, P; };
static NormShape norm_shape(long long rows, int pieces) {
    int W = (pieces + 127) / 128;
    if (rows * W < 2048) W = (pieces + 63) / 64;
    if (W > 16) W = 16;
    const int P = (pieces + 64 * W - 1) / (64 * W);
    return {W, P <= 2 ? P : P <= 4 ? 4 : 8};
}

template <typename F>
static hipError_t by_type(int dt, F f) {
    using std::integral_constant;
    if (dt == DT_F32) return f(integral_constant<int, DT_F32>{});
    if (dt == DT_BF16) return f(integral_constant<int, DT_BF16>{});
    return f(integral_constant<int, DT_F16>{});
}

template <int DT, typename F>
static hipError_t by_pieces(int P, F f) {
    using std::integral_constant;
    if (P == 1) return f(integral_constant<int, 1>{});
    if (P == 2) return f(integral_constant<int, 2>{});
    if constexpr (DT == DT_F32) {
        if (P == 8) return f(integral_constant<int, 8>{});
    }
    return f(integral_constant<int, 4>{});
}

hipError_t norm_launch(const NormArgs& a, int dt, hipStream_t st) {
    return by_type(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        const NormShape s = norm_shape(a.M, (a.D + NormPiece<DT>::N - 1) / NormPiece<DT>::N);
        return by_pieces<DT>(s.P, [&](auto p) {
            return launch_parts(a.M, 64 * s.W, [&](long long first, dim3 grid) {
                hipLaunchKernelGGL((norm_kernel<DT, decltype(p)::value>), grid, dim3(64 * s.W), 0, st, a, (unsigned)first);
            });
        });
    });
}

constexpr int NORM_GRAD_GROUPS = 512;      // workgroups, and so partial sums of d_weight
static int norm_grad_groups(int M) { return M < NORM_GRAD_GROUPS ? M : NORM_GRAD_GROUPS; }

size_t norm_grad_bytes(int M, int D) { return (size_t)norm_grad_groups(M) * D * sizeof(float); }

hipError_t norm_grad_launch(const NormGradArgs& a, int dt, hipStream_t st) {
    const int groups = norm_grad_groups(a.M);
    const hipError_t e = by_type(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        const NormShape s = norm_shape(groups, (a.D + NormPiece<DT>::N - 1) / NormPiece<DT>::N);
        return by_pieces<DT>(s.P, [&](auto p) {
            hipLaunchKernelGGL((norm_grad_kernel<DT, decltype(p)::value>), dim3(groups), dim3(64 * s.W), 0, st, a);
            return hipGetLastError();
        });
    });
    if (e != hipSuccess || a.partial == nullptr) return e;
    hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((a.D + 63) / 64), dim3(1024), 0, st, a.partial, a.d_weight, a.weight_dt, a.D,
                       groups);
    return hipGetLastError();
}

template <int DT, int G, int P, bool TILED>
static hipError_t norm_int8_go(const NormArgs& a, int W, hipStream_t st) {
    static std::atomic<bool> attr[kMaxDev];
    constexpr int MOST = (16 * 64 * kPad + 32) * (int)sizeof(double);
    int dev = 0;
    hipError_t e = current_device(&dev);
    if (e != hipSuccess) return e;
    e = lds_limit_once(attr, dev, reinterpret_cast<const void*>(&norm_int8_kernel<DT, G, P, TILED>), MOST);
    if (e != hipSuccess) return e;
    const long long rows = TILED ? (a.M + 255LL) / 256 * 256 : a.M;
    return launch_parts(rows, 64 * W, [&](long long first, dim3 grid) {
        hipLaunchKernelGGL((norm_int8_kernel<DT, G, P, TILED>), grid, dim3(64 * W), (W * 64 * kPad + 32) * sizeof(double), st, a,
                           (unsigned)first);
    });
}

hipError_t norm_int8_launch(const NormArgs& a, int dt, int G, bool tiled, hipStream_t st) {
    const int waves = (a.D / kChunk + 63) / 64, W = waves <= 16 ? waves : (waves + 1) / 2;
    return by_type(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        const auto go = [&](auto g) {
            constexpr int GG = decltype(g)::value;
            if (waves <= 16)
                return tiled ? norm_int8_go<DT, GG, 1, true>(a, W, st) : norm_int8_go<DT, GG, 1, false>(a, W, st);
            return tiled ? norm_int8_go<DT, GG, 2, true>(a, W, st) : norm_int8_go<DT, GG, 2, false>(a, W, st);
        };
        using std::integral_constant;
        return G == 16 ? go(integral_constant<int, 16>{}) : G == 64 ? go(integral_constant<int, 64>{}) : go(integral_constant<int, 256>{});
    });
}

}  // namespace convrot
