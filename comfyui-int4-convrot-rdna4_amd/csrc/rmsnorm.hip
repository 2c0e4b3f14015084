// Root-mean-square norm of rows, with the residual's addition in front, its gradient, and its rotated 8-bit form.
//
//   h = T(x + residual)          (T: the rows' type; without a residual h = x)
//   y = T(h rstd w),  rstd = 1 / sqrt(mean(h^2) + eps)
// The norm is of the sum as it is kept, so norm and residual stream agree, and the gradient needs h alone.
//
// Squares are added in fp64 (full rate here): they cannot overflow, and no order of the sum shows in the result.  y is
// made in fp32 as ((h 2^n) a) w with rstd = a 2^n: no step overflows where the result does not, and a product with rstd
// that falls below 2^-126 is off by 2^-149 at most before the weight's.

#include "b6t_layout.h"
#include "lanes.h"
#include "rmsnorm.h"
#include "rotate64.h"

namespace convrot {

// Measured on MI355X, graph replays, bf16, us.
// Pieces a lane of a row's norm: 16384 x 5120 with 1, 2 and 4 117, 116 and 119, without residual 92, 62 and 60; 4096 x 13824
// 81, 81 and 82.
constexpr int NORM_PIECES = 2;
// Rows of a team that a single workgroup of several teams takes (us so, and in two launches): two rows 8 x 1024 5.2 and 5.8,
// 16 x 256 3.8 and 4.9, 64 x 64 4.0 and 5.1; three 24 x 256 4.6 and 4.9, 96 x 64 4.7 and 5.1, 12 x 1024 6.6 and 5.8; four 128 x 64
// 5.4 and 5.1, 16 x 1024 7.7 and 5.9.
constexpr int NORM_GRAD_ALONE = 3;
// Waves of a gradient that take a piece a lane each, others two (us, one piece and two).  Below: 64 x 4096 6.4 and 8.1, 256 x 1024
// 6.1 and 6.8, 256 x 2048 7.2 and 7.9, 128 x 4096 7.7 and 8.9.  Above: 2048 x 1024 10.9 and 10.0, 2048 x 2048 17.4 and 16.0,
// 2048 x 4096 27.9 and 24.7, 8192 x 2048 34.5 and 32.6.  Within 5% of the other at the border: 256 x 4096 10.0 and 10.3, 512 x 4096 12.9
// and 13.5, 1024 x 4096 18.5 and 18.0; rows of 5120, in workgroups of five waves and not ten, are 2% to 4% slower so
// above it.
constexpr int NORM_GRAD_FEW = 2048;
// Waves of the 8-bit form that take a chunk a lane each, others two: 64 x 4096 3.8 and 4.6, 512 x 4096 6.2 and 7.2, 1024 x 8192
// without a residual 10.7 and 10.6, 8192 x 5120 45 and 39, 4096 x 16384 89 and 63.  With a residual rows of up to four waves
// always do: 4096 x 4096 26.8 and 29.6, 8192 x 4096 47 and 49; 8192 x 5120 61.7 and 59.5, 3000 x 13824 87 and 65.
constexpr int NORM8_FEW = 4096;

// 16 bytes of a row as floats.  Rows of a width that is no whole number of pieces lie at any multiple of their
// element's size, which loads and stores of 16 bytes may; their last piece ends with the row and shares elements with the
// one before, which both hold and store alike, and which the sums take from one of them (an element at a time would
// wait for memory once more in every place).  TINY: rows narrower than a piece, one element at a time, in kernels of
// their own: beside the others' their branches cost a third of the time.
typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned v2u_any __attribute__((ext_vector_type(2), aligned(2)));

template <int DT, bool TINY = false>
struct NormPiece {
    static constexpr int N = DT == DT_F32 ? 4 : 8, ES = DT == DT_F32 ? 4 : 2;
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
    // the first element of piece i of a row of D; how many of the piece's values belong to the piece before
    static __device__ __forceinline__ int start(int i, int D) { return TINY ? 0 : min(i * N, D - N); }
    static __device__ __forceinline__ int shared(int i, int D) { return TINY ? 0 : i * N - start(i, D); }
    static __device__ __forceinline__ bool there(int i, int D) { return i * N < D; }
    // piece i as it lies there, zeros past the row.  The loads are marked as a stream's: each tensor is read once.
    static __device__ __forceinline__ v4u_mx raw(const void* row, int i, int D) {
        v4u_mx w = {0u, 0u, 0u, 0u};
        if constexpr (TINY) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (j >= D || i != 0) break;
                if constexpr (DT == DT_F32) w[j] = reinterpret_cast<const uint32_t*>(row)[j];
                else w[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[j] << (j % 2 * 16);
            }
            return w;
        } else {
            const v4u_mx v = __builtin_nontemporal_load(
                    reinterpret_cast<const v4u_any*>(reinterpret_cast<const uint8_t*>(row) + start(i, D) * ES));
            return there(i, D) ? v : w;
        }
    }
    static __device__ __forceinline__ void store_raw(void* row, int i, int D, v4u_mx w) {
        if (!there(i, D)) return;
        if constexpr (TINY) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (j >= D) break;
                if constexpr (DT == DT_F32) reinterpret_cast<uint32_t*>(row)[j] = w[j];
                else reinterpret_cast<uint16_t*>(row)[j] = (uint16_t)(w[j / 2] >> (j % 2 * 16));
            }
        } else *reinterpret_cast<v4u_any*>(reinterpret_cast<uint8_t*>(row) + start(i, D) * ES) = w;
    }
};

__device__ __forceinline__ float weight_at(const void* w, int dt, int e) {
    if (dt == DT_F32) return reinterpret_cast<const float*>(w)[e];
    const uint32_t h = reinterpret_cast<const uint16_t*>(w)[e];
    return dt == DT_BF16 ? bf16lo_to_f32(h) : f16bits_to_f32(h);
}
__device__ __forceinline__ void store_weight(void* w, int dt, int e, float v) {
    if (dt == DT_F32) reinterpret_cast<float*>(w)[e] = v;
    else reinterpret_cast<uint16_t*>(w)[e] = (uint16_t)(dt == DT_BF16 ? pack_bf16x2(v, 0.0f) : pack_f16x2(v, 0.0f));
}

// N values of the weight from element e on (ones without a weight); TINY: of a weight of D < N.  The type is asked for once: a
// branch for every pair of values costs the 8-bit form of 8192 x 5120 10 us of 70.
template <int N, bool TINY = false>
__device__ __forceinline__ void load_weight(const void* w, int dt, int e, int D, float (&v)[N]) {
    static_assert(N % 4 == 0, "whole pieces");
    if (w == nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 1.0f;
    } else if constexpr (TINY) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < D ? weight_at(w, dt, j) : 0.0f;
    } else if (dt == DT_F32) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const v4u_mx q = *reinterpret_cast<const v4u_any*>(reinterpret_cast<const float*>(w) + e + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[j + i] = __uint_as_float(q[i]);
        }
    } else {
        v2u_mx q[N / 4];
#pragma unroll
        for (int j = 0; j < N / 4; ++j) q[j] = *reinterpret_cast<const v2u_any*>(reinterpret_cast<const uint16_t*>(w) + e + 4 * j);
        if (dt == DT_BF16) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                v[j] = bf16lo_to_f32(q[j / 4][j / 2 % 2]);
                v[j + 1] = bf16hi_to_f32(q[j / 4][j / 2 % 2]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = f16bits_to_f32(q[j / 4][j / 2 % 2] >> (j % 2 * 16));
        }
    }
}

// 1 / sqrt(v): the instruction's approximation and two Newton steps, a quarter of the library's square root and quotient
__device__ __forceinline__ double rsqrt64(double v) {
    const double y = __builtin_amdgcn_rsq(v);
    if (!(v > 0.0 && v < __builtin_inf())) return y;
    const double e = __builtin_fma(-v * y, y, 1.0), z = __builtin_fma(0.5 * y, e, y);
    return __builtin_fma(0.5 * z, __builtin_fma(-v * z, z, 1.0), z);
}

// rstd = a 2^n, a in [1/2, 1); infinity and NaN as they are, n = 0
struct Rstd { float a; int n; };
__device__ __forceinline__ Rstd split_rstd(double rstd) {
    if (!(rstd < __builtin_inf())) return {(float)rstd, 0};
    return {(float)__builtin_amdgcn_frexp_mant(rstd), __builtin_amdgcn_frexp_exp(rstd)};
}

// A row is a team's: L lanes of a wave (P pieces each), or where L is 64 `waves` waves.  A workgroup has one or more
// whole teams.
template <int L>
struct Team {
    int lanes, number, lane;
    __device__ __forceinline__ explicit Team(int waves)
        : lanes(L < 64 ? L : 64 * waves), number(threadIdx.x / lanes), lane(threadIdx.x - number * lanes) {}
};

// v + the other waves' v of a team, in wave order, for lanes that share v; `slot`: a double of LDS for each wave of the
// workgroup, which no wave reads any more.  All waves of the workgroup come here.
__device__ __forceinline__ double sum_waves(double v, double* slot, int waves) {
    if (waves == 1) return v;
    const int wave = threadIdx.x >> 6, first = wave / waves * waves;
    if ((threadIdx.x & 63) == 0) slot[wave] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < waves; ++i) s += slot[first + i];
    return s;
}

// Bound by memory: 16384 x 5120 bf16 with a residual 115 us, 5.8 TB/s of the four tensors, without 61 us, 5.5 TB/s.  The weight
// is read after the sums: before them its registers cost waves (8192 x 4096 51 us, so 48).  Stores that the caches do not keep
// make this kernel shorter (512 x 4096 5.7 and 5.3, 16384 x 5120 115 and 109) and whoever reads y and h next longer by more:
// with a copy of both 2048 x 4096 24.9 and 28.4, 4096 x 5120 58 and 64, 8192 x 4096 90 and 97.
template <int DT, int P, int L, bool RES, bool TINY>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a, int waves, unsigned first) {
    using V = NormPiece<DT, TINY>;
    constexpr int N = V::N;
    __shared__ double slot[16];
    const Team<L> team(waves);
    const long long row = (long long)(first + blockIdx.x) * (blockDim.x / team.lanes) + team.number;
    if (row >= a.M) return;                                  // teams of several waves are alone in their workgroup
    const size_t at = (size_t)row * a.D * V::ES;
    v4u_mx x[P], r[P];
    float h[P][N];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = p * team.lanes + team.lane;
        x[p] = V::raw(reinterpret_cast<const uint8_t*>(a.x) + at, i, a.D);
        if constexpr (RES) r[p] = V::raw(reinterpret_cast<const uint8_t*>(a.residual) + at, i, a.D);
    }
    const bool ragged = a.D % N != 0;                        // the last piece shares elements
    double ss = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = p * team.lanes + team.lane;
        V::unpack(x[p], h[p]);
        if constexpr (RES) {
            float v[N];
            V::unpack(r[p], v);
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += h[p][j];
            const v4u_mx sum = V::pack(v);
            V::store_raw(reinterpret_cast<uint8_t*>(a.h) + at, i, a.D, sum);
            V::unpack(sum, h[p]);
        }
        if (ragged) {
            const int skip = V::shared(i, a.D);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const double v = j < skip ? 0.0 : (double)h[p][j];
                ss = __builtin_fma(v, v, ss);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) ss = __builtin_fma((double)h[p][j], (double)h[p][j], ss);
        }
    }
    ss = sum_waves(sum_lanes<L>(ss), slot, waves);
    const Rstd s = split_rstd(rsqrt64(ss / a.D + a.eps));
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = p * team.lanes + team.lane;
        float w[N];
        load_weight<N, TINY>(a.weight, a.weight_dt, V::start(i, a.D), a.D, w);
#pragma unroll
        for (int j = 0; j < N; ++j) h[p][j] = __builtin_amdgcn_ldexpf(h[p][j], s.n) * s.a * w[j];
        V::store_raw(reinterpret_cast<uint8_t*>(a.y) + at, i, a.D, V::pack(h[p]));
    }
}

// The gradient: with n = h rstd and g = w d_y,  d_x = rstd (g - n mean(g n)) + d_h,  d_weight = sum over rows of d_y n.
// Teams walk rows, each row's loads sent out before the row before it is worked on, and keep their part of d_weight in
// registers; a workgroup adds its teams' parts in LDS, and a second launch the workgroups', all in order.
// Bound by memory: 8192 x 4096 bf16 with d_h 50 us, 5.4 TB/s of its four tensors, and 4 us of adding up (90 without
// the loads ahead); 110000 x 128 25 us in all, 3.4 TB/s.
//
// What a row takes of a lane's registers is kept as it lies in memory (`again` makes the compiler unpack it a second time
// rather than hold the floats across the sums); rows of four and more pieces a lane are not fetched ahead, read d_h and
// the weight where they are used, and have their part of d_weight in LDS, a slot a piece (2048 x 20000 107 us: 248 with all of
// it in registers that do not hold it, 167 where a row's sums wait for all of its weights).
__device__ __forceinline__ void again(v4u_mx& w) { asm volatile("" : "+v"(w)); }

template <int DT, int P, int L, bool RES, bool TINY>
__global__ __launch_bounds__(1024) void norm_grad_kernel(NormGradArgs a, int waves) {
    using V = NormPiece<DT, TINY>;
    constexpr int N = V::N;
    constexpr bool AHEAD = P <= 2;
    __shared__ double slots[2][2][16];
    extern __shared__ __attribute__((aligned(16))) float sums[];      // [teams, D] where there is more than one; or the slots
    Team<L> team(waves);
    const int teams = blockDim.x / team.lanes;
    const long long step = (long long)gridDim.x * teams;
    const bool ragged = a.D % N != 0;                        // the last piece shares elements
    float w[AHEAD ? P : 1][N], dw[AHEAD ? P : 1][N] = {};
    v4u_mx h[P], g[P], d[P], hn[P], gn[P], dn[P];
    const auto held = [&](int p) { return sums + (size_t)(p * blockDim.x + threadIdx.x) * N; };
    const auto weight = [&](int p, float (&v)[N]) {
        load_weight<N, TINY>(a.weight, a.weight_dt, V::start(p * team.lanes + team.lane, a.D), a.D, v);
    };
    const auto fetch = [&](long long row, v4u_mx (&h)[P], v4u_mx (&g)[P], v4u_mx (&d)[P]) {
        const size_t at = (size_t)(row < a.M ? row : 0) * a.D * V::ES;       // past the end a row that is there, not used
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = p * team.lanes + team.lane;
            h[p] = V::raw(reinterpret_cast<const uint8_t*>(a.h) + at, i, a.D);
            g[p] = V::raw(reinterpret_cast<const uint8_t*>(a.d_y) + at, i, a.D);
            if constexpr (AHEAD && RES) d[p] = V::raw(reinterpret_cast<const uint8_t*>(a.d_h) + at, i, a.D);
        }
    };
    long long row = (long long)blockIdx.x * teams + team.number;
    if (AHEAD) {
#pragma unroll
        for (int p = 0; p < P; ++p) weight(p, w[AHEAD ? p : 0]);
        fetch(row, hn, gn, dn);
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < N; j += 4) *reinterpret_cast<float4*>(held(p) + j) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    const int trips = (int)((a.M - (long long)blockIdx.x * teams + step - 1) / step);      // of the workgroup's first team
    for (int trip = 0; trip < trips; ++trip, row += step) {
        if (AHEAD) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                h[p] = hn[p];
                g[p] = gn[p];
                d[p] = dn[p];
            }
            if (trip + 1 < trips) fetch(row + step, hn, gn, dn);
        } else {
            asm volatile("" : "+v"(team.lane));             // addresses are made again, not kept for every piece
            fetch(row, h, g, d);
        }
        double ss = 0.0, gh = 0.0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float hf[N], gf[N];
            if (!AHEAD) {
                asm volatile("" ::: "memory");               // a piece's weights at a time
                weight(p, w[0]);
            }
            V::unpack(h[p], hf);
            V::unpack(g[p], gf);
            if (ragged) {
                const int skip = V::shared(p * team.lanes + team.lane, a.D);
#pragma unroll
                for (int j = 0; j < N; ++j) hf[j] = j < skip ? 0.0f : hf[j];
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                ss = __builtin_fma((double)hf[j], (double)hf[j], ss);
                gh = __builtin_fma((double)(gf[j] * w[AHEAD ? p : 0][j]), (double)hf[j], gh);
            }
            if (!AHEAD) asm volatile("" : "+v"(ss), "+v"(gh));           // added up before the next piece's are read
        }
        ss = sum_lanes<L>(ss);
        gh = sum_lanes<L>(gh);
        if (!AHEAD || waves > 1) {                           // of more than two pieces a lane, sixteen waves
            double (&s)[2][16] = slots[trip & 1];
            const int wave = threadIdx.x >> 6, first = wave / waves * waves;
            if ((threadIdx.x & 63) == 0) {
                s[0][wave] = ss;
                s[1][wave] = gh;
            }
            __syncthreads();
            ss = gh = 0.0;
            for (int i = 0; i < waves; ++i) {
                ss += s[0][first + i];
                gh += s[1][first + i];
            }
        }
        const double rstd = rsqrt64(ss / a.D + a.eps);
        const Rstd s = split_rstd(rstd);
        const float mean = (float)(gh * rstd / a.D);
        if (row >= a.M) continue;
        const size_t at = (size_t)row * a.D * V::ES;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = p * team.lanes + team.lane;
            float hf[N], gf[N], df[N] = {}, dx[N];
            again(h[p]);
            again(g[p]);
            if (!AHEAD) {
                asm volatile("" ::: "memory");
                weight(p, w[0]);
                if constexpr (RES) d[p] = V::raw(reinterpret_cast<const uint8_t*>(a.d_h) + at, i, a.D);
            }
            V::unpack(h[p], hf);
            V::unpack(g[p], gf);
            if constexpr (RES) V::unpack(d[p], df);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float n = __builtin_amdgcn_ldexpf(hf[j], s.n) * s.a;
                dx[j] = __builtin_amdgcn_ldexpf((gf[j] * w[AHEAD ? p : 0][j] - n * mean) * s.a, s.n) + df[j];
                if constexpr (AHEAD) dw[p][j] = __builtin_fmaf(gf[j], n, dw[p][j]);
                else hf[j] = n;
            }
            if constexpr (!AHEAD) {
#pragma unroll
                for (int j = 0; j < N; j += 4) {
                    float4 v = *reinterpret_cast<const float4*>(held(p) + j);
                    v.x = __builtin_fmaf(gf[j], hf[j], v.x);
                    v.y = __builtin_fmaf(gf[j + 1], hf[j + 1], v.y);
                    v.z = __builtin_fmaf(gf[j + 2], hf[j + 2], v.z);
                    v.w = __builtin_fmaf(gf[j + 3], hf[j + 3], v.w);
                    *reinterpret_cast<float4*>(held(p) + j) = v;
                }
            }
            if (a.d_x != nullptr) V::store_raw(reinterpret_cast<uint8_t*>(a.d_x) + at, i, a.D, V::pack(dx));
        }
    }
    if (a.d_weight == nullptr) return;
    // each lane's part; elements that two pieces share are the same in both
    float* part = teams > 1 ? sums + team.number * a.D : a.partial + (size_t)blockIdx.x * a.D;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = p * team.lanes + team.lane, e = V::start(i, a.D);
        if (!V::there(i, a.D)) continue;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (!TINY || j < a.D) part[e + j] = AHEAD ? dw[AHEAD ? p : 0][j] : held(p)[j];
    }
    if (teams == 1) return;
    __syncthreads();
    for (int e = threadIdx.x; e < a.D; e += blockDim.x) {
        float v = sums[e];
        for (int i = 1; i < teams; ++i) v += sums[i * a.D + e];
        if (gridDim.x == 1) store_weight(a.d_weight, a.weight_dt, e, v);      // no other workgroup has a part
        else a.partial[(size_t)blockIdx.x * a.D + e] = v;
    }
}

// d_weight[e] = the sum of `parts` rows of partial sums: a workgroup takes 16 columns, each of its 16 waves four sixty-fourths of the
// rows, so that a lane's loads are few and all under way at once.
__global__ __launch_bounds__(1024) void norm_weight_grad_kernel(const float* __restrict__ partial, void* __restrict__ d_weight,
                                                                int dt, int D, int parts) {
    __shared__ float part[16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x * 16 + (lane & 15);
    float s = 0.0f;
    if (e < D) {
#pragma unroll 8
        for (int b = wave * 4 + (lane >> 4); b < parts; b += 64) s += partial[(size_t)b * D + e];
    }
    s = all_lanes<64, 16>(s, [](float u, float v) { return u + v; });
    if (lane < 16) part[wave][lane] = s;
    __syncthreads();
    if (threadIdx.x >= 16 || e >= D) return;
    for (int v = 1; v < 16; ++v) s += part[v][lane];
    store_weight(d_weight, dt, e, s);
}

// ---------------------------------------------------------------------------
// The 8-bit form:
//   z = H_G(h w) rstd,  s = fl32(max(max |z|, 1e-10) / 127),  q = rint_even(z / s)
// A lane holds 16 consecutive values.  Everything up to the code is fp64 (full rate here), so a code is the formula's
// nearest one and not a matter of the order of sums; rstd commutes with the rotation, so it is not waited for.  A row
// with a value that is not finite (or zeros over eps = 0) gets scale NaN and codes 0.
// 8192 x 5120 bf16 with a residual 59.5 us, 4.9 TB/s: memory, and VALU instructions 65% of the time (22 an element, of which the
// rotation's are 7); without a residual 39 us, where they are 80%.  LDS for the rotation's transpose holds a CU to 18 waves;
// registers are kept to what five waves a SIMD have (of two chunks a lane: 4096 x 10240 76 us with four, 66 so), but for 32-bit
// values, which would spill.
// ---------------------------------------------------------------------------
template <int DT, int G, int P, int L, bool TILED>
__global__ __launch_bounds__(1024) __attribute__((amdgpu_waves_per_eu(P > 1 && DT != DT_F32 ? 5 : 4))) void norm_int8_kernel(NormArgs a, unsigned first) {
    using V = NormPiece<DT>;
    constexpr int N = V::N, LPG = G / kChunk, PIECES = kChunk / N;
    static_assert(L >= LPG && (L == 64 || P == 1), "groups of whole teams");
    extern __shared__ __attribute__((aligned(16))) double norm_lds[];
    const int waves = __builtin_amdgcn_readfirstlane(blockDim.x >> 6), lane = threadIdx.x & 63;
    const int W = L < 64 ? 1 : waves;                         // of a row
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wv = L < 64 ? 0 : wave;
    double* tbuf = norm_lds + wave * (64 * kPad);
    double* slot = norm_lds + waves * (64 * kPad);            // [2][16]
    uint8_t* cb = reinterpret_cast<uint8_t*>(tbuf);
    const int nchunks = a.D / kChunk, gl = lane % LPG, gfirst = lane - gl;
    const long long row = L < 64 ? (long long)(first + blockIdx.x) * (blockDim.x / L) + threadIdx.x / L : (long long)first + blockIdx.x;
    int8_t* q = reinterpret_cast<int8_t*>(a.y);
    const auto code_at = [&](int c) {
        if constexpr (TILED)
            return reinterpret_cast<uint4*>(q + ((size_t)(row >> 8) * (a.D >> 6) + (c >> 2)) * I8T_CHUNK + i8t_off((int)(row & 255), c & 3));
        else return reinterpret_cast<uint4*>(q + (size_t)row * a.D + (size_t)c * kChunk);
    };
    if (TILED && L == 64 && row >= a.M) {                     // padding rows hold zeros
        for (int c = threadIdx.x; c < nchunks; c += blockDim.x) *code_at(c) = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const bool real = L == 64 || row < a.M;                   // teams without a row go along with the last one's
    const auto chunk = [&](int p) { return L < 64 ? lane % L : (p * W + wv) * 64 + lane; };
    const size_t at = (size_t)(real ? row : a.M - 1) * a.D * V::ES;
    const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x) + at;
    const uint8_t* res = reinterpret_cast<const uint8_t*>(a.residual) + at;
    v4u_mx xs[P][PIECES], rs[P][PIECES];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = chunk(p);                               // lanes past the row's end take its last chunk, and drop it
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const size_t piece = (size_t)(min(c, nchunks - 1) * PIECES + i) * 16;
            xs[p][i] = *reinterpret_cast<const v4u_mx*>(x + piece);
            if (a.residual != nullptr) rs[p][i] = *reinterpret_cast<const v4u_mx*>(res + piece);
        }
    }
    double z[P][kChunk], ss = 0.0, most = 0.0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (L == 64 && (p * W + wv) * 64 >= nchunks) break;   // the wave's
        const int c = chunk(p);
        const bool ok = c < nchunks && real;
        float w[kChunk];
        load_weight<kChunk>(a.weight, a.weight_dt, min(c, nchunks - 1) * kChunk, a.D, w);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            float h[N];
            V::unpack(xs[p][i], h);
            if (a.residual != nullptr) {
                float r[N];
                V::unpack(rs[p][i], r);
#pragma unroll
                for (int j = 0; j < N; ++j) r[j] += h[j];
                const v4u_mx sum = V::pack(r);
                if (ok) *reinterpret_cast<v4u_mx*>(reinterpret_cast<uint8_t*>(a.h) + at + (size_t)(c * PIECES + i) * 16) = sum;
                V::unpack(sum, h);
            }
            double part = 0.0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const double v = (double)h[j];
                z[p][i * N + j] = v * (double)w[i * N + j];
                part = __builtin_fma(v, v, part);
            }
            ss += ok ? part : 0.0;
        }
        rotate_chunk<G>(z[p], tbuf, lane, gl, gfirst);
        double top = 0.0;
#pragma unroll
        for (int i = 0; i < kChunk; ++i) top = fmax(top, fabs(z[p][i]));
        most = ok ? fmax(most, top) : most;
        ss = ok ? __builtin_fma(z[p][0], 0.0, ss) : ss;       // a NaN where a product of the group is not finite: all its sums are not
    }
    ss = sum_lanes<L>(ss);
    most = all_lanes<L>(most, [](double u, double v) { return fmax(u, v); });
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
    const double rstd = rsqrt64(ss / a.D + a.eps);
    const bool finite = ss < __builtin_inf() && rstd < __builtin_inf();
    const float s = finite ? (float)(fmax(most * rstd, 1e-10) * (1.0 / 127.0)) : __builtin_nanf("");
    const double steps = rstd / (double)s;
    const uint32_t keep = finite && real ? 0xffffffffu : 0u;
    const bool put = real || (TILED && row < (a.M + 255LL) / 256 * 256);
    if (L < 64 ? lane % L == 0 && real : threadIdx.x == 0) a.scales[row] = s;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (L == 64 && (p * W + wv) * 64 >= nchunks) break;
        const int c = chunk(p);
        wave_sync();
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
            // low byte of the sum with 1.5 2^52: rint_even; |z steps| <= 127 (1 + 2^-23)
            const uint32_t code = (uint32_t)__double_as_longlong(__builtin_fma(z[p][i], steps, 0x1.8p52));
            const int e = final_elem<G>(gl, i);
            cb[(gfirst + e / kChunk) * kChunk + e % kChunk] = (uint8_t)code;
        }
        wave_sync();
        uint4 v = reinterpret_cast<const uint4*>(cb)[lane];
        v.x &= keep; v.y &= keep; v.z &= keep; v.w &= keep;
        if (c < nchunks && put) *code_at(c) = v;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// How rows of `pieces` are shared out: lanes of a team (64: `waves` waves), pieces a lane.
struct NormShape { int lanes, waves, P; };
static NormShape norm_shape(long long rows, int pieces, int want) {
    if (pieces <= 32) return {pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32, 1, 1};
    int W = (pieces + 64 * want - 1) / (64 * want);
    if (rows * W < 2048) W = (pieces + 63) / 64;             // few rows: a piece a lane
    if (W > 16) W = 16;
    const int P = (pieces + 64 * W - 1) / (64 * W);
    return {64, W, P <= 2 ? P : P <= 4 ? 4 : 8};
}

template <typename F>
static hipError_t by_type(int dt, F f) {
    using std::integral_constant;
    if (dt == DT_F32) return f(integral_constant<int, DT_F32>{});
    if (dt == DT_BF16) return f(integral_constant<int, DT_BF16>{});
    return f(integral_constant<int, DT_F16>{});
}

// f(pieces a lane, lanes of a team, rows narrower than a piece)
template <int DT, typename F>
static hipError_t by_shape(const NormShape& s, int D, F f) {
    using std::integral_constant;
    const integral_constant<int, 64> wave{};
    const integral_constant<int, 1> one{};
    const std::false_type wide{};
    if (D < NormPiece<DT>::N) return f(one, integral_constant<int, 8>{}, std::true_type{});
    if (s.lanes == 8) return f(one, integral_constant<int, 8>{}, wide);
    if (s.lanes == 16) return f(one, integral_constant<int, 16>{}, wide);
    if (s.lanes == 32) return f(one, integral_constant<int, 32>{}, wide);
    if (s.P == 1) return f(one, wave, wide);
    if (s.P == 2) return f(integral_constant<int, 2>{}, wave, wide);
    if constexpr (DT == DT_F32) {
        if (s.P == 8) return f(integral_constant<int, 8>{}, wave, wide);
    }
    return f(integral_constant<int, 4>{}, wave, wide);
}

hipError_t norm_launch(const NormArgs& a, int dt, hipStream_t st) {
    return by_type(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        const NormShape s = norm_shape(a.M, (a.D + NormPiece<DT>::N - 1) / NormPiece<DT>::N, NORM_PIECES);
        const int threads = s.lanes < 64 || s.waves == 1 ? 256 : 64 * s.waves;
        const int rows = threads / (s.lanes < 64 ? s.lanes : 64 * s.waves);
        return by_shape<DT>(s, a.D, [&](auto p, auto l, auto t) {
            constexpr int P = decltype(p)::value, L = decltype(l)::value;
            constexpr bool TINY = decltype(t)::value;
            return launch_parts(((long long)a.M + rows - 1) / rows, threads, [&](long long first, dim3 grid) {
                if (a.residual != nullptr)
                    hipLaunchKernelGGL((norm_kernel<DT, P, L, true, TINY>), grid, dim3(threads), 0, st, a, s.waves, (unsigned)first);
                else
                    hipLaunchKernelGGL((norm_kernel<DT, P, L, false, TINY>), grid, dim3(threads), 0, st, a, s.waves, (unsigned)first);
            });
        });
    });
}

// Teams and workgroups of a gradient, from its shape: workgroups of eight waves or one team.  Each leaves a row of partial
// sums of d_weight, to be read again: as many workgroups as the chip holds at once (16 waves a CU), but past 256, one a
// CU, no more than makes that an eighth of the rows' traffic (8192 x 4096: 512 workgroups 55.6 us, 1024 61.6; 2048 x 13824: 256
// 58.6, 512 69.2; 110000 x 128: 512 30.2, 1024 24.9).  256 workgroups of fewer than 2048 rows M make it 256 / M of them: a
// quarter at 1024 rows, half at 512.  One workgroup where it has several teams and each few rows, which then
// writes d_weight itself.
struct NormGradShape { NormShape team; int teams, groups; };
static NormGradShape norm_grad_shape(int M, int D, int piece) {
    const int pieces = (D + piece - 1) / piece;
    NormShape s = norm_shape(1, pieces, 1);                  // a piece a lane as far as sixteen waves go
    if (s.lanes == 64 && s.P == 1 && s.waves > 1 && (long long)M * s.waves > NORM_GRAD_FEW) s = {64, (s.waves + 1) / 2, 2};
    const int threads = s.lanes < 64 ? 256 : 64 * s.waves < 512 ? 512 / (64 * s.waves) * 64 * s.waves : 64 * s.waves;
    const int teams = threads / (s.lanes < 64 ? s.lanes : 64 * s.waves);
    const long long all = ((long long)M + teams - 1) / teams;
    const int waves = threads / 64, most = 256 * (waves <= 8 ? 16 / waves : 1), few = M / 8 / 256 * 256;
    const int groups = most < few ? most : few > 256 ? few : 256;
    return {s, teams, (int)(teams > 1 && all <= NORM_GRAD_ALONE ? 1 : all < groups ? all : groups)};
}

size_t norm_grad_bytes(int M, int D) {
    const int g4 = norm_grad_shape(M, D, 4).groups, g8 = norm_grad_shape(M, D, 8).groups;
    return (size_t)(g4 > g8 ? g4 : g8) * D * sizeof(float);
}

template <int DT, int P, int L, bool TINY>
static hipError_t norm_grad_go(const NormGradArgs& a, const NormGradShape& s, hipStream_t st) {
    // teams share a workgroup of at most 512 threads, of one piece or two a lane: 512 x 2 pieces x 8 values
    const int threads = s.teams * (L < 64 ? L : 64 * s.team.waves);
    int lds = s.teams > 1 ? s.teams * a.D * (int)sizeof(float) : 0;
    if (lds > 512 * 2 * 8 * (int)sizeof(float)) return hipErrorInvalidValue;
    if constexpr (P > 2) {                                   // the slots: at most 1024 threads' 32 values
        constexpr int N = NormPiece<DT>::N;
        static_assert(1024 * P * N <= NORM_MAX_D, "128 KB");
        if (s.teams > 1 || threads != 1024) return hipErrorInvalidValue;
        static std::atomic<bool> attr[kMaxDev], attr_res[kMaxDev];
        lds = threads * P * N * (int)sizeof(float);
        int dev = 0;
        hipError_t e = current_device(&dev);
        if (e != hipSuccess) return e;
        e = a.d_h != nullptr
                ? lds_limit_once(attr_res, dev, reinterpret_cast<const void*>(&norm_grad_kernel<DT, P, L, true, TINY>), lds)
                : lds_limit_once(attr, dev, reinterpret_cast<const void*>(&norm_grad_kernel<DT, P, L, false, TINY>), lds);
        if (e != hipSuccess) return e;
    }
    if (a.d_h != nullptr)
        hipLaunchKernelGGL((norm_grad_kernel<DT, P, L, true, TINY>), dim3(s.groups), dim3(threads), lds, st, a, s.team.waves);
    else
        hipLaunchKernelGGL((norm_grad_kernel<DT, P, L, false, TINY>), dim3(s.groups), dim3(threads), lds, st, a, s.team.waves);
    return hipGetLastError();
}

static hipError_t norm_weight_grad_launch(const NormGradArgs& a, int parts, hipStream_t st) {
    hipLaunchKernelGGL(norm_weight_grad_kernel, dim3((a.D + 15) / 16), dim3(1024), 0, st, a.partial, a.d_weight, a.weight_dt, a.D, parts);
    return hipGetLastError();
}

hipError_t norm_grad_launch(const NormGradArgs& a, int dt, hipStream_t st) {
    if (a.M == 0) return a.d_weight == nullptr ? hipSuccess : norm_weight_grad_launch(a, 0, st);      // zeros: a sum of no rows
    const NormGradShape s = norm_grad_shape(a.M, a.D, dt == DT_F32 ? 4 : 8);
    const hipError_t e = by_type(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        return by_shape<DT>(s.team, a.D, [&](auto p, auto l, auto t) {
            return norm_grad_go<DT, decltype(p)::value, decltype(l)::value, decltype(t)::value>(a, s, st);
        });
    });
    // several teams of one workgroup have written d_weight themselves
    if (e != hipSuccess || a.d_weight == nullptr || (s.groups == 1 && s.teams > 1)) return e;
    return norm_weight_grad_launch(a, s.groups, st);
}

template <int DT, int G, int P, int L, bool TILED>
static hipError_t norm_int8_go(const NormArgs& a, int waves, hipStream_t st) {
    static std::atomic<bool> attr[kMaxDev];
    constexpr int MOST = (16 * 64 * kPad + 32) * (int)sizeof(double);
    int dev = 0;
    hipError_t e = current_device(&dev);
    if (e != hipSuccess) return e;
    e = lds_limit_once(attr, dev, reinterpret_cast<const void*>(&norm_int8_kernel<DT, G, P, L, TILED>), MOST);
    if (e != hipSuccess) return e;
    const long long rows = TILED ? (a.M + 255LL) / 256 * 256 : a.M, each = L < 64 ? 64 * waves / L : 1;
    return launch_parts((rows + each - 1) / each, 64 * waves, [&](long long first, dim3 grid) {
        hipLaunchKernelGGL((norm_int8_kernel<DT, G, P, L, TILED>), grid, dim3(64 * waves), (waves * 64 * kPad + 32) * sizeof(double), st, a,
                           (unsigned)first);
    });
}

hipError_t norm_int8_launch(const NormArgs& a, int dt, int G, bool tiled, hipStream_t st) {
    const int nchunks = a.D / kChunk, waves = (nchunks + 63) / 64;
    const bool one = waves == 1 || (waves <= 16 && ((long long)a.M * waves < NORM8_FEW || (a.residual != nullptr && waves <= 4)));
    return by_type(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        const auto go = [&](auto g) {
            constexpr int GG = decltype(g)::value;
            const auto shape = [&](auto p, auto l, int w) {
                constexpr int P = decltype(p)::value, L = decltype(l)::value;
                return tiled ? norm_int8_go<DT, GG, P, L, true>(a, w, st) : norm_int8_go<DT, GG, P, L, false>(a, w, st);
            };
            using std::integral_constant;
            const integral_constant<int, 1> p1{};
            // short rows: several of them to a wave, four waves to a workgroup
            if (nchunks <= 16) return shape(p1, integral_constant<int, 16>{}, 4);
            if (nchunks <= 32) return shape(p1, integral_constant<int, 32>{}, 4);
            return one ? shape(p1, integral_constant<int, 64>{}, waves)
                       : shape(integral_constant<int, 2>{}, integral_constant<int, 64>{}, (waves + 1) / 2);
        };
        using std::integral_constant;
        return G == 16 ? go(integral_constant<int, 16>{}) : G == 64 ? go(integral_constant<int, 64>{}) : go(integral_constant<int, 256>{});
    });
}

}  // namespace convrot
