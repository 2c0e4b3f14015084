// What the kernels of the MXFP4 product share: the operands, the map from
// workgroups to tiles (one weight matrix, or one per expert with a ragged set
// of rows each), and the store of a tile.
#pragma once

#include "mxfp4.h"

namespace convrot {

// y[r, n] = sum_k a[row(r), k] w[e(r)][n, k] + bias[e(r)][n] for the R rows of the output.
// a: codes [as_rows, Kp/2], Kp = K rounded up to 256, the padding codes zero; w: codes [E, N, K/2] and scales
// [E, N, K/32].  Scales for staged tiles: as [Ks/16, as_rows, 16] and wp [E, Ks/16, N, 16], Ks = K/32 rounded up
// to 16, 512 k after the other, the bytes of a row in the order of mx_scale_place, the padding 0.  For the others
// as is [as_rows, Ks] and wp is not there.
// offsets NULL: E = 1 and row(r) = r.  Else rows offsets[e] .. offsets[e + 1] - 1 are expert e's, those from
// offsets[E] on come out zero, and row(r) = r, or order[r] / top_k where order is not NULL.
struct MxProblem {
    const uint8_t *a, *as, *w, *ws, *wp;
    const void* bias;
    void* out;
    const int *offsets, *order;
    int R, N, K, Kp, Ks, as_rows, E, top_k;
    int block0;                                            // workgroups of earlier launches of the call
    short dt, bias_dt;                                     // 120 bytes in all: the arguments of a launch in two cache lines
    unsigned k_mul;                                        // n / top_k = n k_mul >> k_shift for 0 <= n < 2^31
    int k_shift;
};

// The kernel of a product: rows and columns of its tile, stages in LDS (0: the kernel for few rows), and whether that
// quantizes x itself.
struct MxKernel {
    int rows, cols, slots;
    bool fused;
};

// l = ceil(log2 d), m = ceil(2^(31 + l) / d): n m >> (31 + l) is n / d for every n < 2^31, and m < 2^32.
inline void mx_set_top_k(MxProblem& p, int d) {
    int l = 0;
    while ((1ll << l) < d) ++l;
    p.top_k = d;
    p.k_shift = 31 + l;
    p.k_mul = (unsigned)(((1ull << p.k_shift) + d - 1) / d);
}

// Place of block b (0 .. 15) of 512 k: a lane of half h of a wave takes blocks 2 s + h of a stage of 256 k, s = 0 .. 3,
// whose bytes are one word.
__host__ __device__ constexpr int mx_scale_place(int b) { return (b & 8) | (b & 1) << 2 | (b >> 1 & 3); }

// A tile of at most BM rows: rows m0 .. m1 - 1 of expert e, or rows to be zeroed (e = E).
struct MxTile { int e, m0, m1; };

// Row tiles at most: every expert's last tile may be short, and so may the zeroed rows'.
inline long long mx_row_tiles(int R, int E, bool ragged, int BM) {
    const long long full = (R + (long long)BM - 1) / BM;
    if (!ragged) return full;
    return R / BM + (E + 1LL < R ? E + 1LL : R);
}

// Row numbers go up to 2^31 - 2: sums of one and a tile's rows are taken unsigned, or as distances.

// Tiles of n rows
template <int BM>
__device__ __forceinline__ int mx_tiles_of(int n) { return (int)(((unsigned)n + (BM - 1)) / BM); }

// End of the tile that begins at row m0 of those before r1
template <int BM>
__device__ __forceinline__ int mx_tile_end(int m0, int r1) { return m0 + min(BM, r1 - m0); }

// Expert e's rows as the wave's lanes hold them, 64 experts a run; expert E is the rows past the last used one.
template <int BM>
struct MxRun {
    int r0, r1, n, sum;                                    // rows, their tiles, tiles of this and the lanes before
    __device__ __forceinline__ MxRun(const MxProblem& p, int e) {
        r0 = e <= p.E ? min(max(p.offsets[e], 0), p.R) : p.R;
        r1 = e < p.E ? min(max(p.offsets[e + 1], r0), p.R) : p.R;
        sum = n = mx_tiles_of<BM>(r1 - r0);
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
    }
};

// Row tiles that there are.
template <int BM>
__device__ __forceinline__ int mx_tile_count(const MxProblem& p) {
    if (p.offsets == nullptr) return mx_tiles_of<BM>(p.R);
    int count = 0;
    for (int e0 = 0; e0 <= p.E; e0 += 64) count += __shfl(MxRun<BM>(p, e0 + (threadIdx.x & 63)).sum, 63);
    return __builtin_amdgcn_readfirstlane(count);
}

// Row tile t, which there is.
template <int BM>
__device__ __forceinline__ MxTile mx_tile(const MxProblem& p, int t) {
    if (p.offsets == nullptr) return {0, t * BM, mx_tile_end<BM>(t * BM, p.R)};
    int base = 0;
    for (int e0 = 0; e0 <= p.E; e0 += 64) {
        const MxRun<BM> run(p, e0 + (threadIdx.x & 63));
        const int first = base + run.sum - run.n;
        const unsigned long long here = __ballot(t >= first && t < first + run.n);
        if (here) {
            const int l = __builtin_ctzll(here);
            const int m0 = __builtin_amdgcn_readfirstlane(__shfl(run.r0 + (t - first) * BM, l));
            return {e0 + l, m0, __builtin_amdgcn_readfirstlane(mx_tile_end<BM>(m0, __shfl(run.r1, l)))};
        }
        base += __shfl(run.sum, 63);
    }
    return {p.E, p.R, p.R};
}

__device__ __forceinline__ float mx_read(const void* p, int dt, size_t i) {
    if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
    const uint32_t h = reinterpret_cast<const uint16_t*>(p)[i];
    return dt == DT_BF16 ? __uint_as_float(h << 16) : f16bits_to_f32(h);
}

// Four neighbouring columns of a row, rounded once to the output type; `vec`: all there and aligned.
__device__ __forceinline__ void mx_store4(void* out, int dt, size_t i, const float (&v)[4], int n, bool vec) {
    if (dt == DT_F32) {
        float* o = reinterpret_cast<float*>(out) + i;
        if (vec) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        else for (int j = 0; j < n; ++j) o[j] = v[j];
    } else {
        const uint2 h = dt == DT_BF16 ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]))
                                      : make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
        uint16_t* o = reinterpret_cast<uint16_t*>(out) + i;
        if (vec) *reinterpret_cast<uint2*>(o) = h;
        else for (int j = 0; j < n; ++j) o[j] = (uint16_t)((j < 2 ? h.x : h.y) >> (16 * (j & 1)));
    }
}

// Row of `a` that output row r takes where there is an order.
__device__ __forceinline__ int mx_source_row(const MxProblem& p, int r) {
    const unsigned slot = (unsigned)min(max(p.order[r], 0), p.R - 1);
    return (int)((unsigned long long)slot * p.k_mul >> p.k_shift);
}

// Zeros in rows m0 .. m1 - 1, columns n0 .. n1 - 1 (n0 a multiple of 16), by the threads of a workgroup: a wave a row at a
// time, 16 bytes a lane where rows are whole pieces of that.
__device__ __forceinline__ void mx_zero(const MxProblem& p, int m0, int m1, int n0, int n1) {
    const int es = p.dt == DT_F32 ? 4 : 2, lane = threadIdx.x & 63;
    for (unsigned m = m0 + (threadIdx.x >> 6); m < (unsigned)m1; m += blockDim.x >> 6) {
        uint8_t* row = reinterpret_cast<uint8_t*>(p.out) + ((size_t)m * p.N + n0) * es;
        const int bytes = (n1 - n0) * es;
        if ((size_t)p.N * es % 16 == 0) {
            for (int i = lane * 16; i < bytes; i += 1024) *reinterpret_cast<v4u_mx*>(row + i) = (v4u_mx){0u, 0u, 0u, 0u};
        } else {
            for (int i = lane * 2; i < bytes; i += 128) *reinterpret_cast<uint16_t*>(row + i) = 0;
        }
    }
}

}  // namespace convrot
