// What the kernels of the MXFP4 product share: the operands, the map from
// workgroups to tiles (one weight matrix, or one per expert with a ragged set
// of rows each), and the store of a tile.
#pragma once

#include "mxfp4.h"

namespace convrot {

// y[r, n] = sum_k a[row(r), k] w[e(r)][n, k] + bias[e(r)][n] for the R rows of the output.
// a: codes [rows, Kp/2] and scales [rows, Kp/32], Kp = K rounded up to 128, the padding codes zero.
// w: codes [E, N, K/2] and scales [E, N, K/32].  offsets NULL: E = 1 and row(r) = r.  Else rows
// offsets[e] .. offsets[e + 1] - 1 are expert e's, those from offsets[E] on come out zero, and
// row(r) = r, or order[r] / top_k where order is not NULL.
struct MxProblem {
    const uint8_t *a, *as, *w, *ws;
    const void* bias;
    void* out;
    const int *offsets, *order;
    int R, N, K, Kp, E, top_k, dt, bias_dt;
};

// A tile of at most BM rows: rows m0 .. m1 - 1 of expert e, or rows to be zeroed (e = E).
struct MxTile { int e, m0, m1; };

// Row tiles at most: every expert's last tile may be short, and so may the zeroed rows'.
inline long long mx_row_tiles(int R, int E, bool ragged, int BM) {
    const long long full = (R + (long long)BM - 1) / BM;
    if (!ragged) return full;
    return R / BM + (E + 1LL < R ? E + 1LL : R);
}

// Row tile `t` of the grid, found by the whole wave from the experts' offsets:
// lane l holds expert l of each run of 64, the tiles are counted with a prefix
// sum over the lanes.  False: past the last tile.
template <int BM>
__device__ __forceinline__ bool mx_tile(const MxProblem& p, int t, MxTile& tile) {
    if (p.offsets == nullptr) {
        tile = {0, t * BM, min(t * BM + BM, p.R)};
        return tile.m0 < p.R;
    }
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int e0 = 0; e0 <= p.E; e0 += 64) {                // expert E: the rows past the last used one
        const int e = e0 + lane;
        const int r0 = e <= p.E ? min(max(p.offsets[e], 0), p.R) : p.R;
        const int r1 = e < p.E ? min(max(p.offsets[e + 1], r0), p.R) : p.R;
        const int n = (r1 - r0 + BM - 1) / BM;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        const int first = base + sum - n;
        const unsigned long long here = __ballot(t >= first && t < first + n);
        if (here) {
            const int l = __builtin_ctzll(here);
            const int m0 = __shfl(r0 + (t - first) * BM, l);
            tile = {e0 + l, m0, min(m0 + BM, __shfl(r1, l))};
            tile.e = __builtin_amdgcn_readfirstlane(tile.e);
            tile.m0 = __builtin_amdgcn_readfirstlane(tile.m0);
            tile.m1 = __builtin_amdgcn_readfirstlane(tile.m1);
            return true;
        }
        base += __shfl(sum, 63);
    }
    return false;
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

// Row of `a` that output row r takes.
__device__ __forceinline__ int mx_source_row(const MxProblem& p, int r) {
    return p.order != nullptr ? min(max(p.order[r], 0), p.R - 1) / p.top_k : r;
}

// Zeros in rows m0 .. m1 - 1, columns n0 .. n1 - 1 (threads of a workgroup).
__device__ __forceinline__ void mx_zero(const MxProblem& p, int m0, int m1, int n0, int n1) {
    const int n = n1 - n0;
    for (long long i = threadIdx.x; i < (long long)(m1 - m0) * n; i += blockDim.x) {
        const size_t o = (size_t)(m0 + i / n) * p.N + n0 + i % n;
        if (p.dt == DT_F32) reinterpret_cast<float*>(p.out)[o] = 0.0f;
        else reinterpret_cast<uint16_t*>(p.out)[o] = 0;
    }
}

}  // namespace convrot
