// The product of MXFP4 rows with MXFP4 weights where there are few rows: operands from
// memory to registers, k split over the waves of a workgroup (mxfp4_gemm.h has the
// operands; mxfp4_staged.hip the kernel for many rows).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 4-bit floats and applies both operands'
// block scales itself: lane l supplies row l % 16, the 32 values of block l / 16 of the
// 128 (16 bytes) and that block's scale byte.  The weight's rows are its first operand,
// so a lane's four results are neighbouring columns of one output row.
//
// Bound by the weight's bytes (a few rows) or by the copies of both operands from L2.
// Eight waves share 16 NF columns by 16 MF rows, each a run of k, so that a CU has
// some 100 KB of loads in flight and a grid of one row tile still fills the card; their
// sums meet in LDS, added in wave order.  With FUSE the workgroup rotates and quantizes
// its rows itself, while its first weights are on the way, which saves a launch and a
// round trip of the codes.
//
// Measured on MI355X, kernel trace: 1 x 5120 -> 13824 rotated 9.9 us (37.6 MB, 3.8 TB/s;
// 1 x 4096 -> 4096 5.2), 4 rows 12.5, 16 rows 10.8 and 2.4 for their codes; one token's four
// experts of 2048 -> 4096 8.1 us.

#include "gemm_common.h"
#include "mxfp4_gemm.h"

namespace convrot {

typedef int v8i_mx __attribute__((ext_vector_type(8)));
typedef float v4f_mx __attribute__((ext_vector_type(4)));

constexpr int FEW_WAVES = 8;

__device__ __forceinline__ v8i_mx mx_operand(v4u_mx c) {
    return (v8i_mx){(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
}

// The 16 values of unit u (K / 16 of them a row) of the tile's rows
template <int DT>
__device__ __forceinline__ void few_load(const MxProblem& p, const uint8_t* x, const MxTile& t, int u, float (&v)[16]) {
    const int per = p.K / 16, r = u / per, k = (u - r * per) * 16;
    const size_t row = p.order != nullptr ? mx_source_row(p, t.m0 + r) : t.m0 + r;
    load16<DT>(x + (row * p.K + k) * (DT == DT_F32 ? 4 : 2), v);
}

// The scale bytes of the tile's columns and rows in LDS, 16 bytes a thread: a byte a lane from memory instead costs a
// third of the time (1 x 5120 -> 13824 12.6 us, 8.2 with none at all).
__device__ __forceinline__ void few_copy16(const uint8_t* src, uint8_t* dst, int bytes) {
    for (int i = threadIdx.x * 16; i < bytes; i += 64 * FEW_WAVES * 16) {
        if (i + 16 <= bytes) {
            v4u_mx w;
            __builtin_memcpy(&w, src + i, 16);             // any alignment
            *reinterpret_cast<v4u_mx*>(dst + i) = w;
        } else {
            for (int j = i; j < bytes; ++j) dst[j] = src[j];
        }
    }
}

constexpr int few_pad(int bytes) { return (bytes + 15) & ~15; }

// Widest rows whose scales are held in LDS; past it they are read from memory.
constexpr int FEW_MAX_K = 32768;

// DT, G: of x, with FUSE.
template <int DT, int G, int MF, int NF, bool FUSE>
__global__ __launch_bounds__(64 * FEW_WAVES) void mxfp4_gemm_few_kernel(MxProblem p, const uint8_t* __restrict__ x) {
    constexpr int BM = 16 * MF, BN = 16 * NF, THREADS = 64 * FEW_WAVES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_few[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles_m = mx_tile_count<BM>(p), tiles_n = (p.N + BN - 1) / BN;
    const int block = p.block0 + (int)blockIdx.x;
    if (block >= tiles_m * tiles_n) return;
    int tm, tn;
    tile_of_block(block, tiles_m, tiles_n, tiles_m, tm, tn);   // an XCD's row tiles of the same columns together
    const MxTile t = mx_tile<BM>(p, tm);
    const int n0 = tn * BN;
    if (t.e == p.E && p.offsets != nullptr) return mx_zero(p, t.m0, t.m1, n0, min(n0 + BN, p.N));
    const int rows = t.m1 - t.m0;

    // x first: its values are needed before the weight's, and loads come back in order
    float v[16];
    const int units = rows * (p.K / 16);
    if constexpr (FUSE) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
        if (tid < units) few_load<DT>(p, x, t, tid, v);
    }

    // Steps of 128 k; this wave's are pairs (whole lines) of them, first .. last - 1.
    const int l16 = lane & 15, g = lane >> 4;
    const int nb = p.K / 32, steps = (p.K + 127) / 128, pairs = (steps + 1) / 2;
    const int first = wave * pairs / FEW_WAVES, last = (wave + 1) * pairs / FEW_WAVES;
    const uint8_t *w[NF], *ws[NF], *a[MF], *as[MF];
#pragma unroll
    for (int j = 0; j < NF; ++j) {                         // columns and rows past the edge repeat the last
        const size_t r = (size_t)t.e * p.N + min(n0 + j * 16 + l16, p.N - 1);
        w[j] = p.w + r * (p.K / 2);
        ws[j] = p.ws + r * nb;
    }
    // LDS: the columns' scales [BN, nb], the rows' scales [rows, srow], with FUSE the rows' codes [rows, stride]
    const bool near = p.K <= FEW_MAX_K;
    const int stride = p.Kp / 2, srow = FUSE ? p.Kp / 32 : p.Ks;
    uint8_t* lds_ws = lds_few;
    uint8_t* lds_s = lds_few + few_pad(BN * nb);
    uint8_t* lds_c = lds_s + few_pad(rows * srow);
    int lrow[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
        lrow[i] = min(i * 16 + l16, rows - 1);
        if constexpr (!FUSE) {
            const size_t r = p.order != nullptr ? mx_source_row(p, t.m0 + lrow[i]) : t.m0 + lrow[i];
            a[i] = p.a + r * stride;
            as[i] = p.as + r * p.Ks;
        }
    }
    struct Step { v4u_mx w[NF], a[MF]; };                  // codes of block 4 st + g
    auto load_w = [&](Step& s, int st) __attribute__((always_inline)) {
        const int blk = st * 4 + g;
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            s.w[j] = *reinterpret_cast<const v4u_mx*>(w[j] + (size_t)min(blk, nb - 1) * 16);   // past K: times codes 0
        }
    };
    auto load_a = [&](Step& s, int st) __attribute__((always_inline)) {
        const int blk = st * 4 + g;
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            if constexpr (FUSE) {
                s.a[i] = *reinterpret_cast<const v4u_mx*>(lds_c + lrow[i] * stride + blk * 16);
            } else {
                s.a[i] = *reinterpret_cast<const v4u_mx*>(a[i] + (size_t)blk * 16);
            }
        }
    };
    Step s[2][2];
    if (first < last) {
        load_w(s[0][0], 2 * first);
        if (2 * first + 1 < steps) load_w(s[0][1], 2 * first + 1);
        if constexpr (!FUSE) {
            load_a(s[0][0], 2 * first);
            if (2 * first + 1 < steps) load_a(s[0][1], 2 * first + 1);
        }
    }
    if constexpr (FUSE) {
        for (int u = tid; u < units; u += THREADS) {           // whole blocks and groups: no lane of one is missing
            if (u >= THREADS) {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0.0f;
                if (u < units) few_load<DT>(p, x, t, u, v);
            }
            rotate16<G>(v);
            uint32_t sb;
            const v2u_mx c = mx_encode16(v, sb);
            const int per = p.K / 16, r = u / per, k16 = u - r * per;
            if (u < units) {
                *reinterpret_cast<v2u_mx*>(lds_c + r * stride + k16 * 8) = c;
                if ((k16 & 1) == 0) lds_s[r * srow + k16 / 2] = (uint8_t)sb;
            }
        }
        const int pad = (p.Kp - p.K) / 32;                 // blocks of zeros behind each row
        for (int i = tid; i < rows * pad; i += THREADS) {
            const int r = i / pad, blk = nb + i - r * pad;
            *reinterpret_cast<v4u_mx*>(lds_c + r * stride + blk * 16) = (v4u_mx){0u, 0u, 0u, 0u};
            lds_s[r * srow + blk] = 0;
        }
    } else if (near) {
        const int per = srow / 16;
        for (int i = tid; i < rows * per; i += THREADS) {
            const int r = i / per;
            const size_t row = p.order != nullptr ? mx_source_row(p, t.m0 + r) : t.m0 + r;
            reinterpret_cast<v4u_mx*>(lds_s)[i] = reinterpret_cast<const v4u_mx*>(p.as + row * srow)[i - r * per];
        }
    }
    const int cols = min(BN, p.N - n0);
    if (near) few_copy16(p.ws + ((size_t)t.e * p.N + n0) * nb, lds_ws, cols * nb);
    __syncthreads();

    v4f_mx acc[NF][MF];
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i) acc[j][i] = (v4f_mx){0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](Step& s, int st) __attribute__((always_inline)) {
        if constexpr (FUSE) load_a(s, st);
        const int blk = st * 4 + g, bw = min(blk, nb - 1);
        int sw[NF], sa[MF];
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            sw[j] = near ? lds_ws[min(j * 16 + l16, cols - 1) * nb + bw] : ws[j][bw];
            if (blk >= nb) sw[j] = 127;                    // past K: the last scale may be NaN
        }
#pragma unroll
        for (int i = 0; i < MF; ++i) {
            if constexpr (FUSE) sa[i] = lds_s[lrow[i] * srow + blk];
            else sa[i] = near ? lds_s[lrow[i] * srow + blk] : as[i][blk];
        }
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
            for (int i = 0; i < MF; ++i)
                acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(s.w[j]), mx_operand(s.a[i]), acc[j][i],
                                                                             4, 4, 0, sw[j], 0, sa[i]);
    };
    auto pair = [&](int pr, int q) __attribute__((always_inline)) {
        if (pr + 1 < last) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (2 * pr + 2 + h < steps) {
                    load_w(s[1 - q][h], 2 * pr + 2 + h);
                    if constexpr (!FUSE) load_a(s[1 - q][h], 2 * pr + 2 + h);
                }
        }
        multiply(s[q][0], 2 * pr);
        if (2 * pr + 1 < steps) multiply(s[q][1], 2 * pr + 1);
    };
    for (int pr = first; pr < last; pr += 2) {
        pair(pr, 0);
        if (pr + 1 < last) pair(pr + 1, 1);
    }

    // the waves' sums, added in wave order
    __syncthreads();                                       // no wave reads codes or scales any more
    float4* part = reinterpret_cast<float4*>(lds_few);
    constexpr int Q = NF * MF * 64;                        // groups of four columns
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i)
            part[wave * Q + (j * MF + i) * 64 + lane] = make_float4(acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]);
    __syncthreads();
    for (int q = tid; q < Q; q += THREADS) {
        float4 o = part[q];
#pragma unroll
        for (int k = 1; k < FEW_WAVES; ++k) {
            const float4 b = part[k * Q + q];
            o.x += b.x; o.y += b.y; o.z += b.z; o.w += b.w;
        }
        const int f = q >> 6, l = q & 63;
        const unsigned m = (unsigned)t.m0 + f % MF * 16 + (l & 15);
        const int n = n0 + f / MF * 16 + (l >> 4) * 4;
        if (m >= (unsigned)t.m1 || n >= p.N) continue;
        float r[4] = {o.x, o.y, o.z, o.w};
        if (p.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N) r[j] += mx_read(p.bias, p.bias_dt, (size_t)t.e * p.N + n + j);
        }
        mx_store4(p.out, p.dt, (size_t)m * p.N + n, r, min(4, p.N - n), p.N % 4 == 0);
    }
}

template <int DT, int G, int MF, int NF, bool FUSE>
static hipError_t few_go(MxProblem p, const void* x, hipStream_t st) {
    static std::atomic<bool> attr[kMaxDev];
    const long long grid = mx_row_tiles(p.R, p.E, p.offsets != nullptr, 16 * MF) * ((p.N + 16 * NF - 1) / (16 * NF));
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    const int sums = FEW_WAVES * NF * MF * 1024;
    const int rows = p.R < 16 * MF ? p.R : 16 * MF;
    const int nb = p.K / 32;
    const int held = p.K > FEW_MAX_K ? 0 : few_pad(16 * NF * nb) + few_pad(rows * (FUSE ? p.Kp / 32 : p.Ks)) + (FUSE ? rows * p.Kp / 2 : 0);
    const int lds = held > sums ? held : sums;
    int dev = 0;
    hipError_t e = current_device(&dev);
    if (e != hipSuccess) return e;
    e = lds_limit_once(attr, dev, reinterpret_cast<const void*>(&mxfp4_gemm_few_kernel<DT, G, MF, NF, FUSE>), 160 << 10);
    if (e != hipSuccess) return e;
    return launch_parts(grid, 64 * FEW_WAVES, [&](long long first, dim3 part) {
        p.block0 = (int)first;
        hipLaunchKernelGGL((mxfp4_gemm_few_kernel<DT, G, MF, NF, FUSE>), part, dim3(64 * FEW_WAVES), lds, st, p,
                           reinterpret_cast<const uint8_t*>(x));
    });
}

// Rows that each workgroup quantizes itself: few of them in a tile, so that the work is less than a launch costs, and their
// codes fit its LDS.  us, in the product and ahead of it: 5120 -> 13824 1 row 9.3 and 12.1, 2 rows 10.6 and 12.2, 4 rows
// 12.9 and 12.5, 8 rows 19.1 and 12.8; 4096 -> 4096 4 rows 6.7 and 8.1, 8 rows 9.3 and 8.3.  Experts' rows are spread over
// the tiles: 2048 -> 4096, 1 token's four 7.5 and 9.4, 2 tokens' eight 11.5 and 14.3.
bool mxfp4_gemm_fused(const MxProblem& p) {
    return p.R <= (p.offsets != nullptr ? 8 : 4) && p.K <= FEW_MAX_K && (long long)p.R * p.Kp <= (64 << 10);
}

// Its tile.  Fused: 16 rows, 32 columns where that leaves a workgroup for each CU.  Else 32 rows, 16 where one tile or an
// expert's rows on average are no more.
MxKernel mxfp4_few_kernel(const MxProblem& p) {
    if (mxfp4_gemm_fused(p)) {
        const long long tiles = mx_row_tiles(p.R, p.E, p.offsets != nullptr, 16) * ((p.N + 31) / 32);
        return {16, tiles >= 256 ? 32 : 16, 0, true};
    }
    const long long rows = p.offsets != nullptr ? 2 * ((p.R + p.E - 1LL) / p.E) : p.R;
    return {rows <= 16 ? 16 : 32, 32, 0, false};
}

template <int DT, int G>
static hipError_t fused_go(const MxProblem& p, const void* x, hipStream_t st) {
    return mxfp4_few_kernel(p).cols == 32 ? few_go<DT, G, 1, 2, true>(p, x, st) : few_go<DT, G, 1, 1, true>(p, x, st);
}

template <int DT>
static hipError_t fused_group(const MxProblem& p, const void* x, int G, hipStream_t st) {
    switch (G) {
        case 0: return fused_go<DT, 0>(p, x, st);
        case 16: return fused_go<DT, 16>(p, x, st);
        case 64: return fused_go<DT, 64>(p, x, st);
        default: return fused_go<DT, 256>(p, x, st);
    }
}

// x as it came, where mxfp4_gemm_fused says so
hipError_t mxfp4_gemm_fused_launch(const MxProblem& p, const void* x, int G, hipStream_t st) {
    switch (p.dt) {
        case DT_F32: return fused_group<DT_F32>(p, x, G, st);
        case DT_BF16: return fused_group<DT_BF16>(p, x, G, st);
        default: return fused_group<DT_F16>(p, x, G, st);
    }
}

// x quantized with scales in rows
hipError_t mxfp4_gemm_few_launch(const MxProblem& p, hipStream_t st) {
    return mxfp4_few_kernel(p).rows == 16 ? few_go<0, 0, 1, 2, false>(p, nullptr, st) : few_go<0, 0, 2, 2, false>(p, nullptr, st);
}

}  // namespace convrot
