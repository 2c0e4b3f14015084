// The MXFP4 product on tiles staged in LDS (mxfp4_gemm.h has the operands).
//
// A workgroup of four waves, 2 x 2, takes BM x BN = 64 FM x 64 FN outputs; a wave
// holds its 32 FM x 32 FN of them in registers and multiplies fragments of 32 rows
// by 64 k (16 bytes a lane) that it reads from LDS.  k runs in stages of 128 (64
// bytes a row), four stages deep, copied from memory by global_load_lds_dwordx4;
// a row's scale bytes come 16 at a time, for four stages.
//
// What bounds it: the copies into LDS.  An MFMA of 32 x 32 x 64 takes 32 cycles,
// so a 256 x 256 tile asks for 32 KB a stage in 1024 cycles.  That is why the tile
// is as large as the registers allow (256 of them are the sums), why four waves
// share it (a wave of 128 x 128 reads 16 KB of fragments for 16 MFMAs, half of
// LDS's rate), and why the rows need no other layout than the public one: 64 bytes
// of a row are whole sectors either way.

#include <type_traits>

#include "gemm_common.h"
#include "mxfp4_gemm.h"

namespace convrot {

typedef int v8i_mx __attribute__((ext_vector_type(8)));
typedef float v16f_mx __attribute__((ext_vector_type(16)));

template <int FM_, int FN_>
struct Staged {
    static constexpr int FM = FM_, FN = FN_;               // 32-row fragments of a wave
    static constexpr int BM = 64 * FM, BN = 64 * FN;
    static constexpr int THREADS = 256, NST = 4;
    static constexpr int STAGE = (BM + BN) * 64;           // codes of 128 k
    static constexpr int SCALES = (BM + BN) * 16;          // scale bytes of 512 k
    static constexpr int RING = NST * STAGE;
    static constexpr int LDS = RING + 2 * SCALES;
    static constexpr int L = FM + FN;                      // copies of a wave and stage (1 KB each)
    static constexpr int LB = L / 2, LA = L - LB;          // those of the first half, in phase B, and the rest
    static constexpr int NS = (L + 3) / 4;                 // copies of scales of a wave and four stages
    static constexpr int SCR = RING / 4;                   // a wave's part of the ring, for the store
};

// The stage's codes in LDS: 64 bytes a row, chunk c (32 k) of row r at 16 (4 r + (c ^ (r / 4 % 4))), so that the 16
// lanes that an LDS read serves at a time, 16 rows of one chunk, touch every bank once.
__device__ __forceinline__ uint32_t staged_off(int row, int chunk) { return row * 64 + ((chunk ^ (row >> 2 & 3)) << 4); }

template <int DT, int FM, int FN>
__global__ __launch_bounds__(256, 1) void mxfp4_gemm_staged_kernel(MxProblem p, int gm_max) {
    using S = Staged<FM, FN>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_mx[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int tiles_m = mx_tile_count<S::BM>(p), tiles_n = (p.N + S::BN - 1) / S::BN;
    if ((int)blockIdx.x >= tiles_m * tiles_n) return;
    int tm, tn;
    tile_of_block(blockIdx.x, tiles_m, tiles_n, min(gm_max, tiles_m), tm, tn);
    const MxTile t = mx_tile<S::BM>(p, tm);
    const int n0 = tn * S::BN, m0 = t.m0;
    if (t.e == p.E && p.offsets != nullptr) return mx_zero(p, m0, t.m1, n0, min(n0 + S::BN, p.N));

    const uint8_t* A = p.a;
    const uint8_t* AS = p.as;
    const uint8_t* W = p.w + ((size_t)t.e * p.N + n0) * (p.K / 2);
    const uint8_t* WS = p.wp + ((size_t)t.e * p.N + n0) * p.Ks;
    if (p.order == nullptr) {
        A += (size_t)m0 * (p.Kp / 2);
        AS += (size_t)m0 * p.Ks;
    }
    // row i of the tile's A rows (is_a), or i - BM of its W rows; rows past the edge repeat the last
    auto row_of = [&](bool is_a, int i) __attribute__((always_inline)) {
        if (!is_a) return min(i - S::BM, p.N - 1 - n0);
        const int r = min(i, t.m1 - 1 - m0);
        return p.order != nullptr ? mx_source_row(p, m0 + r) : r;
    };
    // Copy j of this wave and stage: rows 16 i .. 16 i + 15 of the tile (i = wave L + j), lane l row l / 4 and the
    // chunk that belongs at place l % 4.
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds_mx;
    const int chunk = (lane & 3) ^ (lane >> 4 & 3);
    uint32_t roff[S::L], soff[S::NS];
    const uint8_t* base[S::L];
    const uint8_t* sbase[S::NS];
    uint32_t sdst[S::NS];
#pragma unroll
    for (int j = 0; j < S::L; ++j) {
        const int i = wave * S::L + j;
        const bool is_a = i * 16 < S::BM;
        base[j] = is_a ? A : W;
        roff[j] = (uint32_t)row_of(is_a, i * 16 + (lane >> 2)) * (uint32_t)((is_a ? p.Kp : p.K) / 2);
    }
#pragma unroll
    for (int j = 0; j < S::NS; ++j) {
        const int i = min(wave * S::NS + j, S::L - 1);     // past the last: the last again
        const bool is_a = i * 64 < S::BM;
        sbase[j] = is_a ? AS : WS;
        soff[j] = (uint32_t)row_of(is_a, i * 64 + lane) * (uint32_t)p.Ks;
        sdst[j] = lds0 + S::RING + i * 1024;
    }
    const int nst = p.Kp / 128;
    const uint32_t last_w = p.K / 2 - 16;                  // a chunk past a row of W: its last one (the codes of A are 0)
    auto dma_codes = [&](int st, int j) __attribute__((always_inline)) {
        const uint32_t k = st * 64 + chunk * 16;
        const int i = wave * S::L + j;
        dma16_sv(lds0 + (st % S::NST) * S::STAGE + i * 1024, base[j], roff[j] + (i * 16 < S::BM ? k : min(k, last_w)));
    };
    auto dma_scales = [&](int ss) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < S::NS; ++j) dma16_sv(sdst[j] + (ss & 1) * S::SCALES, sbase[j], soff[j] + ss * 16);
    };

    v16f_mx acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (v16f_mx){0};

    // Fragment reads: k step s (64 k) of a stage takes chunks s (lanes 0..31) and 2 + s (lanes 32..63), so a lane's two
    // scale bytes of a stage are neighbours, and the MFMA of step s takes byte s of them.
    const int l32 = lane & 31, half = lane >> 5;
    const int ra = wm * 32 * FM + l32, rb = S::BM + wn * 32 * FN + l32;
    uint32_t offa[2], offb[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        offa[s] = staged_off(ra, 2 * half + s);
        offb[s] = staged_off(rb, 2 * half + s);
    }
    const uint32_t offsa = S::RING + ra * 16 + 2 * half, offsb = S::RING + rb * 16 + 2 * half;
    struct Frags { v4u_mx a[FM], b[FN]; };
    struct Scales { int a[FM], b[FN]; };
    Frags F[2];
    Scales C[2];
    auto read_frag = [&](Frags& f, uint32_t st, int s, int r) __attribute__((always_inline)) {
        if (r < FN) f.b[r] = *reinterpret_cast<const v4u_mx*>(lds_mx + st + offb[s] + r * 2048);
        else f.a[r - FN] = *reinterpret_cast<const v4u_mx*>(lds_mx + st + offa[s] + (r - FN) * 2048);
    };
    auto read_scale = [&](Scales& c, uint32_t at, int r) __attribute__((always_inline)) {
        if (r < FN) c.b[r] = *reinterpret_cast<const uint16_t*>(lds_mx + at + offsb + r * 512);
        else c.a[r - FN] = *reinterpret_cast<const uint16_t*>(lds_mx + at + offsa + (r - FN) * 512);
    };
    auto mfma_one = [&](const Frags& f, const Scales& c, auto step, int x) __attribute__((always_inline)) {
        constexpr int s = decltype(step)::value;
        const int i = x / FN, j = x % FN;
        const v8i_mx a = {(int)f.a[i].x, (int)f.a[i].y, (int)f.a[i].z, (int)f.a[i].w, 0, 0, 0, 0};
        const v8i_mx b = {(int)f.b[j].x, (int)f.b[j].y, (int)f.b[j].z, (int)f.b[j].w, 0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc[i][j], 4, 4, s, c.b[j], s, c.a[i]);
    };

    // Ring: stage st sits in slot st % 4.  At stage st, phase A multiplies its first 64 k while the second 64 k's
    // fragments are read and the second half of stage st + 3 is copied; then every wave waits for its own copies of
    // stage st + 1 and passes the barrier: stage st + 1 is there, and no wave reads stage st any more.  Phase B
    // multiplies the second 64 k while the first fragments and the scales of stage st + 1 are read and the first half
    // of stage st + 4 is copied into stage st's slot.  Scales of four stages come at the first of the four before.
    dma_scales(0);
#pragma unroll
    for (int st = 0; st < 3; ++st)
        if (st < nst) {
#pragma unroll
            for (int j = 0; j < S::L; ++j) dma_codes(st, j);
        }
    if (nst >= 3) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * S::L));      // scales and stage 0 are there
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    __syncthreads();
    if (nst > 3) {
#pragma unroll
        for (int j = 0; j < S::LB; ++j) dma_codes(3, j);
    }
#pragma unroll
    for (int r = 0; r < S::L; ++r) {
        read_frag(F[0], 0, 0, r);
        read_scale(C[0], 0, r);
    }
    constexpr int X = FM * FN;                             // MFMAs of a phase
    // STEADY: stages st + 4 and below are all there
    auto stage = [&](int st, auto place, auto steady) __attribute__((always_inline)) {
        constexpr int q = decltype(place)::value;          // st % 4
        constexpr bool STEADY = decltype(steady)::value;
        constexpr uint32_t here = q * S::STAGE, next = (q + 1) % 4 * S::STAGE;
        const bool more3 = STEADY || st + 3 < nst, more4 = STEADY || st + 4 < nst;
        const uint32_t sc_next = ((q == 3 ? (st >> 2) + 1 : st >> 2) & 1) * S::SCALES + (q + 1) % 4 * 4;
        if (q == 0 && more4) dma_scales((st >> 2) + 1);
#pragma unroll
        for (int x = 0; x < X; ++x) {
            mfma_one(F[0], C[q & 1], std::integral_constant<int, 0>{}, x);
            __builtin_amdgcn_sched_barrier(0);
            if (x < S::L) read_frag(F[1], here, 1, x);
            if (more3 && x % 2 == 1 && x / 2 < S::LA) dma_codes(st + 3, S::LB + x / 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        // in flight after stage st + 1: stages st + 2 and st + 3, and the scales issued since (in this stage or the
        // one before); vmcnt counts in order of issue, 0xc07f: and no LDS read of this wave outstanding
        if (q == 1 && more3 || q == 0 && more4) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * S::L + S::NS) & 0xc07f);
        else if (more3) __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * S::L) & 0xc07f);
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0) & 0xc07f);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < X; ++x) {
            mfma_one(F[1], C[q & 1], std::integral_constant<int, 1>{}, x);
            __builtin_amdgcn_sched_barrier(0);
            if (x < S::L) {
                read_frag(F[0], next, 0, x);
                read_scale(C[(q + 1) & 1], sc_next, x);
            }
            if (more4 && x % 2 == 1 && x / 2 < S::LB) dma_codes(st + 4, x / 2);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    using T = std::true_type;
    using N = std::false_type;
    int st = 0;
    for (; st + 7 < nst; st += 4) {
        stage(st, std::integral_constant<int, 0>{}, T{});
        stage(st + 1, std::integral_constant<int, 1>{}, T{});
        stage(st + 2, std::integral_constant<int, 2>{}, T{});
        stage(st + 3, std::integral_constant<int, 3>{}, T{});
    }
    for (; st < nst; st += 4) {
        stage(st, std::integral_constant<int, 0>{}, N{});
        if (st + 1 < nst) stage(st + 1, std::integral_constant<int, 1>{}, N{});
        if (st + 2 < nst) stage(st + 2, std::integral_constant<int, 2>{}, N{});
        if (st + 3 < nst) stage(st + 3, std::integral_constant<int, 3>{}, N{});
    }
    __syncthreads();                                       // no copy in flight, no wave reads the ring

    // The store: 32 FM rows of RB bytes at a time in this wave's part of the ring, 16-byte pieces of row r at
    // (piece ^ r % pieces) against bank conflicts, and from there whole pieces of rows to memory.
    float* bias = reinterpret_cast<float*>(lds_mx + S::RING);
    for (int n = tid; n < S::BN; n += S::THREADS)
        bias[n] = p.bias != nullptr && n0 + n < p.N ? mx_read(p.bias, p.bias_dt, (size_t)t.e * p.N + n0 + n) : 0.0f;
    __syncthreads();
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    constexpr int RB = 32 * FN * ES < 256 ? 32 * FN * ES : 256;
    constexpr int CP = RB / ES, PIECES = RB / 16, ROWS = 64 / PIECES;
    static_assert(32 * FM * RB <= S::SCR, "a wave's rows fit its part of the ring");
    uint8_t* scr = lds_mx + wave * S::SCR;
    const bool vec = (p.N * ES) % 16 == 0;
#pragma unroll
    for (int pass = 0; pass < 32 * FN / CP; ++pass) {
#pragma unroll
        for (int jt = pass * (CP / 32); jt < (pass + 1) * (CP / 32); ++jt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = jt * 32 + 8 * g + 4 * half;
                const float4 b = *reinterpret_cast<const float4*>(bias + wn * 32 * FN + c);
                const int at = (c - pass * CP) * ES;
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const int row = i * 32 + l32;
                    const float v0 = acc[i][jt][4 * g] + b.x, v1 = acc[i][jt][4 * g + 1] + b.y;
                    const float v2 = acc[i][jt][4 * g + 2] + b.z, v3 = acc[i][jt][4 * g + 3] + b.w;
                    uint8_t* d = scr + row * RB + (((at >> 4) ^ (row & (PIECES - 1))) << 4) + (at & 15);
                    if constexpr (DT == DT_F32) *reinterpret_cast<float4*>(d) = make_float4(v0, v1, v2, v3);
                    else if constexpr (DT == DT_BF16)
                        *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v0, v1), pack_bf16x2(v2, v3));
                    else *reinterpret_cast<uint2*>(d) = make_uint2(pack_f16x2(v0, v1), pack_f16x2(v2, v3));
                }
            }
        wave_sync();
        const int piece = lane % PIECES;
        const int col = n0 + wn * 32 * FN + pass * CP + piece * (16 / ES);
#pragma unroll
        for (int r0 = 0; r0 < 32 * FM; r0 += ROWS) {
            const int row = r0 + lane / PIECES;
            const int m = m0 + wm * 32 * FM + row;
            const v4u_mx w = *reinterpret_cast<const v4u_mx*>(scr + row * RB + ((piece ^ (row & (PIECES - 1))) << 4));
            if (m < t.m1 && col < p.N) {
                uint8_t* o = reinterpret_cast<uint8_t*>(p.out) + ((size_t)m * p.N + col) * ES;
                if (vec) *reinterpret_cast<v4u_mx*>(o) = w;
                else {
#pragma unroll
                    for (int e = 0; e < 16 / ES; ++e)
                        if (col + e < p.N) {
                            if constexpr (DT == DT_F32) reinterpret_cast<uint32_t*>(o)[e] = w[e];
                            else reinterpret_cast<uint16_t*>(o)[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
                        }
                }
            }
        }
        wave_sync();
    }
}

// 0: not this kernel; else the wave's fragments 16 FM + FN.
static int staged_shape(const MxProblem& p) {
    if (p.R <= 64) return 0;
    // the tokens' rows are addressed by 32-bit offsets from the first
    if (p.order != nullptr && (size_t)(p.R / p.top_k) * (p.Kp / 2) >= (size_t(1) << 32)) return 0;
    const bool ragged = p.offsets != nullptr;
    auto tiles = [&](int bm, int bn) { return mx_row_tiles(p.R, p.E, ragged, bm) * ((p.N + bn - 1) / bn); };
    if (tiles(256, 256) >= 200) return 0x44;
    if (tiles(128, 256) >= 200) return 0x24;
    return 0x22;
}

bool mxfp4_gemm_staged(const MxProblem& p) { return staged_shape(p) != 0; }

template <int DT, int FM, int FN>
static hipError_t staged_go(const MxProblem& p, hipStream_t st) {
    using S = Staged<FM, FN>;
    static std::atomic<bool> attr[kMaxDev];
    int dev = 0;
    hipError_t e = current_device(&dev);
    if (e != hipSuccess) return e;
    e = lds_limit_once(attr, dev, reinterpret_cast<const void*>(&mxfp4_gemm_staged_kernel<DT, FM, FN>), S::LDS);
    if (e != hipSuccess) return e;
    const long long rows = mx_row_tiles(p.R, p.E, p.offsets != nullptr, S::BM);
    const long long grid = rows * ((p.N + S::BN - 1) / S::BN);
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL((mxfp4_gemm_staged_kernel<DT, FM, FN>), dim3((unsigned)grid), dim3(S::THREADS), S::LDS, st, p,
                       tile_group_rows((int)rows));
    return hipGetLastError();
}

template <int DT>
static hipError_t staged_type(const MxProblem& p, hipStream_t st) {
    switch (staged_shape(p)) {
        case 0x44: return staged_go<DT, 4, 4>(p, st);
        case 0x24: return staged_go<DT, 2, 4>(p, st);
        default: return staged_go<DT, 2, 2>(p, st);
    }
}

hipError_t mxfp4_gemm_staged_launch(const MxProblem& p, hipStream_t st) {
    switch (p.dt) {
        case DT_F32: return staged_type<DT_F32>(p, st);
        case DT_BF16: return staged_type<DT_BF16>(p, st);
        default: return staged_type<DT_F16>(p, st);
    }
}

}  // namespace convrot
