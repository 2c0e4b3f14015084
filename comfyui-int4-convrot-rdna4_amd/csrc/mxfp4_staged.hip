// The MXFP4 product on tiles staged in LDS (mxfp4_gemm.h has the operands).
//
// A workgroup of four waves, 2 x 2, takes BM x BN = 64 FM x 64 FN outputs; a wave
// holds its 32 FM x 32 FN of them in registers and multiplies fragments of 32 rows
// by 64 k (16 bytes a lane) that it reads from LDS.  k runs in stages of 256, 128
// bytes a row, in two slots, copied from memory by global_load_lds_dwordx4.
//
// What bounds it: the copies into LDS.  An MFMA of 32 x 32 x 64 takes 32 cycles,
// so a 256 x 256 tile asks for 64 KB a stage in 2048 cycles.  That is why the tile
// is as large as the registers allow (256 of them are the sums), why four waves
// share it (a wave of 128 x 128 reads 32 KB of fragments for 64 MFMAs, half of
// LDS's rate), why a stage takes whole 128-byte lines of the rows (64 bytes a row
// and stage cost twice the requests to L2, 16-byte pieces of the scales' rows a
// quarter more: 8192^3 316 us with both), and why the scales are laid out by
// columns of 512 k first.
//
// Measured on MI355X: 8192 x 5120 -> 13824 279 us in the kernel, 4.2 PFLOP/s; a
// stage takes 2570 cycles, a tile 15000 more to set up (1800), fill (2600) and store
// (11000), at 1.7 GHz, the clock that the card holds under this load.  A
// workgroup that went from tile to tile, copying the next one's first stage while
// it stored, measured slower: loads and stores share one counter, so the next
// tile's first wait is for the stores too.

#include <type_traits>

#include "gemm_common.h"
#include "mxfp4_gemm.h"

namespace convrot {

typedef int v8i_mx __attribute__((ext_vector_type(8)));
typedef float v16f_mx __attribute__((ext_vector_type(16)));

template <int FM_, int FN_, int SLOTS_>
struct Staged {
    static constexpr int FM = FM_, FN = FN_;               // 32-row fragments of a wave
    static constexpr int SLOTS = SLOTS_;                   // stages in LDS: 2 or 4
    static constexpr int BM = 64 * FM, BN = 64 * FN;
    static constexpr int THREADS = 256;
    static constexpr int STAGE = (BM + BN) * 128;          // codes of 256 k
    static constexpr int SCALES = (BM + BN) * 16;          // scale bytes of 512 k
    static constexpr int RING = SLOTS * STAGE;
    static constexpr int LDS = RING + SLOTS * SCALES;      // scales of two stages each: what is read and what is copied
    static constexpr int L = 2 * (FM + FN);                // copies of a wave and stage (1 KB each)
    static constexpr int D3 = (L + 2) / 3, D0 = D3, D1 = L - D3 - D0;   // issued in phase 3 of a stage, 0 and 1 of the next
    static constexpr int NS = (FM + FN + 3) / 4;           // copies of scales of a wave and 512 k
};

// The stage's codes in LDS: 128 bytes a row, chunk c (32 k) of row r at 16 (8 r + (c ^ (r / 2 % 8))), so that the 16
// lanes that an LDS read serves at a time, 16 rows of one chunk, touch every bank once.  The scales' words are not placed
// so: their rows lie 16 bytes apart, and a read of them takes 8 cycles instead of 2.  Of a 256 x 256 tile's wave and stage
// that is 48 of 192 cycles of LDS (by the counters, all of its bank conflicts), of 2570 for the stage.
__device__ __forceinline__ uint32_t staged_off(int row, int chunk) { return row * 128 + ((chunk ^ (row >> 1 & 7)) << 4); }

template <int DT, int FM, int FN, int SLOTS>
__global__ __launch_bounds__(256, 1) void mxfp4_gemm_staged_kernel(MxProblem p, int gm_max) {
    using S = Staged<FM, FN, SLOTS>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_mx[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int tiles_m = mx_tile_count<S::BM>(p), tiles_n = (p.N + S::BN - 1) / S::BN;
    const int block = p.block0 + (int)blockIdx.x;
    if (block >= tiles_m * tiles_n) return;

    // Copy j of this wave and stage: rows 8 i .. 8 i + 7 of the tile (i = wave L + j; the A rows, then the W rows),
    // lane l row l / 8 and the chunk that belongs at place l % 8.
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds_mx;
    const int chunk = (lane & 7) ^ (lane >> 4);            // of an even i; an odd one's is chunk ^ 4
    const int nst = (p.K + 255) / 256;
    // a chunk past a row: its last one (past K the codes of A are 0)
    const uint32_t last_a = p.Kp / 2 - 16, last_w = p.K / 2 - 16;
    const size_t a_step = (size_t)p.as_rows * 16, w_step = (size_t)p.N * 16;      // scales: from 512 k to the next
    // whether copy j is of A: the same for all of a wave's where A's rows are whole waves'
    auto is_a = [&](int j) __attribute__((always_inline)) {
        return (wave * S::L + ((S::BM / 8) % S::L == 0 ? 0 : j)) * 8 < S::BM;
    };
    int tm, tn;
    tile_of_block(block, tiles_m, tiles_n, min(gm_max, tiles_m), tm, tn);
    const MxTile t = mx_tile<S::BM>(p, tm);
    const int n0 = tn * S::BN;
    if (t.e == p.E && p.offsets != nullptr) return mx_zero(p, t.m0, t.m1, n0, min(n0 + S::BN, p.N));
    const uint8_t* A = p.a;
    const uint8_t* AS = p.as;
    const uint8_t* W = p.w + ((size_t)t.e * p.N + n0) * (p.K / 2);
    const uint8_t* WS = p.wp + ((size_t)t.e * (p.Ks / 16) * p.N + n0) * 16;
    if (p.order == nullptr) {
        A += (size_t)t.m0 * (p.Kp / 2);
        AS += (size_t)t.m0 * 16;
    }
    uint32_t roff[S::L], soff[S::NS];
    {
        // rows past the edge repeat the last
        const int last_m = t.m1 - 1 - t.m0, last_n = p.N - 1 - n0;
        int row[S::L + S::NS];
#pragma unroll
        for (int j = 0; j < S::L; ++j) {
            const int i = (wave * S::L + j) * 8 + (lane >> 3);
            row[j] = is_a(j) ? min(i, last_m) : min(i - S::BM, last_n);
        }
#pragma unroll
        for (int j = 0; j < S::NS; ++j) {
            const int i = min(wave * S::NS + j, FM + FN - 1);            // past the last: the last again
            row[S::L + j] = i < FM ? min(i * 64 + lane, last_m) : min(i * 64 + lane - S::BM, last_n);
        }
        if (p.order != nullptr) {
#pragma unroll
            for (int j = 0; j < S::L + S::NS; ++j)
                if (j < S::L ? is_a(j) : wave * S::NS + j - S::L < FM) row[j] = mx_source_row(p, t.m0 + row[j]);
        }
#pragma unroll
        for (int j = 0; j < S::L; ++j) roff[j] = (uint32_t)row[j] * (uint32_t)((is_a(j) ? p.Kp : p.K) / 2);
#pragma unroll
        for (int j = 0; j < S::NS; ++j) soff[j] = (uint32_t)row[S::L + j] * 16u;
    }
    float bias = 0.0f;                                     // of column n0 + tid
    if (p.bias != nullptr) bias = mx_read(p.bias, p.bias_dt, (size_t)t.e * p.N + min(n0 + min(tid, S::BN - 1), p.N - 1));
    auto dma_codes = [&](int st, int slot, int j) __attribute__((always_inline)) {
        const uint32_t k = st * 128 + (j & 1 ? chunk ^ 4 : chunk) * 16;
        dma16_sv(lds0 + slot * S::STAGE + (wave * S::L + j) * 1024, is_a(j) ? A : W,
                 roff[j] + min(k, is_a(j) ? last_a : last_w));
    };
    auto dma_scales = [&](int ss) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < S::NS; ++j) {
            const int i = min(wave * S::NS + j, FM + FN - 1);
            dma16_sv(lds0 + S::RING + ss % SLOTS * S::SCALES + i * 1024,
                     i < FM ? AS + ss * a_step : WS + ss * w_step, soff[j]);
        }
    };
    v16f_mx acc[FM][FN];
    // Fragment reads: k step s (64 k) of a stage is chunks 2 s (lanes 0..31) and 2 s + 1 (lanes 32..63); a lane's four
    // scale bytes of a stage are one word, byte s for step s (mx_scale_place).
    const int l32 = lane & 31, half = lane >> 5;
    const int ra = wm * 32 * FM + l32, rb = S::BM + wn * 32 * FN + l32;
    uint32_t offa[4], offb[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        offa[s] = staged_off(ra, 2 * s + half);
        offb[s] = staged_off(rb, 2 * s + half);
    }
    const uint32_t offsa = S::RING + ra * 16 + 4 * half, offsb = S::RING + rb * 16 + 4 * half;
    struct Frags { v4u_mx a[FM], b[FN]; };
    struct Scales { int a[FM], b[FN]; };
    Frags F[2];
    Scales C[2];
    constexpr int X = FM * FN, Y = FM + FN;                // MFMAs and fragments of a phase
    auto read_frag = [&](Frags& f, uint32_t slot, int s, int r) __attribute__((always_inline)) {
        if (r < FN) f.b[r] = *reinterpret_cast<const v4u_mx*>(lds_mx + slot + offb[s] + r * 4096);
        else f.a[r - FN] = *reinterpret_cast<const v4u_mx*>(lds_mx + slot + offa[s] + (r - FN) * 4096);
    };
    auto read_scale = [&](Scales& c, uint32_t at, int r) __attribute__((always_inline)) {
        if (r < FN) c.b[r] = *reinterpret_cast<const int*>(lds_mx + at + offsb + r * 512);
        else c.a[r - FN] = *reinterpret_cast<const int*>(lds_mx + at + offsa + (r - FN) * 512);
    };
    auto mfma_one = [&](const Frags& f, const Scales& c, auto step, auto zero, int x) __attribute__((always_inline)) {
        constexpr int s = decltype(step)::value;
        const int i = x / FN, j = x % FN;
        const v8i_mx a = {(int)f.a[i].x, (int)f.a[i].y, (int)f.a[i].z, (int)f.a[i].w, 0, 0, 0, 0};
        const v8i_mx b = {(int)f.b[j].x, (int)f.b[j].y, (int)f.b[j].z, (int)f.b[j].w, 0, 0, 0, 0};
        if constexpr (decltype(zero)::value)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, (v16f_mx){0}, 4, 4, s, c.b[j], s, c.a[i]);
        else
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc[i][j], 4, 4, s, c.b[j], s, c.a[i]);
    };
    using T = std::true_type;
    using N = std::false_type;

    // Stage st sits in slot st % SLOTS.  A stage is four phases of 64 k; while phase s multiplies, the fragments of the
    // next one are read.  Before phase 3 every wave waits for its copies of stage st + 1 and for its reads of stage st,
    // and passes the barrier: stage st + 1 is there, and no wave reads stage st's slot any more.  Stage st + SLOTS is
    // copied into it in phase 3 and in phases 0 and 1 of stage st + 1.  With two slots its last copies have phase 2 to
    // arrive in, which two workgroups on a CU, or the long phases of a 256 x 256 tile, hide; four slots give them two
    // stages more.  The scales of 512 k come SLOTS stages ahead.
    // STEADY: stages st + SLOTS and below are all there; START: the first stage.
    auto stage = [&](int st, auto place, auto start, auto steady) __attribute__((always_inline)) {
        constexpr int q = decltype(place)::value;          // st % SLOTS
        constexpr bool STEADY = decltype(steady)::value;
        constexpr uint32_t here = q * S::STAGE, next = (q + 1) % SLOTS * S::STAGE;
        const bool late = STEADY || st + SLOTS < nst, early = STEADY || st + SLOTS - 1 < nst;
        const uint32_t sc_next = ((st + 1) >> 1) % SLOTS * S::SCALES + ((q + 1) & 1) * 8;
        auto phase = [&](auto step, auto zero) __attribute__((always_inline)) {
            constexpr int s = decltype(step)::value;
            constexpr int n = s == 3 ? S::D3 : s == 0 ? S::D0 : s == 1 ? S::D1 : 0;      // copies of this phase
            constexpr int first = s == 3 ? 0 : s == 0 ? S::D3 : S::D3 + S::D0;
            if (s == 0 && q % 2 == 0 && late) dma_scales((st + SLOTS) >> 1);
#pragma unroll
            for (int x = 0; x < X; ++x) {
                mfma_one(F[s & 1], C[q & 1], step, zero, x);
                __builtin_amdgcn_sched_barrier(0);
                // one fragment after each MFMA while there are any, or all of them spread over fewer MFMAs
#pragma unroll
                for (int r = X < Y ? x * Y / X : x; r < (X < Y ? (x + 1) * Y / X : x < Y ? x + 1 : x); ++r) {
                    if (s < 3) read_frag(F[(s + 1) & 1], here, (s + 1) & 3, r);
                    else {
                        read_frag(F[0], next, 0, r);
                        read_scale(C[(q + 1) & 1], sc_next, r);
                    }
                }
                if (s == 3 ? late : early) {
#pragma unroll
                    for (int j = x * n / X; j < (x + 1) * n / X; ++j)
                        dma_codes(s == 3 ? st + SLOTS : st + SLOTS - 1, s == 3 ? q : (q + SLOTS - 1) % SLOTS, first + j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        phase(std::integral_constant<int, 0>{}, start);
        phase(std::integral_constant<int, 1>{}, N{});
        phase(std::integral_constant<int, 2>{}, N{});
        // vmcnt counts in order of issue.  After stage st + 1's copies came those of stages st + 2 .. st + SLOTS - 1, and
        // the scales issued in the even one of this stage and the one before.  0xc07f: no LDS read of this wave either.
        constexpr int AHEAD = (SLOTS - 2) * S::L;
        if (SLOTS > 2 && (q % 2 == 0 ? late : early))
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(AHEAD + S::NS) & 0xc07f);
        else if (SLOTS > 2 && early) __builtin_amdgcn_s_waitcnt(vmcnt_imm(AHEAD) & 0xc07f);
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0) & 0xc07f);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        phase(std::integral_constant<int, 3>{}, N{});
    };

    // LDS traffic of this wave done, and every wave here (vmcnt as it is: copies and stores stay in flight)
    auto lds_barrier = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    // The store goes through the ring, a quarter a wave, in pieces of 32 rows by RB bytes, one after the other: while a
    // piece's stores drain the next one is converted (all pieces at once: 8192 x 5120 -> 13824 315 us, so 309).
    constexpr int RB = 32 * FN * ES < 256 ? 32 * FN * ES : 256, CP = RB / ES, GROUPS = 32 * FN / CP, PIECES = FM * GROUPS;
    constexpr int SCR = 32 * RB, U = RB / 16, ROWS = 64 / U;       // 16-byte units of a row, rows of a wave's store
    static_assert(4 * SCR <= S::RING, "a piece a wave fits the ring");

#pragma unroll
    for (int ss = 0; ss < SLOTS / 2; ++ss)
        if (2 * ss < nst) dma_scales(ss);
#pragma unroll
    for (int st = 0; st < SLOTS - 1; ++st)
        if (st < nst) {
#pragma unroll
            for (int j = 0; j < S::L; ++j) dma_codes(st, st, j);
        }
    if (SLOTS - 1 < nst) {
#pragma unroll
        for (int j = 0; j < S::D3; ++j) dma_codes(SLOTS - 1, SLOTS - 1, j);
        __builtin_amdgcn_s_waitcnt(vmcnt_imm((SLOTS - 2) * S::L + S::D3));      // stage 0 and its scales are there
    } else {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    }
    lds_barrier();
#pragma unroll
    for (int r = 0; r < Y; ++r) {
        read_frag(F[0], 0, 0, r);
        read_scale(C[0], 0, r);
    }
    auto place = [](auto i) { return std::integral_constant<int, decltype(i)::value % SLOTS>{}; };
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    using I4 = std::integral_constant<int, 4>;
    stage(0, std::integral_constant<int, 0>{}, T{}, N{});
    int st = 1;
    for (; st + 2 * SLOTS - 1 < nst; st += SLOTS) {
        stage(st, place(I1{}), N{}, T{});
        stage(st + 1, place(I2{}), N{}, T{});
        if constexpr (SLOTS == 4) {
            stage(st + 2, place(I3{}), N{}, T{});
            stage(st + 3, place(I4{}), N{}, T{});
        }
    }
    for (; st < nst; st += SLOTS) {
        stage(st, place(I1{}), N{}, N{});
        if (st + 1 < nst) stage(st + 1, place(I2{}), N{}, N{});
        if constexpr (SLOTS == 4) {
            if (st + 2 < nst) stage(st + 2, place(I3{}), N{}, N{});
            if (st + 3 < nst) stage(st + 3, place(I4{}), N{}, N{});
        }
    }
    lds_barrier();                                         // no wave reads the ring or the scales any more
    float* biases = reinterpret_cast<float*>(lds_mx + S::RING);
    if (tid < S::BN) biases[tid] = bias;
    lds_barrier();
    {
        int ln = lane;                                     // not the lane's value: no address of the store waits in
        asm volatile("" : "+v"(ln));                       // registers during the main loop
        const int el = ln & 31, eh = ln >> 5, unit = ln % U, prow = ln / U;
        const unsigned m0 = (unsigned)t.m0 + wm * 32 * FM, m1 = t.m1;
        const int c0 = n0 + wn * 32 * FN;
        uint8_t* scr = lds_mx + wave * SCR;
        // piece x: columns c = x / FM, rows i = x % FM; 16-byte unit u of a row at u ^ (row % U) against bank conflicts
        auto store = [&](auto edge) __attribute__((always_inline)) {
            constexpr bool EDGE = decltype(edge)::value;
            const bool vec = (p.N * ES) % 16 == 0;
            float4 bv[CP / 8];
#pragma unroll
            for (int x = 0; x < PIECES; ++x) {
                const int c = x / FM, i = x % FM;
                if (i == 0) {
#pragma unroll
                    for (int y = 0; y < CP / 8; ++y)
                        bv[y] = *reinterpret_cast<const float4*>(biases + wn * 32 * FN + c * CP + y * 8 + 4 * eh);
                }
#pragma unroll
                for (int y = 0; y < CP / 8; ++y) {
                    const int jt = (c * CP + y * 8) / 32, g = y % 4;
                    const int at = (y * 8 + 4 * eh) * ES;
                    const float v0 = acc[i][jt][4 * g] + bv[y].x, v1 = acc[i][jt][4 * g + 1] + bv[y].y;
                    const float v2 = acc[i][jt][4 * g + 2] + bv[y].z, v3 = acc[i][jt][4 * g + 3] + bv[y].w;
                    uint8_t* d = scr + el * RB + (((at >> 4) ^ (el & (U - 1))) << 4) + (at & 15);
                    if constexpr (DT == DT_F32) *reinterpret_cast<float4*>(d) = make_float4(v0, v1, v2, v3);
                    else if constexpr (DT == DT_BF16)
                        *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v0, v1), pack_bf16x2(v2, v3));
                    else *reinterpret_cast<uint2*>(d) = make_uint2(pack_f16x2(v0, v1), pack_f16x2(v2, v3));
                }
                wave_sync();
                // a piece's units read together: one by one, each store waited for its own read
                v4u_mx w[32 / ROWS];
#pragma unroll
                for (int y = 0; y < 32 / ROWS; ++y) {
                    const int row = y * ROWS + prow;
                    w[y] = *reinterpret_cast<const v4u_mx*>(scr + row * RB + ((unit ^ (row & (U - 1))) << 4));
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 32 / ROWS; ++y) {
                    const unsigned m = m0 + i * 32 + y * ROWS + prow;
                    const int col = c0 + c * CP + unit * (16 / ES);
                    uint8_t* o = reinterpret_cast<uint8_t*>(p.out) + ((size_t)m * p.N + col) * ES;
                    // not kept in L2, where the next tiles' operands are
                    if constexpr (!EDGE) __builtin_nontemporal_store(w[y], reinterpret_cast<v4u_mx*>(o));
                    else if (m < m1 && col < p.N) {
                        if (vec) __builtin_nontemporal_store(w[y], reinterpret_cast<v4u_mx*>(o));
                        else {
#pragma unroll
                            for (int e = 0; e < 16 / ES; ++e)
                                if (col + e < p.N) {
                                    if constexpr (DT == DT_F32) reinterpret_cast<uint32_t*>(o)[e] = w[y][e];
                                    else reinterpret_cast<uint16_t*>(o)[e] = (uint16_t)(w[y][e / 2] >> (16 * (e & 1)));
                                }
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                wave_sync();
            }
        };
        if (t.m1 - t.m0 == S::BM && n0 + S::BN <= p.N && (p.N * ES) % 16 == 0) store(N{});
        else store(T{});
    }
}

// The kernel of a product: 0 the one for few rows (mxfp4_gemm.hip), else the tile's columns, 256 or 128.
//
// Up to 32 rows run there (us, there and staged: 4096 columns of K 4096 12.6 and 13.8, 2048 of K 8192 16.2 and 17.9; with
// 64 rows 16 and 14.1, 22.3 and 18).
// Tiles: rounds of the CUs times what a tile takes, fitted to K 1024 to 13824: 256 a side, one a CU, 12.5 + 1.4 us a
// stage of 256 k; 128 a side, two a CU, 3.5 + 1.15 us, three quarters of that where a CU gets one.  us, 256 and 128:
// 13824 columns of K 5120: 512 rows 38.7 and 31.6, 1024 rows 47.4 and 56.6, 1536 rows 82.2 and 78, 8192 rows 307 and 353;
// 8192 columns of K 1024: 2048 rows 23.5 and 23.9, 8192 rows 86 and 74; 8 experts, 4096 columns of K 4096: 1024 rows 40
// and 31, 2048 rows 43.5 and 47.4, 16384 rows 202 and 214.
int mxfp4_gemm_tile(const MxProblem& p) {
    const bool ragged = p.offsets != nullptr;
    if (p.R <= 32) return 0;
    // the tokens' rows are addressed by 32-bit offsets from the first
    if (p.order != nullptr && (size_t)p.as_rows * (p.Kp / 2) >= (size_t(1) << 32)) return 0;
    auto tiles = [&](int side) {                           // half a tile more for each expert that has rows
        const double rows = ragged ? (double)p.R / side + 0.5 * (p.E < p.R ? p.E : p.R) : (double)((p.R + (side - 1LL)) / side);
        return (long long)(rows * ((p.N + side - 1) / side) + 0.5);
    };
    const double stages = (p.K + 255) / 256;
    const long long t128 = tiles(128), rest = t128 % 512;
    const double rounds128 = (double)(t128 / 512) + (rest == 0 ? 0.0 : rest <= 256 ? 0.75 : 1.0);
    return (tiles(256) + 255) / 256 * (12.5 + 1.4 * stages) < rounds128 * (3.5 + 1.15 * stages) ? 256 : 128;
}

bool mxfp4_gemm_staged(const MxProblem& p) { return mxfp4_gemm_tile(p) != 0; }

template <int DT, int FM, int FN, int SLOTS>
static hipError_t staged_go(MxProblem p, hipStream_t st) {
    using S = Staged<FM, FN, SLOTS>;
    static std::atomic<bool> attr[kMaxDev];
    int dev = 0;
    hipError_t e = current_device(&dev);
    if (e != hipSuccess) return e;
    e = lds_limit_once(attr, dev, reinterpret_cast<const void*>(&mxfp4_gemm_staged_kernel<DT, FM, FN, SLOTS>), S::LDS);
    if (e != hipSuccess) return e;
    const long long rows = mx_row_tiles(p.R, p.E, p.offsets != nullptr, S::BM);
    const long long grid = rows * ((p.N + S::BN - 1) / S::BN);
    if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
    return launch_parts(grid, S::THREADS, [&](long long first, dim3 part) {
        p.block0 = (int)first;
        hipLaunchKernelGGL((mxfp4_gemm_staged_kernel<DT, FM, FN, SLOTS>), part, dim3(S::THREADS), S::LDS, st, p,
                           tile_group_rows((int)rows));
    });
}

// The instance that a staged product runs.
MxKernel mxfp4_staged_kernel(const MxProblem& p) {
    if (mxfp4_gemm_tile(p) == 256) return {256, 256, 2, false};
    // One tile a CU or fewer: nothing but its own copies hides a stage's latency, so four slots; and where that leaves half
    // of the CUs idle, tiles of half the rows (256 rows of K 4096 -> 4096: two slots 18, four 17, half the rows 15.1 us).
    const long long tiles = mx_row_tiles(p.R, p.E, p.offsets != nullptr, 128) * ((p.N + 127) / 128);
    if (tiles <= 128) return {64, 128, 4, false};
    return {128, 128, tiles <= 256 ? 4 : 2, false};
}

template <int DT>
static hipError_t staged_type(const MxProblem& p, hipStream_t st) {
    const MxKernel k = mxfp4_staged_kernel(p);
    if (k.rows == 256) return staged_go<DT, 4, 4, 2>(p, st);
    if (k.rows == 64) return staged_go<DT, 1, 2, 4>(p, st);
    return k.slots == 4 ? staged_go<DT, 2, 2, 4>(p, st) : staged_go<DT, 2, 2, 2>(p, st);
}

hipError_t mxfp4_gemm_staged_launch(const MxProblem& p, hipStream_t st) {
    switch (p.dt) {
        case DT_F32: return staged_type<DT_F32>(p, st);
        case DT_BF16: return staged_type<DT_BF16>(p, st);
        default: return staged_type<DT_F16>(p, st);
    }
}

}  // namespace convrot
