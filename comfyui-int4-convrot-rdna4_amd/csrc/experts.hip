// Tokens sorted by expert and back.
//
// A token t has k slots; slot t k + j goes to expert ids[t, j], or to none where
// that id is outside [0, E).  The plan is a stable counting sort of the slots:
//   order[r]      the slot of sorted row r; -1 past the last used row
//   position[s]   the sorted row of slot s; -1 for an unused one
//   offsets[e]    expert e's rows are offsets[e] .. offsets[e + 1] - 1
// Rows follow it: gathered[r] = x[order[r] / k], combined[t] = sum_j w[t, j]
// rows[position[t, j]], and their gradients.  Every sum is taken over a token's
// slots in slot order in fp32: nothing is added atomically, the same inputs give
// the same bits.

#include "mxfp4.h"

namespace convrot {

constexpr int SORT_EACH = 4;               // slots of a lane
constexpr int SORT_FEW = 4, SORT_MANY = 16;                 // waves of a workgroup: of a plan that fits them, of others
constexpr int sort_slots(int waves) { return 64 * SORT_EACH * waves; }      // slots of its run
constexpr int SORT_MAX_E = 1024;

// The experts of a wave's slots w0 + 64 i + lane (-1: none), loaded together.
template <typename ID>
__device__ __forceinline__ void experts_of(const ID* ids, long long w0, int R, int E, int (&e)[SORT_EACH]) {
    ID id[SORT_EACH];
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < SORT_EACH; ++i) {
        const long long s = w0 + 64 * i + lane;
        id[i] = s < R ? ids[s] : (ID)-1;
    }
#pragma unroll
    for (int i = 0; i < SORT_EACH; ++i) e[i] = id[i] >= 0 && id[i] < (ID)E ? (int)id[i] : -1;
}

// counts[b, e]: slots of workgroup b's run that go to expert e
template <typename ID>
__global__ __launch_bounds__(64 * SORT_MANY) void expert_count_kernel(const ID* __restrict__ ids, int* __restrict__ counts,
                                                                    int R, int E) {
    __shared__ int n[SORT_MAX_E];
    int e[SORT_EACH];
    experts_of(ids, (blockIdx.x * (long long)SORT_MANY + (threadIdx.x >> 6)) * (64 * SORT_EACH), R, E, e);
    for (int i = threadIdx.x; i < E; i += 64 * SORT_MANY) n[i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SORT_EACH; ++i)
        if (e[i] >= 0) atomicAdd(&n[e[i]], 1);             // integers: the order does not matter
    __syncthreads();
    for (int i = threadIdx.x; i < E; i += 64 * SORT_MANY) counts[(size_t)blockIdx.x * E + i] = n[i];
}

// Counts of a run -> counts of the runs before it, and behind the last run's the totals.  A workgroup takes 64
// experts, each of its waves a sixteenth of the runs, eight of them read at a time.
__global__ __launch_bounds__(1024) void expert_scan_kernel(int* __restrict__ counts, int E, int runs) {
    __shared__ int part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, x = blockIdx.x * 64 + lane;
    const int b0 = (int)((long long)runs * wave / 16), b1 = (int)((long long)runs * (wave + 1) / 16);
    int sum = 0;
    if (x < E) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) sum += counts[(size_t)b * E + x];
    }
    part[wave][lane] = sum;
    __syncthreads();
    int before = 0;
    for (int v = 0; v < wave; ++v) before += part[v][lane];
    if (x >= E) return;
    for (int b = b0; b < b1; b += 8) {
        int c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = b + i < b1 ? counts[(size_t)(b + i) * E + x] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (b + i < b1) counts[(size_t)(b + i) * E + x] = before;
            before += c[i];
        }
    }
    if (wave == 15) counts[(size_t)runs * E + x] = before;
}

// Workgroup b places its run: expert e's first row there is offsets[e] plus the
// counts of the runs before.  Each wave takes a part of the run, in order, 64
// slots at a time; the lanes that go to one expert find each other by the bits of
// its number, so that one of them counts for all, and their order is the slots'.
// A single run needs no counts from elsewhere (ONE): one launch.  Of a few runs each
// workgroup adds up the counts itself; of more than SCAN_RUNS (SCANNED) that would be the
// square of their number, and a launch between has done it.  Bound by the
// chain of loads, ballots and LDS, so a wave has few slots: 2000 slots of 32
// experts 5.3 us (7.4 with four waves of 512), 64 slots 2.7 (3.4 with sixteen waves).
template <typename ID, bool ONE, int WAVES, bool SCANNED>
__global__ __launch_bounds__(64 * WAVES) void expert_place_kernel(const ID* __restrict__ ids,
                                                                    const int* __restrict__ counts, int* __restrict__ order,
                                                                    int* __restrict__ position, int* __restrict__ offsets,
                                                                    int R, int E, int runs) {
    extern __shared__ int lds_sort[];                      // next[wave][e], then wave_sum
    int* next = lds_sort;
    int* wave_sum = lds_sort + WAVES * E;
    constexpr int THREADS = 64 * WAVES;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long long s0 = blockIdx.x * (long long)sort_slots(WAVES), w0 = s0 + wave * (64 * SORT_EACH);
    int e[SORT_EACH], rank[SORT_EACH], many[SORT_EACH];    // lanes of the same expert before this one; all, of the last
    experts_of(ids, w0, R, E, e);
    for (int i = tid; i < WAVES * E; i += THREADS) next[i] = 0;
    next += wave * E;                                      // this wave's
#pragma unroll
    for (int i = 0; i < SORT_EACH; ++i) {
        if (w0 + 64 * i >= R) break;                       // nothing past here
        unsigned long long same = __ballot(e[i] >= 0);
        for (int bit = 0; (E - 1) >> bit; ++bit) {
            const bool one = (e[i] >> bit) & 1;
            const unsigned long long m = __ballot(one);
            same &= one ? m : ~m;
        }
        rank[i] = __popcll(same & ((1ull << lane) - 1));
        many[i] = e[i] >= 0 && (same >> lane) == 1ull ? rank[i] + 1 : 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SORT_EACH; ++i) {
        if (w0 + 64 * i >= R) break;
        if (many[i]) next[e[i]] += many[i];          // one lane an expert
        wave_sync();
    }
    __syncthreads();
    int used = 0;
    for (int e0 = 0; e0 < E; e0 += THREADS) {
        const int x = e0 + tid;
        int all = 0, before = 0;                           // of all runs, and of those before this one
        int own[WAVES];                                    // of this run's waves; read together
        if (x < E) {
#pragma unroll
            for (int v = 0; v < WAVES; ++v) own[v] = lds_sort[v * E + x];
            if constexpr (ONE) {
#pragma unroll
                for (int v = 0; v < WAVES; ++v) all += own[v];
            } else if constexpr (SCANNED) {
                before = counts[(size_t)blockIdx.x * E + x];
                all = counts[(size_t)runs * E + x];
            } else {
#pragma unroll 8
                for (int b = 0; b < runs; ++b) {
                    const int c = counts[(size_t)b * E + x];
                    before += b < (int)blockIdx.x ? c : 0;
                    all += c;
                }
            }
        }
        int sum = all;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            if (lane >= d) sum += o;
        }
        if (lane == 63) wave_sum[wave] = sum;
        __syncthreads();
        int first = used + sum - all;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
            const int n = wave_sum[v];
            if (v < wave) first += n;
            used += n;
        }
        if (x < E) {
            if (blockIdx.x == 0) offsets[x] = first;
            int at = first + before;                       // each wave's first row of the expert
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                lds_sort[v * E + x] = at;
                at += own[v];
            }
        }
        __syncthreads();
    }
    if (tid == 0 && blockIdx.x == 0) offsets[E] = used;
#pragma unroll
    for (int i = 0; i < SORT_EACH; ++i) {
        if (w0 + 64 * i >= R) break;
        const long long s = w0 + 64 * i + lane;
        int row = -1;
        if (e[i] >= 0) row = next[e[i]] + rank[i];
        wave_sync();
        if (many[i]) next[e[i]] = row + 1;           // the last of them
        wave_sync();
        if (s < R) position[s] = row;
        if (row >= 0) order[row] = (int)s;
    }
    for (int i = tid; i < sort_slots(WAVES); i += THREADS)
        if (s0 + i < R && s0 + i >= used) order[s0 + i] = -1;
}

// Rows by the plan (a row number outside it is taken for an unused slot), 16
// bytes or one element of a row a thread.
template <int DT>
struct RowVec {                              // 16 bytes of a row as floats
    static constexpr int N = DT == DT_F32 ? 4 : 8;
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
};

// One piece of a row: 16 bytes (VEC) or one element, where rows are no whole number of 16 bytes.  8192 tokens of 4095
// bf16 to 4 experts so: gather 156 us, combine 191, its gradient 203; of 4096 in 16 bytes 65, 57 and 121.
template <int DT, bool VEC>
struct Piece {
    static constexpr int N = VEC ? RowVec<DT>::N : 1;
    static constexpr int ES = DT == DT_F32 ? 4 : 2;
    static __device__ __forceinline__ void load(const uint8_t* row, int i, float (&v)[N]) {
        if constexpr (VEC) RowVec<DT>::unpack(reinterpret_cast<const v4u_mx*>(row)[i], v);
        else if constexpr (DT == DT_F32) v[0] = reinterpret_cast<const float*>(row)[i];
        else {
            const uint32_t h = reinterpret_cast<const uint16_t*>(row)[i];
            v[0] = DT == DT_BF16 ? __uint_as_float(h << 16) : f16bits_to_f32(h);
        }
    }
    // Sorted rows, read for the last time where they are combined: the load does not push other data out of the caches,
    // nor wait for it to be written back.  8192 tokens' 4 rows of 4096 bf16, product and combination 254 us, so 209;
    // 4096 tokens' 123 and 117, 512 tokens' 34.3 and 34.8.  Stores of that kind only move the wait to the rows' reader.
    static __device__ __forceinline__ void load_once(const uint8_t* row, int i, float (&v)[N]) {
        if constexpr (VEC) RowVec<DT>::unpack(__builtin_nontemporal_load(reinterpret_cast<const v4u_mx*>(row) + i), v);
        else load(row, i, v);
    }
    static __device__ __forceinline__ void store(uint8_t* row, int i, const float (&v)[N]) {
        if constexpr (VEC) reinterpret_cast<v4u_mx*>(row)[i] = RowVec<DT>::pack(v);
        else if constexpr (DT == DT_F32) reinterpret_cast<float*>(row)[i] = v[0];
        else reinterpret_cast<uint16_t*>(row)[i] = (uint16_t)(DT == DT_BF16 ? pack_bf16x2(v[0], 0.0f) : pack_f16x2(v[0], 0.0f));
    }
};

// Zeros in the rows past the last used one; the workgroups of a call's first launch share them.
template <int DT, bool VEC>
__device__ __forceinline__ void zero_tail(uint8_t* rows, const int* offsets, int R, int E, int D) {
    using P = Piece<DT, VEC>;
    const float z[P::N] = {};
    for (long long r = max(offsets[E], 0) + (long long)blockIdx.x; r < R; r += gridDim.x)
        for (unsigned i = threadIdx.x; i < (unsigned)(D / P::N); i += 256) P::store(rows + (size_t)r * D * P::ES, i, z);
}

// A workgroup takes 256 pieces of one token's row; a token's slots are read four at a time, their rows together.
constexpr int ROW_SLOTS = 4;

// Rows position[t, j0 .. j0 + 3] (-1: none) and with W their weights
__device__ __forceinline__ void slots_of(const int* position, const float* w, long long t, unsigned j0, int k, int R,
                                         int (&r)[ROW_SLOTS], float (&f)[ROW_SLOTS]) {
#pragma unroll
    for (int j = 0; j < ROW_SLOTS; ++j) {
        const bool there = j0 + j < (unsigned)k;
        const int p = there ? position[t * k + j0 + j] : -1;
        r[j] = (unsigned)p < (unsigned)R ? p : -1;
        f[j] = there && w != nullptr ? w[t * k + j0 + j] : 1.0f;
    }
}

// gathered[position[t, j]] = x[t].  Bound by writing the rows: 8192 tokens of 4096
// bf16 to 4 experts each 51 us, 6.6 TB/s (66 behind a kernel whose stores are still on the way).
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void expert_gather_kernel(const uint8_t* __restrict__ x, const int* __restrict__ position,
                                                            const int* __restrict__ offsets, uint8_t* __restrict__ rows, int R,
                                                            int k, int E, int D, int parts, unsigned first) {
    using P = Piece<DT, VEC>;
    const unsigned b = first + blockIdx.x;
    const long long t = b / parts;
    const int i = (b % parts) * 256 + threadIdx.x;
    if (i < D / P::N) {
        float v[P::N];
        P::load(x + (size_t)t * D * P::ES, i, v);
        for (int j = 0; j < k; ++j) {
            const int r = position[t * k + j];
            if ((unsigned)r < (unsigned)R) P::store(rows + (size_t)r * D * P::ES, i, v);
        }
    }
    if (first == 0) zero_tail<DT, VEC>(rows, offsets, R, E, D);
}

// out[t] = sum_j w[t, j] rows[position[t, j]] (w NULL: 1).  Bound by reading the rows, which lie apart: 8192 x 4 rows of
// 4096 bf16 61 us, 5.5 TB/s (75 to 88 with loads that the caches keep).
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void expert_combine_kernel(const uint8_t* __restrict__ rows, const float* __restrict__ w,
                                                             const int* __restrict__ position, uint8_t* __restrict__ out, int R,
                                                             int k, int D, int parts, unsigned first) {
    using P = Piece<DT, VEC>;
    const unsigned b = first + blockIdx.x;
    const long long t = b / parts;
    const int i = (b % parts) * 256 + threadIdx.x;
    if (i >= D / P::N) return;
    float s[P::N] = {};
    for (unsigned j0 = 0; j0 < (unsigned)k; j0 += ROW_SLOTS) {
        int r[ROW_SLOTS];
        float f[ROW_SLOTS], v[ROW_SLOTS][P::N];
        slots_of(position, w, t, j0, k, R, r, f);
#pragma unroll
        for (int j = 0; j < ROW_SLOTS; ++j)
            if (r[j] >= 0) P::load_once(rows + (size_t)r[j] * D * P::ES, i, v[j]);
#pragma unroll
        for (int j = 0; j < ROW_SLOTS; ++j)
            if (r[j] >= 0) {
#pragma unroll
                for (int n = 0; n < P::N; ++n) s[n] = fmaf(f[j], v[j][n], s[n]);
            }
    }
    P::store(out + (size_t)t * D * P::ES, i, s);
}

// d_rows[position[t, j]] = w[t, j] d_out[t]; d_w[t, j] = <d_out[t], rows[position[t, j]]>, 0
// for an unused slot; either may be NULL.  A workgroup takes a token whole: the
// products of a slot are added over its threads in a fixed order.  Bound by memory,
// each row read and written once: 8192 x 4 rows of 4096 bf16 118 us, 5.1 TB/s, the
// rate of a copy (a slot at a time 10% more).
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void expert_combine_grad_kernel(
        const uint8_t* __restrict__ rows, const float* __restrict__ w, const int* __restrict__ position,
        const int* __restrict__ offsets, const uint8_t* __restrict__ d_out, uint8_t* __restrict__ d_rows,
        float* __restrict__ d_w, int R, int k, int E, int D, unsigned first) {
    using P = Piece<DT, VEC>;
    __shared__ float part[4][ROW_SLOTS];
    const long long t = first + blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (unsigned j0 = 0; j0 < (unsigned)k; j0 += ROW_SLOTS) {
        int r[ROW_SLOTS];
        float f[ROW_SLOTS], dot[ROW_SLOTS] = {};
        slots_of(position, w, t, j0, k, R, r, f);
        for (unsigned i = threadIdx.x; i < (unsigned)(D / P::N); i += 256) {
            float g[P::N], v[ROW_SLOTS][P::N];
            P::load(d_out + (size_t)t * D * P::ES, i, g);
            if (d_w != nullptr) {
#pragma unroll
                for (int j = 0; j < ROW_SLOTS; ++j)
                    if (r[j] >= 0) P::load_once(rows + (size_t)r[j] * D * P::ES, i, v[j]);
            }
#pragma unroll
            for (int j = 0; j < ROW_SLOTS; ++j) {
                if (r[j] < 0) continue;
                float d[P::N];
#pragma unroll
                for (int n = 0; n < P::N; ++n) {
                    if (d_w != nullptr) dot[j] = fmaf(v[j][n], g[n], dot[j]);
                    d[n] = f[j] * g[n];
                }
                if (d_rows != nullptr) P::store(d_rows + (size_t)r[j] * D * P::ES, i, d);
            }
        }
        if (d_w == nullptr) continue;
#pragma unroll
        for (int j = 0; j < ROW_SLOTS; ++j) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) dot[j] += __shfl_xor(dot[j], d);
            if (lane == 0) part[wave][j] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < ROW_SLOTS && j0 + threadIdx.x < (unsigned)k)
            d_w[t * k + j0 + threadIdx.x] = (part[0][threadIdx.x] + part[1][threadIdx.x]) +
                                            (part[2][threadIdx.x] + part[3][threadIdx.x]);
        __syncthreads();
    }
    if (first == 0 && d_rows != nullptr) zero_tail<DT, VEC>(d_rows, offsets, R, E, D);
}

int expert_max() { return SORT_MAX_E; }

static int sort_runs(int R) {
    return R <= sort_slots(SORT_FEW) ? 1 : (int)((R + (long long)sort_slots(SORT_MANY) - 1) / sort_slots(SORT_MANY));
}

// counts of every run, and the totals
size_t expert_sort_bytes(int R, int E) { return ((size_t)sort_runs(R) + 1) * E * sizeof(int); }

// Runs whose counts each placing workgroup adds up itself.  us, itself and after the launch between, 32 experts: 16 runs
// 9.9 and 11.8, 64 runs 11.7 and 12.8, 128 runs 14.4 and 13.0, 512 runs 46.5 and 25.3; 1000 experts: 64 runs 16.1 and 16.6.
constexpr int SCAN_RUNS = 64;

template <typename ID, bool ONE, int WAVES, bool SCANNED>
static hipError_t place_go(const ID* ids, const int* counts, int* order, int* position, int* offsets, int R, int E, int runs,
                           hipStream_t st) {
    static std::atomic<bool> attr[kMaxDev];
    constexpr int MOST = WAVES * (SORT_MAX_E + 1) * (int)sizeof(int);
    int dev = 0;
    hipError_t e = current_device(&dev);
    if (e != hipSuccess) return e;
    e = lds_limit_once(attr, dev, reinterpret_cast<const void*>(&expert_place_kernel<ID, ONE, WAVES, SCANNED>), MOST);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((expert_place_kernel<ID, ONE, WAVES, SCANNED>), dim3(runs), dim3(64 * WAVES), WAVES * (E + 1) * sizeof(int), st,
                       ids, counts, order, position, offsets, R, E, runs);
    return hipGetLastError();
}

template <typename ID>
static hipError_t sort_go(const void* ids, int* order, int* position, int* offsets, int* counts, int R, int E, hipStream_t st) {
    const int runs = sort_runs(R);
    const ID* p = reinterpret_cast<const ID*>(ids);
    if (R <= sort_slots(SORT_FEW)) return place_go<ID, true, SORT_FEW, false>(p, counts, order, position, offsets, R, E, runs, st);
    if (runs == 1) return place_go<ID, true, SORT_MANY, false>(p, counts, order, position, offsets, R, E, runs, st);
    hipLaunchKernelGGL((expert_count_kernel<ID>), dim3(runs), dim3(64 * SORT_MANY), 0, st, p, counts, R, E);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (runs <= SCAN_RUNS) return place_go<ID, false, SORT_MANY, false>(p, counts, order, position, offsets, R, E, runs, st);
    hipLaunchKernelGGL(expert_scan_kernel, dim3((E + 63) / 64), dim3(1024), 0, st, counts, E, runs);
    e = hipGetLastError();
    return e != hipSuccess ? e : place_go<ID, false, SORT_MANY, true>(p, counts, order, position, offsets, R, E, runs, st);
}

hipError_t expert_sort_launch(const void* ids, int id_bytes, int* order, int* position, int* offsets, int* counts, int R, int E,
                              hipStream_t st) {
    return id_bytes == 8 ? sort_go<long long>(ids, order, position, offsets, counts, R, E, st)
                         : sort_go<int>(ids, order, position, offsets, counts, R, E, st);
}

// f(type code, vector pieces) for the row type; vector pieces where rows are whole 16-byte pieces
template <typename F>
static hipError_t by_type(int dt, int D, F f) {
    const bool vec = D % (dt == DT_F32 ? 4 : 8) == 0;
    using std::integral_constant;
    using T = std::true_type;
    using N = std::false_type;
    if (dt == DT_F32) return vec ? f(integral_constant<int, DT_F32>{}, T{}) : f(integral_constant<int, DT_F32>{}, N{});
    if (dt == DT_BF16) return vec ? f(integral_constant<int, DT_BF16>{}, T{}) : f(integral_constant<int, DT_BF16>{}, N{});
    return vec ? f(integral_constant<int, DT_F16>{}, T{}) : f(integral_constant<int, DT_F16>{}, N{});
}

// workgroups of 256 pieces that a row takes
template <int DT, bool VEC>
static long long row_parts(int D) { return (D / Piece<DT, VEC>::N + 255LL) / 256; }

hipError_t expert_gather_launch(const void* x, int dt, const int* position, const int* offsets, void* rows, int T, int k, int E,
                                int D, hipStream_t st) {
    return by_type(dt, D, [&](auto d, auto v) {
        constexpr int DT = decltype(d)::value;
        constexpr bool VEC = decltype(v)::value;
        const long long parts = row_parts<DT, VEC>(D);
        if (T * parts > 0xffffffffLL) return hipErrorInvalidValue;
        return launch_parts(T * parts, 256, [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((expert_gather_kernel<DT, VEC>), grid, dim3(256), 0, st, reinterpret_cast<const uint8_t*>(x),
                               position, offsets, reinterpret_cast<uint8_t*>(rows), T * k, k, E, D, (int)parts, (unsigned)first);
        });
    });
}

hipError_t expert_combine_launch(const void* rows, int dt, const float* w, const int* position, void* out, int T, int k, int D,
                                 hipStream_t st) {
    return by_type(dt, D, [&](auto d, auto v) {
        constexpr int DT = decltype(d)::value;
        constexpr bool VEC = decltype(v)::value;
        const long long parts = row_parts<DT, VEC>(D);
        if (T * parts > 0xffffffffLL) return hipErrorInvalidValue;
        return launch_parts(T * parts, 256, [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((expert_combine_kernel<DT, VEC>), grid, dim3(256), 0, st, reinterpret_cast<const uint8_t*>(rows), w,
                               position, reinterpret_cast<uint8_t*>(out), T * k, k, D, (int)parts, (unsigned)first);
        });
    });
}

hipError_t expert_combine_grad_launch(const void* rows, int dt, const float* w, const int* position, const int* offsets,
                                      const void* d_out, void* d_rows, float* d_w, int T, int k, int E, int D, hipStream_t st) {
    return by_type(dt, D, [&](auto d, auto v) {
        return launch_parts(T, 256, [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((expert_combine_grad_kernel<decltype(d)::value, decltype(v)::value>), grid, dim3(256), 0, st,
                               reinterpret_cast<const uint8_t*>(rows), w, position, offsets,
                               reinterpret_cast<const uint8_t*>(d_out), reinterpret_cast<uint8_t*>(d_rows), d_w, T * k, k, E, D,
                               (unsigned)first);
        });
    });
}

}  // namespace convrot
