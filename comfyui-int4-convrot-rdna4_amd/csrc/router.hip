// A router's choice: the experts of each token and their weights.
//
// For a token's logits l[0 .. E - 1] and a bias b (none: 0):
//   s = softmax(l) or 1 / (1 + exp(-l)),  c = s + b
//   groups of E / groups experts are ranked by their greatest c, or the sum of their two greatest; the experts
//   outside the top_groups greatest groups are left out
//   ids = the k experts of the greatest c, greatest first; w = s[ids] (renormalized: over their sum) times `scale`
// An expert whose logit or bias is -inf is not available; a slot that finds none has id -1 and weight 0.
//
// The order is decided in 64 bits: c is cut to 43 bits (past the range to whole 2^-1064), far below what 32-bit scores could
// tell apart, and equal ones go to the lowest index.  Without a bias the order is the logits' own, since scores rise with them; scores
// then rank groups by their sums at most.  A key
// holds both: the low ten bits of a double give way to the index (1023 - e, or e where c is negative, so that of
// equal values the lowest index is the greatest key).  Keys are finite and differ, and the greater and the smaller of
// two are one instruction each, where a pair of value and index would take five.
//
// The work is a token's own and small, so what counts is the length of its chain and the instructions of all tokens:
// L lanes share a token, each with P experts in registers; a lane sorts its keys down to the k greatest, and two
// lanes' sorted lists merge to one in log2(2 k) steps, log2(L) times over.

#include "lanes.h"
#include "router.h"

namespace convrot {

constexpr int RT_MAX_E = 1024;                         // indexes in ten bits
constexpr double RT_NONE = -0x1.fffffffffffffp1023;    // the choice and the key of an expert that is not available
constexpr double RT_MOST = 0x1p1022;                   // the choice of one that is +inf or NaN
// Sums that are equal but for their last bits are often round numbers, the two scores of x and -x for one, which lie where
// the cut parts values: a step of 2^-44 puts them between a quarter and a half into what the 43 bits keep together.
constexpr double RT_ASIDE = 1.0 + 0x1p-44;
constexpr int RT_THREADS = 256;
// Logits of a call that takes 4 experts a lane (us, 4 and 16 a lane): 1 x 256 in groups 4.4 and 6.2, 2048 x 256 6.5 and 6.6,
// 4096 x 256 8.9 and 6.7; 4096 x 128 5.1 and 5.6, 8192 x 128 7.1 and 5.8; 16384 x 32 3.4 and 4.6.
constexpr long long RT_FEW = 1 << 19;

// The greater and the smaller of two keys; fmax would first canonicalize each operand.  The compiler does not know what
// the instruction writes: `settle` keeps the two wait states between it and a move across lanes.
__device__ __forceinline__ double key_max(double a, double b) {
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double key_min(double a, double b) {
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
template <int N>
__device__ __forceinline__ void settle(double (&k)[N]) {
    if constexpr (N == 1) asm volatile("s_nop 1" : "+v"(k[0]));
    else if constexpr (N == 4) asm volatile("s_nop 1" : "+v"(k[0]), "+v"(k[1]), "+v"(k[2]), "+v"(k[3]));
    else {
        static_assert(N == 8 || N == 16, "lists of 1, 4, 8 or 16");
#pragma unroll
        for (int i = 0; i < N; i += 8)
            asm volatile("s_nop 1" : "+v"(k[i]), "+v"(k[i + 1]), "+v"(k[i + 2]), "+v"(k[i + 3]), "+v"(k[i + 4]), "+v"(k[i + 5]),
                         "+v"(k[i + 6]), "+v"(k[i + 7]));
    }
}

// The key of choice c (RT_NONE, or above -2^1000 and at most RT_MOST, no -0) of number e
__device__ __forceinline__ double key_of(double c, int e) {
    const uint64_t u = (uint64_t)__double_as_longlong(c);
    const uint32_t hi = (uint32_t)(u >> 32), lo = (uint32_t)u;
    const uint32_t low = (uint32_t)(1023 - e) ^ ((uint32_t)((int)hi >> 31) & 1023u);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | ((lo & ~1023u) | low)));
}
__device__ __forceinline__ bool is_none(double key) { return key < -0x1p1000; }

// The number that a key was made of; -1 where it is of no expert
__device__ __forceinline__ int key_number(double key) {
    const uint64_t u = (uint64_t)__double_as_longlong(key);
    const int low = (int)(((uint32_t)u ^ (uint32_t)((int)(u >> 32) >> 31)) & 1023u);
    return is_none(key) ? -1 : 1023 - low;
}

// The choice of a logit where the order is the logits' own: -0 counts as 0, a NaN as +inf, -inf is not available
__device__ __forceinline__ double choice_of(float l) { return key_max(key_min((double)l + 0.0, RT_MOST), RT_NONE); }

// exp(x) to 2^-46 of its value for |x| up to 200, 2^-45 up to 708, x at most 708; below -708 rounded to whole 2^-1074 besides,
// 0 from -746 on: x = n ln 2 + r, and of exp(r) on |r| <= ln(2) / 2 the polynomial of degree 10 that is 1 at 0 and meets exp at
// the ten Chebyshev points of the interval (off by 2^-50.5 at most; ln 2 in one double by 2^-55.3 a unit of n).  Sixteen instructions where
// the library's takes forty; the choice keeps 43 bits.
__device__ __forceinline__ double choice_exp(double x) {
    x = x < -746.0 ? -746.0 : x;
    const double t = __builtin_fma(x, 1.4426950408889634, 0x1.8p52);
    const double r = __builtin_fma(t - 0x1.8p52, -0.6931471805599453, x);
    double p = 0x1.28917c89a43a7p-22;
    p = __builtin_fma(p, r, 0x1.72e107c874de9p-19);
    p = __builtin_fma(p, r, 0x1.a019b9149a41cp-16);
    p = __builtin_fma(p, r, 0x1.a01994c849582p-13);
    p = __builtin_fma(p, r, 0x1.6c16c17889ef1p-10);
    p = __builtin_fma(p, r, 0x1.11111123bf154p-7);
    p = __builtin_fma(p, r, 0x1.5555555553d68p-5);
    p = __builtin_fma(p, r, 0x1.5555555550d88p-3);
    p = __builtin_fma(p, r, 0x1.0000000000001p-1);
    p = __builtin_fma(p, r, 0x1.0000000000006p+0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)(uint32_t)(uint64_t)__double_as_longlong(t));
}

// 1 / d of a finite d >= 1 to 2^-46: the instruction's approximation (to 2^-23 at least) and a Newton step
__device__ __forceinline__ double choice_rcp(double d) {
    const double r = __builtin_amdgcn_rcp(d);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

__device__ __forceinline__ float logit_at(const void* p, int dt, size_t i) {
    if (dt == DT_F32) return reinterpret_cast<const float*>(p)[i];
    const uint32_t h = reinterpret_cast<const uint16_t*>(p)[i];
    return dt == DT_BF16 ? __uint_as_float(h << 16) : f16bits_to_f32(h);
}

// Rows whose width is no multiple of 4 lie at any multiple of their element's size, which loads and stores of 8 and 16 bytes may.
typedef float f4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u2_any __attribute__((ext_vector_type(2), aligned(2)));

// Experts e0 .. e0 + P - 1 of a row, -inf past the last: 4 values at a time, of 16 bytes or 8 (where rows allow it 8 of 16),
// and the last one to three one by one.  The loads are sent out before a value is looked at, and the type is asked for once,
// not for every value (16384 x 250 in 16 bits, sigmoid and a bias, 12.2 us; 19.0 one by one).
template <int P>
__device__ __forceinline__ void load_logits(const void* row, int dt, int e0, int E, float (&l)[P]) {
    if (dt == DT_F32) {
        const float* x = reinterpret_cast<const float*>(row) + e0;
        const float none = -__builtin_inff();
#pragma unroll
        for (int p = 0; p < P; p += 4) {
            f4_any v = {none, none, none, none};
            if (e0 + p + 4 <= E) v = *reinterpret_cast<const f4_any*>(x + p);
            else if (E % 4 != 0) {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (e0 + p + i < E) v[i] = x[p + i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) l[p + i] = v[i];
        }
        return;
    }
    const uint16_t* x = reinterpret_cast<const uint16_t*>(row) + e0;
    const uint32_t none = dt == DT_BF16 ? 0xff80ff80u : 0xfc00fc00u;   // -inf twice
    uint32_t v[P / 2];
    if (P % 8 == 0 && E % 8 == 0) {
#pragma unroll
        for (int p = 0; p < P; p += 8) {
            uint4 q = make_uint4(none, none, none, none);
            if (e0 + p < E) q = *reinterpret_cast<const uint4*>(x + p);
            v[p / 2] = q.x; v[p / 2 + 1] = q.y; v[(p / 2 + 2) % (P / 2)] = q.z; v[(p / 2 + 3) % (P / 2)] = q.w;
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; p += 4) {
            u2_any q = {none, none};
            if (e0 + p + 4 <= E) q = *reinterpret_cast<const u2_any*>(x + p);
            else if (E % 4 != 0) {
                const uint32_t high = none & 0xffff0000u;
                if (e0 + p < E) q[0] = x[p] | high;
                if (e0 + p + 1 < E) q[0] = (q[0] & 0xffffu) | (uint32_t)x[p + 1] << 16;
                if (e0 + p + 2 < E) q[1] = x[p + 2] | high;
            }
            v[p / 2] = q[0]; v[p / 2 + 1] = q[1];
        }
    }
    if (dt == DT_BF16) {
#pragma unroll
        for (int p = 0; p < P; ++p) l[p] = p % 2 ? bf16hi_to_f32(v[p / 2]) : bf16lo_to_f32(v[p / 2]);
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) l[p] = f16bits_to_f32(p % 2 ? v[p / 2] >> 16 : v[p / 2]);
    }
}

// The weights' sums of a token's chosen logits.  softmax: exp(l - m); sigmoid: 1 / (1 + exp(-l)) over exp(min(m, 0)), which
// cancels where the weights are renormalized and keeps the greatest from 0.
__device__ __forceinline__ float score_over(float l, float m, bool sigmoid) {
    return sigmoid ? expf(fminf(l, 0.0f) - fminf(m, 0.0f)) / (1.0f + expf(-fabsf(l))) : expf(l - m);
}
__device__ __forceinline__ float sigmoid_of(float l) { return 1.0f / (1.0f + expf(-l)); }

// v[A .. A + N - 1], a list that rises and then falls or the other way round, sorted downwards
template <int A, int N, int K>
__device__ __forceinline__ void sort_bitonic(double (&v)[K]) {
    if constexpr (N > 1) {
#pragma unroll
        for (int i = A; i < A + N / 2; ++i) {
            const double a = v[i], b = v[i + N / 2];
            v[i] = key_max(a, b);
            v[i + N / 2] = key_min(a, b);
        }
        sort_bitonic<A, N / 2>(v);
        sort_bitonic<A + N / 2, N / 2>(v);
    }
}

// v[A .. A + N - 1] sorted downwards: halves, the second turned round, merged
template <int A, int N, int K>
__device__ __forceinline__ void sort_down(double (&v)[K]) {
    if constexpr (N > 1) {
        sort_down<A, N / 2>(v);
        sort_down<A + N / 2, N / 2>(v);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const double a = v[A + i], b = v[A + N - 1 - i];
            v[A + i] = key_max(a, b);
            v[A + N - 1 - i] = key_min(a, b);
        }
        sort_bitonic<A, N / 2>(v);
        sort_bitonic<A + N / 2, N / 2>(v);
    }
}

// The K greatest of a lane's P keys, downwards
template <int K, int P>
__device__ __forceinline__ void greatest(const double (&key)[P], double (&top)[K]) {
    if constexpr (P <= K) {
#pragma unroll
        for (int i = 0; i < K; ++i) top[i] = i < P ? key[i < P ? i : 0] : RT_NONE;
        sort_down<0, P>(top);
    } else {
        double part[K];
#pragma unroll
        for (int i = 0; i < K; ++i) top[i] = key[i];
        sort_down<0, K>(top);
#pragma unroll
        for (int q = K; q < P; q += K) {
#pragma unroll
            for (int i = 0; i < K; ++i) part[i] = key[q + i];
            sort_down<0, K>(part);
#pragma unroll
            for (int i = 0; i < K; ++i) top[i] = key_max(top[i], part[K - 1 - i]);
            sort_bitonic<0, K>(top);
        }
    }
}

// The lists of a token's L lanes made one, which each of them then has
template <int L, int D, int K>
__device__ __forceinline__ void merge_lanes(double (&top)[K]) {
    if constexpr (D < L) {
        double a[K], b[K];
        settle(top);
#pragma unroll
        for (int i = 0; i < K; ++i) neighbours<D>(top[i], a[i], b[i]);
#pragma unroll
        for (int i = 0; i < K; ++i) top[i] = key_max(a[i], b[K - 1 - i]);
        sort_bitonic<0, K>(top);
        merge_lanes<L, 2 * D>(top);
    }
}

// The greatest key of a token's L lanes
template <int L>
__device__ __forceinline__ double greatest_lanes(double key) {
    return all_lanes<L>(key, [](double a, double b) {
        double r[1] = {key_max(a, b)};
        settle(r);
        return r[0];
    });
}

// The two greatest choices of a group that `lanes` lanes share, beside each other
template <int L, int D = 1>
__device__ __forceinline__ void two_lanes(double& one, double& two, int lanes) {
    if constexpr (D < L) {
        if (D >= lanes) return;                                       // the same for every lane
        double v[1] = {one}, w[1] = {two}, a1, b1, a2, b2;
        settle(v);
        settle(w);
        neighbours<D>(v[0], a1, b1);
        neighbours<D>(w[0], a2, b2);
        one = key_max(a1, b1);
        two = key_max(key_min(a1, b1), key_max(a2, b2));
        two_lanes<L, 2 * D>(one, two, lanes);
    }
}

// c[p] of experts outside the top_groups greatest groups -> RT_NONE.  `table`: L P doubles of LDS, the token's own.
template <int L, int P>
__device__ __forceinline__ void keep_groups(double (&c)[P], const RouterArgs& a, int sub, double* table) {
    const int size = a.E / a.groups, e0 = sub * P;
    const int lanes = size / P;
    const auto score = [&](double one, double two) {
        return key_min(a.sum2 && !is_none(two) ? one + two : one, RT_MOST);
    };
    const auto above = [&](double mine) {                             // groups ranked above
        int n = 0;
#pragma unroll 4
        for (int g = 0; g < a.groups; ++g) n += table[g] > mine ? 1 : 0;
        return n;
    };
    if (size % P == 0 && (lanes & (lanes - 1)) == 0) {                // whole lanes, a power of two of them
        double one = RT_NONE, two = RT_NONE;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            two = key_max(two, key_min(one, c[p]));
            one = key_max(one, c[p]);
        }
        two_lanes<L>(one, two, lanes);
        const int g = sub / lanes;
        const double mine = key_of(score(one, two), g);
        if (g < a.groups && sub % lanes == 0) table[g] = mine;
        wave_sync();
        const bool out = above(mine) >= a.top_groups;
#pragma unroll
        for (int p = 0; p < P; ++p) c[p] = out ? RT_NONE : c[p];
        return;
    }
    // any size: a lane reads whole groups; the group's key, and then RT_NONE or not, in the place of its first expert
#pragma unroll
    for (int p = 0; p < P; ++p) table[e0 + p] = c[p];
    wave_sync();
    double mine[P];
#pragma unroll
    for (int q = 0; q < P; ++q) {
        const int g = q * L + sub;
        double one = RT_NONE, two = RT_NONE;
        if (g < a.groups) {
            for (int i = 0; i < size; ++i) {
                const double v = table[g * size + i];
                two = key_max(two, key_min(one, v));
                one = key_max(one, v);
            }
        }
        mine[q] = key_of(score(one, two), g & 1023);
    }
    wave_sync();
#pragma unroll
    for (int q = 0; q < P; ++q)
        if (q * L + sub < a.groups) table[q * L + sub] = mine[q];
    wave_sync();
    bool out[P];
#pragma unroll
    for (int q = 0; q < P; ++q) out[q] = q * L + sub < a.groups && above(mine[q]) >= a.top_groups;
    wave_sync();
#pragma unroll
    for (int q = 0; q < P; ++q)
        if (q * L + sub < a.groups) table[q * L + sub] = out[q] ? RT_NONE : 0.0;
    wave_sync();
#pragma unroll
    for (int p = 0; p < P; ++p)
        if (e0 + p < a.E && is_none(table[(e0 + p) / size])) c[p] = RT_NONE;
}

// L lanes take a token, P experts each, in order.  K: the longest list that is sorted, at least k; 0: any k, one expert
// after the other (4096 tokens' 10 of 512 7.8 us so and 6.6 with lists of 16, 16 of 1024 15.5 and 10.5).
// Few tokens are bound by the chain of one (us, graph replays on MI355X): 1 of 32 experts 2.4, 16 of 256 in groups 4.3 (18
// with a greatest key looked for k times over 16 experts a lane, and groups read from LDS); many by instructions: 16384 tokens
// of 256 experts in 8 groups with sigmoid scores and a bias 12.8 (43 so), 1360 VALU instructions a wave of four tokens,
// three quarters of the cycles; without a bias or groups 6.3.  Their logits are 8 MB, 1.6 us.
template <int L, int P, int K, bool GROUPS>
__global__ __launch_bounds__(RT_THREADS) void choose_kernel(RouterArgs a, unsigned first) {
    __shared__ int chosen_lds[K == 0 ? RT_THREADS * P : 1];           // k <= E <= L P of each token
    __shared__ double table_lds[GROUPS ? RT_THREADS * P : 1];
    const int tid = threadIdx.x, sub = tid % L, e0 = sub * P;
    const long long t = (first + (long long)blockIdx.x) * (RT_THREADS / L) + tid / L;
    if (t >= a.T) return;                                             // a token's lanes are of one wave
    const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + (size_t)t * a.E * (a.dt == DT_F32 ? 4 : 2);
    const bool by_score = a.bias != nullptr || (GROUPS && a.sum2);
    float l[P], b[P];
    load_logits(row, a.dt, e0, a.E, l);
    if (a.bias != nullptr) load_logits(a.bias, DT_F32, e0, a.E, b);
    float m = l[0];                                                   // softmax: the greatest, which the weights may need too
    if (!a.sigmoid && (by_score || !a.renormalize)) {
#pragma unroll
        for (int p = 1; p < P; ++p) m = fmaxf(m, l[p]);
        m = max_lanes<L>(m);
    }
    double c[P];
    bool spoilt = false;                                              // softmax with a NaN: no score is a number
    if (by_score) {
        if (a.sigmoid) {
            bool far = false;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const float x = l[p] < -700.0f ? 700.0f : -l[p];
                c[p] = choice_rcp(1.0 + choice_exp((double)x));
                far |= l[p] < -700.0f && l[p] != -__builtin_inff();
            }
            if (far) {                                                // 1 + exp(-l) leaves the range, exp(l) is the score
#pragma unroll
                for (int p = 0; p < P; ++p) c[p] = l[p] < -700.0f ? choice_exp((double)l[p]) : c[p];
            }
        } else {
            double sum = 0.0;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                c[p] = choice_exp((double)l[p] - (double)m);
                sum += l[p] == -__builtin_inff() ? 0.0 : c[p];
            }
            sum = sum_lanes<L>(sum);
            spoilt = sum != sum;
            const double inv = 1.0 / sum;
#pragma unroll
            for (int p = 0; p < P; ++p) c[p] *= inv;
        }
        // -inf of the logit or the bias, also beside a NaN; scores are no -0, nor is their sum with one
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const float add = l[p] == -__builtin_inff() ? l[p] : a.bias != nullptr ? b[p] : 0.0f;
            const double v = key_min((c[p] + (double)add) * RT_ASIDE, RT_MOST); // of a NaN RT_MOST
            c[p] = add == -__builtin_inff() ? RT_NONE : v;
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) c[p] = choice_of(l[p]);
    }
    if constexpr (GROUPS) {
        keep_groups<L>(c, a, sub, table_lds + tid / L * (L * P));
        if (by_score && a.bias == nullptr) {
#pragma unroll
            for (int p = 0; p < P; ++p) c[p] = is_none(c[p]) ? RT_NONE : choice_of(l[p]);
        }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) c[p] = key_of(c[p], (e0 + p) & 1023);

    // experts j = sub, sub + L, ...: from the sorted list, which every lane has, or from LDS
    constexpr int MINE = K == 0 ? 1 : (K + L - 1) / L;
    double mine[MINE];
    int* chosen = chosen_lds + (K == 0 ? tid / L * (L * P) : 0);
    if constexpr (K > 0) {
        double top[K];
        greatest<K>(c, top);
        merge_lanes<L, 1>(top);
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            mine[i] = RT_NONE;
#pragma unroll
            for (int j = i * L; j < (i + 1) * L && j < K; ++j) mine[i] = sub == j - i * L ? top[j] : mine[i];
        }
    } else {
        double last = __builtin_inf();
        for (int j = 0; j < a.k; ++j) {
            double best = RT_NONE;
#pragma unroll
            for (int p = 0; p < P; ++p) best = key_max(best, c[p] < last ? c[p] : RT_NONE);
            double v[1] = {best};
            settle(v);
            last = greatest_lanes<L>(v[0]);
            if (sub == 0) chosen[j] = key_number(last);
        }
        wave_sync();
    }
    float total = 0.0f;
    if (!a.sigmoid && !a.renormalize) {
#pragma unroll
        for (int p = 0; p < P; ++p) total += l[p] == -__builtin_inff() ? 0.0f : expf(l[p] - m);
        total = sum_lanes<L>(total);
    }
    // the weights, in 32 bits from the chosen logits
    const auto put = [&](int j, int e, float score) {
        a.ids[t * a.k + j] = e;
        a.weights[t * a.k + j] = e >= 0 ? score * a.scale : 0.0f;
    };
    const auto score_of = [&](float v) { return a.sigmoid && !a.renormalize ? sigmoid_of(v) : score_over(v, m, a.sigmoid); };
    const bool over = a.renormalize || !a.sigmoid;                    // over `total`
    if constexpr (K > 0) {
        int e[MINE];
        float v[MINE], s[MINE], top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            e[i] = i * L + sub < a.k ? key_number(mine[i]) : -1;
            v[i] = e[i] >= 0 ? logit_at(row, a.dt, e[i]) : -__builtin_inff();
            top = fmaxf(top, v[i]);
        }
        if (a.renormalize) m = max_lanes<L>(top);
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            s[i] = score_of(v[i]);
            if (a.renormalize && e[i] >= 0) total += s[i];
        }
        if (a.renormalize) total = sum_lanes<L>(total);
        if (spoilt) total = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < MINE; ++i)
            if (i * L + sub < a.k) put(i * L + sub, e[i], over ? s[i] / total : s[i]);
    } else {
        if (a.renormalize) {
            float top = -__builtin_inff();
            for (int j = sub; j < a.k; j += L)
                if (chosen[j] >= 0) top = fmaxf(top, logit_at(row, a.dt, chosen[j]));
            m = max_lanes<L>(top);
            for (int j = sub; j < a.k; j += L)
                if (chosen[j] >= 0) total += score_of(logit_at(row, a.dt, chosen[j]));
            total = sum_lanes<L>(total);
        }
        if (spoilt) total = __builtin_nanf("");
        for (int j = sub; j < a.k; j += L) {
            const float s = chosen[j] >= 0 ? score_of(logit_at(row, a.dt, chosen[j])) : 0.0f;
            put(j, chosen[j], over ? s / total : s);
        }
    }
}

// A row of E in type dt from a token's lanes, every L-th four of each
template <int L, int Q>
__device__ __forceinline__ void store_row(uint8_t* row, int dt, int sub, int E, const float (&v)[Q][4]) {
    const auto at = [&](int q) { return (q * L + sub) * 4; };
    if (dt == DT_F32) {
        float* out = reinterpret_cast<float*>(row);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (at(q) + 4 <= E) *reinterpret_cast<f4_any*>(out + at(q)) = f4_any{v[q][0], v[q][1], v[q][2], v[q][3]};
            else if (E % 4 != 0) {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (at(q) + i < E) out[at(q) + i] = v[q][i];
            }
        }
        return;
    }
    u2_any w[Q];
    if (dt == DT_BF16) {
#pragma unroll
        for (int q = 0; q < Q; ++q) w[q] = u2_any{pack_bf16x2(v[q][0], v[q][1]), pack_bf16x2(v[q][2], v[q][3])};
    } else {
#pragma unroll
        for (int q = 0; q < Q; ++q) w[q] = u2_any{pack_f16x2(v[q][0], v[q][1]), pack_f16x2(v[q][2], v[q][3])};
    }
    uint16_t* out = reinterpret_cast<uint16_t*>(row);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        if (at(q) + 4 <= E) *reinterpret_cast<u2_any*>(out + at(q)) = w[q];
        else if (E % 4 != 0) {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (at(q) + i < E) out[at(q) + i] = (uint16_t)(w[q][i / 2] >> (i % 2 * 16));
        }
    }
}

// d_logits of a token, with p the weights before `scale` and g = scale d_weights:
//   softmax        renormalized p_j (g_j - sum p g), else s_e ([e chosen] g_e - sum s g)
//   sigmoid        renormalized p_j (1 - s_j) (g_j - sum p g), else s_j (1 - s_j) g_j
// and 0 for experts that were not chosen (but for softmax as it is).  Scores are computed again from the logits.
// A lane's experts are every L-th four, so that lanes beside each other write beside each other, in LDS and in memory: 65536
// tokens of 256 experts 11.9 us (20.0 with sixteen experts in a row to a lane), where the stores and the lines that the chosen
// logits lie in are 67 MB; 16384 tokens 5.0 (8.0), of softmax as it is 8.1.
template <int L, int P, int K>
__global__ __launch_bounds__(RT_THREADS) void choose_grad_kernel(RouterGradArgs a, unsigned first) {
    __shared__ float4 d_lds[RT_THREADS * P / 4];
    const int tid = threadIdx.x, sub = tid % L;
    const long long t = (first + (long long)blockIdx.x) * (RT_THREADS / L) + tid / L;
    if (t >= a.T) return;
    float4* fours = d_lds + tid / L * (L * P / 4);
    float* d = reinterpret_cast<float*>(fours);
    const int ES = a.dt == DT_F32 ? 4 : 2;
    const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + (size_t)t * a.E * ES;
    const bool all = !a.sigmoid && !a.renormalize;                     // every logit has a gradient
    // slots j = sub, sub + L, ...; e -1: of no expert
    constexpr int MINE = K == 0 ? P : (K + L - 1) / L;
    int e[MINE];
    float v[MINE], g[MINE], s[MINE], l[P / 4][4], m = -__builtin_inff(), total = 0.0f, mean = 0.0f;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int j = i * L + sub;
        e[i] = j < a.k ? a.ids[t * a.k + j] : -1;
        g[i] = j < a.k ? a.d_weights[t * a.k + j] * a.scale : 0.0f;
    }
    if (all) {
#pragma unroll
        for (int q = 0; q < P / 4; ++q) load_logits(row, a.dt, (q * L + sub) * 4, a.E, l[q]);
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        e[i] = (unsigned)e[i] < (unsigned)a.E ? e[i] : -1;
        v[i] = e[i] >= 0 ? logit_at(row, a.dt, e[i]) : -__builtin_inff();
    }
#pragma unroll
    for (int q = 0; q < P / 4; ++q) fours[q * L + sub] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (all) {
#pragma unroll
        for (int q = 0; q < P; ++q) m = fmaxf(m, l[q / 4][q % 4]);
        m = max_lanes<L>(m);
#pragma unroll
        for (int q = 0; q < P; ++q) {
            float& x = l[q / 4][q % 4];
            x = x == -__builtin_inff() ? 0.0f : expf(x - m);           // from here on
            total += x;
        }
        total = sum_lanes<L>(total);
    } else if (a.renormalize) {
#pragma unroll
        for (int i = 0; i < MINE; ++i) m = fmaxf(m, v[i]);
        m = max_lanes<L>(m);
    }
    const bool over = all || a.renormalize;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        s[i] = e[i] < 0 ? 0.0f : over ? score_over(v[i], m, a.sigmoid) : sigmoid_of(v[i]);
        if (!all) total += s[i];
    }
    if (over) {
        if (!all) total = sum_lanes<L>(total);
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            s[i] = e[i] < 0 ? 0.0f : s[i] / total;
            mean += e[i] < 0 ? 0.0f : s[i] * g[i];
        }
        mean = sum_lanes<L>(mean);
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const float s1 = a.sigmoid ? 1.0f / (1.0f + expf(v[i])) : 1.0f;               // 1 - score
        if (e[i] >= 0) d[e[i]] = s[i] * s1 * (g[i] - (a.renormalize ? mean : 0.0f));
    }
    wave_sync();
    const float share = total == 0.0f ? 0.0f : mean / total;           // no expert: all are 0
    float out[P / 4][4];
#pragma unroll
    for (int q = 0; q < P / 4; ++q) {
        const float4 f = fours[q * L + sub];
        out[q][0] = f.x; out[q][1] = f.y; out[q][2] = f.z; out[q][3] = f.w;
    }
    if (all) {
#pragma unroll
        for (int q = 0; q < P; ++q) out[q / 4][q % 4] -= l[q / 4][q % 4] * share;
    }
    store_row<L>(reinterpret_cast<uint8_t*>(a.d_logits) + (size_t)t * a.E * ES, a.dt, sub, a.E, out);
}

// f(lanes of a token, experts of a lane): 16 experts a lane, the fewest instructions a token, where the tokens fill the
// chip so; else 4, the shortest chain.
template <typename F>
static hipError_t by_lanes(long long T, int E, F f) {
    using std::integral_constant;
    const integral_constant<int, 4> few{};
    const integral_constant<int, 16> many{};
    if (E <= 256 && T * E <= RT_FEW) {
        if (E <= 32) return f(integral_constant<int, 8>{}, few);
        if (E <= 64) return f(integral_constant<int, 16>{}, few);
        if (E <= 128) return f(integral_constant<int, 32>{}, few);
        return f(integral_constant<int, 64>{}, few);
    }
    if (E <= 32) return f(integral_constant<int, 2>{}, many);
    if (E <= 64) return f(integral_constant<int, 4>{}, many);
    if (E <= 128) return f(integral_constant<int, 8>{}, many);
    if (E <= 256) return f(integral_constant<int, 16>{}, many);
    if (E <= 512) return f(integral_constant<int, 32>{}, many);
    return f(integral_constant<int, 64>{}, many);
}

int router_max_experts() { return RT_MAX_E; }

template <int L, int P, int K>
static hipError_t choose_go(const RouterArgs& a, hipStream_t st) {
    return launch_parts((a.T * L + RT_THREADS - 1) / RT_THREADS, RT_THREADS, [&](long long first, dim3 grid) {
        if (a.groups > 1) hipLaunchKernelGGL((choose_kernel<L, P, K, true>), grid, dim3(RT_THREADS), 0, st, a, (unsigned)first);
        else hipLaunchKernelGGL((choose_kernel<L, P, K, false>), grid, dim3(RT_THREADS), 0, st, a, (unsigned)first);
    });
}

hipError_t choose_launch(const RouterArgs& a, hipStream_t st) {
    return by_lanes(a.T, a.E, [&](auto l, auto p) {
        constexpr int L = decltype(l)::value, P = decltype(p)::value;
        if (a.k <= 4) return choose_go<L, P, 4>(a, st);
        if (a.k <= 8) return choose_go<L, P, 8>(a, st);
        if (a.k <= 16) return choose_go<L, P, 16>(a, st);
        return choose_go<L, P, 0>(a, st);
    });
}

template <int L, int P, int K>
static hipError_t choose_grad_go(const RouterGradArgs& a, hipStream_t st) {
    return launch_parts((a.T * L + RT_THREADS - 1) / RT_THREADS, RT_THREADS, [&](long long first, dim3 grid) {
        hipLaunchKernelGGL((choose_grad_kernel<L, P, K>), grid, dim3(RT_THREADS), 0, st, a, (unsigned)first);
    });
}

hipError_t choose_grad_launch(const RouterGradArgs& a, hipStream_t st) {
    return by_lanes(a.T, a.E, [&](auto l, auto p) {
        constexpr int L = decltype(l)::value, P = decltype(p)::value;
        if (a.k <= 8) return choose_grad_go<L, P, 8>(a, st);
        return a.k <= 32 ? choose_grad_go<L, P, 32>(a, st) : choose_grad_go<L, P, 0>(a, st);
    });
}

}  // namespace convrot
