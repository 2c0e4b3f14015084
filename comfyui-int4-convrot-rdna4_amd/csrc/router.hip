// A router's choice: the experts of each token and their weights.
//
// For a token's logits l[0 .. E - 1] and a bias b (none: 0):
//   s = softmax(l) or 1 / (1 + exp(-l)),  c = s + b
//   groups of E / groups experts are ranked by their greatest c, or the sum of their two greatest; the experts
//   outside the top_groups greatest groups are left out
//   ids = the k experts of the greatest c, greatest first; w = s[ids] (renormalized: over their sum) times `scale`
// An expert whose logit or bias is -inf is not available; a slot that finds none has id -1 and weight 0.
//
// The order is decided in 64 bits: c is rounded to 43 bits, far below what 32-bit scores could tell apart, and equal
// ones go to the lowest index.  Without a bias the order is the logits' own, since scores rise with them.  A key
// holds both: the low ten bits of a double give way to the index (1023 - e, or e where c is negative, so that of
// equal values the lowest index is the greatest key); keys differ, and the maximum of doubles is one instruction.

#include "lanes.h"
#include "router.h"

namespace convrot {

constexpr int RT_MAX_E = 1024;                         // indexes in ten bits
constexpr double RT_NONE = -__builtin_inf();           // the key of an expert that is not available
constexpr int RT_THREADS = 256;

__device__ __forceinline__ double key_max(double a, double b) {      // keys are no NaN: without canonicalizing them
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

__device__ __forceinline__ bool ranks_above(double a, double b) { return a > b || (a != a && b == b); }    // a NaN above all

// The key of choice `c` of number e: NaN above +inf above every other value, -inf RT_NONE.
__device__ __forceinline__ double key_of(double c, int e) {
    if (c == RT_NONE) return RT_NONE;
    uint64_t u = (uint64_t)__double_as_longlong(c + 0.0);             // -0 counts as 0
    if (c != c) u = 0x7fe0000000000000ull;
    else if (c == __builtin_inf()) u = 0x7fd0000000000000ull;
    const uint64_t low = (u >> 63) ? (uint64_t)e : (uint64_t)(1023 - e);
    return __longlong_as_double((long long)((u & ~1023ull) | low));
}

// The number that a key was made of; -1 of RT_NONE
__device__ __forceinline__ int key_number(double key) {
    if (key == RT_NONE) return -1;
    const uint64_t u = (uint64_t)__double_as_longlong(key);
    const int low = (int)(u & 1023);
    return (u >> 63) ? low : 1023 - low;
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* p, size_t i) {
    if constexpr (DT == DT_F32) return reinterpret_cast<const float*>(p)[i];
    const uint32_t h = reinterpret_cast<const uint16_t*>(p)[i];
    return DT == DT_BF16 ? __uint_as_float(h << 16) : f16bits_to_f32(h);
}

// Experts e0 .. e0 + P - 1 of a row (-inf past the last).  VEC: E is a multiple of P, so they are there or not together
// and aligned to their size.
template <int DT, int P, bool VEC>
__device__ __forceinline__ void load_logits(const void* row, int e0, int E, float (&l)[P]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int p = 0; p < P; ++p) l[p] = e0 + p < E ? logit_at<DT>(row, e0 + p) : -__builtin_inff();
    } else {
        constexpr int WORDS = P * (DT == DT_F32 ? 4 : 2) / 4;
        uint32_t w[WORDS];
        const bool there = e0 < E;
        if constexpr (WORDS % 4 == 0) {
            const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row) + (size_t)e0 * (DT == DT_F32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < WORDS / 4; ++i) {
                const uint4 v = there ? q[i] : make_uint4(0u, 0u, 0u, 0u);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
        } else {
            static_assert(WORDS == 2, "four 16-bit values");
            const uint2 v = there ? *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(row) + (size_t)e0 * 2)
                                  : make_uint2(0u, 0u);
            w[0] = v.x; w[1] = v.y;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float f;
            if constexpr (DT == DT_F32) f = __uint_as_float(w[p]);
            else if constexpr (DT == DT_BF16) f = (p & 1) ? bf16hi_to_f32(w[p >> 1]) : bf16lo_to_f32(w[p >> 1]);
            else f = f16bits_to_f32((p & 1) ? w[p >> 1] >> 16 : w[p >> 1]);
            l[p] = there ? f : -__builtin_inff();
        }
    }
}

// The weights' sums of a token's chosen logits.  softmax: exp(l - m); sigmoid: 1 / (1 + exp(-l)) over exp(min(m, 0)), which
// cancels where the weights are renormalized and keeps the greatest from 0.
__device__ __forceinline__ float score_over(float l, float m, bool sigmoid) {
    return sigmoid ? expf(fminf(l, 0.0f) - fminf(m, 0.0f)) / (1.0f + expf(-fabsf(l))) : expf(l - m);
}
__device__ __forceinline__ float sigmoid_of(float l) { return 1.0f / (1.0f + expf(-l)); }

// L lanes take a token, P experts each, in order.
template <int DT, int L, int P, bool VEC, bool GROUPS>
__global__ __launch_bounds__(RT_THREADS) void choose_kernel(RouterArgs a, unsigned first) {
    __shared__ int chosen_lds[RT_THREADS * P];                        // k <= E <= L P of each token
    __shared__ double choice_lds[GROUPS ? RT_THREADS * P : 1];
    const int tid = threadIdx.x, sub = tid % L, e0 = sub * P;
    const long long t = (first + (long long)blockIdx.x) * (RT_THREADS / L) + tid / L;
    if (t >= a.T) return;                                             // a token's lanes are of one wave
    int* chosen = chosen_lds + tid / L * (L * P);
    const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + (size_t)t * a.E * (DT == DT_F32 ? 4 : 2);
    float l[P];
    load_logits<DT, P, VEC>(row, e0, a.E, l);
    float m = l[0];
#pragma unroll
    for (int p = 1; p < P; ++p) m = fmaxf(m, l[p]);
    m = max_lanes<L>(m);

    double key[P];
    bool spoilt = false;                                              // a NaN somewhere: no score is a number
    const bool by_score = a.bias != nullptr || (GROUPS && a.sum2);
    if (by_score) {
        double s[P], sum = 0.0;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            s[p] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)l[p])) : exp((double)l[p] - (double)m);
            sum += l[p] == -__builtin_inff() ? 0.0 : s[p];
        }
        if (!a.sigmoid) {
            sum = sum_lanes<L>(sum);
            spoilt = sum != sum;
            const double inv = 1.0 / sum;
#pragma unroll
            for (int p = 0; p < P; ++p) s[p] *= inv;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const bool out = e0 + p >= a.E || l[p] == -__builtin_inff();
            const float b = a.bias != nullptr && e0 + p < a.E ? a.bias[e0 + p] : 0.0f;
            key[p] = out ? RT_NONE : s[p] + (double)b;
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) key[p] = e0 + p < a.E ? (double)l[p] : RT_NONE;
    }

    if constexpr (GROUPS) {
        double* choice = choice_lds + tid / L * (L * P);
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (e0 + p < a.E) choice[e0 + p] = key[p];
        wave_sync();
        const int size = a.E / a.groups;
        for (int g = sub; g < a.groups; g += L) {
            double one = RT_NONE, two = RT_NONE;
            for (int i = 0; i < size; ++i) {
                const double c = choice[g * size + i];
                const bool above = ranks_above(c, one);
                two = above ? one : ranks_above(c, two) ? c : two;
                one = above ? c : one;
            }
            choice[g * size] = key_of(a.sum2 && two != RT_NONE ? one + two : one, g);
        }
        wave_sync();
        double gk[P];
#pragma unroll
        for (int p = 0; p < P; ++p) gk[p] = e0 + p < a.groups ? choice[(e0 + p) * size] : RT_NONE;
        double last = __builtin_inf();
        for (int j = 0; j < a.top_groups; ++j) {
            double best = RT_NONE;
#pragma unroll
            for (int p = 0; p < P; ++p) best = key_max(best, gk[p] < last ? gk[p] : RT_NONE);
            last = all_lanes<L>(best, key_max);
        }
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (e0 + p < a.E && choice[(e0 + p) / size * size] < last) key[p] = RT_NONE;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) key[p] = key_of(key[p], e0 + p);
    double last = __builtin_inf();
    for (int j = 0; j < a.k; ++j) {
        double best = RT_NONE;
#pragma unroll
        for (int p = 0; p < P; ++p) best = key_max(best, key[p] < last ? key[p] : RT_NONE);
        last = all_lanes<L>(best, key_max);
        if (sub == 0) chosen[j] = key_number(last);
    }
    wave_sync();

    // the weights, in 32 bits from the chosen logits
    float total = 0.0f;
    if (a.renormalize) {
        float top = -__builtin_inff();
        for (int j = sub; j < a.k; j += L)
            if (chosen[j] >= 0) top = fmaxf(top, logit_at<DT>(row, chosen[j]));
        m = max_lanes<L>(top);
        for (int j = sub; j < a.k; j += L)
            if (chosen[j] >= 0) total += score_over(logit_at<DT>(row, chosen[j]), m, a.sigmoid);
        total = sum_lanes<L>(total);
    } else if (!a.sigmoid) {
#pragma unroll
        for (int p = 0; p < P; ++p) total += l[p] == -__builtin_inff() ? 0.0f : expf(l[p] - m);
        total = sum_lanes<L>(total);
    }
    if (spoilt) total = __builtin_nanf("");
    for (int j = sub; j < a.k; j += L) {
        const int e = chosen[j];
        float w = 0.0f;
        if (e >= 0) {
            const float v = logit_at<DT>(row, e);
            w = a.sigmoid && !a.renormalize ? sigmoid_of(v) : score_over(v, m, a.sigmoid) / total;
        }
        a.ids[t * a.k + j] = e;
        a.weights[t * a.k + j] = e >= 0 ? w * a.scale : 0.0f;
    }
}

// d_logits of a token, with p the weights before `scale` and g = scale d_weights:
//   softmax        renormalized p_j (g_j - sum p g), else s_e ([e chosen] g_e - sum s g)
//   sigmoid        renormalized p_j (1 - s_j) (g_j - sum p g), else s_j (1 - s_j) g_j
// and 0 for experts that were not chosen (but for softmax as it is).  Scores are computed again from the logits.
template <int DT, int L, int P, bool VEC>
__global__ __launch_bounds__(RT_THREADS) void choose_grad_kernel(RouterGradArgs a, unsigned first) {
    __shared__ float d_lds[RT_THREADS * P];
    const int tid = threadIdx.x, sub = tid % L, e0 = sub * P;
    const long long t = (first + (long long)blockIdx.x) * (RT_THREADS / L) + tid / L;
    if (t >= a.T) return;
    float* d = d_lds + tid / L * (L * P);
    constexpr int ES = DT == DT_F32 ? 4 : 2;
    const uint8_t* row = reinterpret_cast<const uint8_t*>(a.logits) + (size_t)t * a.E * ES;
    const int* ids = a.ids + t * a.k;
    const float* dw = a.d_weights + t * a.k;
    const bool all = !a.sigmoid && !a.renormalize;                     // every logit has a gradient
#pragma unroll
    for (int p = 0; p < P; ++p) d[e0 + p] = 0.0f;
    float l[P], m = -__builtin_inff(), total = 0.0f;
    if (all) {
        load_logits<DT, P, VEC>(row, e0, a.E, l);
#pragma unroll
        for (int p = 0; p < P; ++p) m = fmaxf(m, l[p]);
        m = max_lanes<L>(m);
#pragma unroll
        for (int p = 0; p < P; ++p) total += l[p] == -__builtin_inff() ? 0.0f : expf(l[p] - m);
        total = sum_lanes<L>(total);
    } else if (a.renormalize) {
        for (int j = sub; j < a.k; j += L)
            if ((unsigned)ids[j] < (unsigned)a.E) m = fmaxf(m, logit_at<DT>(row, ids[j]));
        m = max_lanes<L>(m);
        for (int j = sub; j < a.k; j += L)
            if ((unsigned)ids[j] < (unsigned)a.E) total += score_over(logit_at<DT>(row, ids[j]), m, a.sigmoid);
        total = sum_lanes<L>(total);
    }
    float mean = 0.0f;
    if (all || a.renormalize) {
        for (int j = sub; j < a.k; j += L)
            if ((unsigned)ids[j] < (unsigned)a.E)
                mean += score_over(logit_at<DT>(row, ids[j]), m, a.sigmoid) / total * (dw[j] * a.scale);
        mean = sum_lanes<L>(mean);
    }
    wave_sync();
    for (int j = sub; j < a.k; j += L) {
        if ((unsigned)ids[j] >= (unsigned)a.E) continue;
        const float v = logit_at<DT>(row, ids[j]), g = dw[j] * a.scale;
        const float s1 = a.sigmoid ? 1.0f / (1.0f + expf(v)) : 1.0f;                  // 1 - s
        const float p = a.sigmoid && !a.renormalize ? sigmoid_of(v) : score_over(v, m, a.sigmoid) / total;
        d[ids[j]] = all ? p * g : a.renormalize ? p * s1 * (g - mean) : p * s1 * g;
    }
    wave_sync();
    uint8_t* out = reinterpret_cast<uint8_t*>(a.d_logits) + (size_t)t * a.E * ES;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (e0 + p >= a.E) break;
        float v = d[e0 + p];
        if (all && l[p] != -__builtin_inff()) v -= expf(l[p] - m) / total * mean;
        if constexpr (DT == DT_F32) reinterpret_cast<float*>(out)[e0 + p] = v;
        else reinterpret_cast<uint16_t*>(out)[e0 + p] = (uint16_t)(DT == DT_BF16 ? pack_bf16x2(v, 0.0f) : pack_f16x2(v, 0.0f));
    }
}

template <typename F>
static hipError_t by_lanes(int dt, int E, F f) {
    const auto lanes = [&](auto d) {
        constexpr int DT = decltype(d)::value;
        using std::integral_constant;
        const auto vec = [&](auto l) {
            return E % 16 == 0 ? f(integral_constant<int, DT>{}, l, std::true_type{}) : f(integral_constant<int, DT>{}, l, std::false_type{});
        };
        if (E <= 32) return vec(integral_constant<int, 2>{});
        if (E <= 64) return vec(integral_constant<int, 4>{});
        if (E <= 128) return vec(integral_constant<int, 8>{});
        if (E <= 256) return vec(integral_constant<int, 16>{});
        if (E <= 512) return vec(integral_constant<int, 32>{});
        return vec(integral_constant<int, 64>{});
    };
    using std::integral_constant;
    if (dt == DT_F32) return lanes(integral_constant<int, DT_F32>{});
    if (dt == DT_BF16) return lanes(integral_constant<int, DT_BF16>{});
    return lanes(integral_constant<int, DT_F16>{});
}

int router_max_experts() { return RT_MAX_E; }

hipError_t choose_launch(const RouterArgs& a, int dt, hipStream_t st) {
    return by_lanes(dt, a.E, [&](auto d, auto l, auto v) {
        constexpr int DT = decltype(d)::value, L = decltype(l)::value;
        constexpr bool VEC = decltype(v)::value;
        return launch_parts((a.T * L + RT_THREADS - 1) / RT_THREADS, RT_THREADS, [&](long long first, dim3 grid) {
            if (a.groups > 1)
                hipLaunchKernelGGL((choose_kernel<DT, L, 16, VEC, true>), grid, dim3(RT_THREADS), 0, st, a, (unsigned)first);
            else
                hipLaunchKernelGGL((choose_kernel<DT, L, 16, VEC, false>), grid, dim3(RT_THREADS), 0, st, a, (unsigned)first);
        });
    });
}

hipError_t choose_grad_launch(const RouterGradArgs& a, int dt, hipStream_t st) {
    return by_lanes(dt, a.E, [&](auto d, auto l, auto v) {
        constexpr int DT = decltype(d)::value, L = decltype(l)::value;
        constexpr bool VEC = decltype(v)::value;
        return launch_parts((a.T * L + RT_THREADS - 1) / RT_THREADS, RT_THREADS, [&](long long first, dim3 grid) {
            hipLaunchKernelGGL((choose_grad_kernel<DT, L, 16, VEC>), grid, dim3(RT_THREADS), 0, st, a, (unsigned)first);
        });
    });
}

}  // namespace convrot
