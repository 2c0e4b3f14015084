// What the router's kernels are given (router.hip).
#pragma once

#include "common.h"

namespace convrot {

struct RouterArgs {
    const void* logits;        // [T, E]
    const float* bias;         // [E] or NULL
    int* ids;                  // [T, k]
    float* weights;            // [T, k]
    long long T;
    int dt, E, k, groups, top_groups;      // dt: the logits'
    float scale;
    bool sigmoid, sum2, renormalize;
};

struct RouterGradArgs {
    const void* logits;        // [T, E]
    const int* ids;            // [T, k]
    const float* d_weights;    // [T, k]
    void* d_logits;            // [T, E], in the logits' type
    long long T;
    int dt, E, k;
    float scale;
    bool sigmoid, renormalize;
};

int router_max_experts();
hipError_t choose_launch(const RouterArgs& a, hipStream_t st);
hipError_t choose_grad_launch(const RouterGradArgs& a, hipStream_t st);

}  // namespace convrot
