// What the norm's kernels are given (rmsnorm.hip).
#pragma once

#include "common.h"

namespace convrot {

constexpr int NORM_MAX_D = 32768;          // widest row: 16 waves hold it

struct NormArgs {
    const void* x;             // [M, D]
    const void* residual;      // [M, D] or NULL
    const void* weight;        // [D] of type weight_dt, or NULL: 1
    void* h;                   // [M, D] with a residual: x + residual in their type
    void* y;                   // [M, D]; 8-bit codes [M, D] or I8T
    float* scales;             // [M], of 8-bit codes
    double eps;
    int M, D, weight_dt;
};

struct NormGradArgs {
    const void* d_y;           // [M, D]
    const void* d_h;           // [M, D] or NULL: the sum's own gradient
    const void* h;             // [M, D]
    const void* weight;        // [D] or NULL
    void* d_x;                 // [M, D] or NULL
    void* d_weight;            // [D] in the weight's type, or NULL
    float* partial;            // norm_grad_bytes(M, D) bytes where d_weight is asked for
    double eps;
    int M, D, weight_dt;
};

hipError_t norm_launch(const NormArgs& a, int dt, hipStream_t st);
hipError_t norm_int8_launch(const NormArgs& a, int dt, int G, bool tiled, hipStream_t st);
size_t norm_grad_bytes(int M, int D);
hipError_t norm_grad_launch(const NormGradArgs& a, int dt, hipStream_t st);

}  // namespace convrot
