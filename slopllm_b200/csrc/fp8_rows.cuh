// Rows in 8 bits (fp8_rows.cu) and their products with FP8 weights (fp8_gemm_tcgen05.cu); the ctypes mirrors are in `ops/fp8.py`.
#pragma once

#include "common.cuh"

constexpr int FP8_BIAS = 127, FP8_LOW = -60, FP8_HIGH = 60;      // exponents of groups that are written

struct Fp8NormParams {
    const void* x; int ldx;                 // [T, H] bf16 or fp32
    const float* residual; int ldr;         // [T, H], or null
    const void* w;                          // [H] bf16 or fp32
    int H;
    double eps;
    float* res_out;                         // [T, H]
    uint8_t* codes; int ldc;                // [T, H]
    uint8_t* exps; int lde;                 // [T, ceil(H / 128)]
};

struct Fp8RowsParams {
    const void* x; int ldx;                 // [T, K], gated: [T, 2 K]
    int T, K;
    uint8_t* codes; int ldc;
    uint8_t* exps; int lde;
};

struct Fp8ValuesParams {
    const uint8_t* codes; int ldc;
    const uint8_t* exps; int lde;
    int T, K;
    bf16* out;                              // [T, K]
};

struct Fp8LinearParams {
    const uint8_t* exps; int lde;           // exponents of the rows [T, ceil(K / 128)]; rows of 16-byte pieces
    const float* scale; int lds;            // scales of the weights' blocks [ceil(N / 128), >= ceil(K / 128)]
    void* y; int ldy, out_f32;              // [T, N]
    int T, N, K;
    int* err;
};
