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
    void* y; int ldy, out_f32;              // [T, N]; gated: codes [T, N / 2]
    int T, N, K;
    uint8_t* exps_out; int lde_out;         // gated: [T, N / 256]
    int* err;
};

// Many rows, on pairs of SMs, tiles of 256 rows by 128 or 256 columns.  Gated: the activation of N / 2 gate and N / 2 up columns (a multiple of 128 each), in 8 bits.
int fp8_pair(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p, int columns, cudaStream_t s);
int fp8_pair_gated(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p, cudaStream_t s);

__device__ __forceinline__ bool fp8_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// Smallest exponent with which a magnitude (bits of an fp32 number) is at most 448 * 2^exponent, within the limits.
__device__ __forceinline__ int fp8_exponent(uint32_t top) {
    const int e = (int)((top + 0x1fffffu) >> 23) - 127 - 8;   // (a significand above 448's carries into the exponent)
    return max(FP8_LOW, min(FP8_HIGH, e));
}

__device__ __forceinline__ uint32_t fp8_codes(const float (&f)[4]) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
