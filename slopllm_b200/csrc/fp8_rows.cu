// Rows in 8 bits for products with FP8 weights: made from rows, from a residual stream and its norm, from the gate and up rows of a
// feed-forward; and read back.
//
// A row's values lie in groups of 128 (the last may be shorter), as many as a block of the weights has along K: e4m3 codes and one exponent
// byte a group, value = code * 2^(b - 127), with the smallest exponent between -60 and 60 for which the group's largest finite magnitude is at most
// 448 * 2^exponent.  A power of two, because codes times it are exact in bf16, a floating code loses nothing by it, and the exponent depends on
// the largest magnitude's own bits and on nothing that a division could round.  A value that fp32 does not hold as a finite number is the NaN
// code; magnitudes above 448 * 2^60 saturate.  Exponent rows start at multiples of 16 bytes: the product reads sixteen groups at a time.
//
// Codes are the nearest ones of the definition in 64 bits.  fp32 decides all but the values that lie within its error of the middle between two
// codes; those are made again in 64 bits.
#include <algorithm>

#include "fp8_rows.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// Smallest exponent with which a magnitude is at most 448 * 2^exponent, within the limits.
__device__ __forceinline__ int exponent_of(double top) {
    const uint64_t bits = (uint64_t)__double_as_longlong(top);
    const int e = (int)(bits >> 52) - 1023 - 8 + ((bits & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 0);
    return max(FP8_LOW, min(FP8_HIGH, e));
}

// Whether `f`, off by up to `within` of its last places, may lie on the other side of the middle between two codes.  Three bits of the significand
// are kept; below 2^-6 codes have the steps that they have there.
__device__ __forceinline__ bool near_middle(float f, uint32_t within) {
    float a = fabsf(f);
    a = a < 0.015625f ? a + 0.015625f : a;
    return (__float_as_uint(a) & 0xfffffu) - (0x80000u - within) <= 2 * within;
}

// An fp32 number that any rounding to fewer bits takes where it would take `d`: cut off, with the last bit set where something was.
__device__ __forceinline__ float to_odd(double d) {
    const float f = __double2float_rz(d);
    return (double)f == d || !fp8_finite(f) ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// A group in a warp, four values a lane, in fp32 off by up to `within` of their last places (0: exact).  `again(i)`: value i in 64 bits.  The lane's codes;
// `e`: the group's exponent.  `all`: fp32 says nothing.
template <class Again>
__device__ __forceinline__ uint32_t quantize_group(float (&v)[4], uint32_t within, bool all, int& e, Again again) {
    const float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(most, 0.f)));          // (fmaxf passes over NaN)
    if (top == 0x7f800000u) {                                // an infinity: a NaN from here on, and not the largest magnitude
        top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (!fp8_finite(v[i])) v[i] = __uint_as_float(0x7fffffffu);
            else top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
    }
    e = fp8_exponent(top);
    if (within != 0 && (all || (top & 0x7fffffu) - (0x600000u - within) <= 2 * within)) {
        double largest = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double d = fabs(again(i));
            if (d <= (double)FLT_MAX) largest = fmax(largest, d);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) largest = fmax(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        e = exponent_of(largest);
    }
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    bool near = all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] *= down;
        if (within != 0) near |= near_middle(v[i], within);
    }
    if (within != 0 && near) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (all || near_middle(v[i], within)) {
                const double d = again(i);
                v[i] = fabs(d) <= (double)FLT_MAX ? to_odd(d * (double)down) : __uint_as_float(0x7fffffffu);
            }
    }
    return fp8_codes(v);
}

template <bool F32>
__device__ __forceinline__ void load4(const void* row, int i, float (&v)[4]) {
    if (F32) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row) + i);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(row) + i);
        const float2 lo = bf162_to_f2(u.x), hi = bf162_to_f2(u.y);
        v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
    }
}

// ---- residual, norm, rows ------------------------------------------------------------------------------------------------------------

// One block a token; a warp has whole groups, a thread four values of each.  The sum of squares is taken in 64 bits: fp32 rows may be as large
// as fp32 goes, and its rounding would move every code of the row.
template <bool XF32, bool WF32, int Q>
__global__ void __launch_bounds__(1024) fp8_norm_kernel(const __grid_constant__ Fp8NormParams p) {
    pdl_grid_sync();
    __shared__ double sums[33];
    const int t = blockIdx.x, nt = blockDim.x, n4 = p.H / 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const char* const x = reinterpret_cast<const char*>(p.x) + (size_t)t * p.ldx * (XF32 ? 4 : 2);
    float v[Q][4];
    double ss = 0.0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = threadIdx.x + q * nt;
        if (i < n4) load4<XF32>(x, i, v[q]);
        else v[q][0] = v[q][1] = v[q][2] = v[q][3] = 0.f;
    }
    if (p.residual != nullptr) {
        const float4* const r = reinterpret_cast<const float4*>(p.residual + (size_t)t * p.ldr);
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int i = threadIdx.x + q * nt;
            if (i < n4) {
                const float4 a = __ldg(r + i);
                v[q][0] += a.x; v[q][1] += a.y; v[q][2] += a.z; v[q][3] += a.w;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = threadIdx.x + q * nt;
        if (i < n4) reinterpret_cast<float4*>(p.res_out + (size_t)t * p.H)[i] = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fma((double)v[q][j], (double)v[q][j], ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) sums[warp] = ss;
    __syncthreads();
    if (warp == 0) {
        ss = lane < nt / 32 ? sums[lane] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) sums[32] = rsqrt(ss / (double)p.H + p.eps);
    }
    __syncthreads();
    const double inv = sums[32];
    const float inv32 = (float)inv;
    const bool all = !(inv < 1e30);                      // (beyond fp32, or no number)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = threadIdx.x + q * nt;
        if (i - lane >= n4) break;                       // (the same for the whole warp)
        float w[4] = {0.f, 0.f, 0.f, 0.f}, f[4];
        if (i < n4) load4<WF32>(p.w, i, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = v[q][j] * inv32 * w[j];
        int e;
        // three roundings to fp32 (the factor's, two products'): at most 3 last places
        const uint32_t c = quantize_group(f, 4, all, e, [&](int j) { return (double)v[q][j] * inv * (double)w[j]; });
        if (i < n4) reinterpret_cast<uint32_t*>(p.codes + (size_t)t * p.ldc)[i] = c;
        if (lane == 0) p.exps[(size_t)t * p.lde + i / 32] = (uint8_t)(e + FP8_BIAS);
    }
}

// ---- rows, gated rows --------------------------------------------------------------------------------------------------------------------

// The hardware's exponential of base 2 and reciprocal, each within 2^-22 of the result.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A warp has a group of 128 columns and walks over tokens, two at a time.  What fp32 is off by, in units of 2^-24: down to gates of -16 the exponential's
// argument is at most 23.1, its rounding 2^-20 and that of log2(e) 3.1e-7, which makes 15; the exponential and the reciprocal 4 each, the sum and two products 1
// each.  Gates below -16 are made in 64 bits.
template <bool GATED, bool F32>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const __grid_constant__ Fp8RowsParams p, int groups, int abreast) {
    pdl_grid_sync();
    const int lane = threadIdx.x & 31, n4 = p.K / 4, at = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int g = at % groups, i = g * 32 + lane;
    const size_t size = F32 ? 4 : 2;
    const char* const x = reinterpret_cast<const char*>(p.x);
    auto load = [&](int t, float (&a)[4], float (&u)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = u[j] = 0.f;
        if (i < n4) {
            load4<F32>(x + (size_t)t * p.ldx * size, i, a);
            if (GATED) load4<F32>(x + ((size_t)t * p.ldx + p.K) * size, i, u);
        }
    };
    auto store = [&](int t, float (&a)[4], float (&u)[4]) {
        int e;
        uint32_t c;
        if (GATED) {
            auto again = [&](int j) { return (double)a[j] / (1.0 + exp(-(double)a[j])) * (double)u[j]; };
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j] * rcp(1.f + ex2(a[j] * -LOG2E)) * u[j];
            if (fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) < -16.f) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (a[j] < -16.f) v[j] = (float)again(j);
            }
            c = quantize_group(v, 27, false, e, again);
        } else {
            c = quantize_group(a, 0, false, e, [](int) { return 0.0; });
        }
        if (i < n4) reinterpret_cast<uint32_t*>(p.codes + (size_t)t * p.ldc)[i] = c;
        if (lane == 0) p.exps[(size_t)t * p.lde + g] = (uint8_t)(e + FP8_BIAS);
    };
    for (int t = at / groups; t < p.T && at < groups * abreast; t += 2 * abreast) {
        float a0[4], u0[4], a1[4], u1[4];
        load(t, a0, u0);
        const bool two = t + abreast < p.T;                  // (the same for the whole warp)
        if (two) load(t + abreast, a1, u1);
        store(t, a0, u0);
        if (two) store(t + abreast, a1, u1);
    }
}

// ---- reading back ------------------------------------------------------------------------------------------------------------------------

// A thread has sixteen columns and walks over tokens.  Every value is exact in bf16: four significant bits, exponents from -69 to 68.
__global__ void __launch_bounds__(256) fp8_values_kernel(const __grid_constant__ Fp8ValuesParams p, int units, int abreast) {
    pdl_grid_sync();
    const int at = blockIdx.x * 256 + threadIdx.x, i = at % units;
    if (at >= units * abreast) return;
#pragma unroll 2
    for (int t = at / units; t < p.T; t += abreast) {
        const uint4 c = ldg_nc_16(p.codes + (size_t)t * p.ldc + i * 16);
        // (an exponent that no writer leaves is taken to the nearest one)
        const int e = max(FP8_LOW, min(FP8_HIGH, (int)__ldg(p.exps + (size_t)t * p.lde + i / 8) - FP8_BIAS));
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 lo = e4m3x2_to_float2((uint16_t)(w[j] & 0xffffu)), hi = e4m3x2_to_float2((uint16_t)(w[j] >> 16));
            o[2 * j] = f2_to_bf162(lo.x * up, lo.y * up);
            o[2 * j + 1] = f2_to_bf162(hi.x * up, hi.y * up);
        }
        uint4* const dst = reinterpret_cast<uint4*>(p.out + (size_t)t * p.K + i * 16);
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

// How many tokens are worked on at the same time where each is `each` workers: all, as far as the device has room for them.
int tokens_abreast(int T, int each, int room) { return std::max(1, std::min(T, room / each)); }

template <bool XF32, bool WF32>
void launch_norm(const Fp8NormParams& p, int T, cudaStream_t s) {
    const int n4 = p.H / 4;
    // few tokens: a thread has as few values as a block allows; more: eight or sixteen
    const int per = T <= 296 ? (n4 <= 1024 ? 1 : n4 <= 2048 ? 2 : 4) : n4 <= 512 ? 2 : 4;
    const int threads = ((n4 + per - 1) / per + 31) / 32 * 32;
    if (per == 1) sl_launch(fp8_norm_kernel<XF32, WF32, 1>, T, threads, 0, s, p);
    else if (per == 2) sl_launch(fp8_norm_kernel<XF32, WF32, 2>, T, threads, 0, s, p);
    else sl_launch(fp8_norm_kernel<XF32, WF32, 4>, T, threads, 0, s, p);
}

}  // namespace

// H a multiple of 16, at most 16384; rows of x and the residual start at multiples of four values.
SL_API int sl_fp8_add_rmsnorm(const Fp8NormParams* p, int T, int x_f32, int w_f32, cudaStream_t s) {
    if (T == 0) return 0;
    if (T < 0 || p->H <= 0 || p->H % 16 != 0 || p->H > 16384) return -1;
    if (x_f32) {
        if (w_f32) launch_norm<true, true>(*p, T, s);
        else launch_norm<true, false>(*p, T, s);
    } else {
        if (w_f32) launch_norm<false, true>(*p, T, s);
        else launch_norm<false, false>(*p, T, s);
    }
    return SL_LAUNCH_CHECK();
}

// K a multiple of 16; gated: rows are K gates and K values behind them.
SL_API int sl_fp8_rows(const Fp8RowsParams* p, int gated, int f32, cudaStream_t s) {
    if (p->T == 0 || p->K == 0) return 0;
    if (p->T < 0 || p->K < 0 || p->K % 16 != 0) return -1;
    const int groups = (p->K + 127) / 128, abreast = tokens_abreast(p->T, groups, 148 * 48);      // (48 warps an SM)
    const dim3 grid((groups * abreast + 7) / 8);
    if (gated) {
        if (f32) sl_launch(fp8_rows_kernel<true, true>, grid, 256, 0, s, *p, groups, abreast);
        else sl_launch(fp8_rows_kernel<true, false>, grid, 256, 0, s, *p, groups, abreast);
    } else {
        if (f32) sl_launch(fp8_rows_kernel<false, true>, grid, 256, 0, s, *p, groups, abreast);
        else sl_launch(fp8_rows_kernel<false, false>, grid, 256, 0, s, *p, groups, abreast);
    }
    return SL_LAUNCH_CHECK();
}

SL_API int sl_fp8_values(const Fp8ValuesParams* p, cudaStream_t s) {
    if (p->T == 0 || p->K == 0) return 0;
    if (p->T < 0 || p->K < 0 || p->K % 16 != 0) return -1;
    const int units = p->K / 16, abreast = tokens_abreast(p->T, units, 148 * 2048);
    sl_launch(fp8_values_kernel, dim3((units * abreast + 255) / 256), 256, 0, s, *p, units, abreast);
    return SL_LAUNCH_CHECK();
}
