// Rows in 8 bits for products with FP8 weights: made from rows, from a residual stream and its norm, from the gate and up rows of a
// feed-forward; and read back.
//
// A row's values lie in groups of 128 (the last may be shorter), as many as a block of the weights has along K: e4m3 codes and one exponent
// byte a group, value = code * 2^(b - 127), with the smallest exponent between -60 and 60 for which the group's largest finite magnitude is at most
// 448 * 2^exponent.  A power of two, because codes times it are exact in bf16, a floating code loses nothing by it, and the exponent depends on
// the largest magnitude's own bits and on nothing that a division could round.  A value that fp32 does not hold as a finite number is the NaN
// code; magnitudes above 448 * 2^60 saturate.  Exponent rows start at multiples of 16 bytes: the product reads sixteen groups at a time.
//
// Codes are the nearest ones of the definition in 64 bits.  fp32 decides all but the values that lie within its error of the middle between two codes or that
// it does not hold; those are made again in 64 bits.
#include <algorithm>
#include <type_traits>

#include "f32x2.cuh"
#include "fp8_rows.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t INFINITE = 0x7f800000u;                   // bits

// Smallest exponent with which a magnitude is at most 448 * 2^exponent, within the limits.
__device__ __forceinline__ int exponent_of(double top) {
    const uint64_t bits = (uint64_t)__double_as_longlong(top);
    const int e = (int)(bits >> 52) - 1023 - 8 + ((bits & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 0);
    return max(FP8_LOW, min(FP8_HIGH, e));
}

// An fp32 number that any rounding to fewer bits takes where it would take `d`: cut off, with the last bit set where something was.
__device__ __forceinline__ float to_odd(double d) {
    const float f = __double2float_rz(d);
    return (double)f == d || !fp8_finite(f) ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Element i of four registers.
__device__ __forceinline__ float pick(const float (&v)[4], int i) { return i & 2 ? (i & 1 ? v[3] : v[2]) : (i & 1 ? v[1] : v[0]); }
__device__ __forceinline__ void put(float (&v)[4], int i, float x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i == j ? x : v[j];
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Codes of four values times a factor (its bits).
__device__ __forceinline__ uint32_t codes_of(const float (&v)[4], uint32_t factor) {
    const float f = __uint_as_float(factor);
    const f32x2 both = pair(f, f);
    const float2 lo = unpair(mul2(pair(v[0], v[1]), both)), hi = unpair(mul2(pair(v[2], v[3]), both));
    const float x[4] = {lo.x, lo.y, hi.x, hi.y};
    return fp8_codes(x);
}

// A group in a warp, four values a lane, in fp32 off by up to `within` of their last places (0: exact).  `again(i)`: value i in 64 bits.  The lane's codes;
// `e`: the group's exponent.  `all`: fp32 says nothing.
template <class Again>
__device__ __forceinline__ uint32_t quantize_group(float (&v)[4], uint32_t within, bool all, int& e, Again again) {
    const float most = max3(max3(0.f, fabsf(v[0]), fabsf(v[1])), fabsf(v[2]), fabsf(v[3]));
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));          // (max passes over NaN)
    if (within != 0) all |= top >= INFINITE - within - 1;    // (64 bits say which of them fp32 holds)
    if (top == INFINITE) {                                   // an infinity: a NaN from here on, and not the largest magnitude
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
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            const double d = fabs(again(i));
            if (fp8_finite((float)d)) largest = fmax(largest, d);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) largest = fmax(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        e = exponent_of(largest);
    }
    const uint32_t down = (uint32_t)(127 - e) << 23;
    if (within == 0) return codes_of(v, down);
    // The factor off by `within` / 2 + 1 places of 2^-23 either way, which is more than `within` of 2^-24 and the product's rounding: the value in 64 bits
    // lies between the two, and where both have one code it is that one.  (A test of the product's bits for a middle took twice the instructions.)
    const uint32_t low = codes_of(v, down - 2 * (within / 2 + 1)), high = codes_of(v, down + within / 2 + 1);
    uint32_t codes = low;
    if (all || low != high) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i)
            if (all || ((low ^ high) >> (8 * i) & 255u)) {
                const double d = again(i);
                const float f = fp8_finite((float)d) ? to_odd(d * (double)__uint_as_float(down)) : __uint_as_float(0x7fffffffu);
                codes = (codes & ~(255u << (8 * i))) | (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3) << (8 * i);
            }
    }
    return codes;
}

// The same without a branch, for groups that need none; true where `quantize_group` has to do it.
__device__ __forceinline__ bool quantize_quick(const float (&v)[4], uint32_t within, int& e, uint32_t& codes) {
    const float most = max3(max3(0.f, fabsf(v[0]), fabsf(v[1])), fabsf(v[2]), fabsf(v[3]));
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    e = fp8_exponent(top);
    const uint32_t down = (uint32_t)(127 - e) << 23;
    codes = codes_of(v, down - 2 * (within / 2 + 1));
    return (top >= INFINITE - within - 1) | ((top & 0x7fffffu) - (0x600000u - within) <= 2 * within) | (codes != codes_of(v, down + within / 2 + 1));
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

// One block a token; a warp has whole groups, a thread four values of each, so that a group's largest magnitude is one instruction over the warp and the
// row stays in registers between its sum and its codes.  The sum of squares is taken in 64 bits: fp32 rows may be as large as fp32 goes, and its
// rounding would move every code of the row.  Bound by memory: 4096 x 4096, fp32, takes 35 us (6.2 TB/s); few tokens: a launch and three dependent
// waits (2 us).
template <bool XF32, bool WF32, int Q>
__global__ void __launch_bounds__(1024, 1) fp8_norm_kernel(const __grid_constant__ Fp8NormParams p) {
    pdl_grid_sync();
    __shared__ double sums[33];
    const int t = blockIdx.x, nt = blockDim.x, n4 = p.H / 4, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const char* const x = reinterpret_cast<const char*>(p.x) + (size_t)t * p.ldx * (XF32 ? 4 : 2);
    using WRaw = std::conditional_t<WF32, float4, uint2>;
    WRaw gain[Q];                                            // (asked for with the row, used behind the sum)
    float v[Q][4];
    double ss = 0.0;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = threadIdx.x + q * nt;
        gain[q] = WRaw{};
        if (i < n4) {
            load4<XF32>(x, i, v[q]);
            gain[q] = __ldg(reinterpret_cast<const WRaw*>(p.w) + i);
        } else v[q][0] = v[q][1] = v[q][2] = v[q][3] = 0.f;
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
    const bool all = !(inv < 1e30 && inv > 1.2e-38);     // (beyond fp32 or below 2^-126, where its last place is 4 units of 2^-24 and more, or no number)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = threadIdx.x + q * nt;
        if (i - lane >= n4) break;                       // (the same for the whole warp)
        float w[4], f[4];
        if constexpr (WF32) { w[0] = gain[q].x; w[1] = gain[q].y; w[2] = gain[q].z; w[3] = gain[q].w; }
        else {
            const float2 lo = bf162_to_f2(gain[q].x), hi = bf162_to_f2(gain[q].y);
            w[0] = lo.x; w[1] = lo.y; w[2] = hi.x; w[3] = hi.y;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = v[q][j] * inv32 * w[j];
        int e;
        // three roundings to fp32 (the factor's, two products'): at most 3 last places, unless a gain of 2^54 or more brings back what was below 2^-126
        const bool far = __any_sync(0xffffffffu, fmaxf(max3(fabsf(w[0]), fabsf(w[1]), fabsf(w[2])), fabsf(w[3])) >= 0x1p54f);
        const uint32_t c = quantize_group(f, 4, all || far, e, [&](int j) { return (double)pick(v[q], j) * inv * (double)pick(w, j); });
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

// A warp has a group of 128 columns and walks over tokens, some at a time, so that enough loads are on their way.  What fp32 is off by, in units of 2^-24: down
// to gates of -16 the exponential's argument is at most 23.1, its rounding 2^-20 and that of log2(e) 3.1e-7, which makes 15; the exponential and the
// reciprocal 4 each, the sum and two products 1 each.  Gates below -16 are made in 64 bits.
//
// Gated rows are bound by instructions (98 for four values of a lane, issued in two cycles of three) and by their loads in turn: 4096 x 14336 bf16 pairs
// in 64 us, 4.6 TB/s; fp32 pairs in 83, 6.3 TB/s; plain rows in 35, 5.0 TB/s.  Where a group needs 64 bits, a vote and a call leave the way free for the
// others (branches where each is needed: 73).  No faster, before the last instructions went (67): two tokens side by side (73), a warp with adjacent groups of a row
// (75), the next tokens' loads between this one's results (69), five blocks an SM (73: 48 registers a thread do not hold it).
template <bool GATED, bool F32>
struct RowsCfg {
    static constexpr int BLOCKS = GATED ? 4 : 6;                             // resident on an SM
    static constexpr int TOKENS = F32 ? 2 : 4;                               // of a warp at a time
};

__device__ __forceinline__ void values_of(const uint4& r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void values_of(const uint2& r, float (&v)[4]) {
    const float2 lo = bf162_to_f2(r.x), hi = bf162_to_f2(r.y);
    v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
}

constexpr uint32_t GATED_OFF = 27;                           // units of 2^-24, for gates down to
constexpr float GATED_LOW = -16.f;

__device__ __forceinline__ void activation(const float (&a)[4], const float (&u)[4], float (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) {                         // two values to an instruction
        const f32x2 g = pair(a[j], a[j + 1]);
        const float2 z = unpair(mul2(g, pair(-LOG2E, -LOG2E)));
        const float2 d = unpair(add2(pair(ex2(z.x), ex2(z.y)), pair(1.f, 1.f)));
        // `up` before the gate: where a product with `up` leaves the normal range, the gate is above 17 and the reciprocal 1, or the result is below every code
        // (a gate next to 0 left it before a large `up` brought it back)
        const float2 r = unpair(mul2(mul2(pair(rcp(d.x), rcp(d.y)), pair(u[j], u[j + 1])), g));
        v[j] = r.x; v[j + 1] = r.y;
    }
}

// A group of the activation where fp32 does not decide all of it (one in 200): codes and exponent.  A call, so that its registers are not the kernel's.
template <class Raw>
__device__ __noinline__ uint2 gated_group(Raw gate, Raw up) {
    float a[4], u[4], v[4];
    values_of(gate, a);
    values_of(up, u);
    auto again = [&](int j) {
        const double z = pick(a, j);
        return z / (1.0 + exp(-z)) * (double)pick(u, j);
    };
    activation(a, u, v);
#pragma unroll 1
    for (int j = 0; j < 4; ++j)
        if (pick(a, j) < GATED_LOW) put(v, j, (float)again(j));
    int e;
    const uint32_t c = quantize_group(v, GATED_OFF, false, e, again);
    return make_uint2(c, (uint32_t)e);
}

template <bool GATED, bool F32>
__global__ void __launch_bounds__(256, RowsCfg<GATED, F32>::BLOCKS) fp8_rows_kernel(const __grid_constant__ Fp8RowsParams p, int groups, int abreast) {
    pdl_grid_sync();
    constexpr int TOKENS = RowsCfg<GATED, F32>::TOKENS;
    using Raw = std::conditional_t<F32, uint4, uint2>;
    const int lane = threadIdx.x & 31, n4 = p.K / 4, at = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int g = at % groups, i = g * 32 + lane;
    if (at >= groups * abreast) return;
    const Raw* const x = reinterpret_cast<const Raw*>(p.x) + i;              // (rows start at multiples of four values)
    for (int t0 = at / groups; t0 < p.T; t0 += TOKENS * abreast) {
        Raw gate[TOKENS], up[TOKENS];
#pragma unroll
        for (int b = 0; b < TOKENS; ++b) {
            gate[b] = up[b] = Raw{};
            const int t = t0 + b * abreast;
            if (t < p.T && i < n4) {
                gate[b] = __ldg(x + (size_t)t * p.ldx / 4);
                if (GATED) up[b] = __ldg(x + ((size_t)t * p.ldx + p.K) / 4);
            }
        }
#pragma unroll
        for (int b = 0; b < TOKENS; ++b) {
            const int t = t0 + b * abreast;
            if (t >= p.T) break;                             // (the same for the whole warp)
            float a[4];
            values_of(gate[b], a);
            int e;
            uint32_t c;
            if constexpr (GATED) {
                float u[4], v[4];
                values_of(up[b], u);
                activation(a, u, v);
                const bool low = fminf(fminf(a[0], a[1]), fminf(a[2], a[3])) < GATED_LOW;
                if (__any_sync(0xffffffffu, quantize_quick(v, GATED_OFF, e, c) | low)) {
                    const uint2 r = gated_group(gate[b], up[b]);
                    c = r.x;
                    e = (int)r.y;
                }
            } else {
                c = quantize_group(a, 0, false, e, [](int) { return 0.0; });
            }
            if (i < n4) reinterpret_cast<uint32_t*>(p.codes + (size_t)t * p.ldc)[i] = c;
            if (lane == 0) p.exps[(size_t)t * p.lde + g] = (uint8_t)(e + FP8_BIAS);
        }
    }
}

// ---- reading back ------------------------------------------------------------------------------------------------------------------------

// A thread has eight columns (a warp's stores are whole lines: 4096 x 14336 in 31 us; with sixteen, two stores that fill lines in turn, 40) and walks over
// tokens, four at a time.  Every value is exact in bf16: four significant bits, exponents from -69 to 68.
__global__ void __launch_bounds__(256) fp8_values_kernel(const __grid_constant__ Fp8ValuesParams p, int units, int abreast) {
    pdl_grid_sync();
    const int at = blockIdx.x * 256 + threadIdx.x, i = at % units;
    if (at >= units * abreast) return;
    for (int t0 = at / units; t0 < p.T; t0 += 4 * abreast) {
        uint2 codes[4];
        int exps[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = t0 + b * abreast;
            if (t < p.T) {
                codes[b] = __ldg(reinterpret_cast<const uint2*>(p.codes + (size_t)t * p.ldc) + i);
                exps[b] = __ldg(p.exps + (size_t)t * p.lde + i / 16);
            }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = t0 + b * abreast;
            if (t >= p.T) break;
            // (an exponent that no writer leaves is taken to the nearest one)
            const float up = __uint_as_float((uint32_t)(127 + max(FP8_LOW, min(FP8_HIGH, exps[b] - FP8_BIAS))) << 23);
            const float2 x0 = e4m3x2_to_float2((uint16_t)(codes[b].x & 0xffffu)), x1 = e4m3x2_to_float2((uint16_t)(codes[b].x >> 16));
            const float2 x2 = e4m3x2_to_float2((uint16_t)(codes[b].y & 0xffffu)), x3 = e4m3x2_to_float2((uint16_t)(codes[b].y >> 16));
            reinterpret_cast<uint4*>(p.out + (size_t)t * p.K)[i] = make_uint4(f2_to_bf162(x0.x * up, x0.y * up), f2_to_bf162(x1.x * up, x1.y * up),
                                                                             f2_to_bf162(x2.x * up, x2.y * up), f2_to_bf162(x3.x * up, x3.y * up));
        }
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
    const int groups = (p->K + 127) / 128, abreast = tokens_abreast(p->T, groups, 148 * 8 * (gated ? 4 : 6));     // (blocks that are resident)
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
    const int units = p->K / 8, abreast = tokens_abreast(p->T, units, 148 * 2048);
    sl_launch(fp8_values_kernel, dim3((units * abreast + 255) / 256), 256, 0, s, *p, units, abreast);
    return SL_LAUNCH_CHECK();
}
