// Writing and reading back the 8-bit key/value cache (kv8.cuh).
//
//  * kv8_store_kernel: per-head RMS norm and rotate-half of queries and keys, in fp32 from the projection rows to the one rounding of the
//    result; keys and values are scaled by the power of two that brings their largest magnitude to (224, 448] and rounded to e4m3.
//  * kv8_read_kernel: rows of given tokens out of their pages as bf16, which holds them exactly.
#include "kv8.cuh"

namespace {

struct Kv8StoreParams {
    const bf16* q; int ldq;          // [T, n_heads * q_stride]; head h at h * q_stride
    const bf16* k; int ldk;          // [T, n_kv * hd]
    const bf16* v; int ldv;
    const bf16 *q_norm, *k_norm;     // [hd] or null
    const float* freq; float gain;   // [rot_dims / 2] angle per position; factor on cos and sin
    int rot_dims;
    const int* positions; const int* batch_idx;      // [T]; a negative position: nothing is written to the cache
    Kv8Pages pages;
    int n_heads, n_kv, hd, q_stride;
    float eps;
    bf16* q_out;                     // [T, n_heads, hd]
    uint8_t *k_codes, *v_codes, *exps;
};

constexpr double TWO_PI = 6.283185307179586476925;

// grid (T, y), block 256: a warp per row of a head (queries, then keys, then values), P neighbouring values a lane.  VEC: rows are aligned to
// a lane's values.
template <int P, bool VEC>
__global__ void __launch_bounds__(256) kv8_store_kernel(Kv8StoreParams p) {
    pdl_grid_sync();
    __shared__ float2 turn[128];                     // (cos, sin) of each pair
    __shared__ float row[8][32 * P];
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.rot_dims / 2;
    const int pos = p.positions[t];
    // fp32 keeps no digits of the angle of a far position: the product and its remainder are taken in 64 bits
    for (int i = threadIdx.x; i < half; i += 256) {
        const double a = (double)pos * (double)p.freq[i];
        float sn, cs;
        sincosf((float)fma(-rint(a * (1.0 / TWO_PI)), TWO_PI, a), &sn, &cs);
        turn[i] = make_float2(cs * p.gain, sn * p.gain);
    }
    const int slot = pos < 0 ? -1 : kv8_slot(p.pages, 30, p.batch_idx[t], pos);
    __syncthreads();
    const int d0 = lane * P;
    const bool on = d0 < p.hd;
    for (int job = blockIdx.y * 8 + warp; job < p.n_heads + 2 * p.n_kv; job += gridDim.y * 8) {
        const int what = job < p.n_heads ? 0 : job < p.n_heads + p.n_kv ? 1 : 2;         // query, key, value
        const int h = what == 0 ? job : what == 1 ? job - p.n_heads : job - p.n_heads - p.n_kv;
        const bf16* src = what == 0 ? p.q + (size_t)t * p.ldq + (size_t)h * p.q_stride
                                    : (what == 1 ? p.k + (size_t)t * p.ldk : p.v + (size_t)t * p.ldv) + (size_t)h * p.hd;
        auto load = [&](const bf16* from, float (&x)[P]) {
            if (VEC) {
                uint32_t w[P / 2];
                if (P == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(from + d0);
                else if (P == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(from + d0);
                else w[0] = *reinterpret_cast<const uint32_t*>(from + d0);
#pragma unroll
                for (int i = 0; i < P; i += 2) {
                    const float2 f = bf162_to_f2(w[i / 2]);
                    x[i] = f.x;
                    x[i + 1] = f.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) x[i] = __bfloat162float(from[d0 + i]);
            }
        };
        float x[P];
#pragma unroll
        for (int i = 0; i < P; ++i) x[i] = 0.f;
        if (on) load(src, x);
        const bf16* w = what == 0 ? p.q_norm : what == 1 ? p.k_norm : nullptr;
        if (w != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i) ss += x[i] * x[i];
            const float inv = 1.f / sqrtf(warp_sum(ss) / (float)p.hd + p.eps);
            if (on) {
                float g[P];
                load(w, g);
#pragma unroll
                for (int i = 0; i < P; ++i) x[i] = x[i] * inv * g[i];
            }
        }
        if (what < 2 && half > 0) {                  // (warp-uniform)
            __syncwarp();
#pragma unroll
            for (int i = 0; i < P; ++i) row[warp][d0 + i] = x[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int d = d0 + i;
                if (d < half) x[i] = x[i] * turn[d].x - row[warp][d + half] * turn[d].y;
                else if (d < p.rot_dims) x[i] = x[i] * turn[d - half].x + row[warp][d - half] * turn[d - half].y;
            }
        }
        if (what == 0) {
            bf16* dst = p.q_out + ((size_t)t * p.n_heads + h) * p.hd + d0;
            if (on) {
                uint32_t w2[P / 2];
#pragma unroll
                for (int i = 0; i < P; i += 2) w2[i / 2] = f2_to_bf162(x[i], x[i + 1]);
                if (P == 8) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(w2);
                else if (P == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(w2);
                else *reinterpret_cast<uint32_t*>(dst) = w2[0];
            }
            continue;
        }
        float top = 0.f;                             // of the finite values
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (!(fabsf(x[i]) <= FLT_MAX)) x[i] = __int_as_float(0x7fc00000);
            else top = fmaxf(top, fabsf(x[i]));
        }
        top = warp_max(top);
        if (slot < 0) continue;
        // top = m 2^n with m in [1, 2), 448 = 1.75 * 2^8
        const uint32_t bits = __float_as_uint(top);
        const int e = min(KV8_HIGH, max(KV8_LOW, (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0)));
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        uint8_t* dst = (what == 1 ? p.k_codes : p.v_codes) + ((size_t)slot * p.n_kv + h) * p.hd + d0;
        if (on) {
            uint32_t c[(P + 3) / 4] = {};
#pragma unroll
            for (int i = 0; i < P; i += 2)
                c[i / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[i] * inv, x[i + 1] * inv), __NV_SATFINITE, __NV_E4M3) << (i % 4 * 8);
            if (P == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(c[0], c[P / 8]);
            else if (P == 4) *reinterpret_cast<uint32_t*>(dst) = c[0];
            else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)c[0];
        }
        if (lane == 0) p.exps[kv8_exp_at(p.pages, p.n_kv, slot, h) + (what == 1 ? 0 : p.pages.page_size)] = (uint8_t)(e + KV8_BIAS);
    }
}

struct Kv8Rows {
    const uint8_t *k_codes, *v_codes, *exps;
    Kv8Pages pages;
    int n_kv, hd;
};

struct Kv8ReadParams {
    Kv8Rows c;
    const int* ranges;               // [R, 4]: page-table row, first position, count, first row of the result
    int rows;                        // of the result; what would lie behind them is not written (and recorded)
    bf16 *k, *v;                     // [rows, n_kv, hd]
};

// Histories of sequences as bf16 pages of 64 tokens, `per_seq` to a sequence, with a page table, rows of it and positions for a kernel that
// reads such pages.
struct Kv8UnpackParams {
    Kv8Rows c;
    const int *qo_indptr, *positions, *batch_idx;    // token ranges of the sequences, [T], [T]
    int per_seq;
    bf16 *k, *v;                     // [sequences * per_seq * 64, n_kv, hd]
    int *table, *rows_out, *positions_out;           // [sequences, per_seq], [T], [T]
};

// Rows `first` .. first + n - 1 (n <= 64) of page-table row b -> rows of k and v: 16 codes a thread at a time.
__device__ __forceinline__ void read_rows(const Kv8Rows& c, int b, int first, int n, bf16* k, bf16* v) {
    __shared__ int slots[64];
    if (threadIdx.x < n) slots[threadIdx.x] = kv8_slot(c.pages, 31, b, first + threadIdx.x);
    __syncthreads();
    const int per = c.n_kv * c.hd / 16;              // pieces of a row
    for (int x = threadIdx.x; x < 2 * n * per; x += blockDim.x) {
        const int which = x >= n * per ? 1 : 0, y = x - which * n * per, i = y / per, d = (y - i * per) * 16, slot = slots[i];
        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;                  // (a token that is not there reads as zeros)
        if (slot >= 0) {
            const uint4 w = ldg_nc_16((which ? c.v_codes : c.k_codes) + (size_t)slot * c.n_kv * c.hd + d);
            const float s = __uint_as_float((uint32_t)c.exps[kv8_exp_at(c.pages, c.n_kv, slot, d / c.hd) + which * c.pages.page_size] << 23);
            auto two = [&](uint32_t u) {
                const float2 f = e4m3x2_to_float2((uint16_t)u);
                return f2_to_bf162(f.x * s, f.y * s);
            };
            lo = make_uint4(two(w.x & 0xffff), two(w.x >> 16), two(w.y & 0xffff), two(w.y >> 16));
            hi = make_uint4(two(w.z & 0xffff), two(w.z >> 16), two(w.w & 0xffff), two(w.w >> 16));
        }
        uint4* dst = reinterpret_cast<uint4*>((which ? v : k) + (size_t)i * c.n_kv * c.hd + d);
        dst[0] = lo;
        dst[1] = hi;
    }
}

// grid (ceil(longest / 64), R), block 256
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8ReadParams p) {
    pdl_grid_sync();
    const int* r = p.ranges + blockIdx.y * 4;
    const int i0 = blockIdx.x * 64, n = min(64, r[2] - i0), out = r[3] + i0;
    if (n <= 0 || !guard_ok(p.c.pages.guard, 31, out, (long long)p.rows - n + 1)) return;
    const size_t at = (size_t)out * p.c.n_kv * p.c.hd;
    read_rows(p.c, r[0], r[1] + i0, n, p.k + at, p.v + at);
}

// grid (per_seq, sequences), block 256: a page of a sequence's workspace
__global__ void __launch_bounds__(256) kv8_unpack_kernel(Kv8UnpackParams p) {
    pdl_grid_sync();
    const int s = blockIdx.y, page = s * p.per_seq + blockIdx.x, q0 = p.qo_indptr[s], q1 = p.qo_indptr[s + 1], most = p.per_seq * 64;
    if (q0 >= q1) return;
    int n = p.positions[q1 - 1] + 1;                 // positions ascend within a sequence
    if (!guard_ok(p.c.pages.guard, 33, n, (long long)most + 1)) n = most;
    if (threadIdx.x == 0) p.table[page] = page;
    if (blockIdx.x == 0)
        for (int t = q0 + threadIdx.x; t < q1; t += 256) {
            p.rows_out[t] = s;
            p.positions_out[t] = min(p.positions[t], most - 1);
        }
    const int i0 = blockIdx.x * 64;
    n = min(64, n - i0);
    if (n <= 0) return;
    const size_t at = (size_t)page * 64 * p.c.n_kv * p.c.hd;
    read_rows(p.c, p.batch_idx[q0], i0, n, p.k + at, p.v + at);
}

}  // namespace

SL_API int sl_kv8_store(const Kv8StoreParams* p, int T, cudaStream_t s) {
    if (T == 0) return 0;
    if (p->hd < 16 || p->hd > 256 || p->hd % 16 != 0 || p->rot_dims < 0 || p->rot_dims > p->hd || p->rot_dims % 2 != 0 || p->n_kv < 1 || p->n_heads < 1) return -1;
    if ((((uintptr_t)p->k_codes | (uintptr_t)p->v_codes | (uintptr_t)p->q_out) & 15) != 0 || p->pages.page_size < 1) return -1;
    const int P = p->hd <= 64 ? 2 : p->hd <= 128 ? 4 : 8, jobs = p->n_heads + 2 * p->n_kv;
    const uintptr_t at = (uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->q_norm | (uintptr_t)p->k_norm;
    const bool vec = at % (2 * P) == 0 && (p->ldq | p->ldk | p->ldv | p->q_stride) % P == 0;
    const dim3 grid(T, T < 512 ? (jobs + 7) / 8 : 1);                // few tokens: a warp per row; many: the angles once a token
#define SL_KS(PP)                                                                       \
    {                                                                                   \
        if (vec) sl_launch(kv8_store_kernel<PP, true>, grid, 256, 0, s, *p);            \
        else sl_launch(kv8_store_kernel<PP, false>, grid, 256, 0, s, *p);               \
    }
    if (P == 2) SL_KS(2) else if (P == 4) SL_KS(4) else SL_KS(8)
#undef SL_KS
    return SL_LAUNCH_CHECK();
}

static bool kv8_rows_ok(const Kv8Rows& c, const void* k, const void* v) {
    return c.hd >= 16 && c.hd % 16 == 0 && c.n_kv >= 1 && c.pages.page_size >= 1 &&
           (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes | (uintptr_t)k | (uintptr_t)v) & 15) == 0;
}

SL_API int sl_kv8_read(const Kv8ReadParams* p, int ranges, int longest, cudaStream_t s) {
    if (ranges == 0 || longest <= 0) return 0;
    if (!kv8_rows_ok(p->c, p->k, p->v) || ranges > 65535) return -1;
    sl_launch(kv8_read_kernel, dim3((longest + 63) / 64, ranges), 256, 0, s, *p);
    return SL_LAUNCH_CHECK();
}

SL_API int sl_kv8_unpack(const Kv8UnpackParams* p, int sequences, cudaStream_t s) {
    if (sequences == 0) return 0;
    if (!kv8_rows_ok(p->c, p->k, p->v) || sequences > 65535 || p->per_seq < 1) return -1;
    sl_launch(kv8_unpack_kernel, dim3(p->per_seq, sequences), 256, 0, s, *p);
    return SL_LAUNCH_CHECK();
}
