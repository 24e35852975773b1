// Attention of one new token per sequence over the 8-bit key/value cache (kv8.cuh).
//
//  * kv8_rows_kernel: one query head and token a block, on the CUDA cores.
#include "kv8.cuh"

namespace {

struct Kv8DecodeParams {
    const bf16* q;                       // [T, n_heads, hd]
    const uint8_t *k_codes, *v_codes, *exps;
    const int* positions; const int* batch_idx;      // [T]; keys 0..position are visible (a negative one: none, the row is zero)
    Kv8Pages pages;
    int n_heads, n_kv, hd;
    float scale;
    bf16* out;                           // [T, n_heads, hd]
};

constexpr int KT = 64;

// grid (heads, T), block 128
__global__ void __launch_bounds__(128) kv8_rows_kernel(Kv8DecodeParams p) {
    pdl_grid_sync();
    __shared__ float q[256], sc[KT], vs[KT], scratch[33];
    __shared__ int slots[KT];
    const int h = blockIdx.x, t = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, hkv = h / (p.n_heads / p.n_kv);
    const size_t at = ((size_t)t * p.n_heads + h) * p.hd, row = (size_t)p.n_kv * p.hd;
    for (int d = tid; d < p.hd; d += 128) q[d] = __bfloat162float(p.q[at + d]);
    const int n = p.positions[t] + 1, b = p.batch_idx[t];
    float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
    for (int k0 = 0; k0 < n; k0 += KT) {
        const int nk = min(KT, n - k0);
        __syncthreads();
        if (tid < nk) {
            const int s = kv8_slot(p.pages, 32, b, k0 + tid);
            slots[tid] = s;
            vs[tid] = s < 0 ? 0.f : __uint_as_float((uint32_t)p.exps[kv8_exp_at(p.pages, p.n_kv, s, hkv) + p.pages.page_size] << 23);
        }
        __syncthreads();
        for (int k = warp; k < nk; k += 4) {
            const int s = slots[k];
            float a = 0.f;
            if (s >= 0)
                for (int d = lane; d < p.hd; d += 32) a += q[d] * e4m3_to_float(p.k_codes[(size_t)s * row + (size_t)hkv * p.hd + d]);
            a = warp_sum(a);
            if (lane == 0) sc[k] = s < 0 ? 0.f : a * __uint_as_float((uint32_t)p.exps[kv8_exp_at(p.pages, p.n_kv, s, hkv)] << 23) * p.scale;
        }
        __syncthreads();
        const float top = fmaxf(m, block_max(tid < nk ? sc[tid] : -FLT_MAX, scratch));
        const float e = tid < nk ? expf(sc[tid] - top) : 0.f, f = m == -INFINITY ? 0.f : expf(m - top);
        l = l * f + block_sum(e, scratch);
        m = top;
        if (tid < nk) sc[tid] = e * vs[tid];
        __syncthreads();
        for (int i = 0; i < 2; ++i) {
            const int d = tid + i * 128;
            if (d >= p.hd) break;
            float a = o[i] * f;
            for (int k = 0; k < nk; ++k)
                if (slots[k] >= 0) a += sc[k] * e4m3_to_float(p.v_codes[(size_t)slots[k] * row + (size_t)hkv * p.hd + d]);
            o[i] = a;
        }
    }
    for (int i = 0; i < 2; ++i) {
        const int d = tid + i * 128;
        if (d < p.hd) p.out[at + d] = __float2bfloat16(n > 0 ? o[i] / l : 0.f);
    }
}

}  // namespace

SL_API int sl_kv8_decode(const Kv8DecodeParams* p, int T, cudaStream_t s) {
    if (T == 0) return 0;
    if (p->hd < 16 || p->hd > 256 || p->hd % 16 != 0 || p->n_kv < 1 || p->n_heads % p->n_kv != 0 || T > 65535 || p->pages.page_size < 1) return -1;
    sl_launch(kv8_rows_kernel, dim3(p->n_heads, T), 128, 0, s, *p);
    return SL_LAUNCH_CHECK();
}
