// y[T, N] = X[T, K] * W[N, K]^T on the 8-bit tensor cores (tcgen05 kind::f8f6f4), rows and weights both e4m3: X with an exponent byte for each 128 values
// of a row, W with an fp32 scale for each block of 128 x 128.
//
//   y[t, n] = sum over blocks b of  S[n / 128, b] * 2^(E[t, b] - 127) * (sum over the block's k of X[t, k] * W[n, k])
//
// The scales differ from block to block of K, so a block's sums leave the tensor memory 128 values of K later and are added, times their factor, in fp32
// registers: one multiply-add a value and block, beside 128 multiply-adds of the tensor core.
//
// All mbarrier waits are bounded; where one runs out, the error word is set and the blocks still meet at the end.
#include <algorithm>

#include "fp8_rows.cuh"
#include "tcgen05_pair.cuh"

namespace {

constexpr int BK = 128;                                      // values (bytes) of a block of K
enum { WAIT_FREE = 70, WAIT_LANDED, WAIT_READ, WAIT_FETCHED, WAIT_SUMS };       // numbers of waits that run out

__device__ __forceinline__ float two_to(int byte) {          // 2^(byte - 127), for the exponents that writers leave
    return __uint_as_float((uint32_t)(max(FP8_LOW, min(FP8_HIGH, byte - FP8_BIAS)) + 127) << 23);
}
__device__ __forceinline__ float4 ld_cluster(uint32_t at, uint32_t rank) {
    float4 v;
    uint32_t far;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(far) : "memory");
    return v;
}

// ---- few rows: weights are the 128-row operand, rows the columns ---------------------------------------------------------------------------
//
// A block has 128 features, up to BN rows and a share of K; the blocks of a cluster have the shares of the same features and join their sums in shared
// memory, in the order of the shares.  Warp 0 fetches (TMA ring), warp 1 multiplies, warps 2 to 5 have a feature a thread and add up.
template <int BN>
struct Few {
    static constexpr int A_BYTES = 128 * BK, B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES;
    static constexpr int BUFS = BN >= 64 ? 2 : 4;            // accumulators
    static constexpr int COLS = BN * BUFS;
    static constexpr int STAGES = BN >= 128 ? 3 : BN == 64 ? 4 : BN == 32 ? 5 : 5;        // (two blocks an SM)
    static constexpr int RING = STAGES * STAGE;
    static constexpr int PART = BN * 128 * 4;                // a block's sums, in place of the ring
    static constexpr int AREA = RING > PART ? RING : PART;
    static constexpr int FACTORS = 16 * BN * 4;
    static constexpr int SMEM = AREA + FACTORS + 1024 + 256;
};

template <int BN>
__global__ void __launch_bounds__(192) fp8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                                                      const __grid_constant__ Fp8LinearParams p) {
    using C = Few<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* const factors = reinterpret_cast<float*>(smem + C::AREA);        // [16 blocks of K][BN]
    uint64_t* const full = reinterpret_cast<uint64_t*>(smem + C::AREA + C::FACTORS);
    uint64_t* const empty = full + C::STAGES;
    uint64_t* const acc_full = empty + C::STAGES;
    uint64_t* const acc_empty = acc_full + C::BUFS;
    uint32_t* const holder = reinterpret_cast<uint32_t*>(acc_empty + C::BUFS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0 && lane == 0) {
        tc::tma_prefetch_desc(&tmW);
        tc::tma_prefetch_desc(&tmX);
        for (int s = 0; s < C::STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
        for (int b = 0; b < C::BUFS; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], 4); }
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(holder, C::COLS);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *holder;
    pdl_grid_sync();

    const int share = blockIdx.x, shares = gridDim.x, n0 = blockIdx.y * 128, t0 = blockIdx.z * BN;
    const int blocks = (p.K + BK - 1) / BK;
    const int kb0 = (int)((long long)blocks * share / shares), kb1 = (int)((long long)blocks * (share + 1) / shares);
    if (warp == 0) {
        if (tc::elect_one()) {
            int it = 0;
            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                const int s = it % C::STAGES;
                if (!tc::mbar_wait_soon(&empty[s], ((it / C::STAGES) & 1) ^ 1)) { atomicExch(p.err, WAIT_FREE); break; }
                tc::mbar_expect_tx(&full[s], C::STAGE);
                tc::tma_load_2d(smem + s * C::STAGE, &tmW, &full[s], kb * BK, n0);
                tc::tma_load_2d(smem + s * C::STAGE + C::A_BYTES, &tmX, &full[s], kb * BK, t0);
            }
            // nothing is in flight when the block ends or its ring becomes something else
            for (int i = max(0, it - C::STAGES); i < it; ++i)
                if (!tc::mbar_wait(&full[i % C::STAGES], (i / C::STAGES) & 1)) { atomicExch(p.err, WAIT_LANDED); break; }
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = tc::idesc_f8(128, BN);
        const uint64_t base = tc::smem_desc_sw128(tc::smem_u32(smem));
        const uint32_t t_base = tc::warp_uniform(tmem);
        for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
            const int s = it % C::STAGES, buf = it % C::BUFS;
            if (!tc::mbar_wait_soon_warp(&acc_empty[buf], ((it / C::BUFS) & 1) ^ 1)) { if (lane == 0) atomicExch(p.err, WAIT_READ); break; }
            if (!tc::mbar_wait_soon_warp(&full[s], (it / C::STAGES) & 1)) { if (lane == 0) atomicExch(p.err, WAIT_FETCHED); break; }
            tc::fence_after_sync();
            const uint64_t a = tc::desc_at(base, s * C::STAGE), b = tc::desc_at(a, C::A_BYTES);
            if (tc::elect_one()) {
#pragma unroll
                for (int k = 0; k < BK / 32; ++k) tc::mma_f8_ss(t_base + buf * BN, tc::desc_at(a, k * 32), tc::desc_at(b, k * 32), idesc, k > 0 ? 1u : 0u);
                tc::mma_commit(&empty[s]);
                tc::mma_commit(&acc_full[buf]);
            }
            __syncwarp();
        }
    } else {
        const int q = warp & 3, tid = threadIdx.x - 64, feature = q * 32 + lane;
        const float* const scales = p.scale + (size_t)blockIdx.y * p.lds;
        float acc[BN];
#pragma unroll
        for (int j = 0; j < BN; ++j) acc[j] = 0.f;
        bool ok = true;
        for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {     // (warps whose wait ran out keep meeting the others)
            if (it == 0 || (kb & 15) == 0) {                 // factors of up to sixteen blocks: a thread has a row's
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int first = kb & ~15;
                if (tid < BN) {
                    uint4 e = make_uint4(0, 0, 0, 0);
                    if (t0 + tid < p.T) e = __ldg(reinterpret_cast<const uint4*>(p.exps + (size_t)(t0 + tid) * p.lde + first));
                    const uint32_t w[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (first + i >= kb && first + i < kb1)
                            factors[i * BN + tid] = __ldg(scales + first + i) * two_to((w[i / 4] >> (i % 4 * 8)) & 255u);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
            }
            const int buf = it % C::BUFS;
            if (ok) {
                ok = tc::mbar_wait_soon_warp(&acc_full[buf], (it / C::BUFS) & 1);
                if (!ok && lane == 0) atomicExch(p.err, WAIT_SUMS);
            }
            tc::fence_after_sync();
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + buf * BN;
            const float4* const f = reinterpret_cast<const float4*>(factors + (kb & 15) * BN);
#pragma unroll
            for (int c = 0; c < BN; c += 16) {
                uint32_t r[16];
                tc::tmem_ld_32x16(at + c, r);
                tc::tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 g = f[(c + j) / 4];
                    acc[c + j] = fmaf(__uint_as_float(r[j]), g.x, acc[c + j]);
                    acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), g.y, acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), g.z, acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), g.w, acc[c + j + 3]);
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
        }
        // the ring is free: all products of this block have been waited for.  [row][feature]: lanes side by side
        float* const part = reinterpret_cast<float*>(smem);
        if (ok) {
#pragma unroll
            for (int j = 0; j < BN; ++j) part[j * 128 + feature] = acc[j];
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::cluster_sync();
    {
        const int rows = min(BN, p.T - t0), units = rows * 32;
        const uint32_t part = tc::smem_u32(smem);
        for (int u = share * 192 + threadIdx.x; u < units; u += shares * 192) {
            const int t = u / 32, f = u % 32 * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int r = 0; r < shares; ++r) {
                const float4 a = ld_cluster(part + (t * 128 + f) * 4, r);
                v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
            }
            const int n = n0 + f;
            const size_t at = (size_t)(t0 + t) * p.ldy + n;
            if (n + 4 <= p.N) {
                if (p.out_f32) *reinterpret_cast<float4*>((float*)p.y + at) = v;
                else *reinterpret_cast<uint2*>((bf16*)p.y + at) = make_uint2(f2_to_bf162(v.x, v.y), f2_to_bf162(v.z, v.w));
            } else {
                const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) {
                        if (p.out_f32) ((float*)p.y)[at + i] = x[i];
                        else ((bf16*)p.y)[at + i] = __float2bfloat16(x[i]);
                    }
            }
        }
    }
    tc::cluster_sync();                                          // nobody's sums go away while they are read
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, C::COLS);
    }
}

template <int BN>
int launch_few(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p, int shares, cudaStream_t s) {
    CUtensorMap tmW, tmX;
    if (const int rc = make_tmap_2d(&tmW, W, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)ldw, 128, BK)) return rc;
    if (const int rc = make_tmap_2d(&tmX, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.T, (uint64_t)p.K, (uint64_t)ldx, BN, BK)) return rc;
    auto kern = fp8_few_kernel<BN>;
    static SmemOptIn optin;
    if (const int rc = optin((const void*)kern, Few<BN>::SMEM)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(shares, (p.N + 127) / 128, (p.T + BN - 1) / BN);
    cfg.blockDim = 192;
    cfg.dynamicSmemBytes = Few<BN>::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = shares;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_sl_pdl_enabled ? 2 : 1;
    ++g_sl_kernel_launches;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kern, tmW, tmX, p);
    return rc != cudaSuccess ? (int)rc : SL_LAUNCH_CHECK();
}

bool aligned(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p) {
    const int blocks = (p.K + BK - 1) / BK;
    return p.K > 0 && p.K % 16 == 0 && ldx % 16 == 0 && ldw % 16 == 0 && p.lde % 16 == 0 && p.lds >= blocks && p.lde >= blocks &&
           (((uintptr_t)x | (uintptr_t)W | (uintptr_t)p.exps | (uintptr_t)p.y) & 15) == 0;
}

}  // namespace

// x: codes [T, K], rows `ldx` bytes apart; W: codes [N, K], rows `ldw` apart.  K, ldx, ldw and the rows of exponents are multiples of 16 and start there;
// rows of y hold whole pieces of 16 bytes.
SL_API int sl_fp8_linear(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams* params, cudaStream_t s) {
    const Fp8LinearParams& p = *params;
    if (p.T <= 0 || p.N <= 0) return 0;
    if (!aligned(x, ldx, W, ldw, p) || p.ldy % (p.out_f32 ? 4 : 8) != 0 || (p.N + 127) / 128 > 65535) return -1;
    if (p.T > 128) return fp8_pair(x, ldx, W, ldw, p, false, s);
    const int bn = p.T <= 16 ? 16 : p.T <= 32 ? 32 : p.T <= 64 ? 64 : 128;
    const long long tiles = (long long)((p.N + 127) / 128) * ((p.T + bn - 1) / bn);
    const int blocks = (p.K + BK - 1) / BK;
    int shares = 1;
    while (shares < 8 && tiles * shares * 2 <= 296 && blocks >= shares * 4) shares *= 2;
    if (bn == 16) return launch_few<16>(x, ldx, W, ldw, p, shares, s);
    if (bn == 32) return launch_few<32>(x, ldx, W, ldw, p, shares, s);
    if (bn == 64) return launch_few<64>(x, ldx, W, ldw, p, shares, s);
    return launch_few<128>(x, ldx, W, ldw, p, shares, s);
}

// y: codes [T, N / 2] of silu(gate) * up, with exponents exps_out; W: N / 2 gate rows | N / 2 up rows, a multiple of 128 each.
SL_API int sl_fp8_gate_up(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams* params, cudaStream_t s) {
    const Fp8LinearParams& p = *params;
    if (p.T <= 0 || p.N <= 0) return 0;
    if (!aligned(x, ldx, W, ldw, p) || p.N % 256 != 0 || p.ldy % 16 != 0) return -1;
    return fp8_pair(x, ldx, W, ldw, p, true, s);
}
