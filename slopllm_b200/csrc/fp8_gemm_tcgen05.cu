// y[T, N] = X[T, K] * W[N, K]^T on the 8-bit tensor cores (tcgen05 kind::f8f6f4), rows and weights both e4m3: X with an exponent byte for each 128 values
// of a row, W with an fp32 scale for each block of 128 x 128.
//
//   y[t, n] = sum over blocks b of  S[n / 128, b] * 2^(E[t, b] - 127) * (sum over the block's k of X[t, k] * W[n, k])
//
// The scales differ from block to block of K, so a block's sums leave the tensor memory 128 values of K later and are added, times their factor, in fp32
// registers: one multiply-add a value and block, beside 128 multiply-adds of the tensor core.  Few rows here, many on pairs of SMs (fp8_pair_tcgen05.cu).
//
// All mbarrier waits are bounded; where one runs out, the error word is set and the blocks still meet at the end.
#include <algorithm>

#include "f32x2.cuh"
#include "fp8_rows.cuh"
#include "tcgen05_pair.cuh"

namespace {

constexpr int BK = 128;                                      // values (bytes) of a block of K
enum { WAIT_FREE = 80, WAIT_LANDED, WAIT_READ, WAIT_FETCHED, WAIT_SUMS, WAIT_SENT };       // numbers of waits that run out

__device__ __forceinline__ float two_to(int byte) {          // 2^(byte - 127), for the exponents that writers leave
    return __uint_as_float((uint32_t)(max(FP8_LOW, min(FP8_HIGH, byte - FP8_BIAS)) + 127) << 23);
}
// Address of `at` (shared memory of this block) in block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t at, uint32_t rank) {
    uint32_t far;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(at), "r"(rank));
    return far;
}
// A piece of this block's shared memory into another block's, counted by a barrier of that block.
__device__ __forceinline__ void send(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(to), "r"(tc::smem_u32(from)), "r"(bytes), "r"(bar) : "memory");
}
// The wait for what other blocks have sent (bounded).
__device__ __forceinline__ bool wait_sent(uint64_t* bar) {
    const uint32_t at = tc::smem_u32(bar);
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok) : "r"(at) : "memory");
        if (ok) return true;
        if (i == 64) t0 = tc::globaltimer_ns();
        if (i > 64 && (i & 255u) == 255u && tc::globaltimer_ns() - t0 > 2000000000ull) return false;
    }
}
// A meeting of the cluster that passes no memory on: nobody waits for loads and stores in flight (a release does: 6000 cycles beside a full memory).
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// ---- few rows: weights are the 128-row operand, rows the columns ---------------------------------------------------------------------------
//
// A block has 128 features, up to BN rows and a share of K; the blocks of a cluster have the shares of the same features.  Each block completes BN / shares
// of the rows: the others send their sums into its shared memory, and it adds them in the order of the shares.  Warp 0 fetches (TMA ring), warp 1
// multiplies, the others have a feature and up to 32 rows a thread and add up.
//
// Bound by the weights' bytes and by what is around them: a launch (1.2 us), the first bytes (1.5), the joining of the shares (1).  8 rows by 28672 x 4096:
// 22.6 us, 5.2 TB/s; 1 by 6144 x 4096: 7.8 us; 29 by 4096 x 12288: 13.7.  Weights are the operand of 128 rows because those are full whatever the batch.
// 128 rows of X a block were slower than 64 twice (their sums do not fit the registers).
template <int BN>
struct Few {
    static constexpr int A_BYTES = 128 * BK, B_BYTES = BN * BK, STAGE = A_BYTES + B_BYTES;
    static constexpr int BUFS = 4;                           // accumulators
    static constexpr int COLS = BN * BUFS;
    static constexpr int PARTS = BN >= 64 ? 2 : 1, OWN = BN / PARTS;        // threads of a feature, rows of one
    static constexpr int ADDERS = 4 * PARTS, THREADS = 64 + 32 * ADDERS;
    static constexpr int RESIDENT = BN == 16 ? 3 : 2;        // blocks an SM
    static constexpr int STAGES = BN == 32 ? 4 : 3;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int SENT = BN * 128 * 4;                // [share][own row][feature]
    static constexpr int FACTORS = 16 * BN * 4;
    static constexpr int SMEM = RING + SENT + FACTORS + 1024 + 256;
};

template <int BN>
__global__ void __launch_bounds__(Few<BN>::THREADS, Few<BN>::RESIDENT) fp8_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                                                      const __grid_constant__ Fp8LinearParams p) {
    using C = Few<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* const sent = reinterpret_cast<float*>(smem + C::RING);
    float* const factors = reinterpret_cast<float*>(smem + C::RING + C::SENT);             // [16 blocks of K][BN]
    uint64_t* const full = reinterpret_cast<uint64_t*>(smem + C::RING + C::SENT + C::FACTORS);
    uint64_t* const empty = full + C::STAGES;
    uint64_t* const acc_full = empty + C::STAGES;
    uint64_t* const acc_empty = acc_full + C::BUFS;
    uint64_t* const all_sent = acc_empty + C::BUFS;          // the other blocks' sums of this block's rows are there
    uint32_t* const holder = reinterpret_cast<uint32_t*>(all_sent + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int share = blockIdx.x, shares = gridDim.x, n0 = blockIdx.y * 128, t0 = blockIdx.z * BN;
    // `per` rows are completed by a block, `mine` of them are there in this one (shares and BN are powers of two)
    const int rows = min(BN, p.T - t0), per = BN / shares, mine = max(0, min(per, rows - share * per));
    if (warp == 0 && lane == 0) {
        tc::tma_prefetch_desc(&tmW);
        tc::tma_prefetch_desc(&tmX);
        for (int s = 0; s < C::STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
        for (int b = 0; b < C::BUFS; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], C::ADDERS); }
        tc::mbar_init(all_sent, 1);
        tc::mbar_expect_tx(all_sent, shares > 1 ? shares * mine * 128 * 4 : 0);
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
    cluster_arrive_relaxed();                                // the barriers exist (waited for before the first is used from afar)
    pdl_grid_sync();

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
        const int q = warp & 3, tid = threadIdx.x - 64, feature = q * 32 + lane, own = (warp - 2) / 4 * C::OWN;
        const float* const scales = p.scale + (size_t)blockIdx.y * p.lds;
        f32x2 acc[C::OWN / 2];
#pragma unroll
        for (int j = 0; j < C::OWN / 2; ++j) acc[j] = pair(0.f, 0.f);
        bool ok = true;
        for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {     // (warps whose wait ran out keep meeting the others)
            if (it == 0 || (kb & 15) == 0) {                 // factors of up to sixteen blocks: a thread has a row's
                asm volatile("bar.sync 1, %0;" ::"n"(32 * C::ADDERS) : "memory");
                const int from = kb & ~15;
                if (tid < BN) {
                    uint4 e = make_uint4(0, 0, 0, 0);
                    if (t0 + tid < p.T) e = __ldg(reinterpret_cast<const uint4*>(p.exps + (size_t)(t0 + tid) * p.lde + from));
                    const uint32_t w[4] = {e.x, e.y, e.z, e.w};
                    float f[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) f[i] = from + i >= kb && from + i < kb1 ? __ldg(scales + from + i) : 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) factors[i * BN + tid] = f[i] * two_to((w[i / 4] >> (i % 4 * 8)) & 255u);
                }
                asm volatile("bar.sync 1, %0;" ::"n"(32 * C::ADDERS) : "memory");
            }
            const int buf = it % C::BUFS;
            if (ok) {
                ok = tc::mbar_wait_soon_warp(&acc_full[buf], (it / C::BUFS) & 1);
                if (!ok && lane == 0) atomicExch(p.err, WAIT_SUMS);
            }
            tc::fence_after_sync();
            const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + buf * BN + own;
            const ulonglong2* const f = reinterpret_cast<const ulonglong2*>(factors + (kb & 15) * BN + own);
#pragma unroll
            for (int c = 0; c < C::OWN; c += 16) {
                uint32_t r[16];
                tc::tmem_ld_32x16(at + c, r);
                tc::tmem_ld_wait();
                if (c + 16 == C::OWN) {
                    tc::fence_before_sync();
                    if (tc::elect_one()) tc::mbar_arrive(&acc_empty[buf]);
                }
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const ulonglong2 g = f[(c + j) / 4];
                    acc[(c + j) / 2] = fma2(pair(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), g.x, acc[(c + j) / 2]);
                    acc[(c + j) / 2 + 1] = fma2(pair(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), g.y, acc[(c + j) / 2 + 1]);
                }
            }
        }
        if (shares == 1) {
            const int n = n0 + feature;
            if (n < p.N) {
#pragma unroll
                for (int j = 0; j < C::OWN; ++j) {
                    const float2 a = unpair(acc[j / 2]);
                    const float v = j % 2 ? a.y : a.x;
                    const size_t at = (size_t)(t0 + own + j) * p.ldy + n;
                    if (own + j < rows) {
                        if (p.out_f32) ((float*)p.y)[at] = v;
                        else ((bf16*)p.y)[at] = __float2bfloat16(v);
                    }
                }
            }
        } else {
            // [row][feature] in the ring, which is free (all products of this block have been waited for), then a piece to each block.  (Stores into the
            // other blocks' memory, 128 bytes a warp, took 2000 cycles for 64 rows where they went to all blocks in turn, 6500 where not.)
            float* const part = reinterpret_cast<float*>(smem) + own * 128 + feature;
#pragma unroll
            for (int j = 0; j < C::OWN / 2; ++j) {
                const float2 a = unpair(acc[j]);
                part[2 * j * 128] = a.x;
                part[(2 * j + 1) * 128] = a.y;
            }
            tc::fence_proxy_async_smem();
            cluster_wait();
            asm volatile("bar.sync 1, %0;" ::"n"(32 * C::ADDERS) : "memory");
            if (tid < shares) {
                const int r = (share + tid) & (shares - 1), n = min(per, rows - r * per);
                if (n > 0) send(in_block(tc::smem_u32(sent + share * per * 128), r), smem + r * per * 512, n * 512, in_block(tc::smem_u32(all_sent), r));
            }
        }
    }
    tc::fence_before_sync();
    __syncwarp();
    if (shares > 1) {
        if (warp < 2) cluster_wait();
        if (mine > 0 && !__all_sync(0xffffffffu, wait_sent(all_sent)) && lane == 0) atomicExch(p.err, WAIT_SENT);
        __syncwarp();
        cluster_arrive_relaxed();                            // this block has what was sent to it
        for (int u = threadIdx.x; u < mine * 32; u += C::THREADS) {
            const int f = u % 32 * 4, n = n0 + f;
            const float* const at_sent = sent + u / 32 * 128 + f;
            float4 v = *reinterpret_cast<const float4*>(at_sent);
            for (int r = 1; r < shares; ++r) {
                const float4 a = *reinterpret_cast<const float4*>(at_sent + r * per * 128);
                v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
            }
            const size_t at = (size_t)(t0 + share * per + u / 32) * p.ldy + n;
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
    __syncwarp();
    cluster_wait();                                          // nobody leaves before its sums have arrived
    __syncthreads();
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
    cfg.blockDim = Few<BN>::THREADS;
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

// Blocks that share a tile's K: twice as many while every block still has an SM to itself, and on to what is resident at once (some less: clusters leave
// SMs free) where each block keeps so many blocks of K.  Up to 16 rows, with 3 blocks an SM, microseconds with 2, 4 and 8 shares: 4096 x 4096 (32 tiles) 10.9,
// 8.7, 8.4; 9472 x 4096 (74) 12.8, 11.6, 13.7; 12288 x 4096 (96) 14.7, 13.3, 15.5; 4096 x 14336 (32) 23.6, 16.7, 14.9; 18944 x 4096 (148) 17.7, 18.9, 20.7.  With
// 2 blocks an SM instead 4096 x 4096 takes 8.0 (4 shares), but 9472 x 4096 12.1 (2), 12288 x 4096 14.5 (2) and 4096 x 14336 15.5 (4).  More rows, 2 blocks
// an SM: 64 by 4096 x 4096 12.8, 10.4, 10.9; 64 by 9472 x 4096 15.0, 18.4, 21.3; 64 by 4096 x 12288 24.6, 17.4, 16.0; with
// 4 and 8 shares 256 by 1024 x 2048 (32 tiles) 7.2, 8.4.
int shares_of(long long tiles, int blocks, int bn) {
    const int room = bn == 16 ? 384 : 256, least = bn == 16 ? 4 : 6;
    int shares = 1;
    while (shares < 8 && blocks >= 2 * shares && (tiles * shares * 2 <= 148 || (tiles * shares * 2 <= room && blocks >= 2 * shares * least))) shares *= 2;
    return shares;
}

long long cut(long long n, long long by) { return (n + by - 1) / by; }

// Microseconds of the three forms, fitted to what they take (launch and a block of K of one tile, rounds of tiles that run at once).  One SM: tiles of 64 rows
// by 128 columns, 296 at once, whose blocks of K take longer where two share an SM.  Pairs: 256 rows by 128 or 256 columns, 74 at once.
float time_of_few(long long T, long long N, long long K) {
    const long long tiles = cut(T, 64) * cut(N, 128), blocks = cut(K, BK);
    const int shares = shares_of(tiles, (int)blocks, 64);
    const float per = (float)blocks / (float)shares;
    return 5.5f + (float)cut(tiles * shares, 296) * (tiles * shares <= 148 ? 0.34f * per + 1.7f : 0.5f * per + 2.7f);
}
float time_of_pairs(long long T, long long N, long long K, int columns) {
    const long long blocks = cut(K, BK), rounds = cut(cut(T, 256) * cut(N, columns), 74);
    return columns == 128 ? 5.3f + (float)rounds * (0.30f * (float)blocks + 1.4f) : 4.4f + (float)rounds * (0.43f * (float)blocks + 2.f);
}

// Columns of a pair's tile, or 0 for tiles of one SM, which are always the faster form up to 64 rows (64 by 16384 x 2048: 13.5 us, pairs 14.8).
// Microseconds of one SM's tiles and pairs' of 128 and 256 columns: 128 by 6144 x 4096 16.6, 16.6, 20.1; 256 by 6144 x 4096 23.0, 16.6, 20.1; 128 by 24576 x
// 4096 41.8, 38.7, 36.4; 512 by 2321 x 5136 28.8, 19.3, 23.9; 512 by 4096 x 12288 55.6, 37.6, 46.6; 512 by 2048 x 8192 24.4, 25.8, 32.8; 1000 by 2048 x 2048 14.8, 11.4,
// 13.3; 1500 by 2048 x 8192 72, 47, 35; 4096 by 1024 x 8192 85, 51, 38.
int pair_columns(int T, int N, int K) {
    if (T <= 64) return 0;
    const float few = time_of_few(T, N, K), narrow = time_of_pairs(T, N, K, 128), wide = time_of_pairs(T, N, K, 256);
    return few <= std::min(narrow, wide) ? 0 : narrow < wide ? 128 : 256;
}

// Whether the activation of N gate and up columns is made in the pairs' epilogue (1.7 us a round), not by a pass over the fp32 rows of the product (3 us and the
// rows' way through memory).  Microseconds with and without: 192 by 16384 x 2048 17.4, 21.3; 256 by 8192 x 4096 22.8, 20.7; 333 by 8192 x 4096 23.6, 26.6; 1000 by
// 2048 x 8192 35.3, 31.5; 1500 by 2048 x 8192 36.1, 40.5; 65 by 2048 x 2048 14.3, 9.7.
bool gated_on_pairs(int T, int N, int K) {
    if (T <= 64) return false;
    const float wide = time_of_pairs(T, N, K, 256), rounds = (float)cut(cut(T, 256) * cut(N, 256), 74);
    const float apart = std::min(std::min(time_of_few(T, N, K), time_of_pairs(T, N, K, 128)), wide);
    return wide + 1.7f * rounds <= apart + 3.f + 0.95e-6f * (float)T * (float)N;
}

bool aligned(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p) {
    const int blocks = (p.K + BK - 1) / BK;
    return p.K > 0 && p.K % 16 == 0 && ldx % 16 == 0 && ldw % 16 == 0 && p.lde % 16 == 0 && p.lds >= blocks && p.lde >= blocks &&
           (((uintptr_t)x | (uintptr_t)W | (uintptr_t)p.exps | (uintptr_t)p.y) & 15) == 0;
}

}  // namespace

// x: codes [T, K], rows `ldx` bytes apart; W: codes [N, K], rows `ldw` apart.  K, ldx, ldw and the rows of exponents are multiples of 16 and start there;
// rows of y hold whole pieces of 16 bytes (the copy out of a pair's shared memory fills the last one up with zeros).
SL_API int sl_fp8_linear(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams* params, cudaStream_t s) {
    const Fp8LinearParams& p = *params;
    if (p.T <= 0 || p.N <= 0) return 0;
    if (!aligned(x, ldx, W, ldw, p) || p.ldy % (p.out_f32 ? 4 : 8) != 0 || (p.N + 127) / 128 > 65535) return -1;
    if (const int columns = pair_columns(p.T, p.N, p.K)) return fp8_pair(x, ldx, W, ldw, p, columns, s);
    const int bn = p.T <= 16 ? 16 : p.T <= 32 ? 32 : 64;
    if ((p.T + bn - 1) / bn > 65535) return -1;
    const int shares = shares_of((long long)((p.N + 127) / 128) * ((p.T + bn - 1) / bn), (p.K + BK - 1) / BK, bn);
    if (bn == 16) return launch_few<16>(x, ldx, W, ldw, p, shares, s);
    if (bn == 32) return launch_few<32>(x, ldx, W, ldw, p, shares, s);
    return launch_few<64>(x, ldx, W, ldw, p, shares, s);
}

// 1 where gate and up products of this size are made with their activation (sl_fp8_gate_up).
SL_API int sl_fp8_on_pairs(int T, int N, int K) { return gated_on_pairs(T, N, K); }

// y: codes [T, N / 2] of silu(gate) * up, with exponents exps_out; W: N / 2 gate rows | N / 2 up rows, a multiple of 128 each.
SL_API int sl_fp8_gate_up(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams* params, cudaStream_t s) {
    const Fp8LinearParams& p = *params;
    if (p.T <= 0 || p.N <= 0) return 0;
    if (!aligned(x, ldx, W, ldw, p) || p.N % 256 != 0 || p.ldy % 16 != 0) return -1;
    return fp8_pair_gated(x, ldx, W, ldw, p, s);
}
