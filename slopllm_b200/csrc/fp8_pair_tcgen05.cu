// Products of many rows in 8 bits with FP8 weights on pairs of SMs (tcgen05 `cta_group::2`, kind::f8f6f4): the sums of fp8_gemm_tcgen05.cu, and the
// gated activation of a feed-forward, in 8 bits, without its gate and up rows crossing memory.
//
// A pair works on 256 rows by 256 or 128 columns, each SM with its 128 rows of the operand and of the result and half of the weights' rows.  A block of
// 128 values of K is a product by itself in tensor memory (two accumulators of 256 columns, four of 128), because its factor S[n / 128, b] * 2^E[t, b]
// differs from the next one's:
//   warp 0     fetches its SM's operand halves (TMA, five or six blocks of K ahead)
//   warp 1     of the leading SM multiplies
//   warps 4-11 take a block's sums out of tensor memory and add them, times their factor, to fp32 registers: a thread has a row and half of the columns, an
//              instruction for two multiply-adds, while the tensor cores are at the next block (warps 2 and 3 only give their registers)
// Bound by the tensor cores' work beside its feeding: 4096 rows by 12288 x 4096 take 186 us (2.2 PFLOP/s; 0.65 of twice the measured bf16 rate).  The products
// by themselves take 127, with their operands' copies 150, with the sums' way out of tensor memory and no copies 170.  Two products of 128 columns in
// place of one of 256 read an operand twice from shared memory, whose 128 bytes a cycle are all in use (531 and 482 us for 8192 rows by 8192 x 8192); 16
// warps that add up do not have the registers.
//
// Tiles of 128 columns are for calls that have too few of the others to go round: 512 rows by 4096 x 12288 38 us in place of 47.  A block of K takes 0.30 us in
// one, of which 0.18 are the signals between the warps of two SMs (0.24 with those of the copies); of 256 columns 0.43.  The sums of two blocks in a thread's
// registers, so that one is on its way while the other is added, made it slower (0.37).
//
// Persistent over the tiles, one pair per two SMs.  Registers: 384 threads begin with 168 (64512); the first four warps keep 40, the adders take 232
// (5120 + 59392).
//
// All mbarrier waits are bounded; where one runs out, the error word is set and both SMs of the pair still meet at the end.
#include <algorithm>
#include <type_traits>

#include "f32x2.cuh"
#include "fp8_rows.cuh"
#include "tcgen05_pair.cuh"

namespace {

constexpr int BM = 128, BK = 128, ADDERS = 8, THREADS = 128 + ADDERS * 32;
constexpr int X_BYTES = BM * BK;                             // rows of one SM
constexpr int FEW_REGS = 40, MANY_REGS = 232;
static_assert(128 * FEW_REGS + ADDERS * 32 * MANY_REGS <= THREADS * 168, "registers are moved, not made");
constexpr int PIECE = 32 * 128;                              // a warp's part of the result on its way out: 128 bytes of 32 rows
constexpr int OUT = 2 * ADDERS * PIECE;                      // two a warp; gated: half of it for codes, half for sums that threads of a row exchange
static_assert(OUT / 2 >= 2 * 128 * 32 * 4, "32 columns of gate and up sums");
template <int BN>
struct Cut {                                                 // tiles of 256 rows by BN columns
    static constexpr int STAGE = X_BYTES + BN / 2 * BK, STAGES = BN == 256 ? 5 : 6, BUFS = 512 / BN;
    static constexpr int SMEM = STAGES * STAGE + OUT + 1024 + 256;
};
enum { WAIT_FREE = 75, WAIT_LANDED, WAIT_READ, WAIT_FETCHED, WAIT_SUMS };       // numbers of waits that run out

struct Tiles { int m, n, total; };

// silu(g) * u in fp32 (off by some 20 last places where the gate is -16, less above)
__device__ __forceinline__ float silu_mul(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// A warp's piece of the result, shared memory to memory, and the wait until the last one has left shared memory; by the same thread.
__device__ __forceinline__ void bulk_store(const CUtensorMap* map, const void* src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(tc::smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int OTHERS>
__device__ __forceinline__ void bulk_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(OTHERS) : "memory"); }
__device__ __forceinline__ void meet() { asm volatile("bar.sync 1, 256;" ::: "memory"); }      // the adders

template <int BN, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) fp8_pair_kernel(const __grid_constant__ CUtensorMap tmX,
                                                                                    const __grid_constant__ CUtensorMap tmW,
                                                                                    const __grid_constant__ CUtensorMap tmY,
                                                                                    const __grid_constant__ Fp8LinearParams p,
                                                                                    const __grid_constant__ Tiles tiles) {
    static_assert(!GATED || BN == 256, "a block of gate and one of up rows");
    constexpr int STAGE = Cut<BN>::STAGE, STAGES = Cut<BN>::STAGES, BUFS = Cut<BN>::BUFS, OWN = BN / 2;       // columns of a thread
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* const out = smem + STAGES * STAGE;
    uint64_t* const full = reinterpret_cast<uint64_t*>(out + OUT);
    uint64_t* const empty = full + STAGES;
    uint64_t* const acc_full = empty + STAGES;               // [BUFS] a block's sums are there
    uint64_t* const acc_empty = acc_full + BUFS;             // [BUFS] ... are read by both blocks (the leader's counts)
    uint32_t* const holder = reinterpret_cast<uint32_t*>(acc_empty + BUFS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::warp_uniform(tc::cluster_rank());
    if (warp == 0 && lane == 0) {
        tc::tma_prefetch_desc(&tmX);
        tc::tma_prefetch_desc(&tmW);
        tc::tma_prefetch_desc(&tmY);
        for (int s = 0; s < STAGES; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
        for (int b = 0; b < BUFS; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], 2 * ADDERS); }
        tc::mbar_fence_init();
    }
    if (warp == 1) tc::tmem_alloc_pair(holder, BUFS * BN);
    tc::fence_before_sync();
    __syncthreads();
    tc::cluster_sync();                                      // the other block's barriers exist
    tc::fence_after_sync();
    const uint32_t tmem = *holder;
    pdl_grid_sync();

    const int pairs = gridDim.x / 2, first = blockIdx.x / 2, blocks = (p.K + BK - 1) / BK;
    auto coords = [&](int tile, int& m0, int& n0) {
        // bands of eight row tiles, column by column: the band's rows stay in L2 while the weights stream past
        const int band = tile / (8 * tiles.n), in = tile % (8 * tiles.n), rows = min(8, tiles.m - band * 8);
        m0 = (band * 8 + in % rows) * 2 * BM;
        n0 = in / rows * (GATED ? BN / 2 : BN);
    };
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW_REGS));
        if (warp == 0) {
            if (lane == 0) {
                int it = 0;
                bool ok = true;
                for (int tile = first; tile < tiles.total && ok; tile += pairs) {
                    int m0, n0;
                    coords(tile, m0, n0);
                    // the two SMs hold half of a tile's weight rows each; gated: one the gate rows of 128 columns, the other their up rows
                    const int w0 = n0 + (int)rank * (GATED ? p.N / 2 : BN / 2);
                    for (int kb = 0; kb < blocks; ++kb, ++it) {
                        const int s = it % STAGES;
                        if (!tc::mbar_wait_soon(&empty[s], ((it / STAGES) & 1) ^ 1)) { atomicExch(p.err, WAIT_FREE); ok = false; break; }
                        if (rank == 0) tc::mbar_expect_tx(&full[s], 2 * STAGE);
                        const uint32_t bar = tc::in_leader(&full[s]);
                        uint8_t* const x = smem + s * STAGE;
                        tc::tma_load_2d_pair(x, &tmX, bar, kb * BK, m0 + (int)rank * BM);
                        tc::tma_load_2d_pair(x + X_BYTES, &tmW, bar, kb * BK, w0);
                    }
                }
                // Nothing is in flight when the pair ends, also where a wait ran out.  Both SMs' copies of a block signal the leader's `full`, so the
                // leader waits for all that it armed.  Where it armed less than the other SM asked for, commits stop as well and the other SM
                // waits here until the time limit, long after its copies have landed.
                bool landed = true;
                for (int i = std::max(0, it - STAGES); i < it && (landed || rank == 0); ++i)
                    landed &= tc::mbar_wait(rank == 0 ? &full[i % STAGES] : &empty[i % STAGES], (i / STAGES) & 1);
                if (!landed) atomicExch(p.err, WAIT_LANDED);
            }
        } else if (warp == 1) {
            if (rank == 0) {
                constexpr uint32_t idesc = tc::idesc_f8(2 * BM, BN);
                const uint64_t base = tc::smem_desc_sw128(tc::smem_u32(smem));
                const uint32_t t_base = tc::warp_uniform(tmem);
                bool ok = true;
                int it = 0;
                for (int tile = first; tile < tiles.total && ok; tile += pairs)
                    for (int kb = 0; kb < blocks; ++kb, ++it) {
                        const int s = it % STAGES, buf = it % BUFS;
                        // the operands first: they are early, and nothing then stands between an accumulator's return and its next products
                        if (!tc::mbar_wait_soon_warp(&full[s], (it / STAGES) & 1)) { if (lane == 0) atomicExch(p.err, WAIT_FETCHED); ok = false; break; }
                        if (!tc::mbar_wait_soon_warp(&acc_empty[buf], ((it / BUFS) & 1) ^ 1)) { if (lane == 0) atomicExch(p.err, WAIT_READ); ok = false; break; }
                        tc::fence_after_sync();
                        const uint64_t a = tc::desc_at(base, s * STAGE), b = tc::desc_at(a, X_BYTES);
                        if (tc::elect_one()) {
#pragma unroll
                            for (int k = 0; k < BK / 32; ++k)
                                tc::mma_f8_pair(t_base + buf * BN, tc::desc_at(a, k * 32), tc::desc_at(b, k * 32), idesc, k > 0 ? 1u : 0u);
                            tc::commit_pair(&acc_full[buf]);
                            tc::commit_pair(&empty[s]);
                        }
                        __syncwarp();
                    }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY_REGS));
        const int q = warp & 3, half = (warp - 4) >> 2, in_tile = q * 32 + lane;
        bool ok = true;                                      // (threads whose wait ran out keep meeting the others)
        const uint32_t empty_at = tc::in_leader(acc_empty);
        const float* scales;
        const uint4* exps;
        uint4 e_now, e_next;
        float scale;
        auto begin = [&](int tile) {                         // the first factors of a tile are asked for before the last one's result is stored
            int m0, n0;
            coords(tile, m0, n0);
            // scales of columns behind the last are those of the last
            const int scale_row = GATED ? (n0 + half * (p.N / 2)) / 128 : min(n0 + half * OWN, p.N - 1) / 128;
            scales = p.scale + (size_t)scale_row * p.lds;
            exps = reinterpret_cast<const uint4*>(p.exps + (size_t)min(m0 + (int)rank * BM + in_tile, p.T - 1) * p.lde);
            e_next = __ldg(exps);
            scale = __ldg(scales);
        };
        if (first < tiles.total) begin(first);
        int it = 0;
        for (int tile = first; tile < tiles.total; tile += pairs) {
            f32x2 acc[OWN / 2];
#pragma unroll
            for (int i = 0; i < OWN / 2; ++i) acc[i] = pair(0.f, 0.f);
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + half * OWN;
            uint32_t r[OWN == 128 ? 5 : 4][16];
#pragma unroll 1
            for (int kb = 0; kb < blocks; ++kb, ++it) {
                if ((kb & 15) == 0) {                        // the exponents of sixteen blocks of K are a load, one such load ahead
                    e_now = e_next;
                    if (kb + 16 < blocks) e_next = __ldg(exps + kb / 16 + 1);
                }
                const uint32_t word = kb & 8 ? (kb & 4 ? e_now.w : e_now.z) : (kb & 4 ? e_now.y : e_now.x);
                const int e = max(FP8_LOW + FP8_BIAS, min(FP8_HIGH + FP8_BIAS, (int)((word >> ((kb & 3) * 8)) & 255u)));
                const float f = scale * __uint_as_float((uint32_t)e << 23);
                const f32x2 ff = pair(f, f);
                scale = __ldg(scales + min(kb + 1, blocks - 1));
                const uint32_t at = lanes + it % BUFS * BN;
                auto add = [&](const uint32_t (&v)[16], int c) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        acc[c * 8 + i] = fma2(pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), ff, acc[c * 8 + i]);
                };
                if (ok) {
                    ok = tc::mbar_wait_soon_warp(&acc_full[it % BUFS], (it / BUFS) & 1);
                    if (!ok && lane == 0) atomicExch(p.err, WAIT_SUMS);
                }
                tc::fence_after_sync();
                auto back = [&] {
                    tc::tmem_ld_wait();
                    tc::fence_before_sync();
                    if (tc::elect_one()) tc::arrive_cluster_soon(empty_at + it % BUFS * 8);
                };
                // The accumulator goes back as soon as it is read.  Registers hold 80 of 128 columns, so 48 are added up in between.
                if constexpr (OWN == 128) {
#pragma unroll
                    for (int c = 0; c < 5; ++c) tc::tmem_ld_32x16(at + c * 16, r[c]);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 3; ++c) add(r[c], c);
#pragma unroll
                    for (int c = 0; c < 3; ++c) tc::tmem_ld_32x16(at + 80 + c * 16, r[c]);
                    back();
                    add(r[3], 3);
                    add(r[4], 4);
#pragma unroll
                    for (int c = 0; c < 3; ++c) add(r[c], 5 + c);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc::tmem_ld_32x16(at + c * 16, r[c]);
                    back();
#pragma unroll
                    for (int c = 0; c < 4; ++c) add(r[c], c);
                }
            }
            int m0, n0;
            coords(tile, m0, n0);
            const int row0 = m0 + (int)rank * BM + q * 32;
            if (tile + pairs < tiles.total) begin(tile + pairs);
            // 16-byte piece j of this lane's row, as the copy out of shared memory has them (128-byte swizzle)
            auto piece = [&](uint8_t* at, int j) { return reinterpret_cast<uint4*>(at + lane * 128 + ((j ^ (lane & 7)) << 4)); };
            if constexpr (GATED) {
                // Of a row's 128 columns the thread with the gate's sums makes the first 64, the one with the up rows' the others.  They exchange
                // 32 columns at a time, [side][column][row].
                float* const swap = reinterpret_cast<float*>(out + OUT / 2);
                if (half == 0 && lane == 0) bulk_read<0>();     // (codes of the last tile are out before new ones are written behind the first meeting)
                float act[64];
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    float* const mine = swap + half * 32 * 128 + in_tile;
                    const float* const theirs = swap + (half ^ 1) * 32 * 128 + in_tile;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 lo = unpair(acc[c / 2 + i]), hi = unpair(acc[32 + c / 2 + i]);
                        mine[(2 * i) * 128] = half ? lo.x : hi.x;
                        mine[(2 * i + 1) * 128] = half ? lo.y : hi.y;
                    }
                    meet();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 lo = unpair(acc[c / 2 + i]), hi = unpair(acc[32 + c / 2 + i]);
                        const float x = theirs[(2 * i) * 128], y = theirs[(2 * i + 1) * 128];
                        act[c + 2 * i] = half ? silu_mul(x, hi.x) : silu_mul(lo.x, x);
                        act[c + 2 * i + 1] = half ? silu_mul(y, hi.y) : silu_mul(lo.y, y);
                    }
                    meet();
                }
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 64; ++i) top = max(top, fp8_finite(act[i]) ? __float_as_uint(act[i]) & 0x7fffffffu : 0u);
                uint32_t* const tops = reinterpret_cast<uint32_t*>(swap) + in_tile;
                tops[half * 128] = top;
                meet();
                top = max(tops[0], tops[128]);
                const int e = fp8_exponent(top);
                const float down = __uint_as_float((uint32_t)(127 - e) << 23);
                uint8_t* const codes = out + q * PIECE;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t c[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float a = act[16 * j + 4 * i + k];
                            v[k] = fp8_finite(a) ? a * down : __uint_as_float(0x7fffffffu);
                        }
                        c[i] = fp8_codes(v);
                    }
                    *piece(codes, half * 4 + j) = make_uint4(c[0], c[1], c[2], c[3]);
                }
                tc::fence_proxy_async_smem();
                meet();                                      // (also: `tops` is read before it is written again)
                if (half == 0) {
                    if (lane == 0 && row0 < p.T) {
                        bulk_store(&tmY, codes, n0, row0);
                        bulk_commit();
                    }
                    if (row0 + lane < p.T) p.exps_out[(size_t)(row0 + lane) * p.lde_out + n0 / 128] = (uint8_t)(e + FP8_BIAS);
                }
            } else {
                // 128 bytes of each of the warp's rows at a time; rows and columns that are not there are left out by the copy
                uint8_t* const mine = out + (warp - 4) * 2 * PIECE;
                const int col = n0 + half * OWN;
                auto store = [&](auto bits, auto per) {      // `per` values to 16 bytes
                    constexpr int PIECES = OWN / (8 * decltype(per)::value);       // (one of them: the next tile's goes where this one's is)
#pragma unroll
                    for (int c = 0; c < OWN; c += 8 * per) {
                        uint8_t* const here = mine + c / (8 * per) % 2 * PIECE;
                        if (lane == 0) bulk_read<PIECES == 1 ? 0 : 1>();       // (what was in it is out: at most the other one is still on its way)
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; ++j) *piece(here, j) = bits(c + j * per);
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            if (row0 < p.T && col + c < p.N) bulk_store(&tmY, here, col + c, row0);
                            bulk_commit();                   // (an empty group keeps the count)
                        }
                    }
                };
                if (p.out_f32)
                    store([&](int c) {
                        const float2 a = unpair(acc[c / 2]), b = unpair(acc[c / 2 + 1]);
                        return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
                    }, std::integral_constant<int, 4>{});
                else
                    store([&](int c) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float2 a = unpair(acc[c / 2 + i]);
                            w[i] = f2_to_bf162(a.x, a.y);
                        }
                        return make_uint4(w[0], w[1], w[2], w[3]);
                    }, std::integral_constant<int, 8>{});
            }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");          // the result is out
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::cluster_sync();                                      // neither block leaves while the other may still signal it
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_dealloc_pair(tmem, BUFS * BN);
    }
}

// Pairs that the device runs at the same time (a persistent grid must not be larger).
template <int BN, bool GATED>
int max_pairs() {
    static const int n = [] {                                // (made once, whichever thread comes first; the devices are alike)
        cudaFuncSetAttribute(fp8_pair_kernel<BN, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cut<BN>::SMEM);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = 148;
        cfg.blockDim = THREADS;
        cfg.dynamicSmemBytes = Cut<BN>::SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int got = 0;
        if (cudaOccupancyMaxActiveClusters(&got, fp8_pair_kernel<BN, GATED>, &cfg) != cudaSuccess || got < 1) {
            cudaGetLastError();
            got = -1;
        }
        return got;
    }();
    return n;
}

template <int BN, bool GATED>
int launch(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p, cudaStream_t s) {
    CUtensorMap tmX, tmW, tmY;
    if (const int rc = make_tmap_2d(&tmX, x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.T, (uint64_t)p.K, (uint64_t)ldx, BM, BK)) return rc;
    if (const int rc = make_tmap_2d(&tmW, W, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)ldw, BN / 2, BK)) return rc;
    const int size = GATED ? 1 : p.out_f32 ? 4 : 2;
    const auto kind = GATED ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : p.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (const int rc = make_tmap_2d(&tmY, p.y, kind, size, (uint64_t)p.T, (uint64_t)(GATED ? p.N / 2 : p.N), (uint64_t)p.ldy * size, 32, 128 / size)) return rc;
    static SmemOptIn optin;
    if (const int rc = optin((const void*)fp8_pair_kernel<BN, GATED>, Cut<BN>::SMEM)) return rc;
    const int pairs = max_pairs<BN, GATED>();
    if (pairs < 1) return -1;
    const Tiles tiles = {(p.T + 2 * BM - 1) / (2 * BM), (p.N + BN - 1) / BN, ((p.T + 2 * BM - 1) / (2 * BM)) * ((p.N + BN - 1) / BN)};
    sl_launch(fp8_pair_kernel<BN, GATED>, dim3(2 * std::min(tiles.total, pairs)), THREADS, Cut<BN>::SMEM, s, tmX, tmW, tmY, p, tiles);
    return SL_LAUNCH_CHECK();
}

}  // namespace

int fp8_pair(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p, int columns, cudaStream_t s) {
    return columns == 256 ? launch<256, false>(x, ldx, W, ldw, p, s) : launch<128, false>(x, ldx, W, ldw, p, s);
}
int fp8_pair_gated(const void* x, int ldx, const void* W, int ldw, const Fp8LinearParams& p, cudaStream_t s) {
    return launch<256, true>(x, ldx, W, ldw, p, s);
}
