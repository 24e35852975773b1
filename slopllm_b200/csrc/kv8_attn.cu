// Attention of one new token per sequence over the 8-bit key/value cache (kv8.cuh): every cached byte is read once, so what counts is bytes in
// flight and few instructions a byte.
//
// All histories are cut into tiles of 64 keys of one key head (and of up to 8 or 16 of its query heads); the tiles of the whole batch, one
// history behind the other, are dealt out in equal shares to the blocks of a head, so that a batch of ragged histories, one long history and many
// short ones fill the device alike.  Neighbouring blocks take the heads of one share: their rows are neighbours in memory, and are read at
// about the same time.  A history that lies in several shares leaves a partial result in each, which kv8_merge_kernel joins.  Where there is little work,
// kv8_cluster_kernel joins the parts itself.
//
// kv8_decode_kernel: a fetching warp brings tiles (TMA, swizzled) and their exponent bytes through a ring of stages, also across the ends of
// histories; one to three pairs of warps take tiles in turn, a warp 32 keys of one, with softmax states of their own and no barrier before a history's end.
//
//   S^T = K Q^T      keys are the 16-row operand: a lane's 16 bytes of two keys are four steps of the product as they lie, since any order
//                    of the summed dims will do that the queries follow
//   O^T += V^T P^T   a lane's 16 bytes of four keys, two keys' bytes interleaved, are the operand of 8 products: its rows are those dims
//
// e4m3 codes become fp16 exactly (mma.sync f16, fp32 sums); the queries are fp16 times a power of two per head, which loses less than 2^-24 of
// the largest value.  The keys' scales go onto the scores.  The values' scales go into the weights: the reference of a row is the maximum of
// score + exponent (in powers of two), so weights times scales stay within fp16, and the denominator takes the scale out again.  Weights are
// one fp16 term for the products (2^-11 of a weight at most, an eighth of the output's rounding to bf16) and fp32 for the denominator.
#include "kv8.cuh"
#include "tcgen05.cuh"

namespace {

struct Kv8DecodeParams {
    const bf16* q;                       // [T, n_heads, hd]
    const uint8_t *k_codes, *v_codes, *exps;
    const int* positions; const int* batch_idx;      // [T]; keys 0..position are visible (a negative one: none, the row is zero)
    Kv8Pages pages;
    int n_heads, n_kv, hd;
    float scale;
    bf16* out;                           // [T, n_heads, hd]
    float *o_part, *lse_part;            // [blocks x passes, 2, rows, width], [blocks x passes, 2, rows]
    int4* jobs;                          // [blocks x passes] what kv8_merge_kernel joins: token, item, parts, place of the first one
    int T;
    int* err;                            // error word of bounded waits
};

constexpr int KT = 64, MAX_T = 256;              // keys a tile, tokens a launch
// Weights are 2^(score + exponent of the value's scale - reference).  A row's reference is raised to 2^TOP below the largest when one would be above
// 2^(TOP + RAISE), which fp16 holds; fp32 weights reach down to 2^-126, so that two rows whose scales are the format's limits apart (2^120) are told
// apart by weights down to 2^-14 of the largest.  Denominators, from which the scales are taken out, reach further, and are multiplied by the two halves of a
// power of two in turn.
constexpr float TOP = 8.f, RAISE = 7.f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 codes -> fp16 pairs (bytes 0 and 1, bytes 2 and 3).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t f2_to_f16x2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// What kv8_merge_kernel finds in `jobs`: nothing (shares end where histories do), a history, or the history that a block's share ends inside of.
enum class Parts { NONE, BY_ITEM, BY_BLOCK };

// What a block knows of the batch (shared memory).
struct Batch {
    int before[MAX_T + 1];               // tiles of one key head in front of a token
    int row[MAX_T];                      // page-table row
    uint8_t last[MAX_T];                 // keys of the last tile - 1
    int sums[MAX_T / 32];                // of 32 tokens
};

// How the blocks of a launch are dealt out: items (key heads x groups of query heads) i, i + abreast, ... belong to every abreast-th block, and
// the blocks of one item share the tiles of the batch.
struct Deal { int items, abreast, passes; };         // passes: items of a block at most

// The batch's tiles of KT keys of one item, numbered token by token.
struct Tiles {
    const Batch& batch;
    int T, shares;                       // tokens; shares that the tiles are cut into

    // Tiles of token t.
    __device__ __forceinline__ static int note(const Kv8DecodeParams& p, Batch& b, int t) {
        const int pos = p.positions[t];
        b.last[t] = (uint8_t)(pos & (KT - 1));
        b.row[t] = p.batch_idx[t];
        return pos < 0 || !guard_ok(p.pages.guard, KV8_SITE_DECODE, pos / p.pages.page_size, p.pages.pt_width) ? 0 : pos / KT + 1;
    }
    // All threads of the block.
    __device__ __forceinline__ Tiles(Batch& b, const Kv8DecodeParams& p, int most) : batch(b), T(p.T) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        constexpr int ROUNDS = (MAX_T / 32 + 2) / 3;                 // (at least three warps)
        int x[ROUNDS], n = 0;
#pragma unroll
        for (int u = 0; u < ROUNDS; ++u) {
            const int t = (warp + u * warps) * 32 + lane;
            x[u] = t < T ? note(p, b, t) : 0;
        }
#pragma unroll
        for (int u = 0; u < ROUNDS; ++u) {
            const int c = warp + u * warps;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x[u], o);
                if (lane >= o) x[u] += y;
            }
            if (lane == 31 && c * 32 < T) b.sums[c] = x[u];
        }
        if (T > 32) __syncthreads();
#pragma unroll
        for (int u = 0; u < ROUNDS; ++u) {
            const int c = warp + u * warps, t = c * 32 + lane;
            for (int i = u == 0 ? 0 : c - warps; i < c && t < T; ++i) n += b.sums[i];
            if (t < T) b.before[t + 1] = n + x[u];
        }
        if (threadIdx.x == 0) b.before[0] = 0;
        __syncthreads();
        shares = max(1, min(most, total()));
    }
    __device__ __forceinline__ int total() const { return batch.before[T]; }
    __device__ __forceinline__ int count(int t) const { return batch.before[t + 1] - batch.before[t]; }
    // (a division of 64 bits takes some hundred instructions)
    __device__ __forceinline__ int begin(int j) const {
        return total() < 1 << 20 ? (int)((uint32_t)total() * j / (uint32_t)shares) : (int)((long long)total() * j / shares);
    }
    __device__ __forceinline__ int share_of(int w) const {
        return total() < 1 << 20 ? (int)((uint32_t)((w + 1) * shares - 1) / (uint32_t)total()) : (int)(((w + 1ll) * shares - 1) / total());
    }
    struct Place { int t, tile, n; };                // n: tiles of the token
    __device__ __forceinline__ Place at(int w) const {
        int lo = 0, hi = T;                          // the last token with before <= w (tokens without tiles lie in front of it)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (batch.before[mid] <= w) lo = mid;
            else hi = mid;
        }
        return {lo, w - batch.before[lo], count(lo)};
    }
    // The start of the first token that does not begin in front of tile w.
    __device__ __forceinline__ int whole(int w) const {
        if (w >= total()) return total();
        const Place a = at(w);
        return a.tile == 0 ? w : w - a.tile + a.n;
    }
    // The first tile of the next token (there is one).
    __device__ __forceinline__ void next(Place& a) const {
        a.tile = 0;
        do { ++a.t; } while (count(a.t) == 0);
        a.n = count(a.t);
    }
};

// Blocks an SM, and warps of products.  Spilled registers cost more than blocks bring (shared memory leaves no L1 to speak of): the sums of 16 heads of
// 128, or of 8 of 256, take the registers of a block by itself, with two warps on each sub-core.  Heads of 64: four blocks with one pair of warps each
// (200 histories of up to 2500, 16 heads a key head: 55 us; three blocks of two pairs, which spill, 57; five blocks 61; two blocks of three pairs 70).
// Heads of 128: two blocks of two pairs (48 histories of up to 8192: 75 us; three blocks of one pair 78).
constexpr int blocks_per_sm(int width, int tiles) { return width == 64 ? 4 : width * tiles == 128 ? 2 : 1; }

template <int D, int NG>
struct Cfg {
    static constexpr int PER_SM = blocks_per_sm(D, NG), WARPS = PER_SM == 4 ? 2 : PER_SM == 2 ? 4 : 6, THREADS = WARPS * 32 + 32;
    static constexpr int TURNS = WARPS / 2;                              // tiles at a time, a pair of warps to each
    static constexpr int ROW = D < 128 ? D : 128, HALVES = D / ROW;      // bytes of a row in one box, boxes
    static constexpr int STAGES = D == 64 ? 4 : D == 256 ? 4 : NG == 1 ? 5 : 10, HG = 8 * NG;
    static constexpr int CHUNK = D < 128 ? 8 : 16, MT = D / 16;          // neighbouring dims of a lane, 16-dim rows of products
    static constexpr int CODES = KT * D, STAGE = 2 * CODES;              // keys, values
    static constexpr int EXPS = STAGES * STAGE;                          // KT bytes of the keys, KT of the values
    static constexpr int Q = EXPS + STAGES * 2 * KT, Q_BYTES = HG * D * 2;         // two histories' queries
    static constexpr int JOIN = Q + 2 * Q_BYTES, SLOT = NG * MT * 4 * 32 * 4 + 2 * HG * 4;       // sums as they lie in registers, references, denominators
    static constexpr int BATCH = JOIN + WARPS * SLOT;
    static constexpr int BARS = (BATCH + (int)sizeof(Batch) + 7) / 8 * 8;
    static constexpr int TOTAL = BARS + (2 * STAGES + 4) * 8;
};

// A block's part of the work; `smem`: Cfg::TOTAL bytes, aligned to 1024.  CLUSTER: of one history and `item`, shared by so many blocks, of which
// this is number `rank`; its partial result is the first of o_part.  Returns the shares that the tiles are cut into.
template <int D, int NG, int CLUSTER>
__device__ __forceinline__ int decode_block(const CUtensorMap& map_k, const CUtensorMap& map_v, const Kv8DecodeParams& p, const Deal& deal, int box, Parts parts,
                                            uint8_t* smem, int rank, int only) {
    using M = Cfg<D, NG>;
    constexpr int MT = M::MT, WARPS = M::WARPS, THREADS = M::THREADS;
    uint64_t *full = reinterpret_cast<uint64_t*>(smem + M::BARS), *free_ = full + M::STAGES, *q_full = free_ + M::STAGES, *q_free = q_full + 2;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < M::STAGES; ++i) {
            tc::mbar_init(full + i, 1);
            tc::mbar_init(free_ + i, WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(q_full + i, 1);
            tc::mbar_init(q_free + i, WARPS);
        }
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&map_k);
        tc::tma_prefetch_desc(&map_v);
    }
    pdl_grid_sync();
    const int group = p.n_heads / p.n_kv, hg = (group + M::HG - 1) / M::HG;
    const Tiles tiles(*reinterpret_cast<Batch*>(smem + M::BATCH), p, CLUSTER ? CLUSTER : gridDim.x / deal.abreast);
    const bool by_item = parts == Parts::BY_ITEM, by_block = parts == Parts::BY_BLOCK;
    for (int t = CLUSTER ? rank : blockIdx.x; t < p.T; t += CLUSTER ? CLUSTER : gridDim.x)
        if (tiles.count(t) == 0) {
            for (int i = tid; i < p.n_heads * p.hd / 2; i += THREADS) reinterpret_cast<uint32_t*>(p.out + (size_t)t * p.n_heads * p.hd)[i] = 0u;
            if (by_item)
                for (int i = tid; i < deal.items; i += THREADS) p.jobs[t * deal.items + i] = make_int4(0, 0, 0, 0);
        }
    if (by_block && tid < deal.passes) p.jobs[blockIdx.x * deal.passes + tid] = make_int4(0, 0, 0, 0);
    const int share = CLUSTER ? rank : blockIdx.x / deal.abreast, first_item = CLUSTER ? only : blockIdx.x % deal.abreast;
    const int passes = CLUSTER ? 1 : (deal.items - first_item + deal.abreast - 1) / deal.abreast;
    if (share >= tiles.shares) return tiles.shares;
    int s0 = tiles.begin(share), s1 = tiles.begin(share + 1);
    if (!CLUSTER && parts == Parts::NONE) {
        s0 = tiles.whole(s0);
        s1 = tiles.whole(s1);
    }
    const int len = s1 - s0;
    if (len <= 0) return tiles.shares;
    const long long w1 = (long long)len * passes;                // this block's tiles, item by item

    if (warp == WARPS) {
        // ---- fetching: a lane looks up one box of a tile ahead, and sends for it when the tile's turn comes ----
        const int subs = KT / box, batch = 32 / subs;
        struct Ahead {
            int page, key, head;                                 // entry of the page table, first key of the box (-1: nothing to fetch), key head
            const bf16* q;                                       // of a history's first tile: its queries, or null
            uint32_t q_bytes;
        };
        auto look = [&](long long w) -> Ahead {                  // (the entry is not looked at here: it is on its way)
            Ahead a{-1, -1, 0, nullptr, 0u};
            if (w >= w1) return a;
            const int pass = passes == 1 ? 0 : (int)(w / len), s = s0 + (int)(w - (long long)pass * len), item = first_item + pass * deal.abreast;
            const Tiles::Place at = tiles.at(s);
            const int key = at.tile * KT + lane % subs * box, n = at.n * KT - (KT - 1) + tiles.batch.last[at.t];
            const int r_lo = hg == 1 ? 0 : item % hg * M::HG, b = tiles.batch.row[at.t], page = key / p.pages.page_size;
            a.head = hg == 1 ? item : item / hg;
            if (lane % subs == 0 && (s == s0 || at.tile == 0)) {
                a.q = p.q + ((size_t)at.t * p.n_heads + a.head * group + r_lo) * p.hd;
                a.q_bytes = (uint32_t)(min(M::HG, group - r_lo) * p.hd * 2);
            }
            if (key >= n) return a;
            a.key = key;
            if (guard_ok(p.pages.guard, KV8_SITE_DECODE, b, p.pages.pt_rows) && guard_ok(p.pages.guard, KV8_SITE_DECODE, page, p.pages.pt_width))
                a.page = p.pages.page_table[(size_t)b * p.pages.pt_stride + page];
            return a;
        };
        auto of_lane = [](int x, int from) { return __shfl_sync(0xffffffffu, x, from); };
        int issued = 0, asked = 0, st = 0;                       // tiles, histories, stage
        bool ok = true;
        Ahead now, then = look(lane / subs);
        for (long long w = 0; w < w1 && ok; w += batch) {
            now = then;
            const int n = (int)min((long long)batch, w1 - w), off = now.key % p.pages.page_size;
            const uint32_t firsts = __ballot_sync(0xffffffffu, now.q != nullptr), boxes = __ballot_sync(0xffffffffu, now.key >= 0);
            // a page that is not there is recorded; rows in front of the tensor read as zeros
            const bool there = now.key >= 0 && guard_ok(p.pages.guard, KV8_SITE_DECODE, (long long)now.page * p.pages.page_size, p.pages.num_slots);
            const int row = there ? now.page * p.pages.page_size + off : -KT;
            // (exponent bytes of a box start at multiples of 16)
            const uint32_t from = (uint32_t)(((((size_t)(there ? now.page : 0) * p.n_kv + max(now.head, 0)) * 2) * p.pages.page_size + max(off, 0)) / 16);
            for (int i = 0; i < n; ++i, ++issued) {
                if (i == min(n - 1, M::STAGES)) then = look(w + batch + lane / subs);
                const int at = i * subs;
                if (firsts >> at & 1) {
                    const int qb = asked & 1;
                    if (asked >= 2 && !tc::mbar_wait_warp(q_free + qb, (uint32_t)((asked >> 1) + 1) & 1)) { ok = false; break; }
                    if (lane == at) {
                        tc::mbar_expect_tx(q_full + qb, now.q_bytes);
                        tc::bulk_load_1d(smem + M::Q + qb * M::Q_BYTES, now.q, now.q_bytes, q_full + qb);
                    }
                    ++asked;
                }
                if (issued >= M::STAGES && !tc::mbar_wait_warp(free_ + st, (uint32_t)(issued / M::STAGES + 1) & 1)) { ok = false; break; }
                const uint32_t there = boxes >> at & ((1u << subs) - 1), bytes = __popc(there) * box * (2 * D + 2);
                for (int u = 0; u < subs && (there >> u & 1) != 0; ++u) {    // (boxes behind the history are left out)
                    const int row_u = of_lane(row, at + u), head_u = of_lane(now.head, at + u);
                    const uint8_t* from_u = p.exps + (size_t)(uint32_t)of_lane((int)from, at + u) * 16;
                    uint8_t *codes = smem + st * M::STAGE + u * box * M::ROW, *exps = smem + M::EXPS + st * 2 * KT;
                    if (tc::elect_one()) {
                        if (u == 0) tc::mbar_expect_tx(full + st, bytes);
#pragma unroll
                        for (int x = 0; x < M::HALVES; ++x) {
                            tc::tma_load_3d(codes + x * KT * M::ROW, &map_k, full + st, x * 128, head_u, row_u);
                            tc::tma_load_3d(codes + M::CODES + x * KT * M::ROW, &map_v, full + st, x * 128, head_u, row_u);
                        }
                        if (box == KT && p.pages.page_size == KT) {          // the bytes of keys and values are neighbours
                            tc::bulk_load_1d(exps, from_u, 2 * KT, full + st);
                        } else {
                            tc::bulk_load_1d(exps + u * box, from_u, box, full + st);
                            tc::bulk_load_1d(exps + KT + u * box, from_u + p.pages.page_size, box, full + st);
                        }
                    }
                }
                __syncwarp();
                if (++st == M::STAGES) st = 0;
            }
        }
        // nothing is in flight when the block ends, also where a wait ran out
        for (int j = max(0, issued - M::STAGES); j < issued; ++j) ok &= tc::mbar_wait_warp(full + j % M::STAGES, (uint32_t)(j / M::STAGES) & 1);
        for (int j = max(0, asked - 2); j < asked; ++j) ok &= tc::mbar_wait_warp(q_full + (j & 1), (uint32_t)(j >> 1) & 1);
        if (!ok && lane == 0) atomicExch(p.err, KV8_WAIT_FETCH);
        return tiles.shares;
    }

    // ---- products: a pair of warps takes every tile that is its turn, a warp 32 of its keys ----
    const int g = lane >> 2, c4 = lane & 3, k0 = (warp & 1) * 32;
    constexpr int CH = D < 128 ? 1 : D / 64;                         // 16-byte pieces of a key row a lane reads
    // places of a lane's pieces in a tile
    const int ks = D < 128 ? (k0 + g) * 64 + ((c4 ^ (g >> 1 & 3)) << 4) : (k0 + g) * 128;
    int st = 0, turn = warp >> 1, done = 0;                     // 0: this pair's tile; histories behind it
    uint32_t phase = 0;
    bool ok = true;
    const Tiles::Place begin = tiles.at(s0);
    Tiles::Place at = begin;
    for (int s = s0, pass = 0;;) {
        const int item = first_item + pass * deal.abreast, count = min(at.n - at.tile, s1 - s), t = at.t, hkv = item / hg, r_lo = item % hg * M::HG;
        const int nr = min(M::HG, group - r_lo), h0 = hkv * group + r_lo, keys = at.n * KT - (KT - 1) + tiles.batch.last[t];
        // queries as fp16 times 2^-eq: a lane holds head g's dims of its pieces, in the order of the pieces' bytes
        uint32_t q[NG][CH * 4][2];
        float qf[NG][2];                                             // factors on the scores of heads 2 c4 and 2 c4 + 1
        if (ok) ok = tc::mbar_wait_warp(q_full + (done & 1), (uint32_t)(done >> 1) & 1);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const uint8_t* src = smem + M::Q + (done & 1) * M::Q_BYTES + (n * 8 + g) * p.hd * 2;
            uint4 raw[CH][2];
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const int d = D < 128 ? c4 * 16 : (j >> 1) * 128 + (2 * c4 + (j & 1)) * 16;
                raw[j][0] = raw[j][1] = make_uint4(0u, 0u, 0u, 0u);
                if (n * 8 + g < nr && d < p.hd) {
                    raw[j][0] = *reinterpret_cast<const uint4*>(src + d * 2);
                    raw[j][1] = *reinterpret_cast<const uint4*>(src + d * 2 + 16);
                }
                const uint32_t* u = reinterpret_cast<const uint32_t*>(raw[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 f = bf162_to_f2(u[i]);
                    top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int eq = max(-100, (int)(__float_as_uint(top) >> 23) - 127 - 13);          // the largest value: 2^13 to 2^14
            const float down = __uint_as_float((uint32_t)(127 - eq) << 23);
            const float f = __uint_as_float((uint32_t)(127 + eq) << 23) * (p.scale * 1.4426950408889634f);
            qf[n][0] = __shfl_sync(0xffffffffu, f, c4 * 8);
            qf[n][1] = __shfl_sync(0xffffffffu, f, c4 * 8 + 4);
#pragma unroll
            for (int j = 0; j < CH; ++j) {
                const uint32_t* u = reinterpret_cast<const uint32_t*>(raw[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 x = bf162_to_f2(u[i]);
                    q[n][j * 4 + i / 2][i & 1] = f2_to_f16x2(x.x * down, x.y * down);
                }
            }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(q_free + (done & 1));
        ++done;
        float m[NG][2], l[NG][2], acc[NG][MT][4];                    // heads 2 c4 and 2 c4 + 1
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            m[n][0] = m[n][1] = 0.f;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
        }
        bool fresh = true;                                           // no reference yet
        for (int j = at.tile; j < at.tile + count; ++j) {
            const int stage = st;
            // (also where it is another pair's turn: a barrier must not be two phases ahead of who waits for it)
            if (ok) ok = tc::mbar_wait_warp(full + stage, phase);
            if (++st == M::STAGES) { st = 0; phase ^= 1u; }
            const bool mine = turn == 0;
            if (++turn == M::TURNS) turn = 0;
            const uint8_t *kt = smem + stage * M::STAGE, *vt = kt + M::CODES, *exps = smem + M::EXPS + stage * 2 * KT + k0;
            const int nk = mine ? keys - j * KT - k0 : 0;            // of this warp's 32
            if (nk > 0 && nk < 32) {                                 // rows behind the history may hold anything
                for (int i = lane; i < (32 - nk) * (D / 16); i += 32) {
                    const int r = k0 + nk + i / (D / 16), x = i % (D / 16);
                    uint8_t* at16 = smem + stage * M::STAGE + (x * 16 / M::ROW) * KT * M::ROW + r * M::ROW + x * 16 % M::ROW;
                    *reinterpret_cast<uint4*>(at16) = *reinterpret_cast<uint4*>(at16 + M::CODES) = make_uint4(0u, 0u, 0u, 0u);
                }
                tc::fence_proxy_async_smem();                        // (the next copy into these rows comes behind)
                __syncwarp();
            }
            if (nk > 0) {
                // exponents of keys g, g + 8, g + 16, g + 24 (of a key that is not seen: any)
                float kf[4], ev[4], back[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const bool seen = g + u * 8 < nk;
                    const uint32_t eb = seen ? exps[g + u * 8] : KV8_BIAS, vb = seen ? exps[KT + g + u * 8] : KV8_BIAS;
                    kf[u] = __uint_as_float(eb << 23);
                    ev[u] = seen ? __uint_as_float(0x4b000000u | vb) - (8388608.f + KV8_BIAS) : -INFINITY;
                    back[u] = __uint_as_float((2 * KV8_BIAS - vb) << 23);
                }
                float sc[NG][2][4];                                  // keys g and g + 8 of 16, heads 2 c4 and 2 c4 + 1
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int y = 0; y < 2; ++y) sc[n][y][0] = sc[n][y][1] = sc[n][y][2] = sc[n][y][3] = 0.f;
#pragma unroll
                for (int x = 0; x < CH; ++x) {
                    uint4 u[2][2];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint8_t* a0 = kt + (D < 128 ? ks : (x >> 1) * KT * 128 + ks + (((2 * c4 + (x & 1)) ^ g) << 4)) + y * 16 * M::ROW;
                        u[y][0] = *reinterpret_cast<const uint4*>(a0);
                        u[y][1] = *reinterpret_cast<const uint4*>(a0 + 8 * M::ROW);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {                // (independent sums in turn)
                            uint32_t a[4];
                            e4m3x4_to_f16(reinterpret_cast<const uint32_t*>(&u[y][0])[i], a[0], a[2]);
                            e4m3x4_to_f16(reinterpret_cast<const uint32_t*>(&u[y][1])[i], a[1], a[3]);
#pragma unroll
                            for (int n = 0; n < NG; ++n) mma_f16_16816(sc[n][y], a, q[n][x * 4 + i][0], q[n][x * 4 + i][1]);
                        }
                }
                // a lane's dims of keys 2 c4, 2 c4 + 1 and 8 on, of each 16; the first ones are read ahead of the weights
                auto values = [&](int x, int y, uint32_t (&v)[4][M::CHUNK / 4]) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int r = y * 16 + 2 * c4 + (u & 1) + (u >> 1) * 8;
                        if (D < 128) {
                            *reinterpret_cast<uint2*>(v[u]) = *reinterpret_cast<const uint2*>(vt + (k0 + r) * 64 + (((g >> 1) ^ c4) << 4) + (g & 1) * 8);
                        } else {
                            *reinterpret_cast<uint4*>(v[u]) =
                                *reinterpret_cast<const uint4*>(vt + x * KT * 128 + (k0 + r) * 128 + ((g ^ (2 * c4 + (u & 1))) << 4));
                        }
                    }
                };
                constexpr bool AHEAD = D == 64 || NG == 1;           // (where registers are left)
                uint32_t early[2][4][M::CHUNK / 4];
                if (AHEAD) {
                    values(0, 0, early[0]);
                    values(0, 1, early[1]);
                }
                uint32_t pw[NG][4];                                  // weights times scales: head g, keys 2 c4 and 2 c4 + 1 of every 8
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    float x[4][2];                                   // log2 of the weights
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h) x[u][h] = fmaf(sc[n][u >> 1][(u & 1) * 2 + h] * kf[u], qf[n][h], ev[u] - m[n][h]);
                    float top[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) top[h] = fmaxf(fmaxf(x[0][h], x[1][h]), fmaxf(x[2][h], x[3][h]));
                    if (fresh || __any_sync(0xffffffffu, fmaxf(top[0], top[1]) > TOP + RAISE)) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
                            const float up = fresh ? top[h] - TOP : fmaxf(top[h] - TOP, 0.f), root = fresh ? 1.f : ex2(-0.5f * up), f = root * root;
                            m[n][h] += up;
                            l[n][h] = l[n][h] * root * root;
#pragma unroll
                            for (int u = 0; u < 4; ++u) x[u][h] -= up;
#pragma unroll
                            for (int i = 0; i < MT; ++i) { acc[n][i][h] *= f; acc[n][i][2 + h] *= f; }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float e0 = ex2(x[u][0]), e1 = ex2(x[u][1]);
                        l[n][0] = fmaf(e0, back[u], l[n][0]);
                        l[n][1] = fmaf(e1, back[u], l[n][1]);
                        pw[n][u] = transposed8x8(f2_to_f16x2(e0, e1));
                    }
                }
#pragma unroll
                for (int x = 0; x < M::HALVES; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        uint32_t v[4][M::CHUNK / 4];
                        if (AHEAD && x == 0) {
#pragma unroll
                            for (int u = 0; u < 4; ++u)
#pragma unroll
                                for (int i = 0; i < M::CHUNK / 4; ++i) v[u][i] = early[y][u][i];
                        } else {
                            values(x, y, v);
                        }
#pragma unroll
                        for (int i = 0; i < M::CHUNK / 4; ++i)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                uint32_t a[4];
                                e4m3x4_to_f16(__byte_perm(v[0][i], v[1][i], u ? 0x7362 : 0x5140), a[0], a[1]);
                                e4m3x4_to_f16(__byte_perm(v[2][i], v[3][i], u ? 0x7362 : 0x5140), a[2], a[3]);
#pragma unroll
                                for (int n = 0; n < NG; ++n) mma_f16_16816(acc[n][x * 8 + i * 2 + u], a, pw[n][y * 2], pw[n][y * 2 + 1]);
                            }
                    }
            }
            fresh &= nk <= 0;

            __syncwarp();
            if (lane == 0) tc::mbar_arrive(free_ + stage);
        }
        // ---- join the warps: sums as they lie in registers go through shared memory, a warp joins some of the columns ----
        auto together = [] { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); };
        float* const slots = reinterpret_cast<float*>(smem + M::JOIN);
        constexpr int SLOT = M::SLOT / 4, STATE = NG * MT * 4 * 32;
        together();                                                  // (what the previous history left has been read)
#pragma unroll
        for (int n = 0; n < NG; ++n) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], o);
                if (g == 0) {
                    slots[warp * SLOT + STATE + n * 8 + c4 * 2 + h] = fresh ? -INFINITY : m[n][h];
                    slots[warp * SLOT + STATE + M::HG + n * 8 + c4 * 2 + h] = l[n][h];
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) slots[warp * SLOT + ((n * MT + i) * 4 + x) * 32 + lane] = acc[n][i][x];
        }
        together();
        const bool whole = count == at.n;
        const size_t part = CLUSTER ? 0 : ((size_t)blockIdx.x * deal.passes + pass) * 2 + (at.tile == 0 ? 1 : 0);
        if (!CLUSTER && at.tile == 0 && tid == 0) {
            const int4 job = make_int4(t, item, whole ? 1 : tiles.share_of(s + at.n - 1) - share + 1, (int)part >> 1);
            if (by_item) p.jobs[t * deal.items + item] = job;
            else if (by_block && !whole) p.jobs[part >> 1] = job;
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const float* const state = slots + STATE + n * 8 + c4 * 2;
            float top[2], den[2] = {0.f, 0.f}, f[WARPS][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = state[h];
#pragma unroll
                for (int y = 1; y < WARPS; ++y) top[h] = fmaxf(top[h], state[y * SLOT + h]);
#pragma unroll
                for (int y = 0; y < WARPS; ++y) {
                    const float mo = state[y * SLOT + h];
                    const float root = mo == -INFINITY ? 0.f : ex2(0.5f * (mo - top[h]));
                    f[y][h] = root * root;
                    den[h] += state[y * SLOT + M::HG + h] * root * root;
                }
            }
            const float inv[2] = {1.f / den[0], 1.f / den[1]};
            if (!whole && warp == 0 && g == 0)
#pragma unroll
                for (int h = 0; h < 2; ++h) p.lse_part[part * M::HG + n * 8 + c4 * 2 + h] = top[h] + log2f(den[h]);
            for (int i = MT * warp / WARPS; i < MT * (warp + 1) / WARPS; ++i) {
                float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int y = 0; y < WARPS; ++y)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[x] += f[y][x & 1] * slots[y * SLOT + ((n * MT + i) * 4 + x) * 32 + lane];
                const int d = i / (M::CHUNK / 2) * 128 + g * M::CHUNK + i % (M::CHUNK / 2) * 2;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = n * 8 + c4 * 2 + h;
                    if (r >= nr) continue;
                    if (!whole) *reinterpret_cast<float2*>(p.o_part + (part * M::HG + r) * D + d) = make_float2(o[h] * inv[h], o[2 + h] * inv[h]);
                    else if (d < p.hd) *reinterpret_cast<uint32_t*>(p.out + ((size_t)t * p.n_heads + h0 + r) * p.hd + d) = f2_to_bf162(o[h] * inv[h], o[2 + h] * inv[h]);
                }
            }
        }
        s += count;
        if (s < s1) {
            tiles.next(at);
        } else {
            if (++pass == passes) break;
            s = s0;
            at = begin;
        }
    }
    if (!ok && lane == 0) atomicExch(p.err, KV8_WAIT_PRODUCTS);
    return tiles.shares;
}

__device__ __forceinline__ uint8_t* aligned_1024(uint8_t* p) { return reinterpret_cast<uint8_t*>(((uintptr_t)p + 1023) & ~(uintptr_t)1023); }

// grid: blocks of the device
template <int D, int NG>
__global__ void __launch_bounds__(Cfg<D, NG>::THREADS, Cfg<D, NG>::PER_SM) kv8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                               const __grid_constant__ Kv8DecodeParams p, Deal deal, int box, Parts parts) {
    extern __shared__ uint8_t smem_raw[];
    decode_block<D, NG, 0>(map_k, map_v, p, deal, box, parts, aligned_1024(smem_raw), 0, 0);
}

// Little work: a cluster of SIZE blocks to a token and item, which join their parts out of one another's shared memory, in place of a second kernel
// behind parts in global memory (figures: clusters_pay).  grid: tokens x items x SIZE
template <int D, int NG, int SIZE>
__global__ void __cluster_dims__(SIZE) __launch_bounds__(Cfg<D, NG>::THREADS, Cfg<D, NG>::PER_SM)
kv8_cluster_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Kv8DecodeParams p, int items, int box) {
    using M = Cfg<D, NG>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = aligned_1024(smem_raw);
    const int rank = blockIdx.x % SIZE, t = blockIdx.x / SIZE / items, item = blockIdx.x / SIZE % items;
    const size_t row = (size_t)p.n_heads * p.hd;
    p.q += t * row;
    p.out += t * row;
    p.positions += t;
    p.batch_idx += t;
    p.T = 1;
    // (the stages are done with by the time that a block has its part)
    p.o_part = reinterpret_cast<float*>(smem);
    p.lse_part = p.o_part + M::HG * D;
    const int shares = decode_block<D, NG, SIZE>(map_k, map_v, p, Deal{items, 1, 1}, box, Parts::NONE, smem, rank, item);
    if (shares == 1) return;                                         // (all blocks of the cluster)
    auto meet = [] {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    };
    meet();
    const int group = p.n_heads / p.n_kv, hg = (group + M::HG - 1) / M::HG, h0 = item / hg * group + item % hg * M::HG, nr = min(M::HG, group - item % hg * M::HG);
    for (int r = rank; r < nr; r += SIZE)
        for (int d = threadIdx.x * 2; d < p.hd; d += M::THREADS * 2) {
            float lse[SIZE], top = -INFINITY, den = 0.f;
            float2 v[SIZE], o = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < SIZE; ++i) {
                const float* other;
                asm("mapa.u64 %0, %1, %2;" : "=l"(other) : "l"(p.o_part), "r"(i));
                lse[i] = i < shares ? other[M::HG * D + r] : -INFINITY;
                v[i] = i < shares ? *reinterpret_cast<const float2*>(other + r * D + d) : make_float2(0.f, 0.f);
                top = fmaxf(top, lse[i]);
            }
#pragma unroll
            for (int i = 0; i < SIZE; ++i) {
                const float f = lse[i] == -INFINITY ? 0.f : exp2f(lse[i] - top);
                den += f;
                o.x += f * v[i].x;
                o.y += f * v[i].y;
            }
            *reinterpret_cast<uint32_t*>(p.out + (size_t)(h0 + r) * p.hd + d) = f2_to_bf162(o.x / den, o.y / den);
        }
    meet();                                                          // (what the others read is still there)
}

// Joins the partial results of histories that lie in several shares: the first part is its block's second partial result, the others are the first ones of
// the blocks of the item behind it.  Block (i, y): jobs[i], rows y * R .. of its query heads.  A thread has 4 neighbouring values, D / 4 threads a row and
// 512 / (D / 4) / R of the parts in turn.
template <int D, int HG, int R>
__global__ void __launch_bounds__(512) kv8_merge_kernel(Kv8DecodeParams p, Deal deal) {
    constexpr int LANES = D / 4, TURNS = 512 / LANES / R, AHEAD = 4;
    __shared__ float4 sums[512];
    __shared__ float2 state[512 / LANES];            // reference and denominator
    pdl_grid_sync();
    const int4 job = p.jobs[blockIdx.x];
    if (job.z < 2) return;
    const int group = p.n_heads / p.n_kv, hg = (group + HG - 1) / HG, tid = threadIdx.x, t = job.x, item = job.y, n = job.z;
    const int hkv = item / hg, r_lo = item % hg * HG, part_row = tid / LANES, r = blockIdx.y * R + part_row % R, d = tid % LANES * 4;
    const bool on = r < min(HG, group - r_lo);
    float top = -INFINITY, den = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = part_row / R; i0 < n; i0 += TURNS * AHEAD) {
        float lse[AHEAD];
        float4 v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * TURNS;
            const bool there = on && i < n;
            const size_t part = (((size_t)job.w + (size_t)i * deal.abreast * deal.passes) * 2 + (i == 0 ? 1 : 0)) * HG + r;
            lse[u] = there ? p.lse_part[part] : -INFINITY;
            v[u] = there ? *reinterpret_cast<const float4*>(p.o_part + part * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float up = top;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) up = fmaxf(up, lse[u]);
        const float f = top == -INFINITY ? 0.f : exp2f(top - up);
        den *= f;
        o.x *= f; o.y *= f; o.z *= f; o.w *= f;
        top = up;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float e = lse[u] == -INFINITY ? 0.f : exp2f(lse[u] - top);
            den += e;
            o.x += e * v[u].x; o.y += e * v[u].y; o.z += e * v[u].z; o.w += e * v[u].w;
        }
    }
    if (TURNS > 1) {
        sums[tid] = o;
        if (tid % LANES == 0) state[part_row] = make_float2(top, den);
        __syncthreads();
        if (part_row >= R) return;
        float up = top;
#pragma unroll
        for (int i = 1; i < TURNS; ++i) up = fmaxf(up, state[part_row + i * R].x);
        den = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            const float2 s = state[part_row + i * R];
            const float4 v = sums[tid + i * R * LANES];
            const float e = s.x == -INFINITY ? 0.f : exp2f(s.x - up);
            den += e * s.y;
            o.x += e * v.x; o.y += e * v.y; o.z += e * v.z; o.w += e * v.w;
        }
    }
    if (on && d < p.hd)
        *reinterpret_cast<uint2*>(p.out + ((size_t)t * p.n_heads + hkv * group + r_lo + r) * p.hd + d) =
            make_uint2(f2_to_bf162(o.x / den, o.y / den), f2_to_bf162(o.z / den, o.w / den));
}

// Codes as [slots, heads, hd]; boxes of `rows` slots of one head, min(width, 128) bytes wide (what lies behind the head's last byte reads as zero).
int map_codes(CUtensorMap* map, const void* codes, const Kv8DecodeParams* p, int width, int rows) {
    PFN_encodeTiled enc = get_encode_tiled();
    if (enc == nullptr) return -100;
    cuuint64_t dims[3] = {(cuuint64_t)p->hd, (cuuint64_t)p->n_kv, (cuuint64_t)p->pages.num_slots}, strides[2] = {(cuuint64_t)p->hd, (cuuint64_t)p->n_kv * p->hd};
    cuuint32_t box[3] = {(cuuint32_t)(width < 128 ? width : 128), 1, (cuuint32_t)rows}, steps[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               width < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -102;
}

// width of the heads in the kernels, tiles of 8 query heads
struct Shape { int width, tiles; };
Shape shape_of(int n_heads, int n_kv, int hd) {
    const int width = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    return {width, hd <= 128 && n_heads / n_kv > 8 ? 2 : 1};
}
// The items that are walked abreast read neighbouring bytes at the same time, so as many as there are, up to 32 (where a few blocks would be left
// over, at most a ninth of them): 48 histories of up to 8192, 8 key heads of 128: 75 us, one item behind the other 90.
Deal deal_of(const Shape& sh, int n_heads, int n_kv, int blocks) {
    const int items = n_kv * ((n_heads / n_kv + sh.tiles * 8 - 1) / (sh.tiles * 8)), passes = (items + 31) / 32, abreast = (items + passes - 1) / passes;
    return {items, abreast < blocks ? abreast : blocks, abreast < blocks ? passes : (items + blocks - 1) / blocks};
}

// Up to here a history is not cut: faster at every batch measured, while longer ones depend on how evenly the tokens fill the blocks.  16 heads over 8 of 128, us
// whole and cut: 32 tokens of 500 keys 12.0 and 16.6, of up to 500, ragged, 13.2 and 15.2; of 1000 17.1 and 21.4, ragged 17.3 and 20.8, but ragged 1500 21.2
// and 20.9, and 48 ragged 1000 24.6 and 23.6.  (A captured step of the engine tells a power of two of 1024 or more: it is cut.)
constexpr int WHOLE = 512;

// Whether clusters of SIZE are the faster form, for `jobs` tokens x items.  All of them have to run at once, and a block there must not have many more
// keys than here, where the blocks of the device share the batch (histories of half the longest on average) and a second kernel joins.  How many more depends on how
// much of the device the clusters take, since the second kernel costs more with more parts.  Measured on both sides (us, clusters and cut; keys more in brackets):
// * up to a quarter of the blocks: one token, heads of 128 over 8, 4000 keys 10.1 and 10.4 (446), 6000 11.9 and 11.6 (669); of 64 over 8, 3000 9.5 and 9.8 (355), 4000 10.5
//   and 9.9 (473); of 256 over 2, 3500 13.0 and 12.8 (414), two tokens of 4000 13.7 and 12.8 (446); 16 heads a key head: of 128 over 2, one of 2000 11.7 and 11.8
//   (236), of 3000 12.3 and 11.9 (355); of 64 over 4, one of 1500 10.1 and 10.3 (182), of 2000 10.9 and 10.5 (243).
// * two fifths and more: heads of 256 over 2, 4 tokens of 6000 15.8 and 16.9 (588), of 7000 17.5 and 16.9 (686), 7 of up to 8000, ragged, 18.9 and 20.3 (622); of 128 over 8,
//   3 of up to 6000 13.3 and 15.0 (507), of up to 8000 14.8 and 14.6 (676); of 64 over 8, 8 of up to 9000 18.6 and 18.3 (639); 16 heads a key head: of 64 over 4, 8 of up to
//   6000 19.9 and 22.4 (588), of 128 over 2, 4 of up to 6000 15.8 and 16.2 (588); clusters of 4 and 2: heads of 128 over 8, 8 of up to 5000 17.3 and 18.5 (709), 16 of up
//   to 2500 17.7 and 18.1 (709).
// 8 tokens of 1000 keys, 8 key heads of 128 (clusters of 4), 9.7 and 15.1; 16 of 500 (of 2) 9.3, and 11.9 uncut; clusters of 8 for 8 tokens of 2000, more than run
// at once, 20.7, of 4 12.1.
template <int D, int NG, int SIZE>
bool clusters_pay(int longest, long long jobs, int blocks, int smem) {
    const int more = jobs * SIZE * 3 > blocks ? 640 : NG == 2 ? 256 : 400;           // keys
    if (longest <= 2 * KT || jobs * SIZE > blocks || longest * (2 * blocks - jobs * SIZE) > 2ll * more * SIZE * blocks) return false;
    static const int at_once = [=] {                                 // (the devices are alike)
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = SIZE;
        cfg.blockDim = Cfg<D, NG>::THREADS;
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = SIZE;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int got = 0;
        if (cudaOccupancyMaxActiveClusters(&got, kv8_cluster_kernel<D, NG, SIZE>, &cfg) != cudaSuccess) {
            cudaGetLastError();
            got = 0;
        }
        return got;
    }();
    return jobs <= at_once;
}

constexpr int NOT_HERE = -2;             // another form is the faster one

// 0 after the launch of clusters of SIZE, or NOT_HERE, or an error.
template <int D, int NG, int SIZE>
int in_clusters(const CUtensorMap& mk, const CUtensorMap& mv, const Kv8DecodeParams* p, int T, int blocks, const Deal& deal, int box, int longest, int smem,
                cudaStream_t s) {
    static SmemOptIn opt_in;
    const int rc = opt_in((const void*)kv8_cluster_kernel<D, NG, SIZE>, smem);       // (before it is asked how many run at once)
    if (rc != 0) return rc;
    if (!clusters_pay<D, NG, SIZE>(longest, (long long)T * deal.items, blocks, smem)) return NOT_HERE;
    sl_launch(kv8_cluster_kernel<D, NG, SIZE>, T * deal.items * SIZE, Cfg<D, NG>::THREADS, smem, s, mk, mv, *p, deal.items, box);
    return SL_LAUNCH_CHECK();
}

template <int D, int NG>
int launch(const Kv8DecodeParams* all, int T, int blocks, const Deal& deal, int longest, cudaStream_t s) {
    using M = Cfg<D, NG>;
    constexpr int smem = M::TOTAL + 1024;
    static_assert(M::PER_SM * (smem + 1024) <= 228 * 1024, "blocks per SM");
    static SmemOptIn opt_in;
    const int page = all->pages.page_size, box = page % 64 == 0 ? 64 : page % 32 == 0 ? 32 : 16;
    CUtensorMap mk, mv;
    int rc = map_codes(&mk, all->k_codes, all, D, box);
    if (rc == 0) rc = map_codes(&mv, all->v_codes, all, D, box);
    if (rc == 0) rc = opt_in((const void*)kv8_decode_kernel<D, NG>, smem);
    if (rc != 0) return rc;
    rc = in_clusters<D, NG, 8>(mk, mv, all, T, blocks, deal, box, longest, smem, s);
    if (rc == NOT_HERE) rc = in_clusters<D, NG, 4>(mk, mv, all, T, blocks, deal, box, longest, smem, s);
    if (rc == NOT_HERE) rc = in_clusters<D, NG, 2>(mk, mv, all, T, blocks, deal, box, longest, smem, s);
    if (rc != NOT_HERE) return rc;
    for (int t = 0; t < T; t += MAX_T) {
        Kv8DecodeParams p = *all;
        const size_t row = (size_t)p.n_heads * p.hd;
        p.T = T - t < MAX_T ? T - t : MAX_T;
        p.q += t * row;
        p.out += t * row;
        p.positions += t;
        p.batch_idx += t;
        // histories of up to WHOLE tokens are not cut; else, few histories have many parts each: a block a query head; many have few: a block for the one
        // that a share's end cuts
        const int items = p.T * deal.items, rows = p.n_heads / p.n_kv < M::HG ? p.n_heads / p.n_kv : M::HG;
        const Parts parts = longest > 0 && longest <= WHOLE ? Parts::NONE : p.T * 8 <= blocks / deal.abreast && items <= blocks * deal.passes ? Parts::BY_ITEM : Parts::BY_BLOCK;
        sl_launch(kv8_decode_kernel<D, NG>, blocks, M::THREADS, smem, s, mk, mv, p, deal, box, parts);
        if (parts == Parts::BY_ITEM) sl_launch(kv8_merge_kernel<D, M::HG, 1>, dim3(items, rows), 512, 0, s, p, deal);
        else if (parts == Parts::BY_BLOCK) sl_launch(kv8_merge_kernel<D, M::HG, M::HG>, blocks * deal.passes, 512, 0, s, p, deal);
        rc = SL_LAUNCH_CHECK();
        if (rc != 0) return rc;
    }
    return 0;
}

}  // namespace

// Blocks that attention of these sizes is dealt out to, and what their partial results take: 2 `rows` x `width` sums, 2 `rows` references and 16 bytes for
// each of `parts`.
SL_API int sl_kv8_decode_plan(int n_heads, int n_kv, int hd, int* blocks, int* parts, int* rows, int* width) {
    if (hd < 16 || hd > 256 || hd % 16 != 0 || n_kv < 1 || n_heads < n_kv || n_heads % n_kv != 0 || n_heads > 1024) return -1;
    int device = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return (int)e;
    const Shape sh = shape_of(n_heads, n_kv, hd);
    *blocks = sms * blocks_per_sm(sh.width, sh.tiles);
    *parts = *blocks * deal_of(sh, n_heads, n_kv, *blocks).passes;
    *rows = 8 * sh.tiles;
    *width = sh.width;
    return 0;
}

// out = attention of T tokens; `blocks`: of sl_kv8_decode_plan; `longest`: keys of the longest history, if known (a wrong one costs time only).
SL_API int sl_kv8_decode(const Kv8DecodeParams* p, int T, int blocks, int longest, cudaStream_t s) {
    if (T == 0) return 0;
    if (p->hd < 16 || p->hd > 256 || p->hd % 16 != 0 || p->n_kv < 1 || p->n_heads % p->n_kv != 0 || p->n_heads > 1024 || blocks < 1) return -1;
    if (p->pages.page_size < 16 || p->pages.page_size % 16 != 0 || p->o_part == nullptr || p->lse_part == nullptr || p->jobs == nullptr) return -1;
    if ((((uintptr_t)p->q | (uintptr_t)p->k_codes | (uintptr_t)p->v_codes | (uintptr_t)p->exps | (uintptr_t)p->out | (uintptr_t)p->o_part | (uintptr_t)p->jobs) & 15) != 0) return -1;
    const Shape sh = shape_of(p->n_heads, p->n_kv, p->hd);
    const Deal deal = deal_of(sh, p->n_heads, p->n_kv, blocks);
    if ((long long)(p->pages.pt_width) * p->pages.page_size / KT > 0x7fffffff / MAX_T - 1) return -1;        // tiles are counted in 32 bits
    if (sh.width == 64) return sh.tiles == 2 ? launch<64, 2>(p, T, blocks, deal, longest, s) : launch<64, 1>(p, T, blocks, deal, longest, s);
    if (sh.width == 128) return sh.tiles == 2 ? launch<128, 2>(p, T, blocks, deal, longest, s) : launch<128, 1>(p, T, blocks, deal, longest, s);
    return launch<256, 1>(p, T, blocks, deal, longest, s);
}
