// Writing and reading back the 8-bit key/value cache (kv8.cuh).
//
//  * kv8_store_kernel: per-head RMS norm and rotate-half of queries (fp32) and keys (64 bits) from the projection rows to the one rounding of the
//    result; keys and values are scaled by the power of two that brings their largest magnitude to (224, 448] and rounded to e4m3.
//  * kv8_read_kernel: rows of given tokens out of their pages as bf16, which holds them exactly.
#include "f32x2.cuh"
#include "kv8.cuh"
#include "prefill_attn.cuh"

namespace {

struct Kv8StoreParams {
    const bf16* q; int ldq;          // [T, n_heads * q_stride]; head h at h * q_stride
    const bf16* k; int ldk;          // [T, n_kv * hd]
    const bf16* v; int ldv;
    const bf16 *q_norm, *k_norm;     // [hd] or null
    const float* freq; double gain;  // [rot_dims / 2] angle per position; factor on cos and sin
    int rot_dims;
    const int* positions; const int* batch_idx;      // [T]; a negative position: nothing is written to the cache
    Kv8Pages pages;
    int n_heads, n_kv, hd, q_stride;
    double eps;
    bf16* q_out;                     // [T, n_heads, hd]
    uint8_t *k_codes, *v_codes, *exps;
    int T;
};

// 4 bf16 values; VEC: 8 bytes at once
template <bool VEC>
__device__ __forceinline__ uint2 load4(const bf16* p) {
    if (VEC) return *reinterpret_cast<const uint2*>(p);
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    return make_uint2((uint32_t)u[0] | (uint32_t)u[1] << 16, (uint32_t)u[2] | (uint32_t)u[3] << 16);
}
struct Raw { uint2 a, b; };
// Eight values, two to a register pair.
struct Values {
    f32x2 x[4];
    __device__ __forceinline__ explicit Values(const Raw& r) {
        const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = bf162_to_f2(w[i]);
            x[i] = pair(f.x, f.y);
        }
    }
    __device__ __forceinline__ void to(float (&y)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpair(x[i]);
            y[2 * i] = f.x;
            y[2 * i + 1] = f.y;
        }
    }
};

enum Kind { QUERY, KEY, VALUE };

constexpr int WARPS = 4;             // of a block of kv8_store_kernel

// A row of a head has L lanes of 8 values, a warp 32 / L rows of one kind at a time; a lane keeps the angles and weights of its values for all rows.
// EVEN: four of a lane's values and the four that they turn with, so a rotation stays in the lane; else eight neighbours, whose partners come
// through shared memory.  VEC: rows are aligned to 8 bytes.
template <int L, bool VEC, bool EVEN>
struct Writer {
    static constexpr int ROWS = 32 / L;
    const Kv8StoreParams& p;
    int t;                                           // token
    bool placed;                                     // it has a slot: its codes at `codes`, its first head's exponents at `exps` of the cache
    size_t codes, exps;
    int da, db, sub;                                 // the lane's first and fifth value, row of the warp's
    bool on, turning;                                // the lane has values; they are pairs of the rotation (EVEN)
    double* part;                                    // 256 values of the warp (not EVEN)
    const double2* turn;                             // (cos, sin) of each pair
    float cs[EVEN ? 4 : 8], sn[EVEN ? 4 : 8];        // of queries: fp32, whether the warp has keys or not, so that their bits are the token's alone

    // What queries are multiplied with.  EVEN: (a, b) becomes (a aa - b ab, b bb + a ba), weights, cos and sin in one factor; else aa and bb are
    // the weights.
    struct Factors { f32x2 aa[2], ab[2], bb[2], ba[2]; };
    __device__ __forceinline__ Factors factors(const Raw& weights) const {
        Factors f;
        const Values g(weights);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x2 c = EVEN && turning ? pair(cs[2 * i], cs[2 * i + 1]) : pair(1.f, 1.f), s = EVEN ? pair(sn[2 * i], sn[2 * i + 1]) : pair(0.f, 0.f);
            f.aa[i] = mul2(g.x[i], c);
            f.bb[i] = mul2(g.x[2 + i], c);
            f.ab[i] = mul2(mul2(g.x[2 + i], s), pair(-1.f, -1.f));
            f.ba[i] = mul2(g.x[i], s);
        }
        return f;
    }
    __device__ __forceinline__ static Raw load(const bf16* row, int da, int db, bool there) {
        if (!there) return {make_uint2(0u, 0u), make_uint2(0u, 0u)};
        return {load4<VEC>(row + da), load4<VEC>(row + db)};
    }
    template <int KIND>
    __device__ __forceinline__ int heads() const { return KIND == QUERY ? p.n_heads : p.n_kv; }
    // Row of a head (it may lie behind the last one).
    template <int KIND>
    __device__ __forceinline__ const bf16* source(int h) const {
        return KIND == QUERY ? p.q + ((size_t)t * p.ldq + (size_t)h * p.q_stride) : (KIND == KEY ? p.k + (size_t)t * p.ldk : p.v + (size_t)t * p.ldv) + (size_t)h * p.hd;
    }
    template <int KIND>
    __device__ __forceinline__ Raw fetch(int h) const { return load(source<KIND>(h), da, db, on && h < heads<KIND>()); }
    // Keys in 64 bits: a code lies on one side or the other of the middle between two, and fp32's roundings would decide that for one in some 700 thousand
    // (6 of the 4.2 million of 4096 tokens, now none).  `x` is rounded to odd (cut off, with the last bit set where something was), so that the one
    // rounding of it to a code is the value's.
    __device__ __forceinline__ void key(const Raw& raw, const Raw& weights, bool normed, float (&x)[8]) const {
        float g[8];
        Values(raw).to(x);
        Values(weights).to(g);
        double inv = 1.;
        if (normed) {
            double ss = 0.;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fma((double)x[i], (double)x[i], ss);
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const double mean = ss / (double)p.hd + p.eps;
            inv = mean > 3.4028234663852886e38 ? 0. : rsqrt(mean);   // (fp32's largest)
        }
        double z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = normed ? (double)x[i] * inv * (double)g[i] : (double)x[i];
        if (EVEN) {
            if (turning) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const double2 t = turn[da + i];
                    const double a = z[i], b = z[4 + i];
                    z[i] = a * t.x - b * t.y;
                    z[4 + i] = b * t.x + a * t.y;
                }
            }
        } else if (p.rot_dims > 0) {
            const int half = p.rot_dims / 2, at = (threadIdx.x & 31) * 8;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) part[at + i] = z[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = da + i;
                if (d >= p.rot_dims) continue;
                const double2 t = turn[d < half ? d : d - half];
                const double y = part[at + i + (d < half ? half : -half)];
                z[i] = d < half ? z[i] * t.x - y * t.y : z[i] * t.x + y * t.y;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = __double2float_rz(z[i]);
            x[i] = __uint_as_float(__float_as_uint(f) | ((__double2loint(z[i]) & 0x1fffffff) != 0 ? 1u : 0u));
        }
    }
    // Row `h` of the lane, which `raw` holds.
    template <int KIND>
    __device__ __forceinline__ void row(int h, const Raw& raw, const Factors& f, const Raw& weights, bool normed, float per) const {
        Values v(raw);
        const bool there = on && h < heads<KIND>();
        if (KIND == QUERY) {
            if (normed) {
                f32x2 sq = mul2(v.x[0], v.x[0]);
#pragma unroll
                for (int i = 1; i < 4; ++i) sq = fma2(v.x[i], v.x[i], sq);
                const float2 both = unpair(sq);
                float ss = both.x + both.y;
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                // one step of Newton: off by half a step instead of two (a root of an infinite mean is 0 as it is)
                const float mean = fmaf(ss, per, (float)p.eps), r = rsqrtf(mean), inv = r > 0.f ? fmaf(0.5f * r, fmaf(-mean * r, r, 1.f), r) : r;
#pragma unroll
                for (int i = 0; i < 4; ++i) v.x[i] = mul2(v.x[i], pair(inv, inv));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const f32x2 a = v.x[i], b = v.x[2 + i];
                v.x[i] = mul2(a, f.aa[i]);
                v.x[2 + i] = mul2(b, f.bb[i]);
                if (EVEN && turning) {               // (0 times a value that is not finite would not be 0)
                    v.x[i] = fma2(b, f.ab[i], v.x[i]);
                    v.x[2 + i] = fma2(a, f.ba[i], v.x[2 + i]);
                }
            }
        }
        float x[8];
        if (KIND == KEY) key(raw, weights, normed, x);
        else v.to(x);
        if (!EVEN && KIND == QUERY && p.rot_dims > 0) {
            const int half = p.rot_dims / 2, at = (threadIdx.x & 31) * 8;
            float* const part = reinterpret_cast<float*>(this->part);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) part[at + i] = x[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = da + i;
                const float y = part[at + i + (d < half ? half : d < p.rot_dims ? -half : 0)];
                if (d < half) x[i] = x[i] * cs[EVEN ? 0 : i] - y * sn[EVEN ? 0 : i];
                else if (d < p.rot_dims) x[i] = x[i] * cs[EVEN ? 0 : i] + y * sn[EVEN ? 0 : i];
            }
        }
        if (KIND == QUERY) {
            if (there) {
                bf16* dst = p.q_out + (size_t)t * (uint32_t)(p.n_heads * p.hd) + (uint32_t)(h * p.hd);
                *reinterpret_cast<uint2*>(dst + da) = make_uint2(f2_to_bf162(x[0], x[1]), f2_to_bf162(x[2], x[3]));
                *reinterpret_cast<uint2*>(dst + db) = make_uint2(f2_to_bf162(x[4], x[5]), f2_to_bf162(x[6], x[7]));
            }
            return;
        }
        uint32_t top = 0u;                           // magnitudes compare like integers; infinities and NaN are the largest
        constexpr uint32_t INF = 0x7f800000u;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (__any_sync(0xffffffffu, top >= INF)) {   // values that are not finite are NaN, and the others make the scale
            top = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t m = __float_as_uint(x[i]) & 0x7fffffffu;
                if (m >= INF) x[i] = __int_as_float(0x7fc00000);
                else top = max(top, m);
            }
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
        if (!there || !placed) return;
        // top = m 2^n with m in [1, 2), 448 = 1.75 * 2^8
        const int e = min(KV8_HIGH, max(KV8_LOW, (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0)));
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        uint32_t c[2];
#pragma unroll
        for (int i = 0; i < 8; i += 4)
            c[i / 4] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[i] * inv, x[i + 1] * inv), __NV_SATFINITE, __NV_E4M3) |
                       (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[i + 2] * inv, x[i + 3] * inv), __NV_SATFINITE, __NV_E4M3) << 16;
        uint8_t* dst = (KIND == KEY ? p.k_codes : p.v_codes) + codes + (uint32_t)(h * p.hd);
        *reinterpret_cast<uint32_t*>(dst + da) = c[0];
        *reinterpret_cast<uint32_t*>(dst + db) = c[1];
        if (da == 0) p.exps[exps + (size_t)(2 * h + (KIND == KEY ? 0 : 1)) * p.pages.page_size] = (uint8_t)(e + KV8_BIAS);
    }
    // Heads (u, u + step, ..) * ROWS + sub of a kind; the rows of two steps are on their way.
    template <int KIND>
    __device__ __forceinline__ void rows(int u, int step, Raw next) const {
        const int n = heads<KIND>();
        if (u * ROWS >= n) return;
        const bf16* w = KIND == QUERY ? p.q_norm : KIND == KEY ? p.k_norm : nullptr;
        const size_t between = (size_t)step * ROWS * (KIND == QUERY ? p.q_stride : p.hd);
        int h = u * ROWS + sub;
        const bf16* src = source<KIND>(h) + between;
        Raw then = load(src, da, db, on && h + step * ROWS < n);
        Raw g{make_uint2(0x3f803f80u, 0x3f803f80u), make_uint2(0x3f803f80u, 0x3f803f80u)};                   // ones
        if (w != nullptr && on) g = load(w, da, db, true);
        Factors f;
        if (KIND == QUERY) f = factors(g);
        const float per = 1.f / (float)p.hd;
        for (; u * ROWS < n; u += step, h += step * ROWS) {
            const Raw now = next;
            next = then;
            src += between;
            then = load(src, da, db, on && h + 2 * step * ROWS < n);
            row<KIND>(h, now, f, g, w != nullptr, per);
        }
    }
};

// `share` warps to a token, which make its angles for themselves (a block that waits for them waits longer than they take) and take every share-th
// step of its queries, keys and values.  Grid ceil(T * share / WARPS).
// What bounds it is the issue of instructions: queries go two values to an instruction, addresses are made once a token.  Blocks of four warps lie evenly on
// the SMs where those of eight leave a ninth idle (4096 tokens).  4096 tokens, 32 heads over 8 of 128, weights and rotation: 28.8 us, 3.3 TB/s; one token
// 3.8 us.  With keys in fp32 24.8 and 3.0 us; then also with one value to an instruction, 64-bit addresses a row and blocks of eight warps 28.4; rows
// asked for ahead into L2 30.2.
template <int L, bool VEC, bool EVEN>
__global__ void __launch_bounds__(WARPS * 32, 28 / WARPS) kv8_store_kernel(const __grid_constant__ Kv8StoreParams p, int share) {
    pdl_grid_sync();
    using W = Writer<L, VEC, EVEN>;
    __shared__ double2 turns[WARPS][128];                // (cos, sin) of each pair, for keys
    __shared__ float2 turns_q[WARPS][128];               // for queries
    __shared__ double part[EVEN ? 1 : WARPS][EVEN ? 1 : 256];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = p.rot_dims / 2, own = lane % L;
    const long long id = (long long)blockIdx.x * WARPS + warp;
    const int t = (int)(id / share), mine = (int)(id - (long long)t * share);
    if (t >= p.T) return;
    const bool turning = EVEN && own * 8 < p.rot_dims;
    W w{p, t, false, 0, 0, turning ? own * 4 : own * 8, turning ? half + own * 4 : own * 8 + 4, lane / L, own * 8 < p.hd, turning, part[EVEN ? 0 : warp], turns[warp]};
    // steps are numbered through queries, keys and values: this warp's first ones
    const int uq = (p.n_heads + W::ROWS - 1) / W::ROWS, uk = (p.n_kv + W::ROWS - 1) / W::ROWS;
    const int q0 = mine, k0 = (mine + share - uq % share) % share, v0 = (k0 + share - uk % share) % share;
    const Raw q = w.template fetch<QUERY>(q0 * W::ROWS + w.sub), k = w.template fetch<KEY>(k0 * W::ROWS + w.sub), v = w.template fetch<VALUE>(v0 * W::ROWS + w.sub);
    const int pos = p.positions[t], b = p.batch_idx[t];
    // fp32 keeps no digits of the angle of a far position: quarter turns and their remainder are taken in 64 bits (a remainder of an eighth of a turn at
    // most: rounded to fp32 it costs sine and cosine less than their own roundings)
    double2* const turn = turns[warp];
    float2* const turn_q = turns_q[warp];
    const bool keys = k0 * W::ROWS < p.n_kv;         // of this warp
    for (int i = lane; i < half; i += 32) {
        const double a = (double)pos * (double)p.freq[i] * 0.63661977236758134308, whole = rint(a);      // 2 / pi
        const int quarter = (int)(long long)whole;
        float s, c;
        sincospif(0.5f * (float)(a - whole), &s, &c);
        const double gain = quarter & 2 ? -p.gain : p.gain;
        turn_q[i] = make_float2((quarter & 1 ? -s : c) * (float)gain, (quarter & 1 ? c : s) * (float)gain);
        if (keys) {
            double sn, cs;
            sincospi(0.5 * (a - whole), &sn, &cs);
            turn[i] = make_double2((quarter & 1 ? -sn : cs) * gain, (quarter & 1 ? cs : sn) * gain);
        }
    }
    if (pos >= 0) {
        const int slot = kv8_slot(p.pages, KV8_SITE_STORE, b, pos);
        if (slot >= 0) {
            w.placed = true;
            w.codes = (size_t)slot * (uint32_t)(p.n_kv * p.hd);
            w.exps = kv8_exp_at(p.pages, p.n_kv, slot, 0);
        }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < (EVEN ? 4 : 8); ++i) {
        const int d = w.da + i;
        const float2 a = d < half ? turn_q[d] : d < p.rot_dims ? turn_q[d - half] : make_float2(1.f, 0.f);
        w.cs[i] = a.x;
        w.sn[i] = a.y;
    }
    w.template rows<QUERY>(q0, share, q);
    w.template rows<KEY>(k0, share, k);
    w.template rows<VALUE>(v0, share, v);
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

// Histories of sequences as pages of 64 tokens, `per_seq` to a sequence, with a page table, rows of it and positions for a kernel that reads such
// pages.  Keys are bf16; values are, too, or (HALF) fp16: of a page and head whose scales' exponents e are at most NARROW apart, codes times 2^(e - the
// largest), which fp16 holds exactly (2^-9 2^-15 is its smallest number); else the codes alone, with e and 2^-e of each token beside them.
struct Kv8UnpackParams {
    Kv8Rows c;                       // its codes and exponents start at the first key head of a call's
    int heads;                       // key heads of the call: n_kv below
    const int *qo_indptr, *positions, *batch_idx;    // token ranges of the sequences, [T], [T]
    int per_seq;
    bf16 *k, *v;                     // [sequences * per_seq * 64, n_kv, hd]
    int *table, *rows_out, *positions_out;           // [sequences, per_seq], [T], [T]
    int* exps;                       // [sequences, per_seq, n_kv] largest exponent of the values' scales, or KV8_WIDE (HALF)
    float* scales;                   // [sequences, per_seq, n_kv, 2, 64] e and 2^-e, where that is KV8_WIDE
    int* spoiled_pages; uint8_t* spoiled_dims;       // SpoiledValues
};

// 32 bytes at once
__device__ __forceinline__ void store_32(void* p, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

constexpr int READ_ROWS = 4;         // a warp's at a time
constexpr int NARROW = 15;

// NaN codes among four: 0x80 in their bytes.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Rows `first` .. first + n - 1 of page-table row b, `heads` key heads of keys (which 0) or values, -> dst: a warp takes READ_ROWS of them, a lane 16 codes of each at a time.
// HALF: as fp16, divided by 2^top[head]; where that is KV8_WIDE, the codes alone.  CLEAN: NaN codes as zeros, and the first row with one to
// spoiled[head]; returns whether this thread found one.
template <bool HALF, bool CLEAN>
__device__ __forceinline__ bool read_rows(const Kv8Rows& c, int site, int heads, int which, int b, int first, int n, bf16* dst, const int* top, int* spoiled) {
    const int lane = threadIdx.x & 31, per = heads * c.hd / 16, cached = c.n_kv * c.hd / 16, page = c.pages.page_size;
    const uint32_t of_head = (1u << 27) / (uint32_t)(c.hd / 16) + 1;             // x / (hd / 16) is (x * of_head) >> 27: x < 2^14, so it is off by less than 1 / 16
    const uint8_t* codes = which ? c.v_codes : c.k_codes;
    bool found = false;
    for (int i0 = (threadIdx.x >> 5) * READ_ROWS; i0 < n; i0 += (blockDim.x >> 5) * READ_ROWS) {
        // a lane looks up one of the rows
        const int mine = i0 + lane < n && lane < READ_ROWS ? kv8_slot(c.pages, site, b, first + i0 + lane) : -1;
        const unsigned long long my_exps = kv8_exp_at(c.pages, c.n_kv, max(mine, 0), 0) + which * page;
        int slot[READ_ROWS];
        const uint8_t* exps[READ_ROWS];
#pragma unroll
        for (int i = 0; i < READ_ROWS; ++i) {
            slot[i] = __shfl_sync(0xffffffffu, mine, i);
            exps[i] = c.exps + __shfl_sync(0xffffffffu, my_exps, i);
        }
        for (int x = lane; x < per; x += 32) {
            const uint32_t h = __umulhi((uint32_t)x << 5, of_head);
            uint4 u[READ_ROWS];
            float s[READ_ROWS];
#pragma unroll
            for (int i = 0; i < READ_ROWS; ++i)
                if (slot[i] >= 0) {
                    u[i] = ldg_nc_16(codes + ((size_t)slot[i] * (uint32_t)cached + (uint32_t)x) * 16);
                    const int e = exps[i][(size_t)h * (uint32_t)(2 * page)];
                    s[i] = HALF && top[h] == KV8_WIDE ? 1.f : __uint_as_float((uint32_t)(HALF ? e - top[h] : e) << 23);
                } else {
                    u[i] = make_uint4(0u, 0u, 0u, 0u);           // (a token that is not there reads as zeros)
                    s[i] = 0.f;
                }
#pragma unroll
            for (int i = 0; i < READ_ROWS; ++i) {
                if (i0 + i >= n) continue;
                uint32_t in[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
                if (CLEAN && (nan_codes(in[0]) | nan_codes(in[1]) | nan_codes(in[2]) | nan_codes(in[3])) != 0u) {
                    found = true;
                    atomicMin(spoiled + h, i0 + i);
#pragma unroll
                    for (int k = 0; k < 4; ++k) in[k] &= ~((nan_codes(in[k]) >> 7) * 255u);
                }
                uint32_t out[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float2 f = e4m3x2_to_float2((uint16_t)(in[k >> 1] >> (k & 1) * 16));
                    const float2 y = unpair(mul2(pair(f.x, f.y), pair(s[i], s[i])));
                    if (HALF) {
                        const __half2 a = __floats2half2_rn(y.x, y.y);
                        out[k] = *reinterpret_cast<const uint32_t*>(&a);
                    } else {
                        out[k] = f2_to_bf162(y.x, y.y);
                    }
                }
                store_32(dst + ((size_t)(i0 + i) * (uint32_t)per + (uint32_t)x) * 16, out);
            }
        }
    }
    return found;
}

// grid (ceil(longest / 32), R, 2), block 256: 32 rows of keys or of values; a range that is longer is recorded.  9000 tokens of five sequences, 8 heads of 128: 23.5 us, 5.6 TB/s, of which
// two thirds are written
__global__ void __launch_bounds__(256, 4) kv8_read_kernel(Kv8ReadParams p) {
    pdl_grid_sync();
    const int* r = p.ranges + blockIdx.y * 4;
    if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) guard_ok(p.c.pages.guard, KV8_SITE_READ, r[2], (long long)gridDim.x * 32 + 1);
    const int i0 = blockIdx.x * 32, n = min(32, r[2] - i0), out = r[3] + i0;
    if (n <= 0 || !guard_ok(p.c.pages.guard, KV8_SITE_READ, out, (long long)p.rows - n + 1)) return;
    read_rows<false, false>(p.c, KV8_SITE_READ, p.c.n_kv, blockIdx.z, r[0], r[1] + i0, n, (blockIdx.z ? p.v : p.k) + (size_t)out * p.c.n_kv * p.c.hd, nullptr, nullptr);
}

// grid (per_seq, sequences, 2), block 512: a page of a sequence's workspace, keys or values
template <bool HALF>
__global__ void __launch_bounds__(512, 2) kv8_unpack_kernel(Kv8UnpackParams p) {
    pdl_grid_sync();
    __shared__ int top[HALF ? KV8_HEADS : 1];        // exponents of the page's values
    __shared__ int spoiled[KV8_HEADS];               // first row with a value that is not finite
    const int s = blockIdx.y, page = s * p.per_seq + blockIdx.x, q0 = p.qo_indptr[s], q1 = p.qo_indptr[s + 1], most = p.per_seq * 64;
    if (q0 >= q1) return;
    int n = max(p.positions[q1 - 1] + 1, 0);         // positions ascend within a sequence; a negative one has no keys
    if (!guard_ok(p.c.pages.guard, KV8_SITE_PROMPTS, n, (long long)most + 1)) n = most;
    if (blockIdx.z == 0 && threadIdx.x == 0) p.table[page] = page;
    if (blockIdx.x == 0 && blockIdx.z == 0)
        for (int t = q0 + threadIdx.x; t < q1; t += 512) {
            p.rows_out[t] = s;
            p.positions_out[t] = min(p.positions[t], most - 1);
        }
    const int i0 = blockIdx.x * 64, b = p.batch_idx[q0];
    n = min(64, n - i0);
    if (n <= 0) return;
    bf16* dst = (blockIdx.z ? p.v : p.k) + (size_t)page * 64 * p.heads * p.c.hd;
    if (blockIdx.z == 0) {
        read_rows<false, false>(p.c, KV8_SITE_PROMPTS, p.heads, 0, b, i0, n, dst, nullptr, nullptr);
        return;
    }
    const int lane = threadIdx.x & 31, size = p.c.pages.page_size;
    for (int h = threadIdx.x; h < p.heads; h += 512) p.spoiled_pages[(size_t)page * p.heads + h] = spoiled[h] = 64;
    const int s0 = lane < n ? kv8_slot(p.c.pages, KV8_SITE_PROMPTS, b, i0 + lane) : -1, s1 = lane + 32 < n ? kv8_slot(p.c.pages, KV8_SITE_PROMPTS, b, i0 + lane + 32) : -1;
    for (int h = threadIdx.x >> 5; HALF && h < p.heads; h += 16) {
        int e[2], hi = -1, lo = 256;                 // bytes
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int slot = u ? s1 : s0;
            e[u] = slot >= 0 ? p.c.exps[kv8_exp_at(p.c.pages, p.c.n_kv, slot, h) + size] : -1;
            if (e[u] >= 0) {
                hi = max(hi, e[u]);
                lo = min(lo, e[u]);
            }
        }
        hi = __reduce_max_sync(0xffffffffu, hi);
        lo = __reduce_min_sync(0xffffffffu, lo);
        const bool wide = hi - lo > NARROW;          // (not where there are none)
        if (lane == 0) {
            top[h] = wide ? KV8_WIDE : hi - KV8_BIAS;
            p.exps[(size_t)page * p.heads + h] = top[h];
        }
        if (wide) {
            float* const out = p.scales + ((size_t)page * p.heads + h) * 128;
#pragma unroll
            for (int u = 0; u < 2; ++u) {            // (0 and 1 for tokens that are not there)
                const int x = e[u] >= 0 ? max(-126, min(126, e[u] - KV8_BIAS)) : 0;
                out[u * 32 + lane] = (float)x;
                out[64 + u * 32 + lane] = __uint_as_float((uint32_t)(127 - x) << 23);
            }
        }
    }
    __syncthreads();
    if (__syncthreads_or(read_rows<HALF, true>(p.c, KV8_SITE_PROMPTS, p.heads, 1, b, i0, n, dst, top, spoiled)) == 0) return;
    for (int h = threadIdx.x >> 5; h < p.heads; h += 16) {           // (rare: the codes are read once more)
        const size_t at = (size_t)page * p.heads + h;
        if (spoiled[h] == 64) continue;
        if (lane == 0) p.spoiled_pages[at] = spoiled[h];
        for (int d = lane; d < p.c.hd; d += 32) {
            int first = 64;
            for (int t = spoiled[h]; t < n && first == 64; ++t) {
                const int slot = kv8_slot(p.c.pages, KV8_SITE_PROMPTS, b, i0 + t);
                if (slot >= 0 && (p.c.v_codes[((size_t)slot * p.c.n_kv + h) * p.c.hd + d] & 0x7f) == 0x7f) first = t;
            }
            p.spoiled_dims[at * p.c.hd + d] = (uint8_t)first;
        }
    }
}

// Warps that are resident at once; twice as many with half of the steps each take a fifth longer (2048 tokens).
int warps_wanted() {
    static const int sms = [] {                  // (the devices are alike)
        int device = 0, n = 0;
        return cudaGetDevice(&device) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess && n > 0 ? n : 148;
    }();
    return sms * 28;
}

}  // namespace

SL_API int sl_kv8_store(const Kv8StoreParams* p, int T, cudaStream_t s) {
    if (T == 0) return 0;
    if (p->hd < 16 || p->hd > 256 || p->hd % 16 != 0 || p->rot_dims < 0 || p->rot_dims > p->hd || p->rot_dims % 2 != 0 || p->n_kv < 1 || p->n_heads < 1) return -1;
    if ((((uintptr_t)p->k_codes | (uintptr_t)p->v_codes | (uintptr_t)p->q_out) & 15) != 0 || p->pages.page_size < 1) return -1;
    const int L = p->hd <= 64 ? 8 : p->hd <= 128 ? 16 : 32, rows = 32 / L, steps = (p->n_heads + rows - 1) / rows + 2 * ((p->n_kv + rows - 1) / rows);
    const uintptr_t at = (uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->q_norm | (uintptr_t)p->k_norm;
    const bool vec = at % 8 == 0 && (p->ldq | p->ldk | p->ldv | p->q_stride) % 4 == 0, even = p->rot_dims % 8 == 0;
    Kv8StoreParams q = *p;
    q.T = T;
    // warps for all sub-cores, if there are steps for them; no more than need as many steps each
    const int each = (steps - 1) / max(1, min(steps, warps_wanted() / T)) + 1, share = (steps - 1) / each + 1;
    const long long blocks = ((long long)T * share + WARPS - 1) / WARPS;
    if (blocks > 0x7fffffff) return -1;
#define SL_KS(LL)                                                                                          \
    {                                                                                                      \
        if (vec && even) sl_launch(kv8_store_kernel<LL, true, true>, (unsigned)blocks, WARPS * 32, 0, s, q, share);         \
        else if (vec) sl_launch(kv8_store_kernel<LL, true, false>, (unsigned)blocks, WARPS * 32, 0, s, q, share);           \
        else if (even) sl_launch(kv8_store_kernel<LL, false, true>, (unsigned)blocks, WARPS * 32, 0, s, q, share);          \
        else sl_launch(kv8_store_kernel<LL, false, false>, (unsigned)blocks, WARPS * 32, 0, s, q, share);                   \
    }
    if (L == 8) SL_KS(8) else if (L == 16) SL_KS(16) else SL_KS(32)
#undef SL_KS
    return SL_LAUNCH_CHECK();
}

static bool kv8_rows_ok(const Kv8Rows& c, const void* k, const void* v) {
    return c.hd >= 16 && c.hd % 16 == 0 && c.n_kv >= 1 && c.pages.page_size >= 1 &&
           (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) & 15) == 0 && (((uintptr_t)k | (uintptr_t)v) & 31) == 0;
}

SL_API int sl_kv8_read(const Kv8ReadParams* p, int ranges, int longest, cudaStream_t s) {
    if (ranges == 0) return 0;
    if (!kv8_rows_ok(p->c, p->k, p->v) || ranges > 65535) return -1;
    sl_launch(kv8_read_kernel, dim3(max(1, (longest + 31) / 32), ranges, 2), 256, 0, s, *p);
    return SL_LAUNCH_CHECK();
}

// Causal attention of `sequences` token ranges over their histories: the histories' pages into the workspace of `up`, whose memory `attn` reads.
SL_API int sl_kv8_prompts(const Kv8UnpackParams* up, const PagedPrefillParams* attn, int sequences, int max_q, cudaStream_t s) {
    if (sequences == 0 || max_q == 0) return 0;
    if (!kv8_rows_ok(up->c, up->k, up->v) || sequences > 65535 || up->per_seq < 1 || up->heads < 1 || up->heads > up->c.n_kv || up->heads > KV8_HEADS || attn->n_kv != up->heads) return -1;
    const bool half = paged_prefill_in_tcgen05(attn, sequences, max_q);
    const dim3 grid(up->per_seq, sequences, 2);
    if (half) sl_launch(kv8_unpack_kernel<true>, grid, 512, 0, s, *up);
    else sl_launch(kv8_unpack_kernel<false>, grid, 512, 0, s, *up);
    const int rc = SL_LAUNCH_CHECK();
    if (rc != 0) return rc;
    const SpoiledValues spoiled = {up->spoiled_pages, up->spoiled_dims, up->per_seq};
    return half ? paged_prefill_tcgen05(attn, sequences, max_q, s, {up->exps, up->scales, up->per_seq}, spoiled) : paged_prefill(attn, sequences, max_q, s, spoiled);
}
