// Arguments of causal attention of prompts over the paged cache (dense_attn.cu, prefill_attn.cu); the ctypes mirror is `AttnParams`
// (`ops/dense.py`).
#pragma once

#include "common.cuh"

struct PagedPrefillParams {
    const bf16* q;                   // [T, n_heads, hd]
    const bf16* k_cache;             // [num_slots, n_kv, hd]
    const bf16* v_cache;
    const int* positions;            // [T] absolute position of each query (keys 0..pos are visible)
    const int* batch_idx;            // [T]
    const int* page_table; int pt_stride, page_size;
    const int* qo_indptr;            // [B + 1]
    int n_heads, n_kv, hd;
    float sm_scale;
    bf16* out;                       // [T, n_heads, hd]
    int T, num_slots;
    int max_keys;                    // longest history (0: not known)
    int* err;                        // error word of bounded waits
};

// Values as fp16 times a power of two per page and key head, whose exponents are [B, pages of a sequence, n_kv]; where that is KV8_WIDE, one per token, of
// which [B, pages, n_kv, 2, 64] exponents e and factors 2^-e.
constexpr int KV8_WIDE = 1 << 20;
struct HalfValues {
    const int* exps;                 // null: values are bf16
    const float* scales;
    int per_seq;
};

// Values that are not finite are zeros in a workspace, since a product with a weight of 0 would bring them to queries that do not see them.  What was there:
// place in its page of the first token with such a value, [B, pages of a sequence, n_kv], or 64 (none); where it is not 64, the same by dim, [B, pages, n_kv, hd].  A block looks through its
// pages once: three short prompts 31.0 -> 32.4 us with the noting, a chunk of 4096 behind 8192 no longer than before.
struct SpoiledValues {
    const int* pages;                // null: values are as they are
    const uint8_t* dims;
    int per_seq;

    // A whole warp: whether any of the first `keys` keys has one.
    __device__ __forceinline__ bool any(int seq, int n_kv, int hkv, int keys) const {
        bool bad = false;
        for (int j = threadIdx.x & 31; j * 64 < keys; j += 32) bad |= pages[((size_t)seq * per_seq + j) * n_kv + hkv] < 64;
        return __any_sync(0xffffffffu, bad);
    }
    // Whether a query at `pos` sees one of dim d.
    __device__ __noinline__ bool seen(int seq, int n_kv, int hkv, int hd, int pos, int d) const {
        for (int j = 0; j * 64 <= pos; ++j) {
            const size_t at = ((size_t)seq * per_seq + j) * n_kv + hkv;
            const int last = min(pos - j * 64, 63);
            if (pages[at] <= last && dims[at * hd + d] <= last) return true;
        }
        return false;
    }
};

// Whether the tcgen05 kernel takes these arguments (dense_attn.cu).
bool paged_prefill_in_tcgen05(const PagedPrefillParams* p, int B, int max_q);

// Pages of 64 tokens, heads of 64 or 128 values, 16-byte aligned rows (prefill_attn.cu).  `spoiled` goes with HALF values.
int paged_prefill_tcgen05(const PagedPrefillParams* p, int B, int max_q, cudaStream_t s, const HalfValues& half = {nullptr, nullptr, 0},
                          const SpoiledValues& spoiled = {nullptr, nullptr, 0});
// sl_paged_attn_prefill over such a workspace (dense_attn.cu).
int paged_prefill(const PagedPrefillParams* p, int B, int max_q, cudaStream_t s, const SpoiledValues& spoiled);
