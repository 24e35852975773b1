// The 8-bit key/value cache of the grouped-query families (kv8.cu, kv8_attn.cu); the ctypes mirrors are in `ops/kv8.py`.
//
// A token's row of one key head is `hd` e4m3 codes and one exponent byte b, for keys and for values: value = code * 2^(b - 127).  Codes lie at
// [slot, head, :] with slot = page * page_size + offset; exponent bytes at [page, head, 0 (keys) or 1 (values), offset], so that a page's bytes
// of one head are one piece.  The scale is a power of two: 4-bit significands times it are exact in bf16, and a floating code loses
// nothing by it.  A value that is not finite is the NaN code.
#pragma once

#include "common.cuh"

constexpr int KV8_HEADS = 1024;                  // key heads at most
constexpr int KV8_BIAS = 127, KV8_LOW = -60, KV8_HIGH = 60;      // exponents that are written

// Numbers under which the kernels report a place that is not there (guard_ok) and a wait that ran out (error word); no other kernel's.
constexpr int KV8_SITE_STORE = 60, KV8_SITE_READ = 61, KV8_SITE_DECODE = 62, KV8_SITE_PROMPTS = 63;
constexpr int KV8_WAIT_FETCH = 60, KV8_WAIT_PRODUCTS = 61;

// Where a step's tokens lie: checked places of the page table.
struct Kv8Pages {
    const int* page_table; int pt_stride, pt_rows, pt_width, page_size;
    int num_slots;
    int* guard;
};

// Slot of position `pos` of page-table row `b`, or -1 (recorded): a row or page that is not there.
__device__ __forceinline__ int kv8_slot(const Kv8Pages& p, int site, int b, int pos) {
    const int page = pos < 0 ? -1 : pos / p.page_size;
    if (!guard_ok(p.guard, site, b, p.pt_rows) || !guard_ok(p.guard, site, page, p.pt_width)) return -1;
    const long long slot = (long long)p.page_table[(size_t)b * p.pt_stride + page] * p.page_size + pos % p.page_size;
    return guard_ok(p.guard, site, slot, p.num_slots) ? (int)slot : -1;
}
// Place of a slot's exponent byte of the keys; that of the values lies `page_size` bytes on.
__device__ __forceinline__ size_t kv8_exp_at(const Kv8Pages& p, int n_kv, int slot, int h) {
    return ((size_t)(slot / p.page_size) * n_kv + h) * 2 * p.page_size + slot % p.page_size;
}
