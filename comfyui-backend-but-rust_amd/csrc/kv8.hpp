// The paged cache of keys and values in 8 bits: what its kernels share.  Plain C++, so that a host compiler can check it too.
//
// codes int8 [pages][hk][page][d], scales f32 [pages][hk][page / 16]: the largest magnitude A of the 16 tokens' values of that head; a code
// c stands for c A / 127.  Token t of sequence s is slot t % page of page table[s][t / page].  Rows starts[s] .. starts[s + 1] of a call's
// row tensors are the last tokens of sequence s, which holds lens[s].  starts, lens and table are device data that the host has not seen:
// every number from them passes through span() or page_of() before it becomes an address.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#define KV8_FN __host__ __device__ __forceinline__
#else
#define KV8_FN inline
#endif

constexpr int kBlock = 16;      // tokens that share a scale
constexpr int kMostTokens = 1 << 30;

struct Span {
    int first, count, len;      // rows of the call; tokens of the sequence
};
KV8_FN int kv8_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
// Rows outside the call's tensors and above `most` are left out.
KV8_FN Span span(const int32_t* starts, const int32_t* lens, int s, int rows, int most) {
    Span r;
    r.first = kv8_clamp(starts[s], 0, rows);
    r.count = kv8_clamp(starts[s + 1], r.first, rows) - r.first;
    if (r.count > most) r.count = most;
    r.len = kv8_clamp(lens[s], 0, kMostTokens);     // so that positions a block further stay numbers
    return r;
}

// The page of block b (of 16 tokens) of a sequence, or -1 where none holds it.
KV8_FN int page_of(const int32_t* table, int cols, int n_pages, int page_shift, int b) {
    const int at = b >> (page_shift - 4);
    if (b < 0 || at >= cols) return -1;
    const int page = table[at];
    return page >= 0 && page < n_pages ? page : -1;
}
// Element offsets of block b's scale and codes for one head, in a page that page_of() gave.
KV8_FN int64_t scale_at(int page, int hk, int head, int page_shift, int b) {
    const int per = page_shift - 4;
    return (((int64_t)page * hk + head) << per) + (b & ((1 << per) - 1));
}
KV8_FN int64_t codes_at(int page, int hk, int head, int page_shift, int b, int d) { return scale_at(page, hk, head, page_shift, b) * kBlock * d; }

inline bool cache_ok(const void* k, const void* v, const void* ks, const void* vs, int n_pages, int page, int hk, int d) {
    return k && v && ks && vs && n_pages > 0 && hk > 0 && page >= kBlock && page <= 4096 && (page & (page - 1)) == 0 && d >= 16 && d <= 256 && d % 16 == 0 &&
           (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)ks % 4 == 0 && (uintptr_t)vs % 4 == 0;
}
inline bool rows_ok(const void* starts, const void* lens, const void* table, int cols, int n, int rows, int most) {
    return n >= 0 && rows >= 0 && most >= 0 && (n == 0 || (cols > 0 && starts && lens && table));
}
