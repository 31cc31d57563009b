// What the launchers of the paged KV cache (paged.hip) hand to its kernels.
#pragma once
#include "internal.h"

namespace tlhip {

struct PagedCache {
    const void* k;  // [n_pages][hkv][page][D]
    const void* v;
    const int32_t* table;  // [batch][table_stride]
    const int32_t* lens;   // [batch]
    const int32_t* cu;     // [batch + 1], or null: one row per sequence
    int64_t table_stride;
    int64_t page_elems;  // hkv * page * D
    int32_t n_pages, batch, rows;  // rows: packed rows of the call
    int32_t hkv, D, shift;         // page = 1 << shift
    int32_t capacity;              // table_stride * page
};

// Positions of sequence b that the table can hold, and whether kv_lens asks for more.
__device__ __forceinline__ int paged_len(const PagedCache& c, int b, bool* past) {
    const int n = c.lens[b];
    *past = n > c.capacity;
    return min(max(n, 0), c.capacity);
}
// First packed row of sequence b and the number of its rows.
__device__ __forceinline__ int paged_rows(const PagedCache& c, int b, int* first) {
    if (!c.cu) {
        *first = b;
        return 1;
    }
    const int lo = min(max(c.cu[b], 0), c.rows), hi = min(max(c.cu[b + 1], 0), c.rows);
    *first = lo;
    return max(hi - lo, 0);
}

struct PagedAttn {
    PagedCache c;
    const void* q;
    void* out;
    int64_t q_stride;
    int32_t hq, G;
    float scale;
    float* ws;
    bool fuse;  // parts may be joined in the launch that made them: no other call overlaps
};
// q and out are f16 (q16) or f32, the cache f16 (kv16) or f32; not q16 over an f32 cache.
int launch_paged_attention(const PagedAttn& a, bool q16, bool kv16, hipStream_t s);
size_t paged_attention_workspace(int64_t batch, int64_t rows, int hq, int hkv, int D);

}  // namespace tlhip
