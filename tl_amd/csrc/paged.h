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

// Sequences base + lane: packed rows first .. first + n - 1, positions len that the table holds,
// and `shown` positions that its row 0 sees (0 or fewer: none).
struct Seq {
    int first, n, len, shown;
};
// Groups are loaded in order from 0: a sequence's rows begin behind those of all before it, so
// that they never add up to more than the call's, whatever cu holds.
template <bool PACKED>  // otherwise one row per sequence
struct Group {
    Seq q;
    int base, reach;  // reach: the end of the rows of this group and those before
    __device__ __forceinline__ void load(const PagedCache& c, const int32_t* cu, const int32_t* lens, int from) {
        [[maybe_unused]] const int behind = from == 0 ? 0 : reach;
        base = from;
        const int b = from + (int)__lane_id();
        int n = 0, lo = 0, hi = 0;
        if (b < c.batch) {
            n = lens[b], lo = b, hi = b + 1;  // (requested together)
            if constexpr (PACKED) lo = cu[b], hi = cu[b + 1];
        }
        n = min(max(n, 0), INT32_MAX - 32);
        if constexpr (PACKED) {
            lo = min(max(lo, 0), c.rows), hi = min(max(hi, 0), c.rows);
            int top = max(hi, behind);
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) top = max(top, __shfl_up(top, off));  // (lanes below off get their own)
            const int before = __shfl_up(top, 1);
            lo = max(lo, __lane_id() ? before : behind);
            reach = __builtin_amdgcn_readlane(top, 63);
        }
        q.first = lo, q.n = max(hi - lo, 0), q.len = min(n, c.capacity), q.shown = n - q.n + 1;
    }
    __device__ __forceinline__ Seq at(int b) const {
        const int i = b - base;
        return Seq{__builtin_amdgcn_readlane(q.first, i), __builtin_amdgcn_readlane(q.n, i), __builtin_amdgcn_readlane(q.len, i),
                   __builtin_amdgcn_readlane(q.shown, i)};
    }
    // the same, from a later group where b lies there
    __device__ __forceinline__ Seq at(const PagedCache& c, const int32_t* cu, const int32_t* lens, int b) {
        while (b - base >= 64) load(c, cu, lens, base + 64);
        return at(b);
    }
};
// Positions that row i of a sequence sees.
__device__ __forceinline__ int limit_of(const Seq& q, int i) { return max(min(q.shown + i, q.len), 0); }

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
