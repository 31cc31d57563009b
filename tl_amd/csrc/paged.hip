// The paged KV cache: its launchers and their checks, the append and page-copy kernels, and the
// C entries of the host's page book (page_book.h).  The attention kernels are in
// paged_attention.hip.
#include "paged.h"
#include "page_book.h"

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

namespace tlhip {

// ---- append --------------------------------------------------------------------------
// Every new row is read once and written once: HBM bound.  A workgroup takes TOKENS rows, a thread
// the same 8 elements of each (16-byte stores, the loads of all rows requested first); its
// wavefronts find the rows' places for themselves, a lane per sequence.  8192 f32 rows of 8 heads of
// 128 into f16 pages (101 MB): 20.4 us, 4.9 TB/s, with 1 to 4 rows per workgroup alike.
struct AppendArgs {
    PagedCache c;
    const void* kn;
    const void* vn;
    int64_t ks, vs;  // row strides in elements
};

template <typename NT, typename KVT, int TOKENS>
__global__ __launch_bounds__(256) void k_kv_append(const AppendArgs a, const int32_t* __restrict__ table, const int32_t* __restrict__ cu,
                                                   const int32_t* __restrict__ lens) {
    const PagedCache& c = a.c;
    const int t0 = blockIdx.x * TOKENS, page = 1 << c.shift;
    // where each row goes, in elements from the pool's start: -1 nowhere
    int64_t to[TOKENS];
#pragma unroll
    for (int i = 0; i < TOKENS; i++) to[i] = -1;
    Group<true> grp;
    for (int base = 0; base < c.batch; base += 64) {
        grp.load(c, cu, lens, base);
#pragma unroll
        for (int i = 0; i < TOKENS; i++) {
            const uint64_t hit = __ballot(t0 + i >= grp.q.first && t0 + i < grp.q.first + grp.q.n);
            if (!hit) continue;
            const int b = base + __builtin_ctzll(hit);
            const Seq s = grp.at(b);
            const int j = s.shown - 1 + (t0 + i - s.first);  // its position
            if (j < 0 || j >= c.capacity) continue;
            const int p = table[(int64_t)b * c.table_stride + (j >> c.shift)];
            if ((uint32_t)p < (uint32_t)c.n_pages) to[i] = p * c.page_elems + (int64_t)(j & (page - 1)) * c.D;
        }
    }
    const int per = c.D >> 3, row = c.hkv * per;  // chunks of 8 elements
    typedef NT in8 __attribute__((ext_vector_type(8)));
    typedef KVT out8 __attribute__((ext_vector_type(8)));
    for (int u = threadIdx.x; u < 2 * row; u += 256) {
        const bool isv = u >= row;
        const int ch = isv ? u - row : u, h = ch / per;
        const NT* src = (isv ? static_cast<const NT*>(a.vn) + t0 * a.vs : static_cast<const NT*>(a.kn) + t0 * a.ks) + 8 * ch;
        KVT* dst = static_cast<KVT*>(const_cast<void*>(isv ? c.v : c.k)) + (int64_t)h * page * c.D + 8 * (ch - h * per);
        const int64_t step = isv ? a.vs : a.ks;
        in8 x[TOKENS];
#pragma unroll
        for (int i = 0; i < TOKENS; i++)
            if (to[i] >= 0) x[i] = *reinterpret_cast<const in8*>(src + i * step);
#pragma unroll
        for (int i = 0; i < TOKENS; i++)
            if (to[i] >= 0) *reinterpret_cast<out8*>(dst + to[i]) = __builtin_convertvector(x[i], out8);
    }
}

// ---- page copies ---------------------------------------------------------------------
// Bytes read and written once: HBM bound.  The pairs travel in the kernel's arguments (at most
// 4 KiB): nothing to upload, and a captured call keeps its own.  16 bytes per thread, past the
// caches: 768 pages of 128 KiB, K and V (403 MB) 68.4 us, 5.9 TB/s (74.9 us through the caches;
// 79.8 with four loads per thread).
constexpr int COPY_PAIRS = 440;
struct CopyArgs {
    u32x4* k;
    u32x4* v;
    int64_t layer;  // 16-byte words of a layer, and of a page
    int64_t page;
    int32_t src[COPY_PAIRS], dst[COPY_PAIRS];
};

__global__ __launch_bounds__(256) void k_kv_copy(const CopyArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.page) return;
    u32x4* p = (blockIdx.z & 1 ? a.v : a.k) + (blockIdx.z >> 1) * a.layer + i;
    __builtin_nontemporal_store(__builtin_nontemporal_load(p + a.src[blockIdx.y] * a.page), p + a.dst[blockIdx.y] * a.page);
}

// ---- checks --------------------------------------------------------------------------
static int arg_error(const char* what) {
    set_error(TL_HIP_ERR_ARG, "ArgumentError: %s", what);
    return TL_HIP_ERR_ARG;
}
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// (null is aligned: decode has no cu_seqlens)
static int check_ints(const void* table, const void* cu, const void* lens) {
    for (const void* p : {table, cu, lens})
        if (reinterpret_cast<uintptr_t>(p) & 3) return arg_error("page_table, cu_seqlens and kv_lens must be 4-byte aligned");
    return TL_HIP_OK;
}

// Sizes that every entry shares; fills c.
static int check_cache(PagedCache* c, int kv_dtype, int64_t n_pages, int page_size, int hkv, int D, int64_t table_stride,
                       int64_t batch, int64_t rows) {
    if (kv_dtype != TL_HIP_F16 && kv_dtype != TL_HIP_F32) {
        set_error(TL_HIP_ERR_TYPE, "TypeMismatch: cache dtype %d", kv_dtype);
        return TL_HIP_ERR_TYPE;
    }
    if (page_size < 16 || page_size > 32768 || (page_size & (page_size - 1))) return arg_error("page_size must be a power of two from 16 to 32768");
    if (D < 8 || D > 256 || D % 8) return arg_error("head_dim must be a multiple of 8 up to 256");
    if (hkv < 1 || hkv > 1024) return arg_error("n_kv_heads must be 1 to 1024");
    if (n_pages < 1 || n_pages > INT32_MAX) return arg_error("n_pages must be 1 to 2^31 - 1");
    if (batch < 0 || batch > 65536) return arg_error("batch must be 0 to 65536");
    if (rows < 0 || rows > (1 << 24)) return arg_error("n_tokens must be 0 to 2^24");
    if (table_stride < 1 || table_stride * page_size > (1 << 30)) return arg_error("table_stride must be 1 to 2^30 / page_size");
    c->table_stride = table_stride;
    c->page_elems = (int64_t)hkv * page_size * D;
    c->n_pages = (int32_t)n_pages, c->batch = (int32_t)batch, c->rows = (int32_t)rows;
    c->hkv = hkv, c->D = D, c->shift = __builtin_ctz(page_size);
    c->capacity = (int32_t)(table_stride * page_size);
    return TL_HIP_OK;
}

static int check_heads(int hq, int hkv) {
    if (hq < 1 || hq > 4096 || hkv < 1 || hq % hkv) return arg_error("n_heads must be a multiple of n_kv_heads, up to 4096");
    return TL_HIP_OK;
}

// The stream of a call: the library's device current, its first sight outside a capture.
struct OnStream {
    hipStream_t s = nullptr;
    int rc = TL_HIP_OK, back = -1;
    explicit OnStream(void* stream) {
        DeviceState* st = state();
        if (!st) {
            rc = tl_hip_last_status();
            return;
        }
        int cur = -1;
        if (hipGetDevice(&cur) == hipSuccess && cur != st->device && hipSetDevice(st->device) == hipSuccess) back = cur;
        s = stream ? static_cast<hipStream_t>(stream) : cur_stream();
        if (note_stream_syncs(s) && capturing()) {
            rc = arg_error("the first library call on a caller stream cannot be captured; make one call on that stream before capturing it");
            return;
        }
        note_stream(s);
    }
    bool capturing() const {
        hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
        const bool yes = hipStreamIsCapturing(s, &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
        (void)hipGetLastError();
        return yes;
    }
    ~OnStream() {
        if (back >= 0) (void)hipSetDevice(back);
    }
};

static int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TL_HIP_OK : hip_fail(e, what);
}

static int attend(PagedAttn a, int q_dtype, int kv_dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (a.c.batch == 0 || a.c.rows == 0) return TL_HIP_OK;
    const size_t need = paged_attention_workspace(a.c.batch, a.c.rows, a.hq, a.c.hkv, a.c.D);
    if (workspace && (workspace_bytes < need || !aligned16(workspace))) {
        set_error(TL_HIP_ERR_ARG, "ArgumentError: the workspace must hold %zu bytes and be 16-byte aligned", need);
        return TL_HIP_ERR_ARG;
    }
    OnStream on(stream);
    if (on.rc) return on.rc;
    const bool capturing = on.capturing();
    if (!workspace && capturing) return arg_error("a captured call needs a workspace of the caller's");
    void* ws = workspace ? workspace : dev_alloc_on(need, on.s);
    if (!ws) return TL_HIP_ERR_ALLOC;
    a.ws = static_cast<float*>(ws);
    // the arrival counters are the device's: only while calls cannot overlap, and not in a graph
    a.fuse = single_stream() && one_launch_merge() && !capturing;
    const int rc = launch_paged_attention(a, q_dtype == TL_HIP_F16, kv_dtype == TL_HIP_F16, on.s);
    if (!workspace) dev_free_on(ws, on.s);
    return rc;
}

static int check_attention(PagedAttn* a, const void* q, int q_dtype, int64_t q_stride, const void* k, const void* v,
                           int kv_dtype, int64_t n_pages, int page_size, int hq, int hkv, int D, const int32_t* table,
                           int64_t table_stride, const int32_t* cu, const int32_t* lens, int64_t batch, int64_t rows,
                           void* out, float scale) {
    if (int rc = check_heads(hq, hkv)) return rc;
    if (int rc = check_cache(&a->c, kv_dtype, n_pages, page_size, hkv, D, table_stride, batch, rows)) return rc;
    if ((q_dtype != TL_HIP_F32 && q_dtype != TL_HIP_F16) || (q_dtype == TL_HIP_F16 && kv_dtype != TL_HIP_F16)) {
        set_error(TL_HIP_ERR_TYPE, "TypeMismatch: q must be f32, or f16 over an f16 cache");
        return TL_HIP_ERR_TYPE;
    }
    if (batch == 0 || rows == 0) return TL_HIP_OK;
    if (!q || !k || !v || !table || !lens || !out) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: q, pages, page_table, kv_lens or out");
        return TL_HIP_ERR_NULL;
    }
    if (rows * hq > (1 << 26) || batch * hkv > (1 << 22)) return arg_error("n_tokens * n_heads must be at most 2^26, batch * n_kv_heads 2^22");
    const int per16 = q_dtype == TL_HIP_F16 ? 8 : 4;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out)) return arg_error("q, pages and out must be 16-byte aligned");
    if (int rc = check_ints(table, cu, lens)) return rc;
    if (q_stride % per16 || q_stride < (int64_t)hq * D || q_stride > (int64_t(1) << 40))
        return arg_error("q_row_stride must be a multiple of 16 bytes and hold n_heads * head_dim elements");
    if (!std::isfinite(scale)) return arg_error("scale must be finite");
    a->c.k = k, a->c.v = v, a->c.table = table, a->c.lens = lens, a->c.cu = cu;
    a->q = q, a->out = out, a->q_stride = q_stride, a->hq = hq, a->G = hq / hkv, a->scale = scale;
    return TL_HIP_OK;
}

}  // namespace tlhip

using namespace tlhip;

extern "C" {

int tl_hip_launch_kv_append(const void* k_new, const void* v_new, int new_dtype, int64_t k_row_stride,
                            int64_t v_row_stride, void* k_pages, void* v_pages, int kv_dtype, int64_t n_pages,
                            int page_size, int n_kv_heads, int head_dim, const int32_t* page_table,
                            int64_t table_stride, const int32_t* cu_seqlens, const int32_t* kv_lens, int64_t batch,
                            int64_t n_tokens, void* stream) {
    AppendArgs a{};
    if (int rc = check_cache(&a.c, kv_dtype, n_pages, page_size, n_kv_heads, head_dim, table_stride, batch, n_tokens)) return rc;
    if (new_dtype != TL_HIP_F32 && new_dtype != TL_HIP_F16) {
        set_error(TL_HIP_ERR_TYPE, "TypeMismatch: dtype %d of the new rows", new_dtype);
        return TL_HIP_ERR_TYPE;
    }
    if (batch == 0 || n_tokens == 0) return TL_HIP_OK;
    if (!k_new || !v_new || !k_pages || !v_pages || !page_table || !cu_seqlens || !kv_lens) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: rows, pages, page_table, cu_seqlens or kv_lens");
        return TL_HIP_ERR_NULL;
    }
    const int64_t width = (int64_t)n_kv_heads * head_dim, per16 = new_dtype == TL_HIP_F16 ? 8 : 4;
    if (!aligned16(k_new) || !aligned16(v_new) || !aligned16(k_pages) || !aligned16(v_pages)) return arg_error("rows and pages must be 16-byte aligned");
    if (int rc = check_ints(page_table, cu_seqlens, kv_lens)) return rc;
    for (int64_t st : {k_row_stride, v_row_stride})
        if (st % per16 || st < width || st > (int64_t(1) << 40))
            return arg_error("row strides must be multiples of 16 bytes and hold n_kv_heads * head_dim elements");
    a.c.k = k_pages, a.c.v = v_pages, a.c.table = page_table, a.c.lens = kv_lens, a.c.cu = cu_seqlens;
    a.kn = k_new, a.vn = v_new, a.ks = k_row_stride, a.vs = v_row_stride;
    OnStream on(stream);
    if (on.rc) return on.rc;
    // few rows: one per workgroup, for their latency
    const bool n16 = new_dtype == TL_HIP_F16, c16 = kv_dtype == TL_HIP_F16;
#define TLH_APPEND(NT, KVT)                                                                                                \
    (n_tokens <= 512 ? k_kv_append<NT, KVT, 1><<<dim3((unsigned)n_tokens), 256, 0, on.s>>>(a, page_table, cu_seqlens, kv_lens) \
                     : k_kv_append<NT, KVT, 4><<<dim3((unsigned)cdiv(n_tokens, 4)), 256, 0, on.s>>>(a, page_table, cu_seqlens, kv_lens))
    if (n16 && c16) TLH_APPEND(_Float16, _Float16);
    else if (n16) TLH_APPEND(_Float16, float);
    else if (c16) TLH_APPEND(float, _Float16);
    else TLH_APPEND(float, float);
#undef TLH_APPEND
    return launched("append launch");
}

int tl_hip_launch_kv_copy_pages(void* k_pages, void* v_pages, int64_t n_layers, int64_t n_pages, int64_t page_bytes,
                                const int32_t* src, const int32_t* dst, int64_t n_pairs, void* stream) {
    if (n_layers < 1 || n_layers > 32767) return arg_error("n_layers must be 1 to 32767");
    if (n_pages < 1 || n_pages > INT32_MAX) return arg_error("n_pages must be 1 to 2^31 - 1");
    if (page_bytes < 16 || page_bytes % 16 || page_bytes > (int64_t(1) << 31)) return arg_error("page_bytes must be a multiple of 16 up to 2^31");
    if (n_pairs < 0 || n_pairs > n_pages) return arg_error("n_pairs must be 0 to n_pages");
    if (n_pairs == 0) return TL_HIP_OK;
    if (!k_pages || !v_pages || !src || !dst) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: pages, src or dst");
        return TL_HIP_ERR_NULL;
    }
    if (!aligned16(k_pages) || !aligned16(v_pages)) return arg_error("pages must be 16-byte aligned");
    try {
        std::vector<bool> written(n_pages, false);
        for (int64_t i = 0; i < n_pairs; i++) {
            if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages) {
                set_error(TL_HIP_ERR_INDEX, "IndexOutOfBounds: pair %lld names page %d or %d of %lld", (long long)i, src[i], dst[i], (long long)n_pages);
                return TL_HIP_ERR_INDEX;
            }
            if (written[dst[i]]) return arg_error("a page is the destination of two copies");
            written[dst[i]] = true;
        }
        for (int64_t i = 0; i < n_pairs; i++)
            if (written[src[i]]) return arg_error("a page is the source of one copy and the destination of another");
    } catch (const std::bad_alloc&) {
        set_error(TL_HIP_ERR_ALLOC, "AllocationError: no host memory for %lld pairs", (long long)n_pairs);
        return TL_HIP_ERR_ALLOC;
    }
    OnStream on(stream);
    if (on.rc) return on.rc;
    CopyArgs a;
    a.k = static_cast<u32x4*>(k_pages), a.v = static_cast<u32x4*>(v_pages);
    a.page = page_bytes / 16, a.layer = n_pages * a.page;
    for (int64_t i0 = 0; i0 < n_pairs; i0 += COPY_PAIRS) {
        const int n = (int)std::min<int64_t>(COPY_PAIRS, n_pairs - i0);
        std::copy(src + i0, src + i0 + n, a.src);
        std::copy(dst + i0, dst + i0 + n, a.dst);
        k_kv_copy<<<dim3((unsigned)cdiv(a.page, 256), (unsigned)n, (unsigned)(2 * n_layers)), 256, 0, on.s>>>(a);
        if (int rc = launched("page copy launch")) return rc;
    }
    return TL_HIP_OK;
}

int tl_hip_launch_paged_attention_decode(const void* q, int q_dtype, int64_t q_row_stride, const void* k_pages,
                                         const void* v_pages, int kv_dtype, int64_t n_pages, int page_size,
                                         int n_heads, int n_kv_heads, int head_dim, const int32_t* page_table,
                                         int64_t table_stride, const int32_t* kv_lens, int64_t batch, void* out,
                                         float scale, void* workspace, size_t workspace_bytes, void* stream) {
    PagedAttn a{};
    if (int rc = check_attention(&a, q, q_dtype, q_row_stride, k_pages, v_pages, kv_dtype, n_pages, page_size, n_heads, n_kv_heads,
                                 head_dim, page_table, table_stride, nullptr, kv_lens, batch, batch, out, scale))
        return rc;
    return attend(a, q_dtype, kv_dtype, workspace, workspace_bytes, stream);
}

int tl_hip_launch_paged_attention_prefill(const void* q, int q_dtype, int64_t q_row_stride, const void* k_pages,
                                          const void* v_pages, int kv_dtype, int64_t n_pages, int page_size,
                                          int n_heads, int n_kv_heads, int head_dim, const int32_t* page_table,
                                          int64_t table_stride, const int32_t* cu_seqlens, const int32_t* kv_lens,
                                          int64_t batch, int64_t n_tokens, void* out, float scale, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    PagedAttn a{};
    if (int rc = check_attention(&a, q, q_dtype, q_row_stride, k_pages, v_pages, kv_dtype, n_pages, page_size, n_heads, n_kv_heads,
                                 head_dim, page_table, table_stride, cu_seqlens, kv_lens, batch, n_tokens, out, scale))
        return rc;
    if (batch && n_tokens && !cu_seqlens) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: cu_seqlens");
        return TL_HIP_ERR_NULL;
    }
    return attend(a, q_dtype, kv_dtype, workspace, workspace_bytes, stream);
}

size_t tl_hip_paged_attention_workspace(int64_t batch, int64_t n_tokens, int n_heads, int n_kv_heads, int head_dim) {
    PagedCache c;
    if (check_heads(n_heads, n_kv_heads) || check_cache(&c, TL_HIP_F16, 1, 16, n_kv_heads, head_dim, 1, batch, n_tokens)) return 0;
    return paged_attention_workspace(batch, n_tokens, n_heads, n_kv_heads, head_dim);
}

// ---- the page book -------------------------------------------------------------------
static PageBook* book_of(const void* b) {
    if (!b) set_error(TL_HIP_ERR_NULL, "NullPointerError: page book");
    return static_cast<PageBook*>(const_cast<void*>(b));
}
static int book_result(PageBook::Result r, const PageBook* b, int64_t seq) {
    switch (r) {
        case PageBook::OK: return TL_HIP_OK;
        case PageBook::NO_SEQUENCE:
            set_error(TL_HIP_ERR_INDEX, "IndexOutOfBounds: no sequence %lld", (long long)seq);
            return TL_HIP_ERR_INDEX;
        case PageBook::NO_PAGES:
            set_error(TL_HIP_ERR_ALLOC, "AllocationError: too few free pages (%lld)", (long long)b->n_free());
            return TL_HIP_ERR_ALLOC;
        default:
            return arg_error("length outside the sequence");
    }
}
static int no_host_memory() {
    set_error(TL_HIP_ERR_ALLOC, "AllocationError: no host memory for the page book");
    return TL_HIP_ERR_ALLOC;
}

void* tl_hip_page_book_new(int64_t n_pages, int page_size) {
    if (n_pages < 1 || n_pages > INT32_MAX) {
        arg_error("n_pages must be 1 to 2^31 - 1");
        return nullptr;
    }
    if (page_size < 1 || page_size > 32768) {
        arg_error("page_size must be 1 to 32768");
        return nullptr;
    }
    try {
        return new PageBook((int32_t)n_pages, page_size);
    } catch (const std::bad_alloc&) {
        no_host_memory();
        return nullptr;
    }
}

int tl_hip_page_book_release(void* book) {
    delete static_cast<PageBook*>(book);
    return TL_HIP_OK;
}

int64_t tl_hip_page_book_open(void* book) {
    PageBook* b = book_of(book);
    if (!b) return -1;
    try {
        return b->open();
    } catch (const std::bad_alloc&) {
        no_host_memory();
        return -1;
    }
}

int64_t tl_hip_page_book_fork(void* book, int64_t seq) {
    PageBook* b = book_of(book);
    if (!b) return -1;
    try {
        const int64_t id = b->fork(seq);
        if (id < 0) book_result(PageBook::NO_SEQUENCE, b, seq);
        return id;
    } catch (const std::bad_alloc&) {
        no_host_memory();
        return -1;
    }
}

int tl_hip_page_book_close(void* book, int64_t seq) {
    PageBook* b = book_of(book);
    if (!b) return TL_HIP_ERR_NULL;
    try {
        return book_result(b->close(seq), b, seq);
    } catch (const std::bad_alloc&) {
        return no_host_memory();
    }
}

int tl_hip_page_book_grow(void* book, int64_t seq, int64_t n_tokens, int32_t* src, int32_t* dst, int64_t* n_pairs) {
    PageBook* b = book_of(book);
    if (!b) return TL_HIP_ERR_NULL;
    if (!src || !dst || !n_pairs) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: src, dst or n_pairs");
        return TL_HIP_ERR_NULL;
    }
    *n_pairs = 0;
    if (n_tokens < 0) return arg_error("n_tokens below 0");
    try {
        std::vector<PageBook::Pair> moves;
        moves.reserve(1);
        const PageBook::Result r = b->grow(seq, n_tokens, &moves);
        if (r == PageBook::OK && !moves.empty()) {
            *src = moves[0].first;
            *dst = moves[0].second;
            *n_pairs = 1;
        }
        return book_result(r, b, seq);
    } catch (const std::bad_alloc&) {
        return no_host_memory();
    }
}

int tl_hip_page_book_cut(void* book, int64_t seq, int64_t length) {
    PageBook* b = book_of(book);
    if (!b) return TL_HIP_ERR_NULL;
    try {
        return book_result(b->cut(seq, length), b, seq);
    } catch (const std::bad_alloc&) {
        return no_host_memory();
    }
}

int tl_hip_page_book_compact(void* book, int32_t* src, int32_t* dst, int64_t capacity, int64_t* n_pairs) {
    PageBook* b = book_of(book);
    if (!b) return TL_HIP_ERR_NULL;
    if (!n_pairs || (capacity > 0 && (!src || !dst))) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: src, dst or n_pairs");
        return TL_HIP_ERR_NULL;
    }
    *n_pairs = b->to_move();
    if (*n_pairs > capacity) {
        set_error(TL_HIP_ERR_ARG, "ArgumentError: %lld pairs do not fit %lld", (long long)*n_pairs, (long long)capacity);
        return TL_HIP_ERR_ARG;
    }
    try {
        std::vector<PageBook::Pair> moves;
        b->compact(&moves);
        for (size_t i = 0; i < moves.size(); i++) src[i] = moves[i].first, dst[i] = moves[i].second;
        return TL_HIP_OK;
    } catch (const std::bad_alloc&) {
        return no_host_memory();
    }
}

int64_t tl_hip_page_book_length(const void* book, int64_t seq) {
    const PageBook* b = book_of(book);
    if (!b) return -1;
    const int64_t n = b->length(seq);
    if (n < 0) book_result(PageBook::NO_SEQUENCE, b, seq);
    return n;
}

int64_t tl_hip_page_book_free_pages(const void* book) {
    const PageBook* b = book_of(book);
    return b ? b->n_free() : -1;
}

int tl_hip_page_book_row(const void* book, int64_t seq, int32_t* row, int64_t capacity) {
    const PageBook* b = book_of(book);
    if (!b) return TL_HIP_ERR_NULL;
    if (!row && capacity > 0) {
        set_error(TL_HIP_ERR_NULL, "NullPointerError: row");
        return TL_HIP_ERR_NULL;
    }
    const std::vector<int32_t>* pages = b->pages(seq);
    if (!pages) return book_result(PageBook::NO_SEQUENCE, b, seq);
    if ((int64_t)pages->size() > capacity) {
        set_error(TL_HIP_ERR_ARG, "ArgumentError: %zu pages do not fit %lld entries", pages->size(), (long long)capacity);
        return TL_HIP_ERR_ARG;
    }
    std::copy(pages->begin(), pages->end(), row);
    std::fill(row + pages->size(), row + capacity, -1);
    return TL_HIP_OK;
}

}  // extern "C"
