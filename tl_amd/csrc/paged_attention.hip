// Attention over a paged KV cache: one wavefront per (row, head), the general form.
#include "paged.h"

namespace tlhip {

template <typename QT, typename KVT>
__global__ __launch_bounds__(64) void k_paged_rows(const PagedAttn a) {
    const PagedCache& c = a.c;
    const int lane = threadIdx.x, t = blockIdx.x / a.hq, h = blockIdx.x % a.hq;
    int b = 0, first = 0, n = 0;
    for (; b < c.batch; b++) {
        n = paged_rows(c, b, &first);
        if (t >= first && t < first + n) break;
    }
    if (b == c.batch) return;
    bool past;
    const int len = paged_len(c, b, &past);
    const int64_t want = (int64_t)max(c.lens[b], 0) - n + (t - first) + 1;  // positions this row sees
    const int limit = (int)min(want, (int64_t)len);
    const int G = a.hq / c.hkv, page = 1 << c.shift;
    const QT* q = static_cast<const QT*>(a.q) + t * a.q_stride + h * c.D;
    float qv[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) qv[i] = lane + 64 * i < c.D ? (float)q[lane + 64 * i] * (a.scale * 1.44269504088896341f) : 0.f;
    for (int j = 0; j < limit; j++) {
        const int p = c.table[b * c.table_stride + (j >> c.shift)];
        const bool bad = (uint32_t)p >= (uint32_t)c.n_pages;
        const int64_t at = (bad ? 0 : p) * c.page_elems + ((int64_t)(h / G) * page + (j & (page - 1))) * c.D;
        float x = 0.f, v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = lane + 64 * i < c.D;
            x = fmaf(qv[i], in ? (float)static_cast<const KVT*>(c.k)[at + lane + 64 * i] : 0.f, x);
            v[i] = in ? (float)static_cast<const KVT*>(c.v)[at + lane + 64 * i] : 0.f;
        }
        x = wave_allsum(x);
        if (bad) x = NAN;
        const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.f : mn;
        const float al = __builtin_amdgcn_exp2f(m - ms), e = __builtin_amdgcn_exp2f(x - ms);
        m = mn;
        l = fmaf(l, al, e);
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = fmaf(o[i], al, e * v[i]);
    }
    const float inv = limit < want ? NAN : 1.0f / l;
    QT* op = static_cast<QT*>(a.out) + ((int64_t)t * a.hq + h) * c.D;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 64 * i < c.D) op[lane + 64 * i] = (QT)(want <= 0 ? 0.f : o[i] * inv);
}

size_t paged_attention_workspace(int64_t batch, int64_t rows, int hq, int hkv, int D) { return 16; }

int launch_paged_attention(const PagedAttn& a, bool q16, bool kv16, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.c.rows * a.hq));
    if (q16) k_paged_rows<_Float16, _Float16><<<grid, 64, 0, s>>>(a);
    else if (kv16) k_paged_rows<float, _Float16><<<grid, 64, 0, s>>>(a);
    else k_paged_rows<float, float><<<grid, 64, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TL_HIP_OK : hip_fail(e, "paged attention launch");
}

}  // namespace tlhip
