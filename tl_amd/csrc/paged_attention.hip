// Attention over a paged KV cache, for one new token per sequence and for packed rows.
//
// Rows: the (query, head) pairs of a sequence that share a KV head, 16 to a tile.  With scores
// s_j = q . k_j, c = scale log2(e) and a running maximum m of the scores seen, one pass keeps
//   l = sum_j 2^(c (s_j - m)),  o = sum_j 2^(c (s_j - m)) v_j,
// both multiplied by 2^(c (m_old - m_new)) where the maximum rises; out = o / l.  Parts of the
// positions join the same way.
#include "gemm_common.h"
#include "paged.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace tlhip {

typedef _Float16 half4v __attribute__((ext_vector_type(4)));

// ---- which work is whose ---------------------------------------------------------------
// k_paged_tile: sequence b has tiles(b) row tiles per KV head and rounds(b) rounds of KEYS
// positions; the call's work is the line of all (sequence, KV head, tile, round) in that order,
// cut into equal runs, one per workgroup, whatever the lengths.  A tile whose rounds lie in one
// run is finished there; otherwise each run leaves a record (o, m, c, l of 16 rows) in the
// workspace: the run that begins the tile in its slot 1, the others in slot 0, and k_paged_join
// adds them in order.
constexpr int RUNS = 512;  // at most: two workgroups per CU

// A sequence's row of the page table, in the constant address space: no kernel writes it, and its
// entries are the same for a wavefront, so they come by scalar loads.  (As vector loads the wait
// for a page number was a wait for all the keys and values requested before it.)
typedef const __attribute__((address_space(4))) int32_t* table_ptr;
__device__ __forceinline__ table_ptr table_row(const int32_t* table, const PagedCache& c, int b) {
    return (table_ptr)(uintptr_t)(table + (int64_t)b * c.table_stride);
}

struct Work {
    int tiles, rounds;
};
__device__ __forceinline__ Work work_of(const Seq& q, int G, int keys) {
    if (q.n == 0) return {0, 0};
    return {(q.n * G + 15) >> 4, (q.len + keys - 1) / keys};
}
// The line's length fits 31 bits (the launch sees to it).  Sum over lanes 0 .. this one: within 16
// lanes, then lane 15's over the next row, then lane 31's over the upper half.
__device__ __forceinline__ int lane_prefix(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ int run_length(int total, int runs) {
    const uint32_t up = (uint32_t)total + runs - 1;
    const int n = (runs & (runs - 1)) == 0 ? up >> __builtin_ctz(runs) : up / (uint32_t)runs;
    return n < 1 ? 1 : n;
}

// All ones over the f32 or the two f16 of a word that are infinite or NaN, else 0.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    if constexpr (sizeof(T) == 4) return (uint32_t)((int32_t)((w & 0x7F800000u) + 0x00800000u) >> 31);
    const uint32_t top = ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;  // the exponent's carry
    return (top - (top >> 15)) | top;
}

// Adds the parts of a tile's records, in order, and writes its rows: part 0 at byte `first` of the
// workspace, part i at rest + i step.  A thread per four elements, over all parts or, where the rows
// are few, over every `slices`-th and then over the slices.  Eight parts are requested at a time (one
// by one, 64 parts took 44 us).
constexpr int JOIN_ROOM = 7;  // floats of LDS per thread
template <typename QT, int POLICY, int NT>  // NT threads
__device__ __forceinline__ void join_tile(const PagedAttn& a, const Seq& sq, int h, int tile, uint32_t first, uint32_t rest,
                                          uint32_t step, int parts, uint32_t bytes, float* room) {
    const int G = a.G, D = a.c.D, R = min(16, sq.n * G - tile * 16), per = D / 4;
    const uint32_t row = (D + 4) * 4;
    const __amdgpu_buffer_rsrc_t ws = buf_rsrc(a.ws, bytes);
    auto part = [&](int i) { return i == 0 ? first : rest + (uint32_t)i * step; };
    auto word4 = [&](uint32_t at) { return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(ws, at, 0, POLICY)); };
    floatx4* po = reinterpret_cast<floatx4*>(room);
    float *pm = room + 4 * NT, *pl = room + 5 * NT, *pc = room + 6 * NT;
    struct Sum {
        floatx4 o;
        float m, l, cs;
    };
    auto add = [](Sum& t, const floatx4& o, float m, float l) {
        const float mn = fmaxf(t.m, m), ms = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f((t.m - ms) * t.cs), g = __builtin_amdgcn_exp2f((m - ms) * t.cs);
        t.m = mn;
        t.l = fmaf(t.l, f, l * g);
#pragma unroll
        for (int e = 0; e < 4; e++) t.o[e] = fmaf(t.o[e], f, o[e] * g);
    };
    const int items = R * per, slices = max(NT / items, 1);
    auto put = [&](int it, const Sum& t) {
        const int r = it / per, dim = 4 * (it - r * per), orow = tile * 16 + r, oq = orow / G, sees = sq.shown + oq;
        floatx4 o = t.o * (sees > sq.len ? NAN : 1.0f / t.l);
        if (sees <= 0) o = floatx4{0.f, 0.f, 0.f, 0.f};
        QT* op = static_cast<QT*>(a.out) + ((int64_t)(sq.first + oq) * a.hq + h * G + orow - oq * G) * D;
        if constexpr (std::is_same_v<QT, float>) *reinterpret_cast<floatx4*>(op + dim) = o;
        else *reinterpret_cast<half4v*>(op + dim) = half4v{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
    };
    const int slice = slices > 1 ? (int)threadIdx.x / items : 0;
    for (int it = slices > 1 ? (int)threadIdx.x - slice * items : (int)threadIdx.x; it < items && slice < slices; it += NT) {
        const int r = it / per;
        Sum t{{0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.f, 1.f};
        for (int i0 = slice; i0 < parts; i0 += 8 * slices) {
            floatx4 z[8], ml[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                // (an offset at the resource's end reads nothing)
                const uint32_t at = i0 + u * slices < parts ? part(i0 + u * slices) + r * row : bytes;
                z[u] = word4(at + 16 * (it - r * per));
                ml[u] = word4(at + 4 * D);
            }
#pragma unroll
            for (int u = 0; u < 8; u++)
                if (i0 + u * slices < parts) {
                    t.cs = ml[u][2];  // one value for all parts
                    add(t, z[u], ml[u][0], ml[u][1]);
                }
        }
        if (slices == 1) {
            put(it, t);
        } else {
            po[threadIdx.x] = t.o, pm[threadIdx.x] = t.m, pl[threadIdx.x] = t.l;
            if (slice == 0) pc[threadIdx.x] = t.cs;
        }
    }
    if (slices == 1) return;
    __syncthreads();
    const int it = threadIdx.x;
    if (it >= items) return;
    Sum t{po[it], pm[it], pl[it], pc[it]};
    for (int i = 1; i < min(slices, parts); i++) add(t, po[it + i * items], pm[it + i * items], pl[it + i * items]);
    put(it, t);
}
// Runs run0 .. run0 + parts - 1 of k_paged_tile: the first run's record in its slot 1, the others' in slot 0.
template <typename QT, int POLICY, int NT>
__device__ __forceinline__ void join_run(const PagedAttn& a, const Seq& sq, int h, int tile, int run0, int parts, float* room) {
    const uint32_t rec = 16 * (a.c.D + 4) * 4;
    join_tile<QT, POLICY, NT>(a, sq, h, tile, (2 * run0 + 1) * rec, 2 * run0 * rec, 2 * rec, parts, RUNS * 2 * rec, room);
}
// One launch: arrivals at the tile that run `i` began, zero between calls.  The run that arrives
// last joins the tile and sets its counter back.
__device__ uint32_t g_paged_arrive[RUNS];

// ---- 16 rows, keys and values straight from memory into matrix operands ------------------
// A wavefront takes 16 TK positions of a round at a time, the four wavefronts of a workgroup
// the four parts of a round; they add up in LDS at the end of a tile's run.
//   S^T = K Q^T: lane (col, g) = (l % 16, l / 16) holds 16-byte pieces of key 16 t + col, the
//     operand A of the matrix instruction as they stand, and gets the scores of row col at keys
//     16 t + 4 g + e;
//   O^T += V^T P^T with those keys as its k slots, so P stays where the scores are.  The lane
//     loads 4 TK keys' values at the same few dimensions (VE of them, 16 lanes together a
//     whole row): the operand for dimension x of these takes element x of each, and row r of the
//     product is dimension VE r + x.
// f16 caches: products exact in f32; f32 rows enter as two f16 parts (row scaled by a power of
// two, 22 bits), weights as two parts of 2^15 p, so the results keep f32's digits.  f32 caches:
// f32 matrix instructions.
// Long caches are bound by HBM: 32 ragged sequences of up to 8192, 8 KV heads of 128 (543 MB) 91 us,
// 5.9 TB/s; 2 of up to 131072 126 us, 6.5 TB/s.  Short ones by the launch, the reads of lengths,
// table and keys, each waiting for the one before, and the join: one sequence of 512 7.6 us.
template <typename KVT, typename QT, int DP, int TK, int NW>
struct Tile {
    static constexpr bool H16 = std::is_same_v<KVT, _Float16>;
    static constexpr int QP = H16 && std::is_same_v<QT, float> ? 2 : 1;  // parts of a query
    static constexpr int PIECE = 16 / sizeof(KVT);                       // elements per 16 bytes
    static constexpr int KS = DP / (4 * PIECE);                          // pieces of a key per lane
    static constexpr int VE = DP / 16 < PIECE ? DP / 16 : PIECE;         // value elements per load
    static constexpr int VN = DP / 16 / VE;                              // loads per value row and lane
    static constexpr int NA = DP / 16;
    static constexpr int KEYS = 16 * TK * NW;  // positions per round
};

// FULL: head_dim is DP (otherwise the rest of a key's pieces are zeros; the rest of a value's
// make rows of the product that are not stored, and read the row's first elements).
template <typename KVT, typename QT, int DP, int TK, int NW, bool FULL, bool PACKED>
__global__ __launch_bounds__(64 * NW, (DP > 128 ? 1 : 2)) void k_paged_tile(
    const PagedAttn a, const int32_t* __restrict__ table, const int32_t* __restrict__ cu, const int32_t* __restrict__ lens,
    const char* __restrict__ kp, const char* __restrict__ vp) {
    using L = Tile<KVT, QT, DP, TK, NW>;
    constexpr int QP = L::QP, KS = L::KS, VE = L::VE, VN = L::VN, NA = L::NA, KEYS = L::KEYS, EB = sizeof(KVT);
    constexpr bool H16 = L::H16;
    // one token's keys and values are read once; a prompt's by every tile (75 rows over 6 pasts of up
    // to 2000: 17.5 us, 17.7 past the caches)
    constexpr int POLICY = PACKED ? 0 : CPOL_NT;
    typedef KVT vec __attribute__((ext_vector_type(VE)));
    typedef uint32_t words __attribute__((ext_vector_type(sizeof(vec) / 4)));
    typedef KVT piece __attribute__((ext_vector_type(L::PIECE)));
    constexpr int RS = DP + 4;
    __shared__ __attribute__((aligned(16))) float so[NW][16][RS];  // o, then m, l and c
    __shared__ int last_here;
    static_assert(sizeof(so) >= 64 * NW * JOIN_ROOM * 4, "the join's room");
    const PagedCache& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    // arguments in one round of scalar loads (left to the compiler: three dependent rounds)
    asm volatile("" : : "s"(table), "s"(cu), "s"(lens), "s"(kp), "s"(vp), "s"(a.q), "s"(a.out), "s"(a.q_stride), "s"(a.hq), "s"(a.G),
                 "s"(a.scale), "s"(c.table_stride), "s"(c.page_elems), "s"(c.n_pages), "s"(c.batch), "s"(c.rows), "s"(c.hkv),
                 "s"(c.D), "s"(c.shift), "s"(c.capacity));
    const int G = a.G, D = FULL ? DP : c.D, page = 1 << c.shift;
    // run: neighbours on the line stay on one XCD (workgroups go round the eight of them)
    const int runs = gridDim.x, id = blockIdx.x;
    const int run = (runs & 7) == 0 ? (id & 7) * (runs >> 3) + (id >> 3) : id;

    Group<PACKED> grp;
    int total = 0, incl = 0, mine = 0;
    for (int base = 0; base < c.batch; base += 64) {
        grp.load(c, cu, lens, base);
        const Work w = work_of(grp.q, G, KEYS);
        mine = c.hkv * w.tiles * w.rounds;
        incl = lane_prefix(mine);
        total += lane_value(incl, 63);
        // rows of sequences without a position are zeros, and no round's
        for (uint64_t none = __ballot(w.tiles > 0 && w.rounds == 0); none; none &= none - 1) {
            const int i = __builtin_ctzll(none);
            if ((base + i) % runs != run) continue;
            const Seq sq = grp.at(base + i);
            uint32_t* op = reinterpret_cast<uint32_t*>(static_cast<QT*>(a.out) + (int64_t)sq.first * a.hq * D);
            const int64_t words = (int64_t)sq.n * a.hq * D * (int)sizeof(QT) / 4;
            for (int64_t u = threadIdx.x; u < words; u += 64 * NW) op[u] = 0;
        }
    }
    const int len_run = run_length(total, runs);
    if ((int64_t)run * len_run >= total) return;
    int x = run * len_run;
    const int x1 = min(x + len_run, total);
    int b = 0;
    int before = 0;  // line position of sequence b's first round
    for (int base = 0;; base += 64) {
        if (c.batch > 64) {
            grp.load(c, cu, lens, base);
            const Work w = work_of(grp.q, G, KEYS);
            mine = c.hkv * w.tiles * w.rounds;
            incl = lane_prefix(mine);
        }
        const uint64_t hit = __ballot(x < before + incl);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            b = base + at;
            before += lane_value(incl, at) - lane_value(mine, at);
            break;
        }
        before += lane_value(incl, 63);
    }

    while (x < x1) {
        const Seq sq = grp.at(c, cu, lens, b);
        const Work w = work_of(sq, G, KEYS);
        const int here = c.hkv * w.tiles * w.rounds;
        if (x >= before + here) {
            before += here;
            b++;
            continue;
        }
        const uint32_t unit = __builtin_amdgcn_readfirstlane((uint32_t)(x - before) / (uint32_t)w.rounds);
        const int r0 = __builtin_amdgcn_readfirstlane(x - before - (int)unit * w.rounds);
        const int r1 = __builtin_amdgcn_readfirstlane(min(w.rounds, r0 + (x1 - x)));
        const int h = w.tiles == 1 ? unit : unit / w.tiles, tile = unit - h * w.tiles;
        const int begin = x - r0;
        x += r1 - r0;

        // this lane's row; positions that it, that every row and that any row sees
        const int rows = sq.n * G;
        const int r = min(tile * 16 + col, rows - 1), qi = PACKED ? r / G : 0, qh = h * G + r - qi * G;
        const int lim = limit_of(sq, qi);
        const int lim_lo = __builtin_amdgcn_readfirstlane(limit_of(sq, PACKED ? tile * 16 / G : 0));
        const int lim_hi = __builtin_amdgcn_readfirstlane(limit_of(sq, PACKED ? min(tile * 16 + 15, rows - 1) / G : 0));

        const QT* qp = static_cast<const QT*>(a.q) + (int64_t)(sq.first + qi) * a.q_stride + qh * D;
        constexpr int QV = sizeof(QT) * L::PIECE / 16;  // 16-byte words per piece of the row
        uint4 qw[KS][QV];
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < QV; e++) {
                qw[s][e] = make_uint4(0u, 0u, 0u, 0u);
                if (FULL || 4 * L::PIECE * s + L::PIECE * g < D) qw[s][e] = reinterpret_cast<const uint4*>(qp + 4 * L::PIECE * s + L::PIECE * g)[e];
            }

        // positions of this wavefront: blocks of 16 TK from j_first on, every KEYS
        const int64_t head = (int64_t)h * page * D * EB;
        const int j_first = r0 * KEYS + wave * 16 * TK;
        const int j_end = min(r1 * KEYS, lim_hi);
        const int steps = j_first < j_end ? (j_end - j_first + KEYS - 1) / KEYS : 0;
        const table_ptr row = table_row(table, c, b);
        struct Ids {
            int p[TK];
        };
        auto ids_of = [&](int s) __attribute__((always_inline)) {
            Ids d;
#pragma unroll
            for (int t = 0; t < TK; t++)
                d.p[t] = row[__builtin_amdgcn_readfirstlane(max(min(j_first + s * KEYS + 16 * t, lim_hi - 1), 0) >> c.shift)];
            return d;
        };
        struct Buf {
            piece k[TK][KS];
            vec v[4 * TK][VN];
        };
        const uint32_t kof = (uint32_t)(col * D + L::PIECE * g) * EB;  // + 64 s bytes
        const uint32_t vof = (uint32_t)(4 * g * D + VE * col) * EB;    // + e D EB + 16 VE i EB
        [[maybe_unused]] uint32_t kofs[KS], vofs[VN];
        if constexpr (!FULL) {
#pragma unroll
            for (int i = 0; i < KS; i++) kofs[i] = 4 * L::PIECE * i + L::PIECE * g < D ? kof + 64 * i : 0x7FFFFFF0u;
#pragma unroll
            for (int i = 0; i < VN; i++) vofs[i] = 16 * VE * i + VE * col < D ? vof + 16 * VE * i * EB : (uint32_t)(4 * g * D) * EB;
        }
        // a block's 16 keys lie in one page; keys past the last one seen, and blocks past the last
        // step's, lie outside the resources and read as zeros, without a memory access
        auto load = [&](int s, const Ids& d, Buf& f) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < TK; t++) {
                const int j = j_first + s * KEYS + 16 * t;
                const bool none = (uint32_t)d.p[t] >= (uint32_t)c.n_pages;
                const int64_t at = ((none ? 0 : d.p[t]) * c.page_elems + (int64_t)(j & (page - 1)) * D) * EB + head;
                const uint32_t bytes = (uint32_t)__builtin_amdgcn_readfirstlane(none || s >= steps ? 0 : max(min(lim_hi - j, 16), 0) * D * EB);
                const __amdgpu_buffer_rsrc_t rk = buf_rsrc(kp + at, bytes), rv = buf_rsrc(vp + at, bytes);
#pragma unroll
                for (int i = 0; i < KS; i++)
                    f.k[t][i] = __builtin_bit_cast(piece, __builtin_amdgcn_raw_buffer_load_b128(rk, FULL ? kof + 64 * i : kofs[i], 0, POLICY));
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int i = 0; i < VN; i++) {
                        const uint32_t o = (FULL ? vof + 16 * VE * i * EB : vofs[i]) + e * D * EB;
                        if constexpr (sizeof(vec) == 8) f.v[4 * t + e][i] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, POLICY));
                        else f.v[4 * t + e][i] = __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b128(rv, o, 0, POLICY));
                    }
            }
        };
        Buf f0, f1;
        Ids d0 = ids_of(0), d1 = ids_of(1);
        __builtin_amdgcn_sched_barrier(0);
        load(0, d0, f0);
        __builtin_amdgcn_sched_barrier(0);

        float cs = fminf(fabsf(a.scale) * 1.44269504088896341f, FLT_MAX);
        const float sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
        typedef std::conditional_t<H16, half8, floatx4> qvec;
        qvec qf[QP][KS];
        if constexpr (QP == 2) {
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(__builtin_bit_cast(floatx4, qw[s][i / 4])[i % 4]));
            top = lane_pair_max<16>(top);
            top = lane_pair_max<32>(top);
            // the row's largest entry to 2^14 .. 2^15
            const int up = top > 0.f && top <= FLT_MAX ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
            cs = fminf(ldexpf(fabsf(a.scale) * 1.44269504088896341f, -up), FLT_MAX);
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float f = ldexpf(__builtin_bit_cast(floatx4, qw[s][i / 4])[i % 4] * sign, up);
                    qf[0][s][i] = (_Float16)f;
                    qf[1][s][i] = (_Float16)(f - (float)qf[0][s][i]);
                }
        } else {
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < L::PIECE; i++) qf[0][s][i] = __builtin_bit_cast(qvec, qw[s][0])[i] * (QT)sign;
        }
        cs = fmaxf(cs, FLT_MIN);

        float m = -INFINITY, l = 0.f;
        floatx4 acc[NA];
#pragma unroll
        for (int i = 0; i < NA; i++) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};

        auto compute = [&](int s, const Ids& d, Buf& f) __attribute__((always_inline)) {
            const int j0 = j_first + s * KEYS;
            floatx4 st[TK];
#pragma unroll
            for (int t = 0; t < TK; t++) {
                floatx4 z[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int i = 0; i < KS; i++) {
                    if constexpr (H16) {
#pragma unroll
                        for (int p = 0; p < QP; p++) z[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.k[t][i], qf[p][i], z[p], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) z[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(f.k[t][i][e], qf[0][i][e], z[e & 1], 0, 0, 0);
                    }
                }
                st[t] = QP == 2 || !H16 ? z[0] + z[1] : z[0];
            }
            bool odd = false;  // pages that do not exist
#pragma unroll
            for (int t = 0; t < TK; t++) odd |= (uint32_t)d.p[t] >= (uint32_t)c.n_pages;
            const bool edge = j0 + 16 * TK > lim_lo;
            bool fix = false;
            if (__builtin_expect(edge || odd, 0)) {
#pragma unroll
                for (int t = 0; t < TK; t++) {
                    const bool none = (uint32_t)d.p[t] >= (uint32_t)c.n_pages;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (none) st[t][e] = NAN;  // (over values of zero)
                        if (j0 + 16 * t + 4 * g + e >= lim) st[t][e] = -INFINITY;
                    }
                }
                // values that only some rows see: a weight of 0 would not silence an infinity.
                // Infinities and NaN are taken out of the product and added to the rows that see them
                if (lim_lo < lim_hi) {
                    uint32_t wild = 0;
#pragma unroll
                    for (int e = 0; e < 4 * TK; e++)
#pragma unroll
                        for (int i = 0; i < VN; i++) {
                            words u = __builtin_bit_cast(words, f.v[e][i]);
#pragma unroll
                            for (int y = 0; y < (int)(sizeof(vec) / 4); y++) {
                                const uint32_t z = not_finite<KVT>(u[y]);
                                wild |= z;
                                u[y] &= ~z;
                            }
                            f.v[e][i] = __builtin_bit_cast(vec, u);
                        }
                    fix = __ballot(wild != 0) != 0;
                }
            }
            float mt = st[0][0];
#pragma unroll
            for (int t = 0; t < TK; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) mt = fmaxf(mt, st[t][e]);
            mt = lane_pair_max<16>(mt);
            mt = lane_pair_max<32>(mt);
            const float mn = fmaxf(m, mt), ms = mn == -INFINITY ? 0.f : mn;
            if (__ballot(mn != m)) {
                const float al = __builtin_amdgcn_exp2f((m - ms) * cs);
                l *= al;
#pragma unroll
                for (int i = 0; i < NA; i++) acc[i] *= al;
            }
            m = mn;
#pragma unroll
            for (int t = 0; t < TK; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    st[t][e] = __builtin_amdgcn_exp2f(H16 ? fmaf(st[t][e] - ms, cs, 15.0f) : (st[t][e] - ms) * cs);
                    l += st[t][e];
                }
            if constexpr (H16) {
                constexpr int KM = TK == 1 ? 1 : TK / 2;  // matrix instructions per operand
                typedef std::conditional_t<TK == 1, half4v, half8> op;
                constexpr int N = TK == 1 ? 4 : 8;
#pragma unroll
                for (int u = 0; u < KM; u++) {
                    op hi, lo;
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const float p = st[2 * u + e / 4][e % 4];
                        hi[e] = (_Float16)p;
                        lo[e] = (_Float16)(p - (float)hi[e]);
                    }
#pragma unroll
                    for (int i = 0; i < VN; i++)
#pragma unroll
                        for (int y = 0; y < VE; y++) {
                            op av;
#pragma unroll
                            for (int e = 0; e < N; e++) av[e] = f.v[N * u + e][i][y];
                            floatx4& o = acc[i * VE + y];
                            if constexpr (TK == 1) {
                                o = __builtin_amdgcn_mfma_f32_16x16x16f16(av, hi, o, 0, 0, 0);
                                o = __builtin_amdgcn_mfma_f32_16x16x16f16(av, lo, o, 0, 0, 0);
                            } else {
                                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, hi, o, 0, 0, 0);
                                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, lo, o, 0, 0, 0);
                            }
                        }
                }
            } else {
#pragma unroll
                for (int t = 0; t < TK; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int i = 0; i < VN; i++)
#pragma unroll
                            for (int y = 0; y < VE; y++)
                                acc[i * VE + y] = __builtin_amdgcn_mfma_f32_16x16x4f32(f.v[4 * t + e][i][y], st[t][e], acc[i * VE + y], 0, 0, 0);
            }
            if (__builtin_expect(fix, 0)) {
#pragma unroll 1
                for (int k = 0; k < 16 * TK; k++) {
                    int dims = D;
                    asm volatile("" : "+s"(dims));  // its comparisons stay here
                    const int j = j0 + k;
                    if (j >= lim_hi) break;
                    const int p = row[j >> c.shift];
                    if ((uint32_t)p >= (uint32_t)c.n_pages || j >= lim) continue;
                    const KVT* vr = reinterpret_cast<const KVT*>(vp + (p * c.page_elems + (int64_t)(j & (page - 1)) * D) * EB + head);
#pragma unroll
                    for (int i = 0; i < NA; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int dim = 16 * VE * (i / VE) + VE * (4 * g + e) + i % VE;
                            const float v = FULL || dim < dims ? (float)vr[dim] : 0.f;
                            acc[i][e] += __uint_as_float(__float_as_uint(v) & not_finite<float>(__float_as_uint(v)));
                        }
                }
            }
        };

        // the next block's loads are in flight under this one's work; none is conditional, or the
        // waits would count for the path without it
        for (int s = 0; s < steps; s += 2) {
            load(s + 1, d1, f1);
            __builtin_amdgcn_sched_barrier(0);
            const Ids d2 = ids_of(s + 2), d3 = ids_of(s + 3);
            compute(s, d0, f0);
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 >= steps) break;
            load(s + 2, d2, f0);
            __builtin_amdgcn_sched_barrier(0);
            compute(s + 1, d1, f1);
            __builtin_amdgcn_sched_barrier(0);
            d0 = d2, d1 = d3;
        }
        l = lane_pair_sum<16>(l);
        l = lane_pair_sum<32>(l);
        __syncthreads();  // so is free
        if (g == 0) so[wave][col][DP] = m, so[wave][col][DP + 1] = l, so[wave][col][DP + 2] = cs;
        // lane: dimensions 16 VE i + VE (4 g + e) + y of row col
#pragma unroll
        for (int i = 0; i < VN; i++)
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int y = 0; y < VE; y += 4)
                    *reinterpret_cast<floatx4*>(&so[wave][col][16 * VE * i + VE * (4 * g + e) + y]) =
                        floatx4{acc[i * VE + y][e], acc[i * VE + y + 1][e], acc[i * VE + y + 2][e], acc[i * VE + y + 3][e]};
        __syncthreads();
        // thread: row tr, every TPR-th float4 of it
        constexpr int TPR = 4 * NW;
        const int tr = threadIdx.x / TPR, tc = threadIdx.x % TPR;
        const float rc = so[0][tr][DP + 2];
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < NW; v++) M = fmaxf(M, so[v][tr][DP]);
        const float Ms = M == -INFINITY ? 0.f : M;
        float fw[NW], sum = 0.f;
#pragma unroll
        for (int v = 0; v < NW; v++) fw[v] = __builtin_amdgcn_exp2f((so[v][tr][DP] - Ms) * rc), sum = fmaf(so[v][tr][DP + 1], fw[v], sum);
        const bool whole = r0 == 0 && r1 == w.rounds;
        const int orow = tile * 16 + tr, oq = PACKED ? orow / G : 0;
        const uint32_t rec = (uint32_t)(2 * run + (r0 == 0 ? 1 : 0)) * (16 * (D + 4) * 4) + tr * (D + 4) * 4;  // bytes
        const __amdgpu_buffer_rsrc_t ws = buf_rsrc(a.ws, RUNS * 2 * 16 * (D + 4) * 4);
        const int sees = sq.shown + oq;
        const float inv = sees > sq.len ? NAN : 1.0f / sum;
        QT* op = static_cast<QT*>(a.out) + ((int64_t)(sq.first + oq) * a.hq + h * G + orow - oq * G) * D;
        if (orow < rows) {
#pragma unroll
            for (int i = 0; i < (DP + 4 * TPR - 1) / (4 * TPR); i++) {
                const int dim = 4 * TPR * i + 4 * tc;
                if (dim >= D) continue;
                floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int v = 0; v < NW; v++) {
                    const floatx4 z = *reinterpret_cast<const floatx4*>(&so[v][tr][dim]);
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = fmaf(z[e], fw[v], o[e]);
                }
                if (!whole) {
                    // through to where every XCD sees it
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), ws, rec + 4 * dim, 0, CPOL_SC1);
                } else {
                    if (sees <= 0) o = floatx4{0.f, 0.f, 0.f, 0.f};
                    else o *= inv;
                    if constexpr (std::is_same_v<QT, float>) *reinterpret_cast<floatx4*>(op + dim) = o;
                    else *reinterpret_cast<half4v*>(op + dim) = half4v{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
                }
            }
            if (!whole && tc == 0)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, floatx4{M, sum, rc, 0.f}), ws, rec + 4 * D, 0, CPOL_SC1);
        }
        if (a.fuse && !whole) {
            // Every wave waits until its record has reached the point that all XCDs see, then
            // one thread arrives; the records are read past the caches, after the arrival.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const int run0 = (uint32_t)begin / (uint32_t)len_run, parts = (uint32_t)(begin + w.rounds - 1) / (uint32_t)len_run - run0 + 1;
            if (threadIdx.x == 0) {
                const uint32_t old = __hip_atomic_fetch_add(&g_paged_arrive[run0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                const bool end = old == (uint32_t)(parts - 1);
                if (end) __hip_atomic_store(&g_paged_arrive[run0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last_here = end;
            }
            __syncthreads();
            if (last_here) join_run<QT, CPOL_SC1, 64 * NW>(a, sq, h, tile, run0, parts, &so[0][0][0]);
        }
    }
}

// ---- prompts: which work is whose ----
// Tiles of 2^shift rows, `unit` = KV head + n_kv_heads * tile: heads next to each other (on XCDs
// of their own), the tiles that see most first (beyond 64 sequences: of each sequence).  Seven
// prompts, 4001 rows together, 1024 units: 77 us, against 82 with the sequences one by one.
// A call with few units cuts each unit's positions into up to `most` parts, of about four K/V
// tiles at least; a workgroup takes unit index % units, part index / units, and leaves a record
// (o, m, l, c of its rows) in slot unit * most + part, which k_prompt_join adds.
constexpr int SLOTS = 512;
struct Prompt {
    Seq sq;
    int b, h, tile, unit, units;
};
// index: the workgroup's or, with whole, a unit's.
__device__ __forceinline__ bool prompt_tile(const PagedCache& c, const int32_t* cu, const int32_t* lens, int G, int shift, int index,
                                            int most, bool whole, Prompt* p) {
    const int up = (1 << shift) - 1;
    Group<true> grp;
    int total = 0, incl = 0, mine = 0;
    for (int base = 0; base < c.batch; base += 64) {
        grp.load(c, cu, lens, base);
        mine = (grp.q.n * G + up) >> shift;
        incl = lane_prefix(mine);
        total += lane_value(incl, 63);
    }
    p->units = total * c.hkv;  // (rows and heads together are below 2^27)
    if (p->units == 0) return false;
    p->unit = most > 1 && !whole ? index % p->units : index;
    if (p->unit >= p->units) return false;
    p->h = p->unit % c.hkv;
    // tiles before this one; the second 256 units, which share CUs with the first, come shortest
    // first (f32 caches, 3 prompts, 900 rows of 8 x 256 together: 104 us, 117 in plain order)
    int nth = p->unit / c.hkv;
    const int one = 256 / c.hkv, two = min(2 * one, total);
    if (nth >= one && nth < two) nth = one + two - 1 - nth;
    if (c.batch <= 64) {
        // Longest first: tile t of a sequence weighs first + t, its position in tiles.  The nth
        // heaviest of all weighs the most that more than nth tiles weigh or pass.
        const int first = (int)max(min(((int64_t)grp.q.shown * G) >> shift, (int64_t)1 << 29), -((int64_t)1 << 29));
        auto reach = [&](int w) {  // tiles that weigh w or more
            return lane_value(lane_prefix(max(min(first + mine - w, mine), 0)), 63);
        };
        int lo = mine > 0 ? first : 1 << 30, hi = mine > 0 ? first + mine - 1 : -(1 << 30);  // (total is not 0)
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) lo = min(lo, __shfl_xor(lo, off)), hi = max(hi, __shfl_xor(hi, off));
        lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
        while (lo < hi) {
            const int mid = lo + ((hi - lo + 1) >> 1);
            if (reach(mid) > nth) lo = mid;
            else hi = mid - 1;
        }
        int skip = nth - reach(lo + 1);
        uint64_t hit = __ballot(lo >= first && lo - first < mine);
        for (; skip > 0; skip--) hit &= hit - 1;
        p->b = __builtin_ctzll(hit);
        p->tile = lo - lane_value(first, p->b);
        p->sq = grp.at(p->b);
        return true;
    }
    int before = 0;
    for (int base = 0;; base += 64) {
        grp.load(c, cu, lens, base);
        mine = (grp.q.n * G + up) >> shift;
        incl = lane_prefix(mine);
        const uint64_t hit = __ballot(nth < before + incl);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            p->b = base + at;
            const int t = nth - (before + lane_value(incl, at) - lane_value(mine, at));
            p->tile = lane_value(mine, at) - 1 - t;
            break;
        }
        before += lane_value(incl, 63);
    }
    p->sq = grp.at(p->b);
    return true;
}
// Parts of a unit with this many K/V tiles.
__device__ __forceinline__ int prompt_parts(int most, int tiles) { return max(min(most, (tiles + 3) / 4), 1); }

// ---- prompts over f16 caches -------------------------------------------------------------
// A workgroup takes 128 rows, a wavefront 32 of them; 64 positions (32 at head sizes past 128) at
// a time reach LDS by DMA, the next ones under the work on these.  S^T = K Q^T and
// O^T += V^T P^T on v_mfma_f32_32x32x16_f16: lane (col, hf) = (l % 32, l / 32) holds row col's scores at
// keys 8 (i / 4) + 4 hf + i % 4 of 32, which are the k slots of the second product as they stand;
// V^T is read from row-major V by the transposing LDS reads.  Rows that nothing asks for, of
// positions past the last one seen and of dimensions past head_dim, lie outside the buffer
// resources and arrive as zeros.
// 16-byte chunks of K rows are spread by the row, so that 16 rows of one chunk lie in 16
// different places of the banks; chunks of V rows by quarters, for four rows of 64 bytes (no bank
// conflicts counted).
// Bound by the matrix units, at the card's power limit in long calls: 8192 rows over 8192 positions
// and themselves, 32 heads over 8 of 128, f16 rows 1.65 ms, 1000 TFLOP/s; f32 rows take every
// product twice, 7 prompts of 4001 rows together 72 us.
template <int DP>
struct PromptTile {
    static constexpr int KT = DP > 128 ? 32 : 64;
    static constexpr int CPR = DP / 8;       // chunks per row
    static constexpr int U = KT * CPR / 256; // DMA instructions per wavefront and operand
    __device__ static int spread_k(int r) { return CPR == 8 ? (r >> 1) & 7 : r & 15; }
    __device__ static int spread_v(int r) { return CPR == 8 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }
};

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));

// W: groups of four wavefronts.  With two each takes every second tile of the workgroup's, in
// buffers of its own, and the second's sums reach the first through LDS: for calls whose units are
// about as many as the CUs.
template <typename QT, int DP, int W>
__global__ __launch_bounds__(256 * W, (DP > 128 ? 1 : 2)) void k_paged_prompt(
    const PagedAttn a, const int32_t* __restrict__ table, const int32_t* __restrict__ cu, const int32_t* __restrict__ lens,
    const char* __restrict__ kp, const char* __restrict__ vp, int most) {
    using L = PromptTile<DP>;
    constexpr int KT = L::KT, CPR = L::CPR, U = L::U, RPW = KT / 4;
    constexpr int QP = std::is_same_v<QT, float> ? 2 : 1;  // f16 parts of a query, and of a weight
    constexpr int KS = DP / 16, DT = DP / 32, ST = KT / 32;
    struct Stage {
        uint4 k[KT * CPR], v[KT * CPR];
    };
    __shared__ __attribute__((aligned(16))) Stage S[2 * W];
    const PagedCache& c = a.c;
    const int lane = threadIdx.x & 63, wave4 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wave4 & 3, group = W == 1 ? 0 : wave4 >> 2, col = lane & 31, hf = lane >> 5;
    const int G = a.G, D = c.D, page = 1 << c.shift;

    Prompt pt;
    if (!prompt_tile(c, cu, lens, G, 7, blockIdx.x, most, false, &pt)) return;
    const Seq sq = pt.sq;
    const int b = pt.b, h = pt.h, tile = pt.tile;
    const int rows = sq.n * G;
    auto limit = [&](int row) { return limit_of(sq, min(row, rows - 1) / G); };
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int w0 = tile * 128 + wave * 32, r = min(w0 + col, rows - 1), qi = r / G, qh = h * G + r - qi * G;
    const int lim = limit(r), lim_hi = uniform(limit(w0 + 31));
    const int last = uniform(limit(tile * 128 + 127)), all = uniform(limit(tile * 128));  // positions that any, that every row sees
    const bool live = w0 < rows;
    // this part's K/V tiles
    const int tiles = (last + KT - 1) / KT, whole = all / KT, parts = prompt_parts(most, tiles), part = most > 1 ? blockIdx.x / pt.units : 0;
    if (part >= parts) return;
    const int t0 = most > 1 ? (int)((int64_t)tiles * part / parts) : 0, t1 = most > 1 ? (int)((int64_t)tiles * (part + 1) / parts) : tiles;

    // this lane's part of its row: dimensions 16 s + 8 hf ..
    const QT* qp = static_cast<const QT*>(a.q) + (int64_t)(sq.first + qi) * a.q_stride + qh * D;
    const float sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
    float cs = fminf(fabsf(a.scale) * 1.44269504088896341f, FLT_MAX);
    half8 qf[QP][KS];
    if constexpr (QP == 2) {
        float top = 0.f;
        floatx4 qv[KS][2];
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                qv[s][e] = 16 * s + 8 * hf < D ? reinterpret_cast<const floatx4*>(qp + 16 * s + 8 * hf)[e] : floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(qv[s][e][i]));
            }
        top = lane_pair_max<32>(top);
        const int up = top > 0.f && top <= FLT_MAX ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        cs = fminf(ldexpf(fabsf(a.scale) * 1.44269504088896341f, -up), FLT_MAX);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float f = ldexpf(qv[s][i / 4][i % 4] * sign, up);
                qf[0][s][i] = (_Float16)f;
                qf[1][s][i] = (_Float16)(f - (float)qf[0][s][i]);
            }
    } else {
#pragma unroll
        for (int s = 0; s < KS; s++) {
            half8 z = {};
            if (16 * s + 8 * hf < D) z = *reinterpret_cast<const half8*>(qp + 16 * s + 8 * hf);
#pragma unroll
            for (int i = 0; i < 8; i++) qf[0][s][i] = z[i] * (_Float16)sign;
        }
    }
    cs = fmaxf(cs, FLT_MIN);

    // DMA: this wavefront's rows RPW wave .. of a tile, all in one page
    uint32_t ko[U], vo[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int at = u * 64 + lane, rr = at / CPR, ch = at % CPR, tr = wave * RPW + rr;
        const int ck = ch ^ L::spread_k(tr), cv = ch ^ L::spread_v(tr);
        ko[u] = 8 * ck < D ? (uint32_t)(rr * D + 8 * ck) * 2 : 0x7FFFFFF0u;
        vo[u] = 8 * cv < D ? (uint32_t)(rr * D + 8 * cv) * 2 : 0x7FFFFFF0u;
    }
    const table_ptr row = table_row(table, c, b);
    const int64_t head = (int64_t)h * page * D;
    auto page_of = [&](int j0) { return row[uniform(max(min(j0 + wave * RPW, last - 1), 0) >> c.shift)]; };
    auto issue = [&](int j0, int pid, Stage& st) __attribute__((always_inline)) {
        const int j = j0 + wave * RPW;
        const bool none = (uint32_t)pid >= (uint32_t)c.n_pages;
        const int64_t at = ((none ? 0 : pid) * c.page_elems + head + (int64_t)(j & (page - 1)) * D) * 2;
        const uint32_t bytes = (uint32_t)uniform(none ? 0 : max(min(last - j, RPW), 0) * D * 2);
        const __amdgpu_buffer_rsrc_t rk = buf_rsrc(kp + at, bytes), rv = buf_rsrc(vp + at, bytes);
        if (!none) {
#pragma unroll
            for (int u = 0; u < U; u++) buf_dma16(rk, ko[u], 0, &st.k[(wave * U + u) * 64]);
        } else {  // a page that does not exist: NaN scores over zero values
#pragma unroll
            for (int u = 0; u < U; u++) st.k[(wave * U + u) * 64 + lane] = make_uint4(0x7E007E00u, 0x7E007E00u, 0x7E007E00u, 0x7E007E00u);
        }
#pragma unroll
        for (int u = 0; u < U; u++) buf_dma16(rv, vo[u], 0, &st.v[(wave * U + u) * 64]);
    };

    float m = -INFINITY, l = 0.f;
    floatx16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[i][e] = 0.f;

    const int trow = 4 * hf + ((lane & 15) >> 2);  // the key of this lane's address in a transposing read
    auto compute = [&](int j0, const char* st, auto edge) __attribute__((always_inline)) {
        constexpr bool EDGE = decltype(edge)::value;
        floatx16 sc[ST];
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) sc[t][e] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int t = 0; t < ST; t++) {
                const int kr = 32 * t + col;
                const half8 kf = __builtin_bit_cast(half8, reinterpret_cast<const uint4*>(st)[kr * CPR + ((2 * s + hf) ^ L::spread_k(kr))]);
#pragma unroll
                for (int p = 0; p < QP; p++) sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[p][s], sc[t], 0, 0, 0);
            }
        if constexpr (EDGE) {
#pragma unroll
            for (int t = 0; t < ST; t++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (j0 + 32 * t + 8 * (e / 4) + 4 * hf + e % 4 >= lim) sc[t][e] = -INFINITY;
        }
        float mt = sc[0][0];
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) mt = fmaxf(mt, sc[t][e]);
        mt = lane_pair_max<32>(mt);
        // the maximum is raised only where weights would pass 2^8 (times 2^7, f16's range)
        if (__ballot((mt - m) * cs > 8.0f)) {
            const float mn = fmaxf(m, mt), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * cs);
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < DT; i++) acc[i] *= al;
        }
        const float ms = m == -INFINITY ? 0.f : m, bias = fmaf(-ms, cs, 7.0f);
        half8 pf[QP][KT / 16];
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float p = __builtin_amdgcn_exp2f(QP == 2 ? fmaf(sc[t][e] - ms, cs, 7.0f) : fmaf(sc[t][e], cs, bias));
                l += p;
                const _Float16 hi = (_Float16)p;
                pf[0][2 * t + e / 8][e % 8] = hi;
                if constexpr (QP == 2) pf[1][2 * t + e / 8][e % 8] = (_Float16)(p - (float)hi);
            }
        uint32_t wild = 0;
        const _Float16* vh = reinterpret_cast<const _Float16*>(st + sizeof(Stage::k));
#pragma unroll
        for (int s = 0; s < KT / 16; s++)
#pragma unroll
            for (int i = 0; i < DT; i++) {
                const int ch = 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
                uint2 w[2];
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int kr = 16 * s + 8 * y + trow;
                    const _Float16* p = vh + kr * DP + 8 * (ch ^ L::spread_v(kr)) + 4 * (lane & 1);
                    w[y] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p));
                }
                uint4 f = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
                if constexpr (EDGE) {  // infinities and NaN: added below to the rows that see them
                    uint32_t* u = &f.x;
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const uint32_t z = not_finite<_Float16>(u[y]);
                        wild |= z;
                        u[y] &= ~z;
                    }
                }
                const half8 vf = __builtin_bit_cast(half8, f);
#pragma unroll
                for (int p = 0; p < QP; p++) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[p][s], acc[i], 0, 0, 0);
            }
        if constexpr (EDGE) {
            if (__ballot(wild != 0)) {
#pragma unroll 1
                for (int k = 0; k < KT && j0 + k < last; k++) {
                    if (j0 + k >= lim) continue;
#pragma unroll
                    for (int i = 0; i < DT; i++)
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int d = 32 * i + 8 * (e / 4) + 4 * hf + e % 4;
                            const uint32_t v = __float_as_uint((float)vh[k * DP + 8 * ((d >> 3) ^ L::spread_v(k)) + (d & 7)]);
                            acc[i][e] += __uint_as_float(v & not_finite<float>(v));
                        }
                }
            }
        }
    };

    if (t0 < t1) {
        auto buffer = [&](int t) { return W == 1 ? t & 1 : 2 * group + (((t - t0) >> 1) & 1); };
        int pid = page_of((t0 + group) * KT);
        if (W == 1 || t0 + group < t1) issue((t0 + group) * KT, pid, S[buffer(t0)]);
        pid = page_of((t0 + W + group) * KT);
        auto step = [&](int t, auto edge) __attribute__((always_inline)) {  // tiles t .. t + W - 1
            __builtin_amdgcn_s_waitcnt(0xF70);  // vmcnt(0): this tile's DMA has landed
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            const int mine = t + group;
            if (mine + W < t1) {
                issue((mine + W) * KT, pid, S[buffer(t + W)]);
                pid = page_of((mine + 2 * W) * KT);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (live && (W == 1 || mine < t1) && mine * KT < lim_hi) compute(mine * KT, reinterpret_cast<const char*>(&S[buffer(t)]), edge);
        };
        int t = t0;
#pragma unroll 1
        for (; t + W <= min(whole, t1); t += W) step(t, std::false_type{});
#pragma unroll 1
        for (; t < t1; t += W) step(t, std::true_type{});
    }
    l = lane_pair_sum<32>(l);
    if constexpr (W == 2) {
        static_assert(4 * 64 * (16 * DT + 2) * 4 <= (int)sizeof(S), "the second group's sums");
        floatx4* room = reinterpret_cast<floatx4*>(S) + wave * 64 * 4 * DT;
        float* ml = reinterpret_cast<float*>(S) + 4 * 64 * 16 * DT + wave * 128 + lane;
        __syncthreads();  // the tiles are read
        if (group) {
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    room[(4 * i + e) * 64 + lane] = floatx4{acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]};
            ml[0] = m, ml[64] = l;
        }
        __syncthreads();
        if (group) return;
        const float mo = ml[0], mn = fmaxf(m, mo), ms = mn == -INFINITY ? 0.f : mn;
        const float f = __builtin_amdgcn_exp2f((m - ms) * cs), fo = __builtin_amdgcn_exp2f((mo - ms) * cs);
        m = mn;
        l = fmaf(l, f, ml[64] * fo);
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const floatx4 z = room[(4 * i + e) * 64 + lane];
#pragma unroll
                for (int y = 0; y < 4; y++) acc[i][4 * e + y] = fmaf(acc[i][4 * e + y], f, z[y] * fo);
            }
    }
    if (w0 + col >= rows) return;
    const int sees = sq.shown + qi;
    const float inv = sees > sq.len ? NAN : 1.0f / l;
    QT* op = static_cast<QT*>(a.out) + ((int64_t)(sq.first + qi) * a.hq + qh) * D;
    float* rec = a.ws + ((int64_t)(pt.unit * most + part) * 128 + wave * 32 + col) * (D + 4);
    if (parts > 1 && hf == 0) *reinterpret_cast<floatx4*>(rec + D) = floatx4{m, l, cs, 0.f};
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = 32 * i + 8 * e + 4 * hf;
            if (d >= D) continue;
            floatx4 o = {acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]};
            if (parts > 1) {
                *reinterpret_cast<floatx4*>(rec + d) = o;
                continue;
            }
            if (sees <= 0) o = floatx4{0.f, 0.f, 0.f, 0.f};
            else o *= inv;
            if constexpr (std::is_same_v<QT, float>) *reinterpret_cast<floatx4*>(op + d) = o;
            else *reinterpret_cast<half4v*>(op + d) = half4v{(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
        }
}

// ---- prompts over f32 caches -------------------------------------------------------------
// The same with f32 matrix instructions (v_mfma_f32_16x16x4_f32): 64 rows to a workgroup, 16 to a
// wavefront, 16 KiB of keys and of values at a time.  Lane (col, g) holds row col's scores at
// keys 4 g + e of 16; one 16-byte read of a value row feeds four matrix instructions, dimension
// 64 j + 4 r + y in row r of number y.  3 prompts of 1100 rows together, 32 heads over 4 of 64: 38 us
// (2.5 GFLOP, 66 TFLOP/s); while a CU works its matrix units do 59 % of the time.
template <int DP>
__global__ __launch_bounds__(256, 2) void k_paged_prompt_f32(
    const PagedAttn a, const int32_t* __restrict__ table, const int32_t* __restrict__ cu, const int32_t* __restrict__ lens,
    const char* __restrict__ kp, const char* __restrict__ vp, int most) {
    constexpr int CPR = DP / 4, KT = 1024 / CPR, U = 4, RPW = KT / 4, ST = KT / 16, KS = DP / 16, VN = DP / 64;
    struct Stage {
        uint4 k[KT * CPR], v[KT * CPR];
    };
    __shared__ __attribute__((aligned(16))) Stage S[2];
    const PagedCache& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
    const int G = a.G, D = c.D, page = 1 << c.shift;
    Prompt pt;
    if (!prompt_tile(c, cu, lens, G, 6, blockIdx.x, most, false, &pt)) return;
    const Seq sq = pt.sq;
    const int b = pt.b, h = pt.h, tile = pt.tile;
    const int rows = sq.n * G;
    auto limit = [&](int row) { return limit_of(sq, min(row, rows - 1) / G); };
    auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    const int w0 = tile * 64 + wave * 16, r = min(w0 + col, rows - 1), qi = r / G, qh = h * G + r - qi * G;
    const int lim = limit(r), lim_hi = uniform(limit(w0 + 15));
    const int last = uniform(limit(tile * 64 + 63)), all = uniform(limit(tile * 64));  // positions that any, that every row sees
    const bool live = w0 < rows;
    // this part's K/V tiles
    const int tiles = (last + KT - 1) / KT, whole = all / KT, parts = prompt_parts(most, tiles), part = most > 1 ? blockIdx.x / pt.units : 0;
    if (part >= parts) return;
    const int t0 = most > 1 ? (int)((int64_t)tiles * part / parts) : 0, t1 = most > 1 ? (int)((int64_t)tiles * (part + 1) / parts) : tiles;

    const float* qp = static_cast<const float*>(a.q) + (int64_t)(sq.first + qi) * a.q_stride + qh * D;
    const float sign = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
    const float cs = fmaxf(fminf(fabsf(a.scale) * 1.44269504088896341f, FLT_MAX), FLT_MIN);
    floatx4 qf[KS];
#pragma unroll
    for (int s = 0; s < KS; s++) {
        qf[s] = floatx4{0.f, 0.f, 0.f, 0.f};
        if (16 * s + 4 * g < D) qf[s] = *reinterpret_cast<const floatx4*>(qp + 16 * s + 4 * g);
        qf[s] *= sign;
    }

    uint32_t ko[U], vo[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int at = u * 64 + lane, rr = at / CPR, ch = at % CPR, ck = ch ^ ((wave * RPW + rr) & 15);
        ko[u] = 4 * ck < D ? (uint32_t)(rr * D + 4 * ck) * 4 : 0x7FFFFFF0u;
        vo[u] = 4 * ch < D ? (uint32_t)(rr * D + 4 * ch) * 4 : 0x7FFFFFF0u;
    }
    const table_ptr row = table_row(table, c, b);
    const int64_t head = (int64_t)h * page * D;
    auto page_of = [&](int j0) { return row[uniform(max(min(j0 + wave * RPW, last - 1), 0) >> c.shift)]; };
    auto issue = [&](int j0, int pid, Stage& st) __attribute__((always_inline)) {
        const int j = j0 + wave * RPW;
        const bool none = (uint32_t)pid >= (uint32_t)c.n_pages;
        const int64_t at = ((none ? 0 : pid) * c.page_elems + head + (int64_t)(j & (page - 1)) * D) * 4;
        const uint32_t bytes = (uint32_t)uniform(none ? 0 : max(min(last - j, RPW), 0) * D * 4);
        const __amdgpu_buffer_rsrc_t rk = buf_rsrc(kp + at, bytes), rv = buf_rsrc(vp + at, bytes);
        if (!none) {
#pragma unroll
            for (int u = 0; u < U; u++) buf_dma16(rk, ko[u], 0, &st.k[(wave * U + u) * 64]);
        } else {  // a page that does not exist: NaN scores over zero values
#pragma unroll
            for (int u = 0; u < U; u++) st.k[(wave * U + u) * 64 + lane] = make_uint4(0x7FC00000u, 0x7FC00000u, 0x7FC00000u, 0x7FC00000u);
        }
#pragma unroll
        for (int u = 0; u < U; u++) buf_dma16(rv, vo[u], 0, &st.v[(wave * U + u) * 64]);
    };

    float m = -INFINITY, l = 0.f;
    floatx4 acc[KS];
#pragma unroll
    for (int i = 0; i < KS; i++) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int j0, const char* st, auto edge) __attribute__((always_inline)) {
        constexpr bool EDGE = decltype(edge)::value;
        const uint4 *ks = reinterpret_cast<const uint4*>(st), *vs = ks + KT * CPR;
        floatx4 sc[ST][2];
#pragma unroll
        for (int t = 0; t < ST; t++) sc[t][0] = sc[t][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int t = 0; t < ST; t++) {
                const floatx4 kf = __builtin_bit_cast(floatx4, ks[(16 * t + col) * CPR + ((4 * s + g) ^ col)]);
#pragma unroll
                for (int e = 0; e < 4; e++) sc[t][e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[s][e], sc[t][e & 1], 0, 0, 0);
            }
        float mt = -INFINITY;
#pragma unroll
        for (int t = 0; t < ST; t++) {
            sc[t][0] += sc[t][1];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (EDGE && j0 + 16 * t + 4 * g + e >= lim) sc[t][0][e] = -INFINITY;
                mt = fmaxf(mt, sc[t][0][e]);
            }
        }
        mt = lane_pair_max<16>(mt);
        mt = lane_pair_max<32>(mt);
        if (__ballot((mt - m) * cs > 8.0f)) {  // (weights stay below 2^8)
            const float mn = fmaxf(m, mt), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * cs);
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < KS; i++) acc[i] *= al;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        uint32_t wild = 0;
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p = __builtin_amdgcn_exp2f((sc[t][0][e] - ms) * cs);
                l += p;
#pragma unroll
                for (int i = 0; i < VN; i++) {
                    uint4 w = vs[(16 * t + 4 * g + e) * CPR + 16 * i + col];
                    if constexpr (EDGE) {  // infinities and NaN: added below to the rows that see them
                        uint32_t* u = &w.x;
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const uint32_t z = not_finite<float>(u[y]);
                            wild |= z;
                            u[y] &= ~z;
                        }
                    }
                    const floatx4 vf = __builtin_bit_cast(floatx4, w);
#pragma unroll
                    for (int y = 0; y < 4; y++) acc[4 * i + y] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[y], p, acc[4 * i + y], 0, 0, 0);
                }
            }
        if constexpr (EDGE) {
            if (__ballot(wild != 0)) {
#pragma unroll 1
                for (int k = 0; k < KT && j0 + k < last; k++) {
                    if (j0 + k >= lim) continue;
#pragma unroll
                    for (int i = 0; i < KS; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t v = reinterpret_cast<const uint32_t*>(vs)[k * DP + 64 * (i / 4) + 4 * (4 * g + e) + i % 4];
                            acc[i][e] += __uint_as_float(v & not_finite<float>(v));
                        }
                }
            }
        }
    };

    if (t0 < t1) {
        int pid = page_of(t0 * KT);
        issue(t0 * KT, pid, S[t0 & 1]);
        pid = page_of((t0 + 1) * KT);
        auto step = [&](int t, auto edge) __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(0xF70);  // vmcnt(0): this tile's DMA has landed
            __syncthreads();
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < t1) {
                issue((t + 1) * KT, pid, S[(t + 1) & 1]);
                pid = page_of((t + 2) * KT);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (live && t * KT < lim_hi) compute(t * KT, reinterpret_cast<const char*>(&S[t & 1]), edge);
        };
        int t = t0;
#pragma unroll 1
        for (; t < min(whole, t1); t++) step(t, std::false_type{});
#pragma unroll 1
        for (; t < t1; t++) step(t, std::true_type{});
    }
    l = lane_pair_sum<16>(l);
    l = lane_pair_sum<32>(l);
    if (w0 + col >= rows) return;
    const int sees = sq.shown + qi;
    const float inv = sees > sq.len ? NAN : 1.0f / l;
    float* op = static_cast<float*>(a.out) + ((int64_t)(sq.first + qi) * a.hq + qh) * D;
    float* rec = a.ws + ((int64_t)(pt.unit * most + part) * 64 + wave * 16 + col) * (D + 4);
    if (parts > 1 && g == 0) *reinterpret_cast<floatx4*>(rec + D) = floatx4{m, l, cs, 0.f};
#pragma unroll
    for (int i = 0; i < VN; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = 64 * i + 4 * (4 * g + e);
            if (d >= D) continue;
            floatx4 o = {acc[4 * i][e], acc[4 * i + 1][e], acc[4 * i + 2][e], acc[4 * i + 3][e]};
            if (parts > 1) {
                *reinterpret_cast<floatx4*>(rec + d) = o;
                continue;
            }
            if (sees <= 0) o = floatx4{0.f, 0.f, 0.f, 0.f};
            else o *= inv;
            *reinterpret_cast<floatx4*>(op + d) = o;
        }
}

// Adds the parts of cut units, 16 rows to a workgroup: a launch, and one wait per eight parts.
template <typename QT>
__global__ __launch_bounds__(256) void k_prompt_join(const PagedAttn a, const int32_t* __restrict__ cu, const int32_t* __restrict__ lens, int shift, int keys, int most) {
    __shared__ __attribute__((aligned(16))) float room[256 * JOIN_ROOM];
    const PagedCache& c = a.c;
    const int G = a.G, per = 1 << (shift - 4), sub = blockIdx.x & (per - 1);
    Prompt pt;
    if (!prompt_tile(c, cu, lens, G, shift, blockIdx.x / per, most, true, &pt)) return;
    const int rows = pt.sq.n * G, r0 = (pt.tile << shift) + 16 * sub;
    if (r0 >= rows) return;
    const int last = limit_of(pt.sq, min((pt.tile << shift) + (1 << shift) - 1, rows - 1) / G);
    const int parts = prompt_parts(most, (last + keys - 1) / keys);
    if (parts == 1) return;
    const uint32_t row = (c.D + 4) * 4, slot = row << shift, first = (uint32_t)(pt.unit * most) * slot + 16 * sub * row;
    join_tile<QT, 0, 256>(a, pt.sq, pt.h, r0 >> 4, first, first, slot, parts, (uint32_t)SLOTS * slot, room);
}

// The join, one workgroup per (sequence, KV head, tile) that there can be, in the line's order:
// for calls whose parts are not joined where they were made (one sequence of 512: the two launches
// 10.4 us, the one 8.0).
template <typename QT, bool PACKED, int NT>
__global__ __launch_bounds__(NT) void k_paged_join(const PagedAttn a, const int32_t* __restrict__ cu, const int32_t* __restrict__ lens, int keys, int runs) {
    __shared__ __attribute__((aligned(16))) float room[NT * JOIN_ROOM];
    const PagedCache& c = a.c;
    const int G = a.G;
    Group<PACKED> grp;
    Seq sq{};
    int total = 0, units = 0, at = -1, nth = 0;
    int b = -1;
    for (int base = 0; base < c.batch; base += 64) {
        grp.load(c, cu, lens, base);
        const Work w = work_of(grp.q, G, keys);
        const int wu = c.hkv * w.tiles, ww = wu * w.rounds, iu = lane_prefix(wu), iw = lane_prefix(ww);
        const uint64_t hit = __ballot((int)blockIdx.x < units + iu);
        if (b < 0 && hit) {
            const int i = __builtin_ctzll(hit);
            b = base + i;
            sq = grp.at(b);
            nth = (int)blockIdx.x - (units + lane_value(iu, i) - lane_value(wu, i));
            at = total + lane_value(iw, i) - lane_value(ww, i);
        }
        units += lane_value(iu, 63);
        total += lane_value(iw, 63);
    }
    if (b < 0) return;
    const Work w = work_of(sq, G, keys);
    if (w.rounds == 0) return;
    const uint32_t len_run = run_length(total, runs), x = at + nth * w.rounds;
    const int run0 = x / len_run, run1 = (x + w.rounds - 1) / len_run;
    if (run0 == run1) return;
    const int h = (uint32_t)nth / (uint32_t)w.tiles, tile = nth - h * w.tiles;
    join_run<QT, 0, NT>(a, sq, h, tile, run0, run1 - run0 + 1, room);
}

// Units that there can be, for tiles of `tile` rows.
static int64_t units_of(int64_t batch, int64_t rows, int G, int hkv, int tile) { return hkv * (cdiv(rows * G, tile) + batch); }
// Whether a packed call takes the prompt kernels, which read each K/V row an eighth as often as
// 16-row tiles, and need a second launch where their units are cut: with many 16-row tiles, or as
// many rounds of 128 positions in them as the table has room for.  us, 16-row tiles against these,
// f32 rows, 32 heads over 8 of 128, f16 caches: 8 x 128 rows over nothing (1088 tiles) 31 against
// 17; 256 rows (520) over nothing 12 against 20, over 2000 48 against 45, over 16000 372 against
// 146; 8 x 32 rows over 1000 (576) 31 against 35, 8 x 64 (1088) 62 against 43.  f32 caches, 32 over
// 4 of 64: 8 x 16 rows over 1000 (288) 24 against 22, 256 rows over nothing (516) 13 against 19.
static bool takes_prompt(int64_t batch, int64_t rows, int G, int hkv, int64_t capacity, bool kv16) {
    const int64_t tiles = units_of(batch, rows, G, hkv, 16);
    return tiles >= 1024 || tiles * cdiv(capacity, 128) >= (kv16 ? 8192 : 2048);
}
// Whether their units are few: where they alone, about half a tile per sequence short of the most
// there can be, would leave CUs idle.  Then workgroups are twice as wide (f16 caches, head sizes up
// to 128) and units are cut while there are CUs.  256 rows over 16000, 64 units: 447 us whole, 145
// cut into eight, 150 into four with twice the wavefronts, 256 over 2000 43.7 and 41.6; one prompt of
// 900 rows, 232 units: 38 cut in two, 23 with twice the wavefronts; 8 x 128 rows over nothing, 256
// units: 17 whole, 22 cut.
static bool cuts(int64_t batch, int64_t rows, int G, int hkv, int tile) { return hkv * (cdiv(rows * G, tile) + batch / 2) < 256; }

// The records of the runs, or of cut prompts where the packed rows may be such, whatever the table.
size_t paged_attention_workspace(int64_t batch, int64_t rows, int hq, int hkv, int D) {
    const int G = hq / hkv;
    // (where tiles of 64 rows are cut, those of 128 would be)
    const size_t most = rows > batch && cuts(batch, rows, G, hkv, 128) ? SLOTS * 128 : RUNS * 2 * 16;
    return most * (D + 4) * sizeof(float);
}

template <typename KVT, typename QT, int DP, int TK, int NW, bool FULL, bool PACKED>
static int launch_runs(const PagedAttn& a, int64_t units, hipStream_t s) {
    constexpr int KEYS = Tile<KVT, QT, DP, TK, NW>::KEYS;
    // as many runs as there can be rounds, up to eight wavefronts per CU
    const int64_t most = units * cdiv(a.c.capacity, KEYS), cap = RUNS * 4 / NW;
    if (most > INT32_MAX - RUNS) {
        set_error(TL_HIP_ERR_ARG, "ArgumentError: %lld rounds of %d positions are too many for one call", (long long)most, KEYS);
        return TL_HIP_ERR_ARG;
    }
    const int runs = (int)(most < cap ? most : cap);
    k_paged_tile<KVT, QT, DP, TK, NW, FULL, PACKED><<<dim3((unsigned)runs), 64 * NW, 0, s>>>(a, a.c.table, a.c.cu, a.c.lens, static_cast<const char*>(a.c.k), static_cast<const char*>(a.c.v));
    if (!a.fuse) k_paged_join<QT, PACKED, 64 * NW><<<dim3((unsigned)units), 64 * NW, 0, s>>>(a, a.c.cu, a.c.lens, KEYS, runs);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TL_HIP_OK : hip_fail(e, "paged attention launch");
}

template <typename KVT, typename QT, int DP, int TK, bool FULL>
static int launch_tile_of(const PagedAttn& a, hipStream_t s) {
    if (a.c.cu) {
        const int64_t units = units_of(a.c.batch, a.c.rows, a.G, a.c.hkv, 16);
        return launch_runs<KVT, QT, DP, TK, 4, FULL, true>(a, units, s);
    }
    const int64_t units = (int64_t)a.c.hkv * a.c.batch * cdiv(a.G, 16);
    // Few units over long tables: workgroups of eight wavefronts, so that half as many parts are
    // joined.  us, against four: 8 units of 128 over 8192 positions 13.0 against 14.8, f32 caches of
    // one unit 16.3 against 22.7; over 2048 12.2 against 9.4; 256 units up to 8192 95.6 against 92.2.
    if constexpr (DP <= 128)
        if (units < 128 && a.c.capacity >= 4096) return launch_runs<KVT, QT, DP, TK, 8, FULL, false>(a, units, s);
    return launch_runs<KVT, QT, DP, TK, 4, FULL, false>(a, units, s);
}

template <typename KVT, typename QT, int DP, int TK>
static int launch_tile(const PagedAttn& a, hipStream_t s) {
    return a.c.D == DP ? launch_tile_of<KVT, QT, DP, TK, true>(a, s) : launch_tile_of<KVT, QT, DP, TK, false>(a, s);
}

template <typename KVT, typename QT, int DP>
static int launch_prompt(const PagedAttn& a, hipStream_t s) {
    constexpr bool H16 = std::is_same_v<KVT, _Float16>;
    constexpr int ROWS = H16 ? 128 : 64, KEYS = H16 ? PromptTile<DP>::KT : 4096 / DP;
    // Few units: two groups of wavefronts to a workgroup, and parts for the CUs that are left.
    const int64_t units = units_of(a.c.batch, a.c.rows, a.G, a.c.hkv, ROWS);
    const bool cut = cuts(a.c.batch, a.c.rows, a.G, a.c.hkv, ROWS);
    const int64_t likely = a.c.hkv * (cdiv(a.c.rows * (int64_t)a.G, ROWS) + a.c.batch / 2);  // (at least half of units)
    const int most = !cut ? 1 : (int)std::max<int64_t>(H16 && DP <= 128 ? SLOTS / 2 / likely : SLOTS / units, 1);
    const dim3 grid((unsigned)(units * most));
    const char *kp = static_cast<const char*>(a.c.k), *vp = static_cast<const char*>(a.c.v);
    if constexpr (H16 && DP <= 128) {
        if (cut) k_paged_prompt<QT, DP, 2><<<grid, 512, 0, s>>>(a, a.c.table, a.c.cu, a.c.lens, kp, vp, most);
        else k_paged_prompt<QT, DP, 1><<<grid, 256, 0, s>>>(a, a.c.table, a.c.cu, a.c.lens, kp, vp, most);
    } else if constexpr (H16) {
        k_paged_prompt<QT, DP, 1><<<grid, 256, 0, s>>>(a, a.c.table, a.c.cu, a.c.lens, kp, vp, most);
    } else {
        k_paged_prompt_f32<DP><<<grid, 256, 0, s>>>(a, a.c.table, a.c.cu, a.c.lens, kp, vp, most);
    }
    if (most > 1) k_prompt_join<QT><<<dim3((unsigned)(units * (ROWS / 16))), 256, 0, s>>>(a, a.c.cu, a.c.lens, H16 ? 7 : 6, KEYS, most);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TL_HIP_OK : hip_fail(e, "paged attention launch");
}

template <typename KVT, typename QT>
static int launch_kind(const PagedAttn& a, hipStream_t s) {
    constexpr bool H16 = std::is_same_v<KVT, _Float16>;
    if (a.c.cu && a.c.rows > a.c.batch && takes_prompt(a.c.batch, a.c.rows, a.G, a.c.hkv, a.c.capacity, H16)) {
        if (a.c.D <= 64) return launch_prompt<KVT, QT, 64>(a, s);
        if (a.c.D <= 128) return launch_prompt<KVT, QT, 128>(a, s);
        return launch_prompt<KVT, QT, 256>(a, s);
    }
    if (a.c.D <= 64) return launch_tile<KVT, QT, 64, 2>(a, s);
    if (a.c.D == 128) return launch_tile_of<KVT, QT, 128, H16 ? 2 : 1, true>(a, s);
    if (a.c.D < 128) return launch_tile_of<KVT, QT, 128, 1, false>(a, s);  // (two at a time: registers spill)
    return launch_tile<KVT, QT, 256, 1>(a, s);
}

int launch_paged_attention(const PagedAttn& a, bool q16, bool kv16, hipStream_t s) {
    if (q16) return launch_kind<_Float16, _Float16>(a, s);
    if (kv16) return launch_kind<_Float16, float>(a, s);
    return launch_kind<float, float>(a, s);
}

}  // namespace tlhip
