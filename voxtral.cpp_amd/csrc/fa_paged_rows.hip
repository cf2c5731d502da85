// fa_paged_rows.hip — attention of single tokens (and a few at once) over a
// paged cache, split over the rows of every stream, for gfx950.
//
// The paged form of fa_decode.hip's decode step (src/voxtral.cpp:1802 with
// n_tokens = 1), for a ragged batch: up to 16 query rows (tokens x query heads
// of a kv head) share each K/V row that is read. Bound by HBM. Measured, 32/8
// heads of 128: 32 streams of up to 8192 rows 105 us (5.6 TB/s of K and V, 0.89 of a
// large read's rate; without the nontemporal hint at the tiles, which are read once,
// 117), one full stream 10.1 us in a graph (6.5 of them this kernel, 3 the join), the
// first token of a prompt 4.1 (launch cadence).
//
// Work: the rows of all streams together are cut into parts of `chunk` rows,
// a workgroup of four wavefronts for each part and head group; every
// workgroup works the cut out for itself from the sizes on the device (all
// lanes take a stream each), so a captured call follows them. Parts of one
// stream are of one length. The head group is the fastest index: with 8 kv
// heads each XCD reads the rows of one head.
// A wavefront walks tiles of 16 rows (a page holds whole tiles), K and V
// brought to its own LDS slots by global_load_lds, the next tile in flight
// while one is computed, with no barrier on the way:
//   S^T = K Q^T  v_mfma_f32_16x16x32_f16, K rows x query rows: a lane has the
//         scores of 4 rows for one query row,
//   O^T += V^T P^T  v_mfma_f32_16x16x16_f16, whose B operand has just those 4
//         rows of one query row: P goes from the one to the other in place.
// Scores, running maxima and sums in F32; P is rounded to f16 for the second
// product, its sum taken before that rounding.
// The four wavefronts join through LDS; a stream of one part is finished
// there, else each part leaves (O, m, l) and paged_rows_combine joins them
// in order. Short streams are left whole (rows_whole in fa_paged_plan.h).
// Accumulated weights: the kernel leaves its scores (4 bytes a row and query row,
// against 512 of K and V), paged_rows_weights sums 2^(x - lse) when the row sums
// are known, or the workgroup itself where streams are whole: 32 streams of up to
// 8192 rows 105 -> 133 us, of up to 512 11.4 -> 13.8; forming the scores again from
// K (where they do not fit the scratch) took 240. Of the 28 us 16 are the stores,
// 12 the sums (which read the scores with the same hint: 134.7 -> 132.7). Kept in LDS
// and stored 8 tiles at a time they gained 3 %, nontemporal stores lost 2.
#include "fa_paged.h"
#include "fa_paged_plan.h"

namespace vxfa {

constexpr int PR_WAVES = 4;
constexpr int PR_TILE = 16;

struct RowsArgs {
    PagedAttn a;
    RowsPlan p;
    DivMod hpw;               // heads per group
    int32_t groups;           // head groups of a kv head
    int32_t rec;              // floats of a part's record: O [rows][D], m [rows], l [rows]
    int32_t rows;             // query rows of a record
    int32_t items;            // parts in the grid per head group
    int2* cut;                // [n_streams] first part, parts of a stream
    float* recs;              // [head group][part][rec]
    // the scores, for the weights that the rows gather: null, or
    // [head group][stream][query row][xrow], -inf where a row is not seen
    float* x;
    int64_t xrow;
    int32_t whole;            // no stream is cut and no group shared: the weights need no launch of their own
};

// dma16 with a nontemporal hint: rows are read once
__device__ __forceinline__ void dma16_nt(const char* base, uint32_t off, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
}

template <int N>
__device__ __forceinline__ void pr_wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// LDS reads done: their slot may be written again
__device__ __forceinline__ void pr_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ float quad_max(float x) {   // over lanes l ^ 16, l ^ 32
    const int xi = __builtin_bit_cast(int, x);
    const auto r = __builtin_amdgcn_permlane16_swap(xi, xi, false, false);
    return pair32_max(fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1])));
}
__device__ __forceinline__ float quad_sum(float x) {
    const int xi = __builtin_bit_cast(int, x);
    const auto r = __builtin_amdgcn_permlane16_swap(xi, xi, false, false);
    return pair32_sum(__builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]));
}

template <int D>
__global__ __launch_bounds__(64 * PR_WAVES, 2) void paged_rows_kernel(RowsArgs ra) {
    constexpr int KS = D / 32;                 // k steps of the first product
    constexpr int DB = D / 16;                 // 16-dim blocks of O^T
    constexpr int CH = D / 8;                  // 16-byte chunks of a row
    constexpr int RPI = 64 / CH;               // rows of one load instruction
    constexpr int NI = PR_TILE / RPI;          // load instructions per matrix and tile
    constexpr int ROW = 2 * D, MAT = PR_TILE * ROW, TILE = 2 * MAT;
    constexpr int NS = D == 128 ? 2 : 4;       // slots (64 KiB a workgroup: two of them on a CU)
    static_assert(PR_WAVES * 16 * D * 4 <= PR_WAVES * NS * TILE, "the join uses the slots");
    __shared__ __attribute__((aligned(16))) char smem[PR_WAVES * NS * TILE];
    __shared__ float sm[PR_WAVES][16], sl[PR_WAVES][16], slse[16];

    const PagedAttn& a = ra.a;
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int nhg = a.hkv * ra.groups;
    const int hg = (int)blockIdx.x % nhg, item = (int)blockIdx.x / nhg;
    const int hk = hg / ra.groups, sub = hg - hk * ra.groups;
    const Part part = rows_locate(a.b, ra.p, a.window, item);
    if (part.s < 0) return;
    const PagedStream st = part.st;
    if (part.piece == 0 && hg == 0 && threadIdx.x == 0) ra.cut[part.s] = int2{part.first, part.n};

    // ---- this part's tiles, their pages -------------------------------------------
    const int nall = st.t > 0 ? (st.n - part.lo + PR_TILE - 1) / PR_TILE : 0;   // of the stream (none: n <= lo)
    const int tb = (int)((int64_t)nall * part.piece / part.n), te = (int)((int64_t)nall * (part.piece + 1) / part.n);
    const int nk = max((te - tb - wave + PR_WAVES - 1) / PR_WAVES, 0);   // the wavefront's: tb + wave + 4 k
    const int lg = a.b.ps_log2;
    // lane l: the page of tile (k & ~63) + l; bit l: whether it is there (of the 64
    // tiles before, too, which may not all be computed yet)
    int ids = 0;
    uint64_t there = 0, there_before = 0;
    int ids_from = 0;
    auto load_ids = [&](int k0) {
        const int t = min(tb + wave + PR_WAVES * (k0 + lane), te - 1);
        ids = paged_page(a.b, part.s, (part.lo + PR_TILE * t) >> lg);
        there_before = there;
        there = __ballot(ids >= 0);
        ids_from = k0;
    };

    // ---- Q: B operand, column = query row lane % 16, dims 32 ks + 8 (lane / 16) ..
    const int row = lane & 15, quad = lane >> 4;
    const int tok = (int)ra.hpw.div((uint32_t)row), hr = row - tok * (int)ra.hpw.d;
    const int G = a.hq / a.hkv;
    const int h = hk * G + sub * (int)ra.hpw.d + hr;
    const bool valid = tok < min(st.t, a.b.max_nq) && sub * (int)ra.hpw.d + hr < G;
    half8 q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        q[ks] = half8{};
        if (valid)
            q[ks] = load_q8(a.q, (int64_t)(st.q0 + tok) * a.q_nb1 + (int64_t)h * a.q_nb2 + (32 * ks + 8 * quad) * (a.q_f16 ? 2 : 4),
                            a.q_f16);
    }
    if (nk > 0) load_ids(0);
    // (the queries have to be here before the first loads below: a wait for them
    // in the loop would wait for those too)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(q[ks]));
    const float slope = valid ? paged_slope(a, h) : 0.f;
    const int p = valid ? st.n - st.t + tok : -1;                       // rows [first, p] are seen
    const int first = a.window > 0 ? max(p - a.window + 1, 0) : 0;

    // ---- loads: row r of a tile, LDS chunk c holds chunk c ^ swizzle(r) -----------
    // K: the 16 rows that an operand read takes of one chunk column fall on 16
    // bank groups; V: the transposing reads take 32 bytes of 16 rows.
    const uint32_t lds0 = lds_offset(smem) + wave * NS * TILE;
    char* const mine = smem + wave * NS * TILE;
    auto swk = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    auto swv = [](int r) { return D == 128 ? (r & 7) << 1 : ((r >> 1) & 3) << 1; };
    auto issue = [&](int k) {
        if ((k & 63) == 0 && k > 0) load_ids(k);
        const int page = max(__builtin_amdgcn_readlane(ids, k & 63), 0);   // (absent: page 0, not used)
        const int j0 = part.lo + PR_TILE * (tb + wave + PR_WAVES * k);
        const int last = min(st.n - 1 - j0, PR_TILE - 1);                  // rows past the stream read its last one
        const int64_t at = a.kv.at(page, hk, j0 & ((1 << lg) - 1));
        const char *kp = a.kv.k + at, *vp = a.kv.v + at;
        const uint32_t slot = lds0 + (k & (NS - 1)) * TILE;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = RPI * i + lane / CH, c = lane % CH;
            dma16_nt(kp, (uint32_t)min(r, last) * (uint32_t)a.kv.nb1 + ((c ^ swk(r)) * 16), slot + RPI * i * ROW);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = RPI * i + lane / CH, c = lane % CH;
            dma16_nt(vp, (uint32_t)min(r, last) * (uint32_t)a.kv.nb1 + ((c ^ swv(r)) * 16), slot + MAT + RPI * i * ROW);
        }
    };
    for (int k = 0; k < min(nk, NS - 1); ++k) issue(k);

    floatx4 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int kaddr = row * ROW, ksw = swk(row);
    const int vr = 4 * quad + (row >> 2);      // the row this lane addresses, 8 bytes 16 db + 4 (row % 4) of it
    const int vaddr = MAT + vr * ROW + (row & 1) * 8, vsw = swv(vr);

    float* const xs = ra.x && valid ? ra.x + (((int64_t)hg * a.b.n_streams + part.s) * ra.rows + row) * ra.xrow : nullptr;
    for (int k = 0; k < nk; ++k) {
        pr_wait_lds();
        if (k + NS - 1 < nk) {
            issue(k + NS - 1);
            pr_wait_vm<2 * NI * (NS - 1)>();
        } else {
            pr_wait_vm<0>();
        }
        if (!(((k >= ids_from ? there : there_before) >> (k & 63)) & 1)) continue;   // an absent page
        const char* slot = mine + (k & (NS - 1)) * TILE;
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const half8 kr = *(const half8*)(slot + kaddr + (((4 * ks + quad) ^ ksw) * 16));
            s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr, q[ks], s, 0, 0, 0);
        }
        const int j0 = part.lo + PR_TILE * (tb + wave + PR_WAVES * k) + 4 * quad;
        float x[4], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + i;
            x[i] = fmaf(slope, (float)(j - p), a.capk != 0.f ? paged_wide_cap(a.c * s[i], a.cap, a.capk) : paged_score(a, s[i]));
            x[i] = j >= first && j <= p ? x[i] : -INFINITY;
            mx = fmaxf(mx, x[i]);
        }
        if (xs) *(floatx4*)(xs + j0) = floatx4{x[0], x[1], x[2], x[3]};
        mx = quad_max(mx);
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx), al = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] *= al;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        half4 pv;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e = exp2_fast(x[i] - ms);
            l += e;
            pv[i] = (_Float16)e;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const half4 vt = lds_read_tr16(slot + vaddr + (((2 * db + ((row >> 1) & 1)) ^ vsw) * 16));
            o[db] = __builtin_amdgcn_mfma_f32_16x16x16f16(vt, pv, o[db], 0, 0, 0);
        }
    }

    // ---- join the wavefronts -------------------------------------------------------
    l = quad_sum(l);
    pr_wait_lds();
    __syncthreads();
    // (query row r at r D of the wavefront's part; chunks of 4 dims swizzled by row)
    float* const xo = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int db = 0; db < DB; ++db)
        *(floatx4*)(xo + (wave * 16 + row) * D + 4 * ((4 * db + quad) ^ (row & 7))) = o[db];
    if (quad == 0) { sm[wave][row] = m; sl[wave][row] = l; }
    __syncthreads();
    const int nrow = min(min(st.t, a.b.max_nq) * (int)ra.hpw.d, 16);
    float* const rec = ra.recs + ((int64_t)hg * ra.items + item) * ra.rec;
    for (int e = (int)threadIdx.x; e < nrow * (D / 4); e += 64 * PR_WAVES) {
        const int r = e / (D / 4), c = e % (D / 4);
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < PR_WAVES; ++w) M = fmaxf(M, sm[w][r]);
        const float Ms = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < PR_WAVES; ++w) {
            const float f = exp2_fast(sm[w][r] - Ms);
            L = fmaf(f, sl[w][r], L);
            const floatx4 y = *(const floatx4*)(xo + (w * 16 + r) * D + 4 * (c ^ (r & 7)));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(f, y[i], x[i]);
        }
        if (part.n == 1) {
            const int tk = (int)ra.hpw.div((uint32_t)r), hh = r - tk * (int)ra.hpw.d;
            if (sub * (int)ra.hpw.d + hh < G) {
                const int64_t at = (int64_t)(st.q0 + tk) * a.hq + hk * G + sub * (int)ra.hpw.d + hh;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                paged_store4(a, at * D + 4 * c, x * inv);
                if (a.lse && c == 0) {
                    const float lse = L == 0.f ? INFINITY : M + log2f(L);
                    a.lse[at] = lse;
                    slse[r] = lse;
                }
            }
        } else {
            *(floatx4*)(rec + r * D + 4 * c) = x;
            if (c == 0) {
                rec[ra.rows * D + r] = M;
                rec[ra.rows * (D + 1) + r] = L;
            }
        }
    }
    // a whole stream's rows have their weights at once (as paged_rows_weights does)
    if (ra.whole) {
        __syncthreads();
        const float* x = ra.x + ((int64_t)hg * a.b.n_streams + part.s) * ra.rows * ra.xrow;
        for (int j = (int)threadIdx.x; j < st.n; j += 64 * PR_WAVES) {
            const int page = paged_page(a.b, part.s, j >> lg);
            if (page < 0) continue;
            float sum = 0.f;
            if (j >= part.lo)
                for (int r = 0; r < nrow; ++r) sum += exp2_fast(x[r * ra.xrow + j] - slse[r]);
            const int64_t at = 4 * (int64_t)(j & ((1 << lg) - 1));
            const float old = a.w_in ? *(const float*)((const char*)a.w_in + page * a.wi_nb3 + hk * a.wi_nb2 + at) : 0.f;
            *(float*)((char*)a.w_out + page * a.wo_nb3 + hk * a.wo_nb2 + at) = old + sum;
        }
    }
}

// Joins the parts of a stream: a wavefront per (token, query head, 32 dims), 8
// lanes of 4 dims for every eighth part, all loads of 8 parts a lane at once.
template <int D>
__global__ __launch_bounds__(64) void paged_rows_combine(RowsArgs ra) {
    const PagedAttn& a = ra.a;
    const int lane = (int)threadIdx.x, f = lane & 7, grp = lane >> 3;
    // kv head fastest, as in the kernel that wrote the records
    const int hk = (int)blockIdx.x % a.hkv, rest = (int)blockIdx.x / a.hkv;
    const int g = rest / (D / 32), sl = rest % (D / 32);
    const int i = (int)blockIdx.y, s = (int)blockIdx.z;
    const PagedStream st = paged_stream(a.b, s);
    // (one stream's parts begin at 0: its records are on their way before their number
    // is known)
    const bool one = a.b.n_streams == 1;
    const int2 cut = ra.cut[s];
    if (!one && (i >= min(st.t, a.b.max_nq) || cut.y <= 1)) return;
    const int first = one ? 0 : cut.x, nload = one ? ra.items : cut.y;
    const int sub = (int)ra.hpw.div((uint32_t)g), r = i * (int)ra.hpw.d + g - sub * (int)ra.hpw.d;
    const float* rec = ra.recs + ((int64_t)(hk * ra.groups + sub) * ra.items + first) * ra.rec;
    float M = -INFINITY, L = 0.f;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = grp; p0 < nload; p0 += 64) {
        float m[8], l[8];
        floatx4 o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float* q = rec + (int64_t)min(p0 + 8 * u, nload - 1) * ra.rec;
            o[u] = *(const floatx4*)(q + r * D + 32 * sl + 4 * f);
            m[u] = q[ra.rows * D + r];
            l[u] = q[ra.rows * (D + 1) + r];
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (p0 + 8 * u >= cut.y) {   // (what is loaded there may be anything)
                m[u] = -INFINITY;
                l[u] = 0.f;
                o[u] = floatx4{0.f, 0.f, 0.f, 0.f};
            }
            mn = fmaxf(mn, m[u]);
        }
        const float ms = mn == -INFINITY ? 0.f : mn, al = exp2_fast(M - ms);
        L *= al;
        x *= al;
        M = mn;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float w = exp2_fast(m[u] - ms);
            L = fmaf(w, l[u], L);
#pragma unroll
            for (int c = 0; c < 4; ++c) x[c] = fmaf(w, o[u][c], x[c]);
        }
    }
    if (one && (i >= min(st.t, a.b.max_nq) || cut.y <= 1)) return;
    const float mm = quad_max(fmaxf(M, row_ror<8>(M))), ms = mm == -INFINITY ? 0.f : mm;
    const float w = exp2_fast(M - ms);
    auto all = [](float y) { return quad_sum(y + row_ror<8>(y)); };
    L = all(L * w);
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = all(x[c] * w);
    if (grp == 0) {
        const int64_t at = (int64_t)(st.q0 + i) * a.hq + hk * (a.hq / a.hkv) + g;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        paged_store4(a, at * D + 32 * sl + 4 * f, x * inv);
        if (a.lse && sl == 0 && f == 0) a.lse[at] = L == 0.f ? INFINITY : mm + log2f(L);
    }
}

// The weights that the rows gather from scores that paged_rows_kernel left: a
// thread per 4 rows (of one page) and kv head sums 2^(x - lse) over the query
// rows.
__global__ __launch_bounds__(256) void paged_rows_weights(RowsArgs ra) {
    const PagedAttn& a = ra.a;
    const int s = (int)blockIdx.y, hk = (int)blockIdx.x % a.hkv, j = ((int)blockIdx.x / a.hkv * 256 + (int)threadIdx.x) * 4;
    const PagedStream st = paged_stream(a.b, s);
    if (j >= st.n) return;
    const int page = paged_page(a.b, s, j >> a.b.ps_log2);
    if (page < 0) return;
    const int left = min(st.n - j, 4), r = j & ((1 << a.b.ps_log2) - 1);
    const int G = a.hq / a.hkv, hpw = (int)ra.hpw.d;
    const float* wi = a.w_in ? (const float*)((const char*)a.w_in + page * a.wi_nb3 + hk * a.wi_nb2) + r : nullptr;
    float* wo = (float*)((char*)a.w_out + page * a.wo_nb3 + hk * a.wo_nb2) + r;
    float old[4] = {0.f, 0.f, 0.f, 0.f};
    if (wi) {
#pragma unroll
        for (int c = 0; c < 4; ++c) old[c] = c < left ? wi[c] : 0.f;
    }
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    if (j + 3 >= rows_first(st, a.window)) {       // (a multiple of 16, as the tiles are)
        for (int sub = 0; sub < ra.groups; ++sub) {
            const float* x = ra.x + ((int64_t)(hk * ra.groups + sub) * a.b.n_streams + s) * ra.rows * ra.xrow + j;
            const int heads = min(hpw, G - sub * hpw), nrow = min(st.t, a.b.max_nq) * hpw;
            // (four query rows' loads at once)
            for (int r0 = 0; r0 < nrow; r0 += 4) {
                floatx4 y[4];
                float lse[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int i = (int)ra.hpw.div((uint32_t)(r0 + u)), h = r0 + u - i * hpw;
                    const bool in = r0 + u < nrow && h < heads;
                    y[u] = __builtin_nontemporal_load((const floatx4*)(x + (int64_t)(in ? r0 + u : 0) * ra.xrow));
                    lse[u] = a.lse[(int64_t)(st.q0 + (in ? i : 0)) * a.hq + hk * G + sub * hpw + (in ? h : 0)];
                    if (!in) lse[u] = INFINITY;    // (weight 0)
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int c = 0; c < 4; ++c) sum[c] += exp2_fast(y[u][c] - lse[u]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (c < left) wo[c] = old[c] + sum[c];
}

bool paged_rows_takes(const PagedAttn& a) {
    return (int64_t)a.b.max_nq * rows_heads(a.hq / a.hkv) <= 16;
}

hipError_t launch_paged_rows(const PagedAttn& a, int head_dim, hipStream_t st, bool& weighed) {
    weighed = false;
    if (!paged_rows_takes(a)) return hipErrorInvalidValue;
    RowsArgs ra;
    ra.a = a;
    const int G = a.hq / a.hkv, hpw = rows_heads(G);
    ra.hpw = DivMod::make((uint32_t)hpw);
    ra.groups = (G + hpw - 1) / hpw;
    ra.rows = hpw * (a.b.max_nq > 0 ? a.b.max_nq : 1);
    ra.rec = (ra.rows * (head_dim + 2) + 3) & ~3;
    const int nhg = a.hkv * ra.groups;
    const size_t cut = ((size_t)a.b.n_streams * sizeof(int2) + 255) & ~(size_t)255;
    if (cut > a.ws_bytes) return hipErrorOutOfMemory;    // (65535 streams at most: half a MiB)
    ra.cut = reinterpret_cast<int2*>(a.ws);
    size_t used = cut;
    // scores, if they leave the records' usual room; else the weights form them again
    ra.x = nullptr;
    ra.xrow = ((int64_t)a.b.max_nkv + 15) & ~(int64_t)15;
    const double xb = (double)nhg * a.b.n_streams * ra.rows * (double)ra.xrow * sizeof(float);
    const size_t usual = (size_t)(512 + (size_t)a.b.n_streams * nhg) * ra.rec * sizeof(float);
    if (a.w_out && a.b.max_nkv > 0 && xb + (double)used + (double)usual <= (double)a.ws_bytes) {
        ra.x = reinterpret_cast<float*>(a.ws + used);
        used += ((size_t)xb + 255) & ~(size_t)255;
        weighed = true;
    }
    ra.recs = reinterpret_cast<float*>(a.ws + used);
    const int64_t room = used < a.ws_bytes ? (int64_t)((a.ws_bytes - used) / ((size_t)ra.rec * sizeof(float))) / nhg : 0;
    ra.p = rows_plan(a.b, nhg, head_dim, room, ra.items);
    // (streams without tokens have a part then, too: their rows' weights are taken over)
    ra.whole = ra.x && !ra.p.cuts && ra.groups == 1;
    ra.p.empty = ra.whole;
    const int64_t nwg = (int64_t)ra.items * nhg;
    if (nwg > 0x7fffffff / 256) return hipErrorNotSupported;
    const dim3 grid((unsigned)nwg), block(64 * PR_WAVES);
    if (head_dim == 128) hipLaunchKernelGGL((paged_rows_kernel<128>), grid, block, 0, st, ra);
    else hipLaunchKernelGGL((paged_rows_kernel<64>), grid, block, 0, st, ra);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (ra.p.cuts) {
        const dim3 cg((unsigned)(a.hq * (head_dim / 32)), (unsigned)a.b.max_nq, (unsigned)a.b.n_streams);
        if (head_dim == 128) hipLaunchKernelGGL((paged_rows_combine<128>), cg, dim3(64), 0, st, ra);
        else hipLaunchKernelGGL((paged_rows_combine<64>), cg, dim3(64), 0, st, ra);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (!ra.x || ra.whole) return e;
    const int64_t gx = ((int64_t)a.b.max_nkv + 1023) / 1024 * a.hkv;   // (paged_weights_fit's are more)
    hipLaunchKernelGGL(paged_rows_weights, dim3((unsigned)gx, (unsigned)a.b.n_streams), dim3(256), 0, st, ra);
    return hipGetLastError();
}

}  // namespace vxfa
