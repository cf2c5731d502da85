// fa_paged_walk.hip — attention of single tokens (and a few at once) over pages of 8
// bits, and of any tokens over chosen blocks of pages of F16 or 8 bits, for gfx950.
//
// As fa_paged_rows.hip: the rows in parts, a workgroup for each part and head group, up to 16
// query rows (tokens x query heads of a kv head; one token's heads over chosen
// blocks, which each token has its own) share each K/V row; S^T = K Q^T and O^T
// += V^T P^T on MFMA, P passed from the one to the other in place. Bound by HBM.
// What differs:
//   Rows are not transposed in LDS: they go to the registers that feed the MFMA as they lie
//   in memory (K of 8 bits through a DMA slot, for whole lines). A wavefront walks steps of two
//   tiles of 16 rows (each of one page and one scale), the next steps' loads in flight. K: a
//   lane has 16 bytes of row lane % 16 (which dims a k step takes is free, if K and Q
//   agree). V: a lane reads, of rows 4 (lane / 16) .. + 3 of both tiles, the dims DPL (lane
//   % 16) .. + DPL - 1, DPL = D / 16: byte e of those eight rows is the operand of output
//   block e, whose row i stands for dim DPL i + e. So the transposition is the choice of
//   bytes that the conversion makes anyway (v_perm_b32).
//   8 bits: a whole number is exact in f16; K's scale multiplies the score, in F32. V's is
//   taken into the exponent: with x' = x + log2(s) the weights P' = 2^(x' - max x') are those that
//   multiply whole numbers, and f16 rounds them as it rounds P: by half a step, or, of rows whose P s
//   lies more than 2^14 below the largest, by 2^-25 of that; the sum of the softmax adds P' / s, in F32.
//   Chosen blocks: which tile is which row is read from the list, 32 steps at a time, a
//   lane each, with the page and the scales. A call's tokens are cut into equal parts of
//   their lists where they are few.
// Measured, 32/8 heads of 128, 8 bits: 32 uneven streams of up to 8192 rows 56-58 us (290-320
// MB: 5.3-5.5 TB/s; of F16 101) and 5 the join; 8192 rows of one stream 7.0 + 2.3 (a step a
// wavefront: three dependent loads, sizes, pages, rows). 32 lists of 2048 rows 25.3 (5.0
// TB/s); of F16 pages, 4 tokens each of 8 streams, 1024 rows, 20.2 (6.7 TB/s: tokens of a
// stream choose many of the same blocks, which the L2 has).
#include "fa_paged_join.h"
#include "fa_paged_q8.h"

namespace vxfa {

struct WalkArgs {
    RowsArgs r;               // (x, xrow, whole not used; cut: all rows only)
    PagedScales sc;
    const int32_t* list;      // chosen blocks: [token][hkv][top]
    int32_t top, lg;
    int32_t parts;            // of a token's list: the first `longer` of them one tile more than `tiles`
    int32_t tiles, longer;
};

template <int W>
struct Words {
    uint32_t w[W];
};
// NT: with a nontemporal hint. (All rows are read once: 32 streams of up to 8192 rows 77.5 -> 69.4 us for V's, 69.4 ->
// 67.2 for K's. Chosen ones may be read again: 32 lists of 2048 rows 28.7 -> 27.8 without V's, 26.2 without K's.)
template <int W, bool NT>
__device__ __forceinline__ Words<W> load_words(const char* p) {
    Words<W> r;
    if constexpr (W == 4) {
        const u32x4 x = NT ? __builtin_nontemporal_load((const u32x4*)p) : *(const u32x4*)p;
        r.w[0] = x[0]; r.w[1] = x[1]; r.w[2] = x[2]; r.w[3] = x[3];
    } else if constexpr (W == 2) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 x = NT ? __builtin_nontemporal_load((const u32x2*)p) : *(const u32x2*)p;
        r.w[0] = x[0]; r.w[1] = x[1];
    } else {
        r.w[0] = NT ? __builtin_nontemporal_load((const uint32_t*)p) : *(const uint32_t*)p;
    }
    return r;
}

// PLAIN: scores without cap and slopes.
template <int D, bool I8, bool LISTED, int NW, bool PLAIN, int HW>
static __global__ __launch_bounds__(64 * NW, I8 ? 4 : (NW == 8 ? 2 : 3)) void paged_walk_kernel(WalkArgs wa) {
    constexpr int KC = I8 ? D / 64 : D / 32;          // 16-byte chunks of a K row that a lane reads
    constexpr int KS = D / 32;                        // k steps of the first product
    constexpr int DPL = D / 16;                       // dims of V that a lane reads, blocks of O^T
    constexpr int VW = I8 ? DPL / 4 : DPL / 2;        // words of them
    constexpr int LA = I8 ? 2 : 1;                    // steps that K is requested ahead
    constexpr int CH = D / 16, RPI = 64 / CH, NI = 16 / RPI;   // 8 bits: chunks of a row, rows of a load of K, loads of a tile
    constexpr int KSTEP = 2 * 16 * D;                 // bytes of a step's K in LDS
    __shared__ __attribute__((aligned(16))) float xo[NW * 16 * D];
    static_assert(NW * LA * KSTEP <= NW * 16 * D * 4 || !I8, "K's slots lie where the wavefronts are joined");
    __shared__ float sm[NW][16], sl[NW][16];

    const RowsArgs& ra = wa.r;
    const PagedAttn& a = ra.a;
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    constexpr int NS = NW / HW;
    const int stripe = wave / HW;
    const int nhg = a.hkv * ra.groups, nhw = nhg / HW;
    const int hg0 = (int)blockIdx.x % nhw * HW, item = (int)blockIdx.x / nhw;
    const int hg = hg0 + wave % HW;
    const int hk = hg / ra.groups, sub = hg - hk * ra.groups;
    const int lg = a.b.ps_log2;

    // ---- the part: stream, first of its tokens, rows [first, p] seen by each ----------
    PagedStream st;
    int s, tok0 = 0, ntok, lo = 0, tb, te, np;
    if constexpr (LISTED) {
        const int t = item / wa.parts, piece = item - t * wa.parts;
        const PagedUnit u = paged_token(a.b, t);
        if (u.s < 0) return;
        s = u.s;
        st = u.st;
        tok0 = u.i;
        ntok = 1;
        np = wa.parts;
        tb = wa.tiles * piece + min(piece, wa.longer);
        te = tb + wa.tiles + (piece < wa.longer ? 1 : 0);
        if (a.b.n_pages == 0) te = tb;                // (no page that tiles which are not there could read)
    } else {
        const Part part = rows_locate(a.b, ra.p, a.window, item);
        if (part.s < 0) return;
        s = part.s;
        st = part.st;
        ntok = min(st.t, a.b.max_nq);
        lo = part.lo;
        np = part.n;
        if (part.piece == 0 && hg0 == 0 && threadIdx.x == 0) ra.cut[s] = int2{part.first, part.n};
        const int nall = st.t > 0 ? (st.n - lo + 15) / 16 : 0;                // of the stream (none: n <= lo)
        const int q = np == 1 ? nall : (int)((uint32_t)max(nall, 0) / (uint32_t)np), more = nall - q * np;
        tb = q * part.piece + min(part.piece, more);
        te = tb + q + (part.piece < more ? 1 : 0);
    }
    const int nk = max((te - tb - 2 * stripe + 2 * NS - 1) / (2 * NS), 0);      // steps: tiles tb + 2 (wave + NW k) and the next

    // ---- Q: B operand, column = query row lane % 16 -------------------------------
    const int row = lane & 15, quad = lane >> 4;
    const int tok = (int)ra.hpw.div((uint32_t)row), hr = row - tok * (int)ra.hpw.d;
    const int G = a.hq / a.hkv;
    const int h = hk * G + sub * (int)ra.hpw.d + hr;
    const bool valid = tok < ntok && sub * (int)ra.hpw.d + hr < G;
    half8 q[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        q[ks] = half8{};
        // (8 bits: the two halves of a lane's 16 dims; F16: its 8 dims)
        const int d = I8 ? 64 * (ks >> 1) + 16 * quad + 8 * (ks & 1) : 32 * ks + 8 * quad;
        if (valid)
            q[ks] = load_q8(a.q, (int64_t)(st.q0 + tok0 + tok) * a.q_nb1 + (int64_t)h * a.q_nb2 + d * (a.q_f16 ? 2 : 4), a.q_f16);
    }
    const float slope = !PLAIN && valid ? paged_slope(a, h) : 0.f;
    const int p = valid ? st.n - st.t + tok0 + tok : -1;                      // rows [first, p] are seen
    const int first = a.window > 0 ? max(p - a.window + 1, 0) : 0;
    // rows [sfirst, slast] are seen by all tokens, none past pend by any
    const int pend = st.n - st.t + tok0 + ntok - 1, slast = pend - ntok + 1;
    const int sfirst = a.window > 0 ? max(pend - a.window + 1, 0) : 0;

    // ---- tiles: lane l has tile 2 (wave + NW (ids_from + l / 2)) + l % 2 of the part -----
    // (and of the 32 steps before, which may not all be computed yet, first row and scales)
    int64_t offs = 0;
    int j0s = 0, j0s_before = 0;
    float sks = 1.f, svs = 1.f, sks_before = 1.f, svs_before = 1.f;
    uint64_t there = 0;
    int ids_from = 0;
    auto load_ids = [&](int k0) {
        j0s_before = j0s;
        sks_before = sks;
        svs_before = svs;
        const int t = tb + 2 * (stripe + NS * (k0 + (lane >> 1))) + (lane & 1);
        int j0 = -1;
        if (t < te) {
            if constexpr (LISTED) {
                const int per = wa.lg - 4;
                const int b = wa.list[((int64_t)(st.q0 + tok0) * a.hkv + hk) * wa.top + (t >> per)];
                // (a block past the token's row: none of its rows are seen)
                if (b >= 0 && b <= (max(pend, 0) >> wa.lg)) j0 = (b << wa.lg) + ((t & ((1 << per) - 1)) << 4);
                if (j0 > pend || j0 + 15 < sfirst) j0 = -1;
            } else {
                j0 = lo + 16 * t;
            }
        }
        const int page = j0 >= 0 ? paged_page(a.b, s, j0 >> lg) : -1;
        there = __ballot(page >= 0);
        j0s = max(j0, 0);
        const int r = j0s & ((1 << lg) - 1);
        offs = page >= 0 ? a.kv.at(page, hk, r) : a.kv.at(0, hk, 0);
        if constexpr (I8) {
            sks = svs = 1.f;
            if (page >= 0) {
                const int64_t at = wa.sc.at(page, hk, r);
                sks = scale_in_range(*(const float*)(wa.sc.k + at));
                svs = scale_in_range(*(const float*)(wa.sc.v + at));
            }
        }
        ids_from = k0;
    };

    // Loads. 8 bits: K of step k + 2 goes to LDS (whole rows with a nontemporal hint; a lane's own
    // 64 bytes of 16 rows apart would be half lines) when step k is done, V of step k + 1
    // to registers right after, so whoever has V has K of the step after; F16: K of step k + 1 to registers when S of
    // step k is done, its V after P V. One step's registers hold what is in flight, and four
    // (F16: three) wavefronts a SIMD hide the rest.
    u32x4 kr[2][KC];
    Words<VW> vr[2][4];
    uint32_t live = 0, live1 = 0, live2 = 0;          // of step k, of the next ones: bit i: tile i is there
    int64_t at[2] = {0, 0}, at1[2] = {0, 0};          // of the steps that V is requested of next, K was last: where the tiles lie
    char* const mine = (char*)xo + wave * LA * KSTEP;
    const uint32_t lds0 = lds_offset(mine);
    const uint32_t koff = I8 ? 0u : (uint32_t)row * (uint32_t)a.kv.nb1 + 16 * quad;
    const uint32_t voff = 4 * quad * (uint32_t)a.kv.nb1 + 4 * VW * row;
    // (chunk c of row r of a tile lies at c ^ swz(r): 16 rows of one chunk column in 16 bank groups)
    auto swz = [](int r) { return D == 128 ? r & 7 : (r >> 2) & 3; };
    auto issue_k = [&](int k) {
        if (k >= ids_from + 32) load_ids(k);
        const int l = 2 * ((k - ids_from) & 31);
        live1 = live2;
        live2 = (uint32_t)(there >> l) & 3u;
        at[0] = at1[0];
        at[1] = at1[1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // (a tile that is not there: the head's first rows of page 0, which are not used)
            const int alo = __builtin_amdgcn_readlane((int)(uint32_t)offs, l + i), ahi = __builtin_amdgcn_readlane((int)(offs >> 32), l + i);
            at1[i] = ((int64_t)ahi << 32) | (uint32_t)alo;
            const char* const kp = a.kv.k + at1[i];
            if constexpr (I8) {
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    const int r = RPI * n + lane / CH;
                    const uint32_t off = (uint32_t)r * (uint32_t)a.kv.nb1 + (((lane % CH) ^ swz(r)) * 16), to = lds0 + (k & 1) * KSTEP + i * 16 * D + 1024 * n;
                    if constexpr (LISTED) dma16(kp, off, to);
                    else dma16_nt(kp, off, to);
                }
            } else {
#pragma unroll
                for (int c = 0; c < KC; ++c) kr[i][c] = *(const u32x4*)(kp + (koff + 64 * c));
            }
        }
    };
    auto issue_v = [&](int k, const int64_t (&from)[2]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const char* const vp = a.kv.v + from[i];
            // (F16: rows past the stream's last may hold anything, and read that one)
            const int left = I8 ? 15 : max(min(st.n - 1 - __builtin_amdgcn_readlane(j0s, 2 * ((k - ids_from) & 31) + i), 15), 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t vo = voff + (uint32_t)r * (uint32_t)a.kv.nb1;
                if constexpr (!I8) vo = (uint32_t)min(4 * quad + r, left) * (uint32_t)a.kv.nb1 + 4 * VW * row;
                vr[i][r] = load_words<VW, !LISTED>(vp + vo);
            }
        }
    };

    floatx4 o[DPL];
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    // step k; more: of how many after it (up to LA) there are
    auto step = [&](int k, auto more) {
        constexpr int MORE = decltype(more)::value;
        const bool any = live != 0;
        floatx4 sc[2];
        const bool now = k >= ids_from;
        const int lt = 2 * ((k - ids_from) & 31);
        auto lane_of = [&](float x, int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lt + i)); };
        int j0[2];
        float sk[2], sv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            j0[i] = __builtin_amdgcn_readlane(now ? j0s : j0s_before, lt + i);
            sk[i] = I8 ? lane_of(now ? sks : sks_before, i) : 1.f;
            sv[i] = I8 ? lane_of(now ? svs : svs_before, i) : 1.f;
        }
        if constexpr (I8) {
            // K of this step is here; at most that of the next one and V of this one are not
            pr_wait_vm<8 + (MORE > 0 ? 2 * NI : 0)>();
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int c = 0; c < KC; ++c)
                    kr[i][c] = *(const u32x4*)(mine + (k & 1) * KSTEP + i * 16 * D + row * D + (((4 * c + quad) ^ swz(row)) * 16));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                half8 x;
                if constexpr (I8) x = half8_of_bytes(kr[i][ks >> 1][2 * (ks & 1)], kr[i][ks >> 1][2 * (ks & 1) + 1]);
                else x = __builtin_bit_cast(half8, kr[i][ks]);
                sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[ks], sc[i], 0, 0, 0);
            }
        }
        if constexpr (!I8 && MORE > 0) issue_k(k + 1);
        if (any) {
            float x[8], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float lsv = I8 ? __builtin_amdgcn_logf(sv[i]) : 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float z;
                    if constexpr (PLAIN) {
                        z = I8 ? fmaf(sc[i][r], a.c * sk[i], lsv) : a.c * sc[i][r];
                    } else {
                        const float y = I8 ? sc[i][r] * sk[i] : sc[i][r];
                        z = fmaf(slope, (float)(j0[i] + 4 * quad + r - p), a.capk != 0.f ? paged_wide_cap(a.c * y, a.cap, a.capk) : paged_score(a, y));
                        if constexpr (I8) z += lsv;
                    }
                    x[4 * i + r] = z;
                }
                // (a tile that all tokens see whole needs no masks)
                if (!((live >> i) & 1) || j0[i] < sfirst || j0[i] + 15 > slast) {
                    const bool on = (live >> i) & 1;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = j0[i] + 4 * quad + r;
                        x[4 * i + r] = (on & (j >= first) & (j <= p)) ? x[4 * i + r] : -INFINITY;
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[4 * i + r]);
            }
            mx = quad_max(mx);
            if (__any(mx > m)) {
                const float mn = fmaxf(m, mx), al = exp2_fast(m - (mn == -INFINITY ? 0.f : mn));
                m = mn;
                l *= al;
#pragma unroll
                for (int e = 0; e < DPL; ++e) o[e] *= al;
            }
            const float ms = m == -INFINITY ? 0.f : m;
            half8 pv;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = exp2_fast(x[4 * i + r] - ms);
                    sum += e;
                    pv[4 * i + r] = (_Float16)e;
                }
                l = I8 ? fmaf(sum, __builtin_amdgcn_rcpf(512.f * sv[i]), l) : l + sum;
            }
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int e = 0; e < DPL / VW; ++e) {
                    half8 vt;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 4; r += 2) {
                            const uint32_t w0 = vr[i][r].w[w], w1 = vr[i][r + 1].w[w];
                            half2 y;
                            if constexpr (I8) {
                                y = halves_over_512(__builtin_amdgcn_perm(w1 ^ 0x80808080u, w0 ^ 0x80808080u, 0x0C040C00u + 0x00010001u * e));
                            } else {
                                // (of a tile that is not there zeros)
                                const uint32_t z = __builtin_amdgcn_perm(w1, w0, 0x05040100u + 0x02020202u * e);
                                y = __builtin_bit_cast(half2, (live >> i) & 1 ? z : 0u);
                            }
                            vt[4 * i + r] = y[0];
                            vt[4 * i + r + 1] = y[1];
                        }
                    const int eb = w * (DPL / VW) + e;
                    o[eb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pv, o[eb], 0, 0, 0);
                }
        }
        if constexpr (I8) {
            pr_wait_lds();                            // (this step's slot has been read)
            if constexpr (MORE > 1) issue_k(k + 2);
            if constexpr (MORE == 1) { at[0] = at1[0]; at[1] = at1[1]; live1 = live2; }
            if constexpr (MORE > 0) issue_v(k + 1, at);
            live = live1;
        } else {
            if constexpr (MORE > 0) issue_v(k + 1, at1);
            live = live2;
        }
    };

    if (nk > 0) {
        load_ids(0);
        issue_k(0);
        issue_v(0, at1);
        live = live2;
        int k = 0;
        if constexpr (I8) {
            if (nk > 1) issue_k(1);
            for (; k < nk - 2; ++k) step(k, std::integral_constant<int, 2>{});
        }
        for (; k < nk - 1; ++k) step(k, std::integral_constant<int, 1>{});
        step(nk - 1, std::integral_constant<int, 0>{});
    }

    // ---- join the wavefronts -------------------------------------------------------
    l = quad_sum(l);
    if constexpr (I8) {
        pr_wait_lds();
        __syncthreads();                              // (K's slots have been read)
    }
    // (query row r at r D of the wavefront's part; chunks of 4 dims swizzled by row; element i
    // of block e is dim DPL (4 quad + i) + e)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DPL / 4; ++c) {
            const floatx4 y = {o[4 * c][i], o[4 * c + 1][i], o[4 * c + 2][i], o[4 * c + 3][i]};
            *(floatx4*)(xo + (wave * 16 + row) * D + 4 * ((DPL / 4 * (4 * quad + i) + c) ^ (row & 7))) = y;
        }
    if (quad == 0) { sm[wave][row] = m; sl[wave][row] = l; }
    __syncthreads();
    const int nrow = min(ntok * (int)ra.hpw.d, 16);
    for (int e0 = (int)threadIdx.x; e0 < HW * nrow * (D / 4); e0 += 64 * NW) {
        const int wh = HW == 1 ? 0 : e0 / (nrow * (D / 4)), e = e0 - wh * nrow * (D / 4);
        const int hk = (hg0 + wh) / ra.groups, sub = hg0 + wh - hk * ra.groups;
        float* const rec = ra.recs + ((int64_t)(hg0 + wh) * ra.items + item) * ra.rec;
        const int r = e / (D / 4), c = e % (D / 4);
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NS; ++w) M = fmaxf(M, sm[w * HW + wh][r]);
        const float Ms = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NS; ++w) {
            const float f = exp2_fast(sm[w * HW + wh][r] - Ms);
            L = fmaf(f, sl[w * HW + wh][r], L);
            const floatx4 y = *(const floatx4*)(xo + ((w * HW + wh) * 16 + r) * D + 4 * (c ^ (r & 7)));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf(f, y[i], x[i]);
        }
        if (np == 1) {
            const int tk = (int)ra.hpw.div((uint32_t)r), hh = r - tk * (int)ra.hpw.d;
            if (sub * (int)ra.hpw.d + hh < G) {
                const int64_t at = (int64_t)(st.q0 + tok0 + tk) * a.hq + hk * G + sub * (int)ra.hpw.d + hh;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                paged_store4(a, at * D + 4 * c, x * inv);
            }
        } else {
            *(floatx4*)(rec + r * D + 4 * c) = x;
            if (c == 0) {
                rec[ra.rows * D + r] = M;
                rec[ra.rows * (D + 1) + r] = L;
            }
        }
    }
}

static void heads_of(const PagedAttn& a, int tokens, int head_dim, RowsArgs& ra) {
    ra.a = a;
    const int G = a.hq / a.hkv, hpw = rows_heads(G);
    ra.hpw = DivMod::make((uint32_t)hpw);
    ra.groups = (G + hpw - 1) / hpw;
    ra.rows = hpw * tokens;
    ra.rec = (ra.rows * (head_dim + 2) + 3) & ~3;
    ra.x = nullptr;
    ra.xrow = 0;
    ra.whole = 0;
}

template <int D, bool I8, bool LISTED, int NW, int HW = 1>
static void launch_walk(const WalkArgs& wa, dim3 grid, hipStream_t st) {
    const PagedAttn& a = wa.r.a;
    if (a.cap == 0.f && a.n2 == 0) hipLaunchKernelGGL((paged_walk_kernel<D, I8, LISTED, NW, true, HW>), grid, dim3(64 * NW), 0, st, wa);
    else hipLaunchKernelGGL((paged_walk_kernel<D, I8, LISTED, NW, false, HW>), grid, dim3(64 * NW), 0, st, wa);
}

// Whether a workgroup's wavefronts take four neighbouring heads, each all rows of the part, or one
// head's rows in turn: neighbouring heads' rows are neighbouring lines, which memory gives
// faster at once, but a wavefront's walk is four times as long. By the bounds' rows x heads; one -> four heads,
// 8 kv heads of 128: 8 even streams of 8192 (half a million) 31.5 -> 33.0 us, 12 of them 43.8 -> 43.4, 16 58.6 -> 50.5,
// 4 of 32768 59.3 -> 49.9; 32 uneven ones of up to 2048 24.0 -> 24.4, of 8192 60.4 -> 56.3; 20 heads of 64: 8 uneven ones of
// 1500 21.6 -> 21.6, 32 of 2048 35.3 -> 28.7, of 8192 117 -> 84; one stream of 32768 31 -> 29, of 131072 109 -> 83.
// Rows far below their bounds, whose parts are short, lose by it: at hd 128 2 streams of 512 8.0 -> 9.8, 4 of 8192
// 19 -> 23, 16 of 2048 20.5 -> 23.7, 32 of 512 14.9 -> 16.6; at hd 64 2 to 32 of 512 10 % more to 10 % less. So one
// stream of 128 keeps one head a workgroup: it would gain at 131072 rows (56 -> 51), but lose below its
// bound: 8192 rows 9.8 -> 11.1, 300 7.6 -> 9.4 (hd 64: 13.2 -> 13.5, 7.4 -> 8.2).
static bool rows_wide(const PagedBatch& b, int nhg, int head_dim) {
    return nhg % 4 == 0 && (b.n_streams > 1 || head_dim == 64) && (double)b.n_streams * b.max_nkv * nhg >= 786432.0;
}

hipError_t launch_paged_rows_q8(const PagedBlocks& pb, int head_dim, hipStream_t st) {
    const PagedAttn& a = pb.a;
    if (!paged_rows_takes(a)) return hipErrorInvalidValue;
    WalkArgs wa;
    heads_of(a, a.b.max_nq > 0 ? a.b.max_nq : 1, head_dim, wa.r);
    wa.sc = pb.sc;
    wa.list = nullptr;
    wa.top = wa.lg = wa.tiles = wa.longer = 0;
    wa.parts = 1;
    RowsArgs& ra = wa.r;
    const int nhg = a.hkv * ra.groups;
    const size_t cut = ((size_t)a.b.n_streams * sizeof(int2) + 255) & ~(size_t)255;
    if (cut > a.ws_bytes) return hipErrorOutOfMemory;    // (65535 streams at most: half a MiB)
    ra.cut = reinterpret_cast<int2*>(a.ws);
    ra.recs = reinterpret_cast<float*>(a.ws + cut);
    const int64_t room = (int64_t)((a.ws_bytes - cut) / ((size_t)ra.rec * sizeof(float))) / nhg;
    ra.p = rows_plan(a.b, nhg, head_dim, room, ra.items, true);
    const bool wide = ra.p.cuts && rows_wide(a.b, nhg, head_dim) && 4096 / nhg + 1 + (int64_t)a.b.n_streams <= room;
    if (wide) {
        ra.p.small = 2048 / nhg > 0 ? 2048 / nhg : 1;
        ra.p.large = 4096 / nhg > 0 ? 4096 / nhg : 1;
        const int64_t most = (int64_t)ra.p.large + a.b.n_streams;
        ra.items = (int32_t)most;
    }
    const int64_t nwg = (int64_t)ra.items * nhg;
    if (nwg > kMaxGridX) return hipErrorNotSupported;
    const dim3 grid((unsigned)(wide ? nwg / 4 : nwg));
    if (head_dim == 128 && wide) launch_walk<128, true, false, 4, 4>(wa, grid, st);
    else if (head_dim == 128) launch_walk<128, true, false, 4>(wa, grid, st);
    else if (wide) launch_walk<64, true, false, 4, 4>(wa, grid, st);
    else launch_walk<64, true, false, 4>(wa, grid, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !ra.p.cuts) return e;
    const dim3 cg((unsigned)(a.hq * (head_dim / 32)), (unsigned)a.b.max_nq, (unsigned)a.b.n_streams);
    if (head_dim == 128) hipLaunchKernelGGL((paged_rows_combine<128, false>), cg, dim3(64), 0, st, ra, 0);
    else hipLaunchKernelGGL((paged_rows_combine<64, false>), cg, dim3(64), 0, st, ra, 0);
    return hipGetLastError();
}

template <int D, bool I8>
static void launch_listed(const WalkArgs& wa, int nw, dim3 grid, hipStream_t st) {
    if (nw == 4) launch_walk<D, I8, true, 4>(wa, grid, st);
    else launch_walk<D, I8, true, 8>(wa, grid, st);
}

hipError_t launch_paged_blocks(const PagedBlocks& pb, int head_dim, hipStream_t st) {
    const PagedAttn& a = pb.a;
    WalkArgs wa;
    heads_of(a, 1, head_dim, wa.r);
    wa.sc = pb.sc;
    wa.list = pb.list;
    wa.top = pb.top;
    wa.lg = pb.lg;
    RowsArgs& ra = wa.r;
    ra.cut = nullptr;
    ra.recs = reinterpret_cast<float*>(a.ws);
    const int nhg = a.hkv * ra.groups;
    // A list stays whole, 8 wavefronts a workgroup, where there are workgroups for the CUs or it is
    // short: a cut's join is a launch of its own. Else 4, and parts for two workgroups a CU, of a
    // step for each wavefront at least. Cut -> whole, 32/8 heads of 128, 8 (16) bits, us: 32 tokens of 2048 rows
    // 32.2 -> 27.8 (47.9 -> 43.1), of 256 11.1 -> 7.1; 16 of 2048 20.4 -> 23.7 (27.5 -> 26.2), of 512 10.1 -> 8.6
    // (11.4 -> 10.1); 1 of 2048 7.8 -> 16.9, of 1024 7.7 -> 10.6, of 512 7.8 -> 7.6 (7.7 -> 8.5).
    // (512 and more workgroups: 4 wavefronts 46.8, 8 49.4; 16 wavefronts were slower everywhere.)
    const int64_t wgs = (int64_t)a.b.tokens * nhg, tiles = (int64_t)pb.top << (pb.lg - 4);
    const bool one = wgs >= 256 || tiles <= 32;
    const int nw = one && wgs < 512 ? 8 : 4;
    int64_t parts = one ? 1 : (512 + wgs - 1) / wgs;
    if (parts > (tiles + 7) / 8) parts = (tiles + 7) / 8;
    const int64_t room = (int64_t)(a.ws_bytes / ((size_t)ra.rec * sizeof(float))) / wgs;
    if (parts > room) parts = room;
    if (parts < 1) parts = 1;
    wa.parts = (int32_t)parts;
    wa.tiles = (int32_t)(tiles / parts);
    wa.longer = (int32_t)(tiles % parts);
    ra.items = (int32_t)(a.b.tokens * parts);
    const int64_t nwg = wgs * parts;
    if (nwg > kMaxGridX || (parts > 1 && a.b.tokens > 65535)) return hipErrorNotSupported;
    const dim3 grid((unsigned)nwg);
    if (head_dim == 128 && pb.sc.k) launch_listed<128, true>(wa, nw, grid, st);
    else if (head_dim == 128) launch_listed<128, false>(wa, nw, grid, st);
    else if (pb.sc.k) launch_listed<64, true>(wa, nw, grid, st);
    else launch_listed<64, false>(wa, nw, grid, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || parts == 1) return e;
    const dim3 cg((unsigned)(a.hq * (head_dim / 32)), (unsigned)a.b.tokens);
    if (head_dim == 128) hipLaunchKernelGGL((paged_rows_combine<128, true>), cg, dim3(64), 0, st, ra, wa.parts);
    else hipLaunchKernelGGL((paged_rows_combine<64, true>), cg, dim3(64), 0, st, ra, wa.parts);
    return hipGetLastError();
}

}  // namespace vxfa
