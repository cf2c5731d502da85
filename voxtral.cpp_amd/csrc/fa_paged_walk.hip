// fa_paged_walk.hip — attention of single tokens (and a few at once) over pages of 8
// bits, and of any tokens over chosen blocks of pages of F16 or 8 bits, for gfx950.
//
// As fa_paged_rows.hip: the rows in parts, a workgroup for each part and head group, up to 16
// query rows (tokens x query heads of a kv head; one token's heads over chosen
// blocks, which each token has its own) share each K/V row; S^T = K Q^T and O^T
// += V^T P^T on MFMA, P passed from the one to the other in place. Bound by HBM.
// What differs:
//   Rows go from memory to the registers that feed the MFMA, without LDS. A wavefront
//   walks steps of two tiles of 16 rows (each of one page and one scale), the next
//   steps' loads in flight. K: a lane reads 16 bytes of row lane % 16 (which dims a k step
//   takes is free, if K and Q agree). V: a lane reads, of rows 4 (lane / 16) .. + 3 of
//   both tiles, the dims DPL (lane % 16) .. + DPL - 1, DPL = D / 16: byte e of those eight rows is
//   the operand of output block e, whose row i stands for dim DPL i + e. So the
//   transposition is the choice of bytes that the conversion makes anyway (v_perm_b32).
//   8 bits: a whole number is exact in f16; K's scale multiplies the score, in F32. V's is
//   taken into the exponent: with x' = x + log2(s) the weights P' = 2^(x' - max x') are those that
//   multiply whole numbers, so f16 rounds them as it rounds P, however the scales of
//   blocks differ; the sum of the softmax adds P' / s, in F32.
//   Chosen blocks: which tile is which row is read from the list, 32 steps at a time, a
//   lane each, with the page and the scales. A call's tokens are cut into equal parts of
//   their lists where they are few.
#include "fa_paged_join.h"
#include "fa_paged_q8.h"

namespace vxfa {

struct WalkArgs {
    RowsArgs r;               // (x, xrow, whole not used; cut: all rows only)
    PagedScales sc;
    const int32_t* list;      // chosen blocks: [token][hkv][top]
    int32_t top, lg;
    int32_t parts;            // of a token's list
};

template <int W>
struct Words {
    uint32_t w[W];
};
template <int W>
__device__ __forceinline__ Words<W> load_words(const char* p) {
    Words<W> r;
    if constexpr (W == 4) {
        const u32x4 x = __builtin_nontemporal_load((const u32x4*)p);
        r.w[0] = x[0]; r.w[1] = x[1]; r.w[2] = x[2]; r.w[3] = x[3];
    } else if constexpr (W == 2) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 x = __builtin_nontemporal_load((const u32x2*)p);
        r.w[0] = x[0]; r.w[1] = x[1];
    } else {
        r.w[0] = __builtin_nontemporal_load((const uint32_t*)p);
    }
    return r;
}

template <int D, bool I8, bool LISTED, int NW>
static __global__ __launch_bounds__(64 * NW, 2) void paged_walk_kernel(WalkArgs wa) {
    constexpr int KC = I8 ? D / 64 : D / 32;          // 16-byte chunks of a K row that a lane reads
    constexpr int KS = D / 32;                        // k steps of the first product
    constexpr int DPL = D / 16;                       // dims of V that a lane reads, blocks of O^T
    constexpr int VW = I8 ? DPL / 4 : DPL / 2;        // words of them
    constexpr int PF = I8 ? 3 : 2;                    // steps in registers
    __shared__ __attribute__((aligned(16))) float xo[NW * 16 * D];
    __shared__ float sm[NW][16], sl[NW][16];

    const RowsArgs& ra = wa.r;
    const PagedAttn& a = ra.a;
    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int nhg = a.hkv * ra.groups;
    const int hg = (int)blockIdx.x % nhg, item = (int)blockIdx.x / nhg;
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
        const int nall = wa.top << (wa.lg - 4);
        tb = (int)((int64_t)nall * piece / np);
        te = (int)((int64_t)nall * (piece + 1) / np);
    } else {
        const Part part = rows_locate(a.b, ra.p, a.window, item);
        if (part.s < 0) return;
        s = part.s;
        st = part.st;
        ntok = min(st.t, a.b.max_nq);
        lo = part.lo;
        np = part.n;
        if (part.piece == 0 && hg == 0 && threadIdx.x == 0) ra.cut[s] = int2{part.first, part.n};
        const int nall = st.t > 0 ? (st.n - lo + 15) / 16 : 0;                // of the stream (none: n <= lo)
        tb = (int)((int64_t)nall * part.piece / np);
        te = (int)((int64_t)nall * (part.piece + 1) / np);
    }
    const int nk = max((te - tb - 2 * wave + 2 * NW - 1) / (2 * NW), 0);      // steps: tiles tb + 2 (wave + NW k) and the next

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
    const float slope = valid ? paged_slope(a, h) : 0.f;
    const int p = valid ? st.n - st.t + tok0 + tok : -1;                      // rows [first, p] are seen
    const int first = a.window > 0 ? max(p - a.window + 1, 0) : 0;
    const int pend = st.n - st.t + tok0 + ntok - 1;                           // the last row that any token sees

    // ---- tiles: lane l has tile 2 (wave + NW (ids_from + l / 2)) + l % 2 of the part -----
    int64_t offs = 0;
    int j0s = 0;
    float sks = 1.f, svs = 1.f;
    uint64_t there = 0;
    int ids_from = 0;
    auto load_ids = [&](int k0) {
        const int t = tb + 2 * (wave + NW * (k0 + (lane >> 1))) + (lane & 1);
        int j0 = -1;
        if (t < te) {
            if constexpr (LISTED) {
                const int per = wa.lg - 4;
                const int b = wa.list[((int64_t)(st.q0 + tok0) * a.hkv + hk) * wa.top + (t >> per)];
                // (a block past the token's row: none of its rows are seen)
                if (b >= 0 && b <= (max(pend, 0) >> wa.lg)) j0 = (b << wa.lg) + ((t & ((1 << per) - 1)) << 4);
                const int low = a.window > 0 ? max(pend - a.window + 1, 0) : 0;
                if (j0 > pend || j0 + 15 < low) j0 = -1;
            } else {
                j0 = lo + 16 * t;
            }
        }
        const int page = j0 >= 0 ? paged_page(a.b, s, j0 >> lg) : -1;
        there = __ballot(page >= 0);
        j0s = max(j0, 0);
        const int r = j0s & ((1 << lg) - 1);
        offs = page >= 0 ? a.kv.at(page, hk, r) : 0;
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

    struct Step {
        u32x4 k[2][KC];
        Words<VW> v[2][4];
        int j0[2];
        float sk[2], sv[2];
        uint32_t live;
    } buf[PF];
    // byte offsets of what the lane reads, from a tile's first row
    const uint32_t koff = (uint32_t)row * (uint32_t)a.kv.nb1 + 16 * quad;
    const uint32_t voff = 4 * quad * (uint32_t)a.kv.nb1 + 4 * VW * row;
    auto issue = [&](Step& b, int k) {
        if (k < nk && k >= ids_from + 32) load_ids(k);
        const int l = 2 * ((k - ids_from) & 31);
        b.live = k < nk ? (uint32_t)(there >> l) & 3u : 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int alo = __builtin_amdgcn_readlane((int)(uint32_t)offs, l + i), ahi = __builtin_amdgcn_readlane((int)(offs >> 32), l + i);
            b.j0[i] = __builtin_amdgcn_readlane(j0s, l + i);
            if constexpr (I8) {
                b.sk[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, sks), l + i));
                b.sv[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, svs), l + i));
            }
            // (a tile that is not there, or past the last step: all lanes read the pool's first bytes)
            const bool on = (b.live >> i) & 1;
            const int64_t at = on ? ((int64_t)ahi << 32) | (uint32_t)alo : 0;
            const uint32_t mask = on ? ~0u : 0u;
            const char *kp = a.kv.k + at, *vp = a.kv.v + at;
            const uint32_t ko = koff & mask;
#pragma unroll
            for (int c = 0; c < KC; ++c) b.k[i][c] = __builtin_nontemporal_load((const u32x4*)(kp + (ko + (64 * c & mask))));
            // (F16: rows past the stream's last may hold anything, and read that one)
            const int left = I8 ? 15 : min(st.n - 1 - b.j0[i], 15);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t vo = voff + (uint32_t)r * (uint32_t)a.kv.nb1;
                if constexpr (!I8) vo = (uint32_t)min(4 * quad + r, left) * (uint32_t)a.kv.nb1 + 4 * VW * row;
                b.v[i][r] = load_words<VW>(vp + (vo & mask));
            }
        }
    };

    floatx4 o[DPL];
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    auto compute = [&](const Step& b) {
        if (b.live == 0) return;
        floatx4 sc[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                half8 kr;
                if constexpr (I8) kr = half8_of_bytes(b.k[i][ks >> 1][2 * (ks & 1)], b.k[i][ks >> 1][2 * (ks & 1) + 1]);
                else kr = __builtin_bit_cast(half8, b.k[i][ks]);
                sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kr, q[ks], sc[i], 0, 0, 0);
            }
        }
        float x[8], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool on = (b.live >> i) & 1;
            const float lsv = I8 ? __builtin_amdgcn_logf(b.sv[i]) : 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = b.j0[i] + 4 * quad + r;
                const float y = I8 ? sc[i][r] * b.sk[i] : sc[i][r];
                float z = fmaf(slope, (float)(j - p), a.capk != 0.f ? paged_wide_cap(a.c * y, a.cap, a.capk) : paged_score(a, y));
                if constexpr (I8) z += lsv;
                z = on && j >= first && j <= p ? z : -INFINITY;
                x[4 * i + r] = z;
                mx = fmaxf(mx, z);
            }
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
            l = I8 ? fmaf(sum, __builtin_amdgcn_rcpf(b.sv[i]), l) : l + sum;
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
                        const uint32_t w0 = b.v[i][r].w[w], w1 = b.v[i][r + 1].w[w];
                        half2 y;
                        if constexpr (I8) {
                            y = halves_of_bytes(__builtin_amdgcn_perm(w1, w0, 0x0C040C00u + 0x00010001u * e));
                        } else {
                            // (of a tile that is not there zeros)
                            const uint32_t z = __builtin_amdgcn_perm(w1, w0, 0x05040100u + 0x02020202u * e);
                            y = __builtin_bit_cast(half2, (b.live >> i) & 1 ? z : 0u);
                        }
                        vt[4 * i + r] = y[0];
                        vt[4 * i + r + 1] = y[1];
                    }
                const int eb = w * (DPL / VW) + e;
                o[eb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pv, o[eb], 0, 0, 0);
            }
    };

    if (nk > 0) {
        load_ids(0);
#pragma unroll
        for (int u = 0; u < PF; ++u) issue(buf[u], u);
        for (int k = 0; k < nk; k += PF) {
#pragma unroll
            for (int u = 0; u < PF; ++u) {
                compute(buf[u]);
                issue(buf[u], k + u + PF);
            }
        }
    }

    // ---- join the wavefronts -------------------------------------------------------
    l = quad_sum(l);
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
    float* const rec = ra.recs + ((int64_t)hg * ra.items + item) * ra.rec;
    for (int e = (int)threadIdx.x; e < nrow * (D / 4); e += 64 * NW) {
        const int r = e / (D / 4), c = e % (D / 4);
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][r]);
        const float Ms = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = exp2_fast(sm[w][r] - Ms);
            L = fmaf(f, sl[w][r], L);
            const floatx4 y = *(const floatx4*)(xo + (w * 16 + r) * D + 4 * (c ^ (r & 7)));
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

// Joins the parts of a token's list, in order: a wavefront per (token, query head), a
// lane per 4 dims and, at D 64, half of the wavefront idle.
template <int D>
static __global__ __launch_bounds__(64) void paged_walk_join(WalkArgs wa) {
    const RowsArgs& ra = wa.r;
    const PagedAttn& a = ra.a;
    const int lane = (int)threadIdx.x;
    const int h = (int)blockIdx.x % a.hq, t = (int)blockIdx.x / a.hq;
    if (paged_token(a.b, t).s < 0) return;
    const int G = a.hq / a.hkv, hk = h / G, g = h - hk * G;
    const int sub = (int)ra.hpw.div((uint32_t)g), r = g - sub * (int)ra.hpw.d;
    const float* rec = ra.recs + ((int64_t)(hk * ra.groups + sub) * ra.items + (int64_t)t * wa.parts) * ra.rec;
    float M = -INFINITY;
    for (int i = 0; i < wa.parts; ++i) M = fmaxf(M, rec[(int64_t)i * ra.rec + ra.rows * D + r]);
    const float Ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    const int c = lane % (D / 4);
    for (int i = 0; i < wa.parts; ++i) {
        const float* q = rec + (int64_t)i * ra.rec;
        const float f = exp2_fast(q[ra.rows * D + r] - Ms);
        L = fmaf(f, q[ra.rows * (D + 1) + r], L);
        const floatx4 y = *(const floatx4*)(q + r * D + 4 * c);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = fmaf(f, y[k], x[k]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (lane < D / 4) paged_store4(a, ((int64_t)t * a.hq + h) * D + 4 * c, x * inv);
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

hipError_t launch_paged_rows_q8(const PagedBlocks& pb, int head_dim, hipStream_t st) {
    const PagedAttn& a = pb.a;
    if (!paged_rows_takes(a)) return hipErrorInvalidValue;
    WalkArgs wa;
    heads_of(a, a.b.max_nq > 0 ? a.b.max_nq : 1, head_dim, wa.r);
    wa.sc = pb.sc;
    wa.list = nullptr;
    wa.top = wa.lg = 0;
    wa.parts = 1;
    RowsArgs& ra = wa.r;
    const int nhg = a.hkv * ra.groups;
    const size_t cut = ((size_t)a.b.n_streams * sizeof(int2) + 255) & ~(size_t)255;
    if (cut > a.ws_bytes) return hipErrorOutOfMemory;    // (65535 streams at most: half a MiB)
    ra.cut = reinterpret_cast<int2*>(a.ws);
    ra.recs = reinterpret_cast<float*>(a.ws + cut);
    ra.p = rows_plan(a.b, nhg, head_dim, (int64_t)((a.ws_bytes - cut) / ((size_t)ra.rec * sizeof(float))) / nhg, ra.items);
    const int64_t nwg = (int64_t)ra.items * nhg;
    if (nwg > kMaxGridX) return hipErrorNotSupported;
    const dim3 grid((unsigned)nwg);
    if (head_dim == 128) hipLaunchKernelGGL((paged_walk_kernel<128, true, false, 4>), grid, dim3(256), 0, st, wa);
    else hipLaunchKernelGGL((paged_walk_kernel<64, true, false, 4>), grid, dim3(256), 0, st, wa);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !ra.p.cuts) return e;
    const dim3 cg((unsigned)(a.hq * (head_dim / 32)), (unsigned)a.b.max_nq, (unsigned)a.b.n_streams);
    if (head_dim == 128) hipLaunchKernelGGL((paged_rows_combine<128>), cg, dim3(64), 0, st, ra);
    else hipLaunchKernelGGL((paged_rows_combine<64>), cg, dim3(64), 0, st, ra);
    return hipGetLastError();
}

template <int D, bool I8>
static void launch_listed(const WalkArgs& wa, unsigned nwg, hipStream_t st) {
    hipLaunchKernelGGL((paged_walk_kernel<D, I8, true, 4>), dim3(nwg), dim3(256), 0, st, wa);
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
    // parts of a list: workgroups for two a CU, and at least a step for each wavefront
    const int64_t wgs = (int64_t)a.b.tokens * nhg, tiles = (int64_t)pb.top << (pb.lg - 4);
    int64_t parts = (512 + wgs - 1) / wgs;
    if (parts > (tiles + 7) / 8) parts = (tiles + 7) / 8;
    const int64_t room = (int64_t)(a.ws_bytes / ((size_t)ra.rec * sizeof(float))) / wgs;
    if (parts > room) parts = room;
    if (parts < 1) parts = 1;
    wa.parts = (int32_t)parts;
    ra.items = (int32_t)(a.b.tokens * parts);
    const int64_t nwg = wgs * parts;
    if (nwg > kMaxGridX || (parts > 1 && (int64_t)a.b.tokens * a.hq > kMaxGridX)) return hipErrorNotSupported;
    if (head_dim == 128 && pb.sc.k) launch_listed<128, true>(wa, (unsigned)nwg, st);
    else if (head_dim == 128) launch_listed<128, false>(wa, (unsigned)nwg, st);
    else if (pb.sc.k) launch_listed<64, true>(wa, (unsigned)nwg, st);
    else launch_listed<64, false>(wa, (unsigned)nwg, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || parts == 1) return e;
    const dim3 cg((unsigned)(a.b.tokens * a.hq));
    if (head_dim == 128) hipLaunchKernelGGL((paged_walk_join<128>), cg, dim3(64), 0, st, wa);
    else hipLaunchKernelGGL((paged_walk_join<64>), cg, dim3(64), 0, st, wa);
    return hipGetLastError();
}

}  // namespace vxfa
