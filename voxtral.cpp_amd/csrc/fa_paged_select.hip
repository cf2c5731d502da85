// fa_paged_select.hip — bounds of the keys of a paged cache's blocks, and the blocks
// that each token's queries choose by them, for gfx950.
//
// A block's keys lie, dim for dim, between lo and hi, so no key's product with a query
// q is larger than sum_d max(q_d lo_d, q_d hi_d) = sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d.
// With bounds and queries in 8 bits at scales that are powers of two that is one
// product of whole numbers, of length 2 D, on v_mfma_i32_16x16x64_i8: exact, so the choice depends on
// no order of sums. Bound by the bytes of the bounds: 2 D + 4 a block and kv head.
#include "fa_paged_q8.h"

namespace vxfa {

typedef int intx4 __attribute__((ext_vector_type(4)));

// ---- bounds ------------------------------------------------------------------------
// A wavefront per block and kv head: rows of 16-byte chunks, a lane's dims' extremes in
// registers, joined over the lanes that have the same dims.
template <int D, bool I8>
__global__ __launch_bounds__(256) void paged_bounds_kernel(PagedBounds a) {
    constexpr int DPL = I8 ? 16 : 8, CH = D / DPL, RPI = 64 / CH;   // dims of a lane, lanes of a row, rows of a load
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int nh = (a.hkv + 3) / 4, lg = a.out.lg;
    const int h = (int)blockIdx.x % nh * 4 + wave;
    const PagedUnit u = paged_unit(a.b, (int)blockIdx.x / nh, [&](const PagedStream& s) { return blocks_count(s, a.b.max_nq, lg); });
    if (u.s < 0 || h >= a.hkv) return;
    const int row0 = (blocks_first(u.st, lg) + u.i) << lg, rows = min(u.st.n - row0, 1 << lg);
    const int page = paged_page(a.b, u.s, row0 >> a.b.ps_log2);
    if (page < 0) return;
    const int at = row0 & ((1 << a.b.ps_log2) - 1);
    const char* const src = a.kv.k + a.kv.at(page, h, at) + 16 * (lane % CH);
    float hi[DPL], lo[DPL];
#pragma unroll
    for (int i = 0; i < DPL; ++i) { hi[i] = -INFINITY; lo[i] = INFINITY; }
    constexpr int U = 4;
    for (int r0 = 0; r0 < rows; r0 += U * RPI) {
        u32x4 w[U];
        float s[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            // (rows past the last read that one again)
            const int rb = min(r0 + RPI * j, rows - 1), r = min(r0 + RPI * j + lane / CH, rows - 1);
            w[j] = *(const u32x4*)(src + (int64_t)r * a.kv.nb1);
            s[j] = 1.f;
            if constexpr (I8) s[j] = scale_in_range(*(const float*)(a.sc.k + a.sc.at(page, h, at + rb)));   // (16 rows hold the load's)
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int i = 0; i < DPL; ++i) {
                float x;
                if constexpr (I8) x = (float)((int)(w[j][i >> 2] << (24 - 8 * (i & 3))) >> 24) * s[j];
                else x = (float)__builtin_bit_cast(half8, w[j])[i];
                hi[i] = fmaxf(hi[i], x);
                lo[i] = fminf(lo[i], x);
            }
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
#pragma unroll
        for (int k = CH; k < 64; k *= 2) {
            hi[i] = fmaxf(hi[i], shfl_xor(hi[i], k));
            lo[i] = fminf(lo[i], shfl_xor(lo[i], k));
        }
        m = fmaxf(m, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
    }
    const int e = exp_for(__builtin_bit_cast(float, wave_max(__builtin_bit_cast(int, m))));
    const float f = two_to(-e);
    uint32_t bh[DPL / 4], bl[DPL / 4];
#pragma unroll
    for (int i = 0; i < DPL; ++i) {
        const uint32_t x = (uint32_t)(int)fminf(fmaxf(ceilf(hi[i] * f), -127.f), 127.f) & 255u;
        const uint32_t y = (uint32_t)(int)fminf(fmaxf(floorf(lo[i] * f), -127.f), 127.f) & 255u;
        bh[i / 4] = (i & 3) ? bh[i / 4] | x << (8 * (i & 3)) : x;
        bl[i / 4] = (i & 3) ? bl[i / 4] | y << (8 * (i & 3)) : y;
    }
    const int bi = at >> lg;
    if (lane < CH) {
        uint32_t* const dh = (uint32_t*)(a.out.b + page * a.out.nb3 + h * a.out.nb2 + bi * a.out.nb1 + DPL * lane);
#pragma unroll
        for (int i = 0; i < DPL / 4; ++i) { dh[i] = bh[i]; dh[D / 4 + i] = bl[i]; }
    }
    if (lane == 0) *(float*)(a.out.s + page * a.out.s_nb3 + h * a.out.s_nb2 + 4 * (int64_t)bi) = two_to(e);
}

hipError_t launch_paged_bounds(const PagedBounds& a, hipStream_t st) {
    if (a.b.tokens <= 0 || a.b.n_streams <= 0 || a.b.max_nkv <= 0) return hipSuccess;
    const int64_t grid = blocks_bound(a.b, a.out.lg) * ((a.hkv + 3) / 4);
    if (grid > kMaxGridX) return hipErrorNotSupported;
    const dim3 g((unsigned)grid), b(256);
    if (a.d == 128 && a.sc.k) hipLaunchKernelGGL((paged_bounds_kernel<128, true>), g, b, 0, st, a);
    else if (a.d == 128) hipLaunchKernelGGL((paged_bounds_kernel<128, false>), g, b, 0, st, a);
    else if (a.d == 64 && a.sc.k) hipLaunchKernelGGL((paged_bounds_kernel<64, true>), g, b, 0, st, a);
    else if (a.d == 64) hipLaunchKernelGGL((paged_bounds_kernel<64, false>), g, b, 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

// ---- choice ------------------------------------------------------------------------
// A workgroup per tile of tokens of one stream, kv head and segment of blocks. Columns
// of the product: tokens x query heads of the group (padded to a power of two, gp;
// groups above 16 in passes), rows: 16 blocks a wavefront and step. Scores, as
// unsigned keys that order as they do, go to LDS; a wavefront per token finds the key of
// the last block to be chosen, bit by bit from the highest in which two keys
// differ, counting keys by ballots, and stops where a threshold leaves just as many
// as are wanted; then it lists them in order. Streams of more blocks than a segment: each
// segment leaves its best (key, block) and paged_select_join chooses among those.

constexpr int SL_NT = 512;
constexpr uint32_t kForced = 0xFFFFFFFFu;              // a first or last block
struct SelectArgs {
    PagedSelect a;
    int32_t gp_log2;           // log2 of the columns of a token
    int32_t tiles;             // tokens of a tile
    int32_t seg, segs;         // blocks of a segment (a multiple of 16), segments
    int32_t keep;              // pairs that a segment leaves: min(top, seg)
    uint2* pairs;              // [token][hkv][segment][keep], key 0: none
};

// orders as the floats do, above 0
__device__ __forceinline__ uint32_t score_key(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One wavefront: of n keys key(i) (0: no candidate) the `want` largest, of equal ones the first;
// put(rank, i) of each, in order. Returns how many. REGS: 64 REGS keys or fewer, kept in registers.
template <int REGS, class K, class P>
__device__ __forceinline__ int wave_choose(int n, int want, int lane, K key, P put) {
    uint32_t reg[REGS > 0 ? REGS : 1];
    if constexpr (REGS > 0) {
#pragma unroll
        for (int c = 0; c < REGS; ++c) reg[c] = 64 * c + lane < n ? key(64 * c + lane) : 0u;
    }
    auto each = [&](auto f) {
        if constexpr (REGS > 0) {
#pragma unroll
            for (int c = 0; c < REGS; ++c)
                if (64 * c < n) f(64 * c + lane, reg[c]);
        } else {
            for (int i = 0; i < n; i += 64) f(i + lane, i + lane < n ? key(i + lane) : 0u);
        }
    };
    auto count = [&](uint32_t t) -> int {
        int r = 0;
        each([&](int, uint32_t k) { r += __popcll(__ballot(k >= t)); });
        return r;
    };
    uint32_t hi = 0, lo = 0xFFFFFFFFu;
    int all = 0, forced = 0;
    each([&](int, uint32_t k) {
        all += __popcll(__ballot(k != 0));
        forced += __popcll(__ballot(k == kForced));
        const bool in = k != 0 && k != kForced;
        hi = max(hi, in ? k : 0u);
        lo = min(lo, in ? k : 0xFFFFFFFFu);
    });
    uint32_t t = 1;            // chosen: keys above t, and `eq` of those that are t
    int eq = 0x7fffffff;
    if (all > want) {
        if (forced >= want) {
            t = kForced;
            eq = want;
        } else {
            // (unsigned maximum and minimum over the lanes, as signed ones)
            hi = (uint32_t)wave_max((int)(hi ^ 0x80000000u)) ^ 0x80000000u;
            lo = ~((uint32_t)wave_max((int)(~lo ^ 0x80000000u)) ^ 0x80000000u);
            const uint32_t diff = hi ^ lo;
            int bit = diff ? 31 - __builtin_clz(diff) : -1;
            t = bit >= 31 ? 0u : hi >> (bit + 1) << (bit + 1);
            for (; bit >= 0; --bit) {
                const uint32_t c = t | 1u << bit;
                const int m = count(c);
                if (m >= want) t = c;
                if (m == want) break;
            }
            if (bit < 0) eq = want - (t == 0xFFFFFFFFu ? 0 : count(t + 1));
        }
    }
    int done = 0, eqs = 0;
    const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
    each([&](int i, uint32_t k) {
        const uint64_t same = __ballot(k == t && k != 0);
        const bool take = k != 0 && (k > t || (k == t && eqs + __popcll(same & below) < eq));
        const uint64_t b = __ballot(take);
        if (take) put(done + __popcll(b & below), i);
        eqs += __popcll(same);
        done += __popcll(b);
    });
    return done;
}
template <class K, class P>
__device__ __forceinline__ int wave_choose_any(int n, int want, int lane, K key, P put) {
    if (n <= 256) return wave_choose<4>(n, want, lane, key, put);
    if (n <= 1024) return wave_choose<16>(n, want, lane, key, put);
    return wave_choose<0>(n, want, lane, key, put);
}

template <int D>
__global__ __launch_bounds__(SL_NT) void paged_select_blocks(SelectArgs sa) {
    constexpr int KS = 2 * D / 64, QS = D / 64;       // k steps of the product, of a query
    extern __shared__ uint32_t keys[];                // [token][segment]
    const PagedSelect& a = sa.a;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int hk = (int)blockIdx.x % a.hkv, rest = (int)blockIdx.x / a.hkv;
    const int seg = rest % sa.segs, tile = rest / sa.segs;
    const PagedUnit u = paged_unit(a.b, tile, [&](const PagedStream& s) { return (min(s.t, a.b.max_nq) + sa.tiles - 1) / sa.tiles; });
    if (u.s < 0) return;
    const int lg = a.in.lg, bpp = a.b.ps_log2 - lg;   // log2 of the blocks of a page
    const int i0 = u.i * sa.tiles, ntok = min(min(u.st.t, a.b.max_nq) - i0, sa.tiles);
    const int p0 = u.st.n - u.st.t + i0;              // row of the first token
    auto low_of = [&](int p) -> int { return a.window > 0 ? max(p - a.window + 1, 0) >> lg : 0; };
    const int end = ((p0 + ntok - 1) >> lg) + 1;      // blocks seen by any token (none: 0 or less)
    const int sb = low_of(p0) + seg * sa.seg, n = min(end - sb, sa.seg);   // this segment's
    const int G = a.hq / a.hkv, gp = 1 << sa.gp_log2;

    // ---- queries in 8 bits: column lane % 16, dims 64 ks + 16 (lane / 16) .. ----------
    const int col = lane & 15, quad = lane >> 4;
    const int tk = col >> sa.gp_log2, g0 = col & (gp - 1);
    const int passes = (G + gp - 1) >> sa.gp_log2;
    const int p = p0 + tk, low = low_of(p), last = p >> lg;
    const int nt = (max(n, 0) + 15) / 16;
    for (int pass = 0; pass < passes; ++pass) {
        const int g = g0 + (pass << sa.gp_log2);
        const bool valid = tk < ntok && g < G;
        half8 q[2 * QS];
#pragma unroll
        for (int c = 0; c < 2 * QS; ++c) {
            q[c] = half8{};
            if (valid)
                q[c] = load_q8(a.q, (int64_t)(u.st.q0 + i0 + tk) * a.q_nb1 + (int64_t)(hk * G + g) * a.q_nb2 +
                                        (64 * (c >> 1) + 16 * quad + 8 * (c & 1)) * (a.q_f16 ? 2 : 4), a.q_f16);
        }
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < 2 * QS; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf((float)q[c][i]));
        m = fmaxf(m, shfl_xor(m, 16));
        m = fmaxf(m, shfl_xor(m, 32));
        const int e = exp_for(m);
        const float f = two_to(-e), fs = valid ? two_to(e) : 0.f;
        intx4 qb[KS];
#pragma unroll
        for (int ks = 0; ks < QS; ++ks)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t up = 0, dn = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = (float)q[2 * ks + (w >> 1)][4 * (w & 1) + i] * f;
                    const int r = x == x ? (int)fminf(fmaxf(rintf(x), -127.f), 127.f) : 0;
                    up |= (uint32_t)(max(r, 0) & 255) << (8 * i);
                    dn |= (uint32_t)(min(r, 0) & 255) << (8 * i);
                }
                qb[ks][w] = (int)up;
                qb[QS + ks][w] = (int)dn;
            }
        for (int t = wave; t < nt; t += SL_NT / 64) {
            // the lane's row of the operand: block b
            const int b = min(sb + 16 * t + col, end - 1);
            const int page = paged_page(a.b, u.s, b >> bpp), bi = b & ((1 << bpp) - 1);
            const char* const src = a.in.b + max(page, 0) * a.in.nb3 + hk * a.in.nb2 + bi * a.in.nb1 + 16 * quad;
            intx4 kb[KS], acc = {0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kb[ks] = *(const intx4*)(src + 64 * ks);
            const float s = *(const float*)(a.in.s + max(page, 0) * a.in.s_nb3 + hk * a.in.s_nb2 + 4 * (int64_t)bi);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kb[ks], qb[ks], acc, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // block of the result's row, its scale and page from the lane that read it
                const int r = 4 * quad + i, at = 16 * t + r, bl = sb + at;
                const float sr = __shfl(s, r, 64);
                const int pr = __shfl(page, r, 64);
                float y = valid ? (float)acc[i] * fs : -INFINITY;
                for (int k = 1; k < gp; k *= 2) y = fmaxf(y, shfl_xor(y, k));
                if (g0 != 0 || tk >= ntok || at >= n) continue;
                uint32_t key = pr < 0 ? 0u : score_key(y * sr);
                if (pass > 0) key = max(key, keys[tk * sa.seg + at]);
                if (pass + 1 == passes) {
                    if (bl < low + a.n_sink || bl > last - a.n_recent) key = kForced;
                    if (bl < low || bl > last) key = 0u;
                }
                keys[tk * sa.seg + at] = key;
            }
        }
    }
    __syncthreads();
    for (int t = wave; t < ntok; t += SL_NT / 64) {
        const uint32_t* const key = keys + t * sa.seg;
        const int64_t row = (int64_t)(u.st.q0 + i0 + t) * a.hkv + hk;
        auto get = [&](int i) -> uint32_t { return key[i]; };
        if (sa.segs == 1) {
            int32_t* const out = a.list + row * a.top;
            const int k = wave_choose_any(max(n, 0), a.top, lane, get, [&](int r, int i) { out[r] = sb + i; });
            for (int r = k + lane; r < a.top; r += 64) out[r] = -1;
        } else {
            uint2* const out = sa.pairs + (row * sa.segs + seg) * sa.keep;
            const int k = wave_choose_any(max(n, 0), sa.keep, lane, get, [&](int r, int i) { out[r] = uint2{key[i], (uint32_t)(sb + i)}; });
            for (int r = k + lane; r < sa.keep; r += 64) out[r] = uint2{0u, 0u};
        }
    }
}

// Among the segments' best: a wavefront per token and kv head.
__global__ __launch_bounds__(256) void paged_select_join(SelectArgs sa) {
    const PagedSelect& a = sa.a;
    const int lane = (int)threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if (row >= (int64_t)a.b.tokens * a.hkv) return;
    if (paged_token(a.b, (int)(row / a.hkv)).s < 0) return;
    const uint2* const in = sa.pairs + row * sa.segs * sa.keep;
    int32_t* const out = a.list + row * a.top;
    const int k = wave_choose_any(sa.segs * sa.keep, a.top, lane, [&](int i) -> uint32_t { return in[i].x; },
                                  [&](int r, int i) { out[r] = (int32_t)in[i].y; });
    for (int r = k + lane; r < a.top; r += 64) out[r] = -1;
}

hipError_t launch_paged_select(const PagedSelect& a, hipStream_t st) {
    if (a.b.tokens <= 0 || a.b.n_streams <= 0 || a.b.max_nq <= 0 || a.hq <= 0) return hipSuccess;
    SelectArgs sa;
    sa.a = a;
    const int G = a.hq / a.hkv;
    sa.gp_log2 = 0;
    while ((1 << sa.gp_log2) < G && sa.gp_log2 < 4) ++sa.gp_log2;
    sa.tiles = 16 >> sa.gp_log2;
    if (sa.tiles > a.b.max_nq) sa.tiles = a.b.max_nq;
    // blocks that a tile's tokens see at most
    int64_t rows = a.b.max_nkv;
    if (a.window > 0 && rows > (int64_t)a.window + sa.tiles) rows = (int64_t)a.window + sa.tiles + (1 << a.in.lg);
    const int64_t nb = (rows + (1 << a.in.lg) - 1) >> a.in.lg;
    int64_t most = 16384 / sa.tiles / 16 * 16;          // (64 KiB of keys)
    if (most > kSelectSeg) most = kSelectSeg;
    sa.segs = (int32_t)((nb + most - 1) / most);
    if (sa.segs < 1) sa.segs = 1;
    sa.seg = (int32_t)(((nb + sa.segs - 1) / sa.segs + 15) / 16 * 16);
    if (sa.seg < 16) sa.seg = 16;
    sa.keep = a.top < sa.seg ? a.top : sa.seg;
    sa.pairs = reinterpret_cast<uint2*>(a.ws);
    if (sa.segs > 1 && (double)a.b.tokens * a.hkv * sa.segs * sa.keep * sizeof(uint2) > (double)a.ws_bytes) return hipErrorOutOfMemory;
    const int64_t per = ((int64_t)a.b.max_nq + sa.tiles - 1) / sa.tiles;
    int64_t tiles = (int64_t)a.b.tokens / sa.tiles + a.b.n_streams;
    if (tiles > per * a.b.n_streams) tiles = per * a.b.n_streams;
    if (tiles > a.b.tokens) tiles = a.b.tokens;
    const int64_t grid = tiles * sa.segs * a.hkv, jgrid = ((int64_t)a.b.tokens * a.hkv + 3) / 4;
    if (grid > kMaxGridX / 2 || jgrid > kMaxGridX) return hipErrorNotSupported;
    const size_t lds = (size_t)sa.tiles * sa.seg * sizeof(uint32_t);
    if (a.d == 128) hipLaunchKernelGGL((paged_select_blocks<128>), dim3((unsigned)grid), dim3(SL_NT), lds, st, sa);
    else if (a.d == 64) hipLaunchKernelGGL((paged_select_blocks<64>), dim3((unsigned)grid), dim3(SL_NT), lds, st, sa);
    else return hipErrorInvalidValue;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || sa.segs == 1) return e;
    hipLaunchKernelGGL(paged_select_join, dim3((unsigned)jgrid), dim3(256), 0, st, sa);
    return hipGetLastError();
}

}  // namespace vxfa
