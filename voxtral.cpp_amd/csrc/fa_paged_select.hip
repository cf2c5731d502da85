// fa_paged_select.hip — bounds of the keys of a paged cache's blocks, and the blocks
// that each token's queries choose by them, for gfx950.
//
// A block's keys lie, dim for dim, between lo and hi, so no key's product with a query
// q is larger than sum_d max(q_d lo_d, q_d hi_d) = sum_d max(q_d, 0) hi_d + min(q_d, 0) lo_d.
// With bounds and queries in 8 bits at scales that are powers of two that is one
// product of whole numbers, of length 2 D, on v_mfma_i32_16x16x64_i8: exact, so the choice depends on
// no order of sums. The choice is bound by a chain of loads (sizes, pages, queries, bounds), each of
// about a microsecond, and the search; the first bounds are asked for after the queries are converted, which
// each wavefront does for all columns (about 270 of its 661 VALU instructions), so the chain is longer than it has to be: one stream of 128 blocks 8.7 us in a graph, of 512 12.9, 32 uneven ones of up
// to 512 18 (19 MB of bounds: 4 us at what a large copy reaches), of up to 2048 41 (76 MB). Bounds of
// a token's block 4.3 us, of 8192 tokens' keys of 16 bits in blocks of 32 4.6 (17 MB: 3.4).
#include <algorithm>

#include "fa_paged_join.h"
#include "fa_paged_q8.h"

namespace vxfa {

typedef int intx4 __attribute__((ext_vector_type(4)));

// ---- bounds ------------------------------------------------------------------------
// A wavefront per block and kv head. A lane has 4 dims of every second (D 64: fourth) row, their
// extremes in registers (of the smallest, the negative's largest), which one lane swap (two) joins:
// with 16 dims a lane the joining took most of the time (8192 tokens in blocks of 16 rows of 8 bits
// 9.7 us, not 5.1). ROWS: of a round, whose loads are in flight together.
template <int D, bool I8, int ROWS>
__global__ __launch_bounds__(256) void paged_bounds_kernel(PagedBounds a) {
    constexpr int CH = D / 4, RPI = 64 / CH, U = ROWS / RPI;   // lanes of a row, rows of a load, loads of a round
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int nh = (a.hkv + 3) / 4, lg = a.out.lg;
    const int h = (int)blockIdx.x % nh * 4 + wave;
    const PagedUnit u = paged_unit(a.b, (int)blockIdx.x / nh, [&](const PagedStream& s) { return blocks_count(s, a.b.max_nq, lg); });
    if (u.s < 0 || h >= a.hkv) return;
    const int row0 = (blocks_first(u.st, lg) + u.i) << lg, rows = min(u.st.n - row0, 1 << lg);
    const int page = paged_page(a.b, u.s, row0 >> a.b.ps_log2);
    if (page < 0) return;
    const int at = row0 & ((1 << a.b.ps_log2) - 1);
    const char* const src = a.kv.k + a.kv.at(page, h, at) + (I8 ? 4 : 8) * (lane % CH);
    float hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) hi[i] = lo[i] = -INFINITY;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    for (int r0 = 0; r0 < rows; r0 += ROWS) {
        u32x2 w[U];
        float s[ROWS / 16];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            // (rows past the last read that one again)
            const char* const from = src + (int64_t)min(r0 + RPI * j + lane / CH, rows - 1) * a.kv.nb1;
            if constexpr (I8) w[j][0] = *(const uint32_t*)from;
            else w[j] = *(const u32x2*)from;
        }
        if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < ROWS / 16; ++j) s[j] = scale_in_range(*(const float*)(a.sc.k + a.sc.at(page, h, at + min(r0 + 16 * j, rows - 1))));
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x;
                // (16 rows hold a load's; those past the last are of the scale of the last one's 16)
                if constexpr (I8) x = (float)((int)(w[j][0] << (24 - 8 * i)) >> 24) * s[RPI * j / 16];
                else x = (float)__builtin_bit_cast(half4, w[j])[i];
                hi[i] = fmaxf(hi[i], x);
                lo[i] = fmaxf(lo[i], -x);
            }
    }
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi[i] = CH == 32 ? pair32_max(hi[i]) : quad_max(hi[i]);
        lo[i] = -(CH == 32 ? pair32_max(lo[i]) : quad_max(lo[i]));
        if (hi[i] < lo[i]) hi[i] = lo[i] = 0.f;           // (no number among the block's keys: all NaN)
        m = fmaxf(m, fmaxf(fabsf(hi[i]), fabsf(lo[i])));
    }
    const int e = exp_for(__builtin_bit_cast(float, wave_max(__builtin_bit_cast(int, m))));
    const float f = two_to(-e);
    uint32_t bh = 0, bl = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bh |= ((uint32_t)(int)fminf(fmaxf(ceilf(hi[i] * f), -127.f), 127.f) & 255u) << (8 * i);
        bl |= ((uint32_t)(int)fminf(fmaxf(floorf(lo[i] * f), -127.f), 127.f) & 255u) << (8 * i);
    }
    const int bi = at >> lg;
    uint32_t* const dst = (uint32_t*)(a.out.b + page * a.out.nb3 + h * a.out.nb2 + bi * a.out.nb1);
    // (the second half of the lanes, or the second row of them, has the same: it stores the lower ones)
    if (lane < 2 * CH) dst[lane] = lane < CH ? bh : bl;
    if (lane == 0) *(float*)(a.out.s + page * a.out.s_nb3 + h * a.out.s_nb2 + 4 * (int64_t)bi) = two_to(e);
}

template <int D, bool I8>
static void launch_bounds(const PagedBounds& a, unsigned grid, hipStream_t st) {
    if (a.out.lg >= 6) hipLaunchKernelGGL((paged_bounds_kernel<D, I8, 64>), dim3(grid), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_bounds_kernel<D, I8, 16>), dim3(grid), dim3(256), 0, st, a);
}

hipError_t launch_paged_bounds(const PagedBounds& a, hipStream_t st) {
    if (a.b.max_nq <= 0 || a.b.n_streams <= 0 || a.b.max_nkv <= 0) return hipSuccess;
    // (max_nq rows, wherever they begin, or all)
    const int64_t per = std::min((((int64_t)a.b.max_nq - 2) >> a.out.lg) + 2, (((int64_t)a.b.max_nkv - 1) >> a.out.lg) + 1);
    const int64_t grid = a.b.n_streams * per * ((a.hkv + 3) / 4);
    if (grid > kMaxGridX) return hipErrorNotSupported;
    if (a.d == 128 && a.sc.k) launch_bounds<128, true>(a, (unsigned)grid, st);
    else if (a.d == 128) launch_bounds<128, false>(a, (unsigned)grid, st);
    else if (a.d == 64 && a.sc.k) launch_bounds<64, true>(a, (unsigned)grid, st);
    else if (a.d == 64) launch_bounds<64, false>(a, (unsigned)grid, st);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

// ---- choice ------------------------------------------------------------------------
// A workgroup of 16 wavefronts per tile of tokens of one stream, kv head and segment of
// blocks. Columns of the product: tokens x query heads of the group (padded to a power of two,
// gp; groups above 16 in passes), rows: 16 blocks a wavefront and step, two steps' loads in
// flight. Scores, as unsigned keys that order as they do, go to LDS. The key of the last block to be
// chosen is found bit by bit from the highest in which two keys differ, by counting keys
// (ballots), and the search stops where a threshold leaves just as many as are wanted; then
// they are listed in order: by a wavefront per token where there are several and few blocks, else by all
// of them, token by token. Streams of more blocks than a segment: each segment leaves its best
// (key, block) and paged_select_join chooses among those.

constexpr int SL_WAVES = 16;                           // wavefronts of a workgroup at most
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

// LDS of the wavefronts that choose together.
struct ChooseRoom {
    uint32_t cnt[3][8];        // counts of keys from seven thresholds on, in turn
    uint32_t first[4][SL_WAVES], over[SL_WAVES], same[SL_WAVES];
};

__device__ __forceinline__ uint32_t wave_largest(uint32_t x) { return (uint32_t)wave_max((int)(x ^ 0x80000000u)) ^ 0x80000000u; }

// Of n keys key(i) (0: no candidate) the `want` largest, of equal ones the first; put(rank, i) of each,
// in order. Returns how many. TEAM: all that many wavefronts of the workgroup, each with keys 64 REGS wave .. in
// registers, three bits of the threshold a round (a round is a barrier); 0:
// one wavefront, a bit a round, REGS 0: any number of keys, read again each time.
template <int TEAM, int REGS, class K, class P>
__device__ __forceinline__ int choose(ChooseRoom* room, int wave, int lane, int n, int want, K key, P put) {
    constexpr int NT = TEAM > 0 ? TEAM : 1;
    const int at = TEAM ? 64 * REGS * wave : 0;
    uint32_t reg[REGS > 0 ? REGS : 1];
    if constexpr (REGS > 0) {
#pragma unroll
        for (int c = 0; c < REGS; ++c) reg[c] = at + 64 * c + lane < n ? key(at + 64 * c + lane) : 0u;
    }
    auto each = [&](auto f) {
        if constexpr (REGS > 0) {
#pragma unroll
            for (int c = 0; c < REGS; ++c)
                if (at + 64 * c < n) f(at + 64 * c + lane, reg[c]);
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
    hi = wave_largest(hi);
    lo = ~wave_largest(~lo);
    if constexpr (TEAM > 0) {
        __syncthreads();       // (the keys are here; the room is free)
        if (lane < 4) room->first[lane][wave] = lane == 0 ? (uint32_t)all : (lane == 1 ? (uint32_t)forced : (lane == 2 ? hi : lo));
        if (wave == 0 && lane < 24) (&room->cnt[0][0])[lane] = 0;
        __syncthreads();
        const int w = lane & (NT - 1);
        all = wave_sum(lane < NT ? (int)room->first[0][w] : 0);
        forced = wave_sum(lane < NT ? (int)room->first[1][w] : 0);
        hi = wave_largest(room->first[2][w]);
        lo = ~wave_largest(~room->first[3][w]);
    }
    uint32_t t = 1;            // chosen: keys above t, and `eq` of those that are t
    int eq = 0x7fffffff;
    if (all > want) {
        if (forced >= want) {
            t = kForced;
            eq = want;
        } else {
            const uint32_t diff = hi ^ lo;
            int bit = diff ? 31 - __builtin_clz(diff) : -1;
            t = bit >= 31 ? 0u : hi >> (bit + 1) << (bit + 1);
            bool exact = false;
            if constexpr (TEAM > 0) {
                // m: keys from t on
                int m = all, turn = 0;
                for (; bit >= 0 && !exact; bit -= 3, turn = turn == 2 ? 0 : turn + 1) {
                    const int sh = max(bit - 2, 0);
                    uint32_t mine = 0;
#pragma unroll
                    for (int j = 0; j < 7; ++j) {
                        const uint32_t c = (uint32_t)count(t + ((uint32_t)(j + 1) << sh));
                        mine = lane == j ? c : mine;
                    }
                    if (lane < 7) atomicAdd(&room->cnt[turn][lane], mine);
                    __syncthreads();
                    const int c = lane < 7 ? (int)room->cnt[turn][lane] : 0;
                    // (the counts fall from threshold to threshold; those past the remaining bits
                    // count first and last blocks only)
                    const int best = __popcll(__ballot(lane < 7 && c >= want));
                    if (best > 0) {
                        t += (uint32_t)best << sh;
                        m = __builtin_amdgcn_readlane(c, best > 0 ? best - 1 : 0);
                    }
                    exact = m == want;
                    // (read before the last barrier but one, written after the next)
                    if (wave == 0 && lane < 8) room->cnt[turn == 0 ? 2 : turn - 1][lane] = 0;
                }
            } else {
                for (; bit >= 0 && !exact; --bit) {
                    const uint32_t c = t | 1u << bit;
                    const int m = count(c);
                    if (m >= want) t = c;
                    exact = m == want;
                }
            }
            if (!exact) {
                eq = want - count(t + 1);              // (t is below kForced)
                if constexpr (TEAM > 0) {
                    __syncthreads();
                    if (lane == 0) room->over[wave] = (uint32_t)(want - eq);
                    __syncthreads();
                    eq = want - wave_sum(lane < NT ? (int)room->over[lane & (NT - 1)] : 0);
                }
            }
        }
    }
    const uint64_t below = lane ? ~0ull >> (64 - lane) : 0ull;
    int eqs = 0, done = 0;
    if constexpr (TEAM > 0) {
        // what the wavefronts before this one take
        int same = 0, over = 0;
        each([&](int, uint32_t k) {
            same += __popcll(__ballot(k == t && k != 0));
            over += __popcll(__ballot(k > t));
        });
        __syncthreads();
        if (lane == 0) { room->over[wave] = (uint32_t)over; room->same[wave] = (uint32_t)same; }
        __syncthreads();
        const int w = lane & (NT - 1);
        const int o = lane < wave ? (int)room->over[w] : 0, e = lane < wave ? (int)room->same[w] : 0;
        eqs = wave_sum(e);
        done = wave_sum(o) + min(eqs, eq);
    }
    each([&](int i, uint32_t k) {
        const uint64_t same = __ballot(k == t && k != 0);
        const bool take = k != 0 && (k > t || (k == t && eqs + __popcll(same & below) < eq));
        const uint64_t b = __ballot(take);
        if (take) put(done + __popcll(b & below), i);
        eqs += __popcll(same);
        done += __popcll(b);
    });
    return min(all, want);
}
template <class K, class P>
__device__ __forceinline__ int wave_choose(int n, int want, int lane, K key, P put) {
    if (n <= 256) return choose<0, 4>(nullptr, 0, lane, n, want, key, put);
    if (n <= 512) return choose<0, 8>(nullptr, 0, lane, n, want, key, put);
    if (n <= 1024) return choose<0, 16>(nullptr, 0, lane, n, want, key, put);
    return choose<0, 0>(nullptr, 0, lane, n, want, key, put);
}

// the largest over the gp columns of a token, in each of them (gp: 1, 2, 4, 8 or 16 neighbouring lanes)
__device__ __forceinline__ float columns_max(float x, int gp) {
    auto with = [](float y, auto ctl) { return fmaxf(y, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, y), decltype(ctl)::value, 0xF, 0xF, true))); };
    if (gp > 1) x = with(x, std::integral_constant<int, 0xB1>{});     // lane ^ 1
    if (gp > 2) x = with(x, std::integral_constant<int, 0x4E>{});     // lane ^ 2
    if (gp > 4) x = with(x, std::integral_constant<int, 0x141>{});    // the other 4 of 8
    if (gp > 8) x = with(x, std::integral_constant<int, 0x140>{});    // the other 8 of 16
    return x;
}

template <int D, int NW>
__global__ __launch_bounds__(64 * NW) void paged_select_blocks(SelectArgs sa) {
    constexpr int KS = 2 * D / 64, QS = D / 64, U = 2;   // k steps of the product, of a query; steps in flight
    extern __shared__ uint32_t keys[];                // [token][segment]
    __shared__ ChooseRoom room;
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
    const int sb = low_of(p0) + seg * sa.seg, n = max(min(end - sb, sa.seg), 0);   // this segment's
    const int G = a.hq / a.hkv, gp = 1 << sa.gp_log2;

    // the lane's block of steps t0, t0 + NW, ..: its page and place (asked for a round ahead)
    const int col = lane & 15, quad = lane >> 4;
    const int nt = (n + 15) / 16;
    int page[U], place[U];
    auto find = [&](int t0) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int b = max(min(sb + 16 * (t0 + NW * j) + col, end - 1), 0);
            page[j] = nt > 0 ? paged_page(a.b, u.s, b >> bpp) : -1;
            place[j] = b & ((1 << bpp) - 1);
        }
    };
    find(wave);

    // ---- queries in 8 bits: column lane % 16, dims 64 ks + 16 (lane / 16) .. ----------
    const int tk = col >> sa.gp_log2, g0 = col & (gp - 1);
    const int passes = (G + gp - 1) >> sa.gp_log2;
    const int p = p0 + tk, low = low_of(p), last = p >> lg;
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
        // (scores times 2^-32, which leaves their order: with infinities in query and keys they reach 2^150, of the
        // least numbers 2^-94)
        const float f = two_to(-e), fs = valid ? two_to(e - 32) : 0.f;
        intx4 qb[KS];
#pragma unroll
        for (int ks = 0; ks < QS; ++ks)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    r[i] = (uint32_t)(int)__builtin_amdgcn_fmed3f(rintf((float)q[2 * ks + (w >> 1)][4 * (w & 1) + i] * f), -127.f, 127.f);
                const uint32_t lo = __builtin_amdgcn_perm(r[1], r[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(r[3], r[2], 0x04000C0Cu), x = lo | hi;
                // bytes of all ones where a number is below 0
                const uint32_t below = ((x >> 7) & 0x01010101u) * 255u;
                qb[ks][w] = (int)(x & ~below);
                qb[QS + ks][w] = (int)(x & below);
            }
        for (int t0 = wave; t0 < nt; t0 += U * NW) {
            intx4 kb[U][KS];
            float s[U];
            int there[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                there[j] = page[j];
                const char* const src = a.in.b + max(page[j], 0) * a.in.nb3 + hk * a.in.nb2 + place[j] * a.in.nb1 + 16 * quad;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) kb[j][ks] = *(const intx4*)(src + 64 * ks);
                // (no NaN: of some the keys lie so high that the search's thresholds pass 32 bits)
                s[j] = scale_in_range(*(const float*)(a.in.s + max(page[j], 0) * a.in.s_nb3 + hk * a.in.s_nb2 + 4 * (int64_t)place[j]));
            }
            find(t0 + U * NW < nt ? t0 + U * NW : wave);   // (the next pass begins again)
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int t = t0 + NW * j;
                if (t >= nt) break;
                intx4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kb[j][ks], qb[ks], acc, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // block of the result's row, its scale and page from the lane that read it
                    const int r = 4 * quad + i, at = 16 * t + r, bl = sb + at;
                    const float sr = __shfl(s[j], r, 64);
                    const int pr = __shfl(there[j], r, 64);
                    const float y = columns_max(valid ? (float)acc[i] * fs : -INFINITY, gp);
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
    }
    __syncthreads();
    const int want = sa.segs == 1 ? a.top : sa.keep;
    auto lists = [&](int t, auto choice, int lane0, int step) {
        const uint32_t* const key = keys + t * sa.seg;
        const int64_t row = (int64_t)(u.st.q0 + i0 + t) * a.hkv + hk;
        auto get = [&](int i) -> uint32_t { return key[i]; };
        if (sa.segs == 1) {
            int32_t* const out = a.list + row * a.top;
            const int k = choice(get, [&](int r, int i) { out[r] = sb + i; });
            for (int r = k + lane0; r < a.top; r += step) out[r] = -1;
        } else {
            uint2* const out = sa.pairs + (row * sa.segs + seg) * sa.keep;
            const int k = choice(get, [&](int r, int i) { out[r] = uint2{key[i], (uint32_t)(sb + i)}; });
            for (int r = k + lane0; r < sa.keep; r += step) out[r] = uint2{0u, 0u};
        }
    };
    // a wavefront per token, or all of them for one after another
    if (NW < SL_WAVES || n <= 512 || (ntok >= 4 && n <= 1024)) {
        for (int t = wave; t < ntok; t += NW) lists(t, [&](auto get, auto put) { return wave_choose(n, want, lane, get, put); }, lane, 64);
    } else if constexpr (NW == SL_WAVES) {
        for (int t = 0; t < ntok; ++t)
            lists(t, [&](auto get, auto put) { return choose<NW, kSelectSeg / (64 * NW)>(&room, wave, lane, n, want, get, put); }, (int)threadIdx.x, 64 * NW);
    }
}

// Among the segments' best: a workgroup per token and kv head, of one wavefront (up to 1024 pairs) or 16
// (up to 16384; beyond, one of them reads the pairs again and again: 65536 blocks, top 1024 86 us, 69632 1.28 ms).
template <int NW>
__global__ __launch_bounds__(64 * NW) void paged_select_join(SelectArgs sa) {
    __shared__ ChooseRoom room;
    const PagedSelect& a = sa.a;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    if (paged_token(a.b, (int)(row / a.hkv)).s < 0) return;
    const int n = sa.segs * sa.keep;
    const uint2* const in = sa.pairs + row * n;
    int32_t* const out = a.list + row * a.top;
    auto get = [&](int i) -> uint32_t { return in[i].x; };
    auto put = [&](int r, int i) { out[r] = (int32_t)in[i].y; };
    int k;
    if constexpr (NW == 1) {
        k = wave_choose(n, a.top, lane, get, put);
    } else if (n <= 4096) {
        k = choose<NW, 4>(&room, wave, lane, n, a.top, get, put);
    } else if (n <= 16384) {
        k = choose<NW, 16>(&room, wave, lane, n, a.top, get, put);
    } else {
        if (wave > 0) return;
        k = wave_choose(n, a.top, lane, get, put);
        for (int r = k + lane; r < a.top; r += 64) out[r] = -1;
        return;
    }
    for (int r = k + (int)threadIdx.x; r < a.top; r += 64 * NW) out[r] = -1;
}

hipError_t launch_paged_select(const PagedSelect& a, hipStream_t st) {
    if (a.b.tokens <= 0 || a.b.n_streams <= 0 || a.b.max_nq <= 0 || a.hq <= 0) return hipSuccess;
    if (a.d != 128 && a.d != 64) return hipErrorInvalidValue;
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
    const int64_t per = ((int64_t)a.b.max_nq + sa.tiles - 1) / sa.tiles;
    int64_t tiles = (int64_t)a.b.tokens / sa.tiles + a.b.n_streams;
    if (tiles > per * a.b.n_streams) tiles = per * a.b.n_streams;
    if (tiles > a.b.tokens) tiles = a.b.tokens;
    // Few workgroups with many blocks: segments of 128 and more, for up to a workgroup a CU, and no more
    // pairs than one wavefront of the join holds. Whole -> cut, a stream, 8 kv heads of 128: 512
    // blocks 16.1 -> 12.9 us, 2048 32.2 -> 20.9 (segments of 256: 16.1, 19.3), 8192 50 -> 24.9 (with
    // segments of 256 alone, whose pairs the join read again and again, 115); 8 streams of 512 16.1 -> 13.5.
    constexpr int64_t kSeg = 128;
    if (nb >= 4 * kSeg && tiles * a.hkv < 128) {
        int64_t cuts = 256 / (tiles * a.hkv);
        if (cuts > 1024 / a.top) cuts = 1024 / a.top;
        int64_t seg = cuts > 1 ? (nb + cuts - 1) / cuts : nb;
        if (seg < kSeg) seg = kSeg;
        if (seg < most) most = seg;
    }
    sa.segs = (int32_t)((nb + most - 1) / most);
    if (sa.segs < 1) sa.segs = 1;
    sa.seg = (int32_t)(((nb + sa.segs - 1) / sa.segs + 15) / 16 * 16);
    if (sa.seg < 16) sa.seg = 16;
    sa.keep = a.top < sa.seg ? a.top : sa.seg;
    sa.pairs = reinterpret_cast<uint2*>(a.ws);
    if (sa.segs > 1 && (double)a.b.tokens * a.hkv * sa.segs * sa.keep * sizeof(uint2) > (double)a.ws_bytes) return hipErrorOutOfMemory;
    const int64_t grid = tiles * sa.segs * a.hkv, jgrid = (int64_t)a.b.tokens * a.hkv;
    if (grid > kMaxGridX / 4 || (sa.segs > 1 && jgrid > kMaxGridX / 4)) return hipErrorNotSupported;
    const size_t lds = (size_t)sa.tiles * sa.seg * sizeof(uint32_t);
    // (Each wavefront forms all the columns' queries: with several tokens to choose for, 4 of them, 256
    // tokens over 256 blocks 23.6 -> 16.7 us; with one token 16, whose loads are all in flight at once, 512
    // blocks of 32 streams 23.9 -> 18.1.)
    if (sa.tiles >= 4 && sa.seg <= 512) {
        if (a.d == 128) hipLaunchKernelGGL((paged_select_blocks<128, 4>), dim3((unsigned)grid), dim3(256), lds, st, sa);
        else hipLaunchKernelGGL((paged_select_blocks<64, 4>), dim3((unsigned)grid), dim3(256), lds, st, sa);
    } else {
        if (a.d == 128) hipLaunchKernelGGL((paged_select_blocks<128, SL_WAVES>), dim3((unsigned)grid), dim3(64 * SL_WAVES), lds, st, sa);
        else hipLaunchKernelGGL((paged_select_blocks<64, SL_WAVES>), dim3((unsigned)grid), dim3(64 * SL_WAVES), lds, st, sa);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || sa.segs == 1) return e;
    if (sa.segs * sa.keep <= 1024) hipLaunchKernelGGL((paged_select_join<1>), dim3((unsigned)jgrid), dim3(64), 0, st, sa);
    else hipLaunchKernelGGL((paged_select_join<SL_WAVES>), dim3((unsigned)jgrid), dim3(64 * SL_WAVES), 0, st, sa);
    return hipGetLastError();
}

}  // namespace vxfa
