// fa_paged_chunk.h — attention of chunks of new tokens over a paged cache, a
// ragged batch in one launch, for gfx950. (A translation unit per head dim and
// type of the pages: fa_paged_chunk.hip, fa_paged_chunk64.hip; of 8 bits _q8.)
//
// The paged form of fa_prefill_group.hip, whose loop it has: a workgroup of 8
// (hd 64: 4) wavefronts of 32 query rows, the heads of a kv group by as many row
// tiles, shares K/V blocks of 32 rows in a ring of LDS steps filled by
// global_load_lds; P V runs one block behind, so that no MFMA waits for the
// softmax beside it; P is taken against the running maximum, and its sum tells
// when a score has passed that by more than 2^8.
// What differs:
//   Work. Streams have their own lengths, on the device. Every workgroup finds
//   its tile and piece of a tile's rows itself (chunk_locate in fa_paged_plan.h:
//   all lanes weigh a piece length each). Long streams come first, and long
//   tiles within a stream.
//   Rows. A load instruction fills 4 (8) rows, which lie in one 16-row granule
//   and so in one page: its base is a scalar. The granules' pages are read, and
//   their addresses worked out, 64 at a time, a lane each. Absent pages and rows
//   past the stream's last granule read a row of zeros.
//   Scores. MOD 1: with the distance term, two FMAs a score where the plain
//   softmax has one (slope j + (slope (kv0 - p) - m), then c s + that); MOD 2: with
//   a cap, too, MOD 3 with one above kNarrowCap. These walk a tile's blocks from the
//   last: far rows lie lower by the distance, so from the first on the running maximum
//   would rise by more than 2^8 in every block of a steep head, and every block's
//   softmax be done twice.
//   The sum of P is taken in F32 before P is rounded: its logarithm is what the
//   accumulated weights are divided by.
//   hd 64, up to 256 workgroups: two groups of 4 wavefronts, each with half of the
//   piece's blocks and a ring of its own, joined through LDS: alone on its CU a
//   workgroup has one wavefront a SIMD, and the chain of a block's dependent steps
//   takes 0.6 us (600 tokens on 3000 rows, 20 heads: 41.3 -> 35.5 us; with 320
//   workgroups, of which the LDS of a CU holds one at 136 KiB each, 41 -> 50).
// What bounds it, 32/8 heads of 128: 8192 tokens 554-579 us, 0.95-0.99 PFLOP/s (power,
// as fa_prefill_group.hip; matrix pipe busy 49 % of the cycles); with slopes 565,
// with a cap 750-775 (the VALU: exp2 and reciprocal a score more), with a wide one 1060
// (the series beside them). 600 tokens on 3000
// rows 53 us, 3 pieces: 38 blocks of ~0.9 us, ~8 before and after, 7 for the join.
// 16 streams of up to 512 tokens and 4096 rows, half of them single tokens, cap and
// slopes 208-220 us: 416 workgroups of 8 to 128 blocks, one a CU; VALU 56 % busy.
// With a cap the hd 128 kernel takes all 256 VGPRs and spills 6: 28 bytes of scratch
// a lane.
//
// KV8: pages of 8 bits, value = scale[granule] whole number. Whole numbers are exact
// in f16, so the products stay those above, on whole numbers, and the scales are
// applied in F32: K's multiplies the score; V's goes into the exponent, P' = 2^(x +
// log2 s - m), so that f16 rounds P s as it rounds P (by 2^-25 of the largest where
// they lie more than 2^14 below it), and the sum adds P' / s. A step's bytes come by global_load_lds a step ahead into a
// region of their own, and each is turned into f16 once, when the workgroup stores
// the step to the ring (v_perm_b32, one f16 operation for two): in every wavefront's
// fragments it would be done 8 times. The scales of 32 steps' granules lie in a table
// in LDS. With a cap the softmax of a block stands ahead of the next block's S, whose
// registers it then has: 223 VGPRs, no scratch.
// The conversions are VALU work beside MFMAs, and the stores of the ring meet bank
// conflicts (8 cycles a store of 16 bytes a lane; storing the two halves in turn by row
// changed neither the count nor the time). Graph, F16 -> 8 bits on one card: 8192 tokens 574-582 -> 605-610 us
// (0.91 PFLOP/s), 600 on 3000 rows 55.7 -> 57, 100 on 8192 44 -> 39; the mixed batch above
// 264 -> 300 on one set of lengths (215 on the shortest); 2000 on 4000 with a cap 181 ->
// 203, wide 261 -> 270; hd 64, 4000 tokens 72 -> 83. Raw numbers in registers instead of LDS:
// spills of 4 to 42; five steps ahead with a ring of three slots 581 -> 591; the reciprocal
// scale read again at its use 605 -> 619.
#pragma once

#include "fa_paged_plan.h"
#include "fa_paged_q8.h"

#include <type_traits>

namespace vxfa {

template <int HD, int KVGROUPS = 1>
struct PC {
    static constexpr int D = HD;
    static constexpr int KS = D / 16;             // S-MFMA k-steps
    static constexpr int DB = D / 32;             // O^T row blocks
    static constexpr int BK = 32;                 // rows per block
    static constexpr int ROW = D * 2;             // bytes per K/V row
    static constexpr int BLK = BK * ROW;          // bytes of one matrix block
    static constexpr int STEP = 2 * BLK;          // one matrix of a 64-row step
    static constexpr int NS = 4;                  // ring slots
    static constexpr int NW = D / 16;             // wavefronts of 32 query rows (8 or 4)
    static constexpr int KVG = KVGROUPS;          // groups of them, each with its share of the blocks
    static constexpr int NT = 64 * NW * KVG;
    static constexpr int RECO = 64 * 16 * DB;     // floats of O in a wavefront's record
    static constexpr int REC = RECO + 64;         // and (m, l) of 32 rows
};
constexpr float PC_TAU_SUM = 256.0f;              // 2^8

struct ChunkArgs {
    PagedAttn a;
    ChunkPlan p;
    float* rec;                // records [head group][slot][wavefront]
    ChunkTile* tiles;          // what the joining launch needs of every tile; [0].s: their number first
    int32_t nhg;
    PagedScales sc;            // of pages of 8 bits
};

static __device__ const char pc_zeros[256] = {0};

template <int N>
__device__ __forceinline__ void pc_wait_vm() {
    static_assert(N >= 0 && N < 16, "vmcnt range");
    __builtin_amdgcn_s_waitcnt(N | (7 << 4) | (15 << 8));
}

// MOD: 1 the scores have a distance term, 2 a cap (and a slope, or 0), 3 a wide one. QF16: q is F16.
// KV8: pages of 8 bits.
template <int HD, int KVGROUPS, bool QF16, int MOD, bool KV8>
static __global__ __launch_bounds__((PC<HD, KVGROUPS>::NT), 2) void paged_chunk_kernel(ChunkArgs ca) {
    using P = PC<HD, KVGROUPS>;
    constexpr int D = P::D, KS = P::KS, DB = P::DB, BK = P::BK, ROW = P::ROW, BLK = P::BLK, STEP = P::STEP, NS = P::NS,
                  NW = P::NW, REC = P::REC;
    // K steps, V steps, and with 8 wavefronts half of the Q staging. The first block
    // past the ring is zeros from step 0 on: V of a block dead for a wavefront's rows.
    constexpr int ZERO = 2 * NS * STEP, KVG = P::KVG;
    // KV8: the whole numbers of a step, and the scales of 32 steps' granules
    constexpr int RAW = ZERO + BLK, TAB = RAW + 2 * NW * 1024;
    constexpr int REGION = KV8 ? TAB + 2048 : ZERO + (NW == 8 ? 4 : 1) * BLK;     // a group's
    constexpr bool REV = MOD != 0;                        // blocks from the last
    __shared__ __attribute__((aligned(16))) char smem_all[KVG * REGION];

    const PagedAttn& a = ca.a;
    const int tid = (int)threadIdx.x;
    const int lane = tid & 63;
    const int grp = KVG == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6) / NW;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) - grp * NW;
    char* const smem = smem_all + grp * REGION;
    const int hg = (int)blockIdx.x % ca.nhg;
    const int item = (int)blockIdx.x / ca.nhg;
    const int hpw = 1 << ca.p.hpw_log2;
    const int bm = 32 * (NW >> ca.p.hpw_log2);            // positions per workgroup
    const ChunkItem it = chunk_locate(a.b, ca.p, a.window, bm, item);
    if (hg == 0 && tid == 0) {
        if (item == 0) ca.tiles[0].s = it.tiles;
        if (it.s >= 0 && it.piece == 0) ca.tiles[1 + it.tile_no] = ChunkTile{it.s, it.tile, it.n, it.slot};
    }
    if (it.s < 0) return;
    const PagedStream st = it.st;
    const int nq = min(st.t, a.b.max_nq);
    const int past = st.n - st.t;                         // token i lies in row past + i
    const int h = hg * hpw + (wave & (hpw - 1));
    const int hk = hg * hpw / (a.hq / a.hkv);
    const int q0 = it.tile * bm;                          // the workgroup's first token
    const int r0 = q0 + 32 * (wave >> ca.p.hpw_log2);     // the wavefront's
    const int nl = lane & 31, hh = lane >> 5;
    const int qrow = r0 + nl;
    const bool qvalid = qrow < nq;
    const bool active = r0 < nq;
    const int qld = min(qrow, nq - 1);

    // ---- rows that the lane's token sees, the workgroup's, this piece's blocks ---
    const int prow = past + qld;
    const int rlo = a.window > 0 ? max(prow - a.window + 1, 0) : 0;
    const int lo = a.window > 0 ? max(past + q0 - a.window + 1, 0) : 0;
    const int hi = max(past + min(q0 + bm, nq), 0);       // (n at most)
    const int blo = lo / BK;
    const int nblk = hi > lo ? (hi + BK - 1) / BK - blo : 0;
    int bs = blo, nb = nblk;
    if (it.n > 1) {
        const int len = ((nblk + it.n - 1) / it.n + 1) & ~1;   // whole steps
        bs = blo + min(it.piece * len, nblk);
        nb = min(len, blo + nblk - bs);
    }
    // the group's share: whole steps, the first group's the longer
    int steps = (nb + 1) >> 1;                            // of the first group
    if constexpr (KVG == 2) {
        const int n0 = min(((nb + 1) / 2 + 1) & ~1, nb);
        steps = (n0 + 1) >> 1;
        bs += grp ? n0 : 0;
        nb = grp ? nb - n0 : n0;
    }

    // ---- Q loads: whole rows of the wavefront's 32, through LDS below -------------
    constexpr int QL = QF16 ? KS : 2 * KS;           // 16-byte loads per lane
    constexpr int QCH = QF16 ? D / 8 : D / 4;        // 16-byte chunks per row
    floatx4 qraw[QL];
    {
        const char* qp = (const char*)a.q + (int64_t)h * a.q_nb2 + (int64_t)st.q0 * a.q_nb1;
#pragma unroll
        for (int u = 0; u < QL; ++u) {
            const int row = min(r0 + (64 / QCH) * u + lane / QCH, nq - 1);
            qraw[u] = __builtin_nontemporal_load((const floatx4*)(qp + (int64_t)row * a.q_nb1) + lane % QCH);
        }
    }

    // ---- step loads: global -> LDS ring ----------------------------------------
    // Instruction i (0, 1) of wavefront w fills rows [RPI (w + NW i), + RPI) of
    // the step; lane l writes LDS chunk l % CH of row + l / CH, which holds the
    // row's chunk (l % CH) ^ swizzle(row).
    constexpr int CH = D / 8, RPI = 64 / CH;
    static_assert(2 * NW * RPI == 2 * BK && 16 % RPI == 0, "two instructions per matrix and step, rows of a granule");
    const int nstep = (nb + 1) >> 1;
    const int lg = a.b.ps_log2;
    // (step u and block t count in the order of the walk)
    auto step_row = [&](int u) -> int { return (bs + 2 * (REV ? nstep - 1 - u : u)) * BK; };
    auto block_row = [&](int t) -> int { return step_row(t >> 1) + (REV ? 1 - (t & 1) : t & 1) * BK; };
    auto block_lds = [&](int t) -> int { return (REV ? (t ^ 1) : t) & (2 * NS - 1); };
    // lane l: where granule l of the 16 steps from ids_from on lies from K's and V's
    // bases (the page's part worked out here, 64 lanes at once: the products on the
    // scalar unit cost every wavefront 6 % of its issue slots); bit l of `there`: it is
    // there (and of the 16 steps before, which may not all be computed yet)
    int64_t offs = -1;
    int ids_from = 0;
    uint64_t there = 0, there_before = 0;
    floatx4 scales = {1.f, 0.f, 1.f, 0.f};                // KV8: of the lane's granule K's, log2 of V's, 1 / V's
    auto load_ids = [&](int u0) {
        const int u = u0 + (lane >> 2), row = step_row(u) + 16 * (lane & 3);
        const int p = u < nstep && row < st.n ? paged_page(a.b, it.s, row >> lg) : -1;
        offs = p >= 0 ? a.kv.at(p, hk, row & ((1 << lg) - 1)) : -1;
        if constexpr (KV8) {
            scales = floatx4{1.f, 0.f, 1.f, 0.f};
            if (wave == NW - 1 && p >= 0) {
                const int64_t at = ca.sc.at(p, hk, row & ((1 << lg) - 1));
                const float sv = scale_in_range(*(const float*)(ca.sc.v + at));
                scales = floatx4{scale_in_range(*(const float*)(ca.sc.k + at)), __builtin_amdgcn_logf(sv), __builtin_amdgcn_rcpf(sv), 0.f};
            }
        }
        there_before = there;
        there = __ballot(p >= 0);
        ids_from = u0;
    };
    // (written by the last wavefront, 3 steps ahead of their use; the half that is
    // overwritten was of the 16 steps before the last 16)
    auto put_scales = [&](int u0) {
        if constexpr (KV8)
            if (wave == NW - 1) *(floatx4*)(smem + TAB + 1024 * ((u0 >> 4) & 1) + 16 * lane) = scales;
    };
    const uint32_t lds0 = lds_offset(smem);
    const int lrow = lane / CH;
    uint32_t ldk[2], ldv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = RPI * (wave + NW * i) + lrow;
        ldk[i] = (uint32_t)(r & 15) * (uint32_t)a.kv.nb1 + ((lane % CH) ^ swz_k<D>(r)) * 16;
        ldv[i] = (uint32_t)(r & 15) * (uint32_t)a.kv.nb1 + ((lane % CH) ^ swz_v<D>(r)) * 16;
    }
    auto issue = [&](int u) {
        if ((u & 15) == 0) load_ids(u);
        const int kv0 = step_row(u);
        const uint32_t kd = lds0 + (u & (NS - 1)) * STEP, vd = kd + NS * STEP;
        const char *kp[2], *vp[2];
        bool plain = kv0 + 2 * BK <= st.n;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int g = 4 * (u & 15) + RPI * (wave + NW * i) / 16;
            const int lo = __builtin_amdgcn_readlane((int)(uint32_t)offs, g), hi = __builtin_amdgcn_readlane((int)(offs >> 32), g);
            const int64_t at = ((int64_t)hi << 32) | (uint32_t)lo;
            plain = plain && hi >= 0;
            kp[i] = a.kv.k + at;
            vp[i] = a.kv.v + at;
        }
        if (plain) {
#pragma unroll
            for (int i = 0; i < 2; ++i) dma16(kp[i], ldk[i], kd + RPI * (wave + NW * i) * ROW);
#pragma unroll
            for (int i = 0; i < 2; ++i) dma16(vp[i], ldv[i], vd + RPI * (wave + NW * i) * ROW);
        } else {
            // rows of zeros in place of an absent granule and behind the last row, whose
            // own instruction reads it for those behind it (worked out here rather than
            // held across the loop; the empty asm keeps it here)
            int ln = lane;
            asm volatile("" : "+v"(ln));
            uint32_t ok[2], ov[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int rs = RPI * (wave + NW * i), r = rs + ln / CH;
                ok[i] = ((ln % CH) ^ swz_k<D>(r)) * 16;
                ov[i] = ((ln % CH) ^ swz_v<D>(r)) * 16;
                if (__builtin_amdgcn_readlane((int)(offs >> 32), 4 * (u & 15) + rs / 16) < 0 || kv0 + rs >= st.n) {
                    kp[i] = vp[i] = pc_zeros;
                } else {
                    const uint32_t rr = (uint32_t)min(r & 15, (st.n - 1 - kv0) - (rs & ~15)) * (uint32_t)a.kv.nb1;
                    ok[i] += rr;
                    ov[i] += rr;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) dma16(kp[i], ok[i], kd + RPI * (wave + NW * i) * ROW);
#pragma unroll
            for (int i = 0; i < 2; ++i) dma16(vp[i], ov[i], vd + RPI * (wave + NW * i) * ROW);
        }
    };
    // KV8: a lane's 16 bytes of K and V of a step (a row has CH / 2 lanes) go to LDS as they are,
    // and a step later through its registers to the ring as f16: converted once, not
    // by each wavefront that reads them. (Kept in registers for that step they cost 4 to 20 spills; five steps ahead
    // in LDS, with a ring of three slots, 8192 tokens took 591 us instead of 581.)
    constexpr int CH8 = D / 16, RPW = 64 / CH8;
    static_assert(NW * RPW == 2 * BK && (16 % RPW == 0), "a wavefront's rows lie in one granule");
    const uint32_t raw0 = RAW + 2048 * wave;
    struct Raw {
        u32x4 k, v;
    };
    // where the wavefront's rows of step u lie (absent: zeros, all rows the same ones)
    auto find8 = [&](int u, const char*& kp, const char*& vp) -> uint32_t {
        if ((u & 15) == 0) {
            load_ids(u);
            if (u > 0) put_scales(u);
        }
        const int g = 4 * (u & 15) + RPW * wave / 16;
        const int lo = __builtin_amdgcn_readlane((int)(uint32_t)offs, g), hi = __builtin_amdgcn_readlane((int)(offs >> 32), g);
        const int64_t at = ((int64_t)hi << 32) | (uint32_t)lo;
        kp = hi < 0 ? pc_zeros : a.kv.k + at;
        vp = hi < 0 ? pc_zeros : a.kv.v + at;
        int ln = lane;
        asm volatile("" : "+v"(ln));                      // (worked out here rather than held across the loop)
        return ((uint32_t)(RPW * wave + ln / CH8) & (hi < 0 ? 0u : 15u)) * (uint32_t)a.kv.nb1 + 16 * (ln % CH8);
    };
    auto load8 = [&](int u, Raw& w) {
        const char *kp, *vp;
        const uint32_t off = find8(u, kp, vp);
        w.k = *(const u32x4*)(kp + off);
        w.v = *(const u32x4*)(vp + off);
    };
    auto issue8 = [&](int u) {
        const char *kp, *vp;
        const uint32_t off = find8(u, kp, vp);
        dma16(kp, off, lds0 + raw0);
        dma16(vp, off, lds0 + raw0 + 1024);
    };
    auto store8 = [&](int u, const Raw& w) {
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int r = RPW * wave + ln / CH8, j = 2 * (ln % CH8);
        char* const kd = smem + (u & (NS - 1)) * STEP + r * ROW;
        char* const vd = kd + NS * STEP;
#pragma unroll
        for (int i = 0; i < 2; ++i) *(half8*)(kd + (((j + i) ^ swz_k<D>(r)) * 16)) = half8_of_bytes(w.k[2 * i], w.k[2 * i + 1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) *(half8*)(vd + (((j + i) ^ swz_v<D>(r)) * 16)) = half8_of_bytes(w.v[2 * i], w.v[2 * i + 1]);
    };
    Raw first0, first1;
    if constexpr (KV8) {
        if (nstep > 0) load8(0, first0);
        if (nstep > 1) load8(1, first1);
        if (nstep > 2) issue8(2);
    } else {
        for (int u = 0; u < min(nstep, 2); ++u) issue(u);
    }

    // ---- Q operand: row qrow, dims 16 ks + 8 hh .. + 7, in f16; the sign of the
    // scale folded in (0 for scale 0) -----------------------------------------------
    const float c = a.c != 0.f ? fabsf(a.c) : 1.0f;
    half8 qb[KS];
    {
        const float sg = a.c < 0.f ? -1.0f : (a.c > 0.f ? 1.0f : 0.0f);
        // 16-byte chunk j of row r at j ^ (r % CH); wavefronts 0-3 in ring slot 3
        // (filled from step 0 on), 4-7 past the ring (KV8: in slot 2, which is, too)
        const int w2 = wave & 1, slot = KV8 && wave >= 4 ? 2 : 3;
        char* qs = smem + (wave >= 4 && !KV8 ? 2 * NS * STEP + (wave - 4) * BLK : ((wave & 2) ? NS + slot : slot) * STEP + w2 * BLK);
#pragma unroll
        for (int u = 0; u < QL; ++u) {
            const int r = (64 / QCH) * u + lane / QCH, j = lane % QCH;
            if constexpr (QF16) {
                *(half8*)(qs + r * ROW + ((j ^ (r % CH)) * 16)) = __builtin_bit_cast(half8, qraw[u]) * (_Float16)sg;
            } else {
                half4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (_Float16)(qraw[u][e] * sg);
                *(half4*)(qs + r * ROW + (((j >> 1) ^ (r % CH)) * 16) + (j & 1) * 8) = y;
            }
        }
        __builtin_amdgcn_wave_barrier();   // (one wavefront's LDS accesses run in order)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qb[ks] = *(const half8*)(qs + nl * ROW + (((2 * ks + hh) ^ (nl % CH)) * 16));
        __builtin_amdgcn_wave_barrier();
    }
    if constexpr (KV8) {
        put_scales(0);
        if (nstep > 0) store8(0, first0);
        if (nstep > 1) store8(1, first1);
    }
    // the block of zeros (past the ring: by the wavefront whose rows it held)
    if constexpr (NW == 8) {
        if (wave == 4) {
#pragma unroll
            for (int i = 0; i < BLK / 1024; ++i) *(half8*)(smem + ZERO + 1024 * i + 16 * lane) = half8{};
        }
    } else {
        static_assert(NW == 8 || BLK == 16 * 64 * NW, "one 16-byte store per thread of the group");
        *(half8*)(smem + ZERO + 16 * (64 * wave + lane)) = half8{};
    }

    // ---- operand reads (layouts of fa_prefill.hip) ----------------------------------
    int kbase;
    {
        const int am = nl >> 3, ahb = (nl >> 2) & 1, ab = nl & 3;
        const int krow = ahb ? 16 + ((am + 2) & 3) * 4 + ab : 4 * am + ab;
        kbase = krow * ROW + (hh ^ swz_k<D>(krow)) * 16;
    }
    int vbase;
    {
        const int vq = (lane & 15) >> 2;
        const int clo = 2 * ((lane & 31) >> 4) + ((lane & 3) >> 1);
        vbase = NS * STEP + ((hh ? 24 : 0) + vq) * ROW + (clo ^ swz_v<D>(vq)) * 16 + (lane & 1) * 8;
    }
    auto read_k = [&](int t, half8 (&kr)[KS]) {
        const int base = kbase + block_lds(t) * BLK;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kr[ks] = *(const half8*)(smem + (base ^ (32 * ks)));
    };
    auto read_v = [&](int at, half8 (&vr)[2][DB]) {
        const int base = vbase + at;
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const char* p = smem + (base ^ (8 * ROW * cc + 64 * db));
                const half4 lo4 = lds_read_tr16(p);
                const half4 hi4 = lds_read_tr16(p + 4 * ROW);
                vr[cc][db] = half8{lo4[0], lo4[1], lo4[2], lo4[3], hi4[0], hi4[1], hi4[2], hi4[3]};
            }
    };
    auto s_mfma = [&](floatx16& s, const half8 (&kr)[KS]) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[0], qb[0], floatx16{}, 0, 0, 0);
#pragma unroll
        for (int ks = 1; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[ks], qb[ks], s, 0, 0, 0);
    };
    floatx16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = floatx16{};
    auto pv_mfma = [&](const half8 (&p)[2], const half8 (&vr)[2][DB]) {
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vr[cc][db], p[cc], o[db], 0, 0, 0);
    };

    // ---- masks ------------------------------------------------------------------
    const int last = min(st.n, (bs + nb) * BK) - 1;       // this piece's last row
    const int rhi = min(prow, last);
    // a block inside [hlo, hhi] is seen whole by the wavefront's tokens, one
    // outside [dlo, dhi] by none
    const int hlo = __builtin_amdgcn_readlane(rlo, 31), hhi = __builtin_amdgcn_readlane(rhi, 0);
    const int dlo = __builtin_amdgcn_readlane(rlo, 0), dhi = __builtin_amdgcn_readlane(rhi, 31);
    // (masked: the wavefront's tokens do not see all of the block; returns where its
    // V is read: the zeros when no token of the wavefront sees any, as P x V has
    // to be 0 there whatever V holds)
    bool masked = false, gone = false;                    // gone: the lane's granule of the block is absent
    auto mask_test = [&](int t) -> int {
        const int kv0 = block_row(t), u = t >> 1;
        const uint32_t here = (uint32_t)((u >= ids_from ? there : there_before) >> (4 * (u & 15) + 2 * (REV ? 1 - (t & 1) : t & 1))) & 3u;
        masked = !(kv0 >= hlo && kv0 + BK - 1 <= hhi && here == 3u);
        gone = !((here >> hh) & 1);                       // (a lane's 16 rows are one granule)
        if (kv0 > dhi || kv0 + BK <= dlo || here == 0) return ZERO - NS * STEP;
        return block_lds(t) * BLK;
    };
    auto dead = [&](int t, int j) -> bool {
        const int kv = block_row(t) + pf_kv_of(hh, j);
        return gone || kv < rlo || kv > rhi;
    };

    // ---- softmax ------------------------------------------------------------------
    // P = 2^(x - m), x the score in log2 units: c s; MOD 1: c s + slope (j - p);
    // MOD 2: cap - 2 cap / (1 + 2^(c s)) + slope (j - p); MOD 3: paged_wide_cap of c s + slope (j - p)
    const float slope = MOD ? __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, paged_slope(a, h)))) : 0.f;
    float m = -INFINITY, l = 0.f;
    // KV8: the block's scales for the lane's granule: K's times c; log2 of V's, which is added to the
    // scores (P are then the weights of whole numbers, and rounded as such);
    // 1 / V's, which the sum of P takes back
    float cs = c, lsv = 0.f, isv = 1.f;
    auto scales_of = [&](int t) {
        if constexpr (KV8) {
            const int u = t >> 1;
            const floatx4 x = *(const floatx4*)(smem + TAB + 1024 * ((u >> 4) & 1) + 16 * (4 * (u & 15) + 2 * (REV ? 1 - (t & 1) : t & 1) + hh));
            cs = c * x[0];
            lsv = x[1];
            isv = x[2];
        }
    };
    // element j of block t, plus `base`
    auto terms = [&](int t, float base, float (&e)[2]) {
        if constexpr (KV8) base += lsv;
        if constexpr (MOD == 0) {
            e[0] = e[1] = base;
        } else {
            const int d0 = block_row(t) - prow;
            if constexpr (MOD == 2) base += a.cap;
            e[0] = fmaf(slope, (float)(d0 + (hh ? 24 : 0)), base);
            e[1] = fmaf(slope, (float)(d0 + (hh ? 8 : 0) + (KV8 ? 8 : 0)), base);   // (KV8: of element 8, not 0)
        }
    };
    auto score = [&](float s, const float (&e)[2], int j) -> float {
        if constexpr (MOD == 0) return fmaf(s, cs, e[0]);
        float tj;
        if constexpr (KV8) {
            // (multiples that are constants of the instruction: 3, 5, 6 and 7 would each take a register)
            const float e4 = (j & 7) < 3 ? e[j >> 3] : fmaf(slope, 4.f, e[j >> 3]), e8 = (j & 7) < 7 ? e4 : fmaf(slope, 4.f, e4);
            constexpr float f[8] = {0.f, 1.f, 2.f, -1.f, 0.f, 1.f, 2.f, -1.f};
            tj = f[j & 7] == 0.f ? e4 : fmaf(slope, f[j & 7], e8);
        } else {
            tj = fmaf(slope, (float)j, e[j >> 3]);
        }
        if constexpr (MOD == 1) return fmaf(s, cs, tj);
        if constexpr (MOD == 3) return paged_wide_cap(s * cs, a.cap, a.capk) + tj;
        return fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(1.f + exp2_fast(s * cs)), tj);
    };
    // a few scores at a time: with all 16 in flight the registers do not do
    auto few = [](int j) {
        if (MOD >= 2 ? (j & 3) == 3 : MOD == 1 && (j & 7) == 7) __builtin_amdgcn_sched_barrier(0x3FC);   // VALU may not cross
    };
    auto exps = [&](const floatx16& sc, half8 (&p)[2], int t) -> float {
        float nm = (m == -INFINITY) ? 0.f : -m;
        asm("" : "+v"(nm));
        float e[2], ls[4] = {0.f, 0.f, 0.f, 0.f};
        terms(t, nm, e);
        auto all = [&](auto with_mask) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                float y = exp2_fast(score(sc[j], e, j));
                if constexpr (decltype(with_mask)::value) y = dead(t, j) ? 0.f : y;
                ls[j & 3] += y;
                p[j >> 3][j & 7] = (_Float16)y;
                few(j);
            }
        };
        // (MOD 0 and 1: a removed score is -inf already)
        if (MOD >= 2 && masked) all(std::true_type{});
        else all(std::false_type{});
        return (ls[0] + ls[1]) + (ls[2] + ls[3]);
    };
    auto block_max = [&](const floatx16& sc, int t) -> float {
        float e[2], r = -INFINITY;
        terms(t, 0.f, e);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float x = score(sc[j], e, j);
            r = fmaxf(r, MOD >= 2 && dead(t, j) ? -INFINITY : x);
            few(j);
        }
        return pair32_max(r);
    };
    auto mask_fix = [&](floatx16& sc, int t) {
        if (MOD < 2 && masked) {
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[j] = dead(t, j) ? -INFINITY : sc[j];
        }
    };
    auto raise = [&](float mx) {
        const float mnew = fmaxf(m, mx);
        const float ms = (mnew == -INFINITY) ? 0.f : mnew;
        const float alpha = exp2_fast(m - ms);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[db][j] *= alpha;
        l *= alpha;
        m = mnew;
    };
    // (a row that has seen no score yet takes the exact path; rows past the chunk
    // take no part in the choice)
    auto softmax = [&](const floatx16& sc, half8 (&p)[2], int t) {
        float ls = exps(sc, p, t);
        const bool up = (!(ls <= PC_TAU_SUM) || m == -INFINITY) && qvalid;
        if (__any(up)) {
            raise(block_max(sc, t));
            ls = exps(sc, p, t);
        }
        l = KV8 ? fmaf(ls, isv, l) : l + ls;
    };

    // before step 0: steps 0 and 1 (step 2's loads may stay in flight)
    if constexpr (!KV8) {
        if (nstep > 2) {
            issue(2);
            pc_wait_vm<4>();
        } else {
            pc_wait_vm<0>();
        }
    }
    __syncthreads();

    {
        half8 kr[KS], vr[2][DB], pa[2], pb[2];
        floatx16 sa, sb;
        // PV of the block before the first adds zero
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
            pb[cc] = half8{};
#pragma unroll
            for (int db = 0; db < DB; ++db) vr[cc][db] = half8{};
        }
        if (nb > 0) {
            read_k(0, kr);
            s_mfma(sa, kr);
            scales_of(0);
            mask_test(0);
            mask_fix(sa, 0);
            m = block_max(sa, 0);
        }
        // half t: PV(t - 1), S(t + 1) and the softmax of S(t)
        auto half = [&](int t, floatx16& scur, floatx16& snext, half8 (&pcur)[2], half8 (&pprev)[2]) {
            const int va = mask_test(t);
            scales_of(t);
            mask_fix(scur, t);
            if constexpr (KV8 && MOD >= 2) {
                // (a cap's softmax takes the registers: S(t + 1) after it)
                pv_mfma(pprev, vr);
                softmax(scur, pcur, t);
                __builtin_amdgcn_sched_barrier(0);
                read_v(va, vr);
                read_k(t + 1, kr);
                s_mfma(snext, kr);
                return;
            }
            read_k(t + 1, kr);
            pv_mfma(pprev, vr);
            __builtin_amdgcn_sched_barrier(0x6);   // VALU and SALU may cross
            read_v(va, vr);
            s_mfma(snext, kr);
            softmax(scur, pcur, t);
        };
        // (whole steps: a second block past nb has no live score, and the last
        // half's S is not used)
        for (int u = 0; u < (KVG == 1 ? nstep : steps); ++u) {
            if constexpr (KV8) {
                // (step u - 2 had the slot, and has been read)
                if (u + 2 < nstep) {
                    pc_wait_vm<0>();
                    asm volatile("" ::: "memory");
                    Raw w;
                    w.k = *(const u32x4*)(smem + raw0 + 16 * lane);
                    w.v = *(const u32x4*)(smem + raw0 + 1024 + 16 * lane);
                    store8(u + 2, w);
                    // (the whole numbers have been read: the next ones may come)
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    if (u + 3 < nstep) issue8(u + 3);
                }
                __builtin_amdgcn_sched_barrier(0);
            } else {
                if (u + NS - 1 < nstep) issue(u + NS - 1);
            }
            if (active && (KVG == 1 || u < nstep)) {
                half(2 * u, sa, sb, pa, pb);
                half(2 * u + 1, sb, sa, pb, pa);
            }
            // K of step u + 2 and V of step u + 1 have landed: at most the
            // loads of step u + 3 and V of step u + 2 are in flight
            if constexpr (!KV8) {
                if (u + 3 < nstep) pc_wait_vm<6>();
                else if (u + 2 < nstep) pc_wait_vm<2>();
                else pc_wait_vm<0>();
            }
            __syncthreads();
        }
        if (nb > 0) pv_mfma(pb, vr);
    }

    // ---- output, or this piece's record --------------------------------------------
    float lt = pair32_sum(l);
    if constexpr (KVG == 2) {
        // the second group's O, m and l through LDS (its ring has been read)
        static_assert(KVG == 1 || NW * 64 * (16 * DB + 2) * 4 <= REGION, "the join's room");
        float* const x = reinterpret_cast<float*>(smem_all) + wave * 64 * (16 * DB + 2);
        __syncthreads();
        if (grp == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int a4 = 0; a4 < 4; ++a4)
                    *(floatx4*)(x + (4 * db + a4) * 256 + 4 * lane) =
                        floatx4{o[db][4 * a4], o[db][4 * a4 + 1], o[db][4 * a4 + 2], o[db][4 * a4 + 3]};
            *(float2*)(x + 64 * 16 * DB + 2 * lane) = float2{m, lt};
        }
        __syncthreads();
        if (grp == 1) return;
        const float2 ml = *(const float2*)(x + 64 * 16 * DB + 2 * lane);
        const float mn = fmaxf(m, ml.x), ms = mn == -INFINITY ? 0.f : mn;
        const float w0 = exp2_fast(m - ms), w1 = exp2_fast(ml.x - ms);
        m = mn;
        lt = lt * w0 + ml.y * w1;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int a4 = 0; a4 < 4; ++a4) {
                const floatx4 y = *(const floatx4*)(x + (4 * db + a4) * 256 + 4 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[db][4 * a4 + e] = fmaf(y[e], w1, o[db][4 * a4 + e] * w0);
            }
    }
    if (it.n == 1) {
        const float inv = (lt == 0.f) ? 0.f : 1.0f / lt;
        if (qvalid) {
            const int64_t row = (int64_t)(st.q0 + qrow) * a.hq + h;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int a4 = 0; a4 < 4; ++a4)
                    paged_store4(a, row * D + 32 * db + 8 * a4 + 4 * hh,
                                 floatx4{o[db][4 * a4] * inv, o[db][4 * a4 + 1] * inv, o[db][4 * a4 + 2] * inv,
                                         o[db][4 * a4 + 3] * inv});
            if (a.lse && hh == 0) a.lse[row] = lt == 0.f ? INFINITY : m + log2f(lt);
        }
    } else if (active) {
        float* rec = ca.rec + (((int64_t)hg * ca.p.room + it.slot + it.piece) * NW + wave) * REC;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int a4 = 0; a4 < 4; ++a4)
                *(floatx4*)(rec + (4 * db + a4) * 256 + 4 * lane) =
                    floatx4{o[db][4 * a4], o[db][4 * a4 + 1], o[db][4 * a4 + 2], o[db][4 * a4 + 3]};
        if (hh == 0) *(float2*)(rec + P::RECO + 2 * nl) = float2{m, lt};
    }
}

// Joins the pieces of a tile in order: a wavefront per 32 output dims of a
// wavefront's tile, four records' loads in flight.
template <int HD>
static __global__ __launch_bounds__(64 * PC<HD>::DB) void paged_chunk_combine(ChunkArgs ca) {
    using P = PC<HD>;
    constexpr int D = P::D, NW = P::NW, REC = P::REC, UP = 4;
    const PagedAttn& a = ca.a;
    const int lane = (int)threadIdx.x & 63, db = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int nl = lane & 31, hh = lane >> 5;
    const int hg = (int)blockIdx.x % ca.nhg, wt = (int)blockIdx.x / ca.nhg;
    const int tile_no = wt / NW, wave = wt % NW;
    if (tile_no >= ca.tiles[0].s) return;
    const ChunkTile tl = ca.tiles[1 + tile_no];
    if (tl.n <= 1) return;
    const PagedStream st = paged_stream(a.b, tl.s);
    const int nq = min(st.t, a.b.max_nq);
    const int hpw = 1 << ca.p.hpw_log2;
    const int h = hg * hpw + (wave & (hpw - 1));
    const int r0 = tl.tile * 32 * (NW >> ca.p.hpw_log2) + 32 * (wave >> ca.p.hpw_log2);
    if (r0 >= nq) return;
    const float* rec = ca.rec + (((int64_t)hg * ca.p.room + tl.slot) * NW + wave) * REC;
    const int64_t stride = (int64_t)NW * REC;
    float M = -INFINITY, L = 0.f;
    floatx4 acc[4];
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) acc[a4] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < tl.n; p0 += UP) {
        float2 ml[UP];
        floatx4 v[UP][4];
#pragma unroll
        for (int i = 0; i < UP; ++i) {
            const float* r = rec + min(p0 + i, tl.n - 1) * stride;
            ml[i] = *(const float2*)(r + P::RECO + 2 * nl);
#pragma unroll
            for (int a4 = 0; a4 < 4; ++a4) v[i][a4] = *(const floatx4*)(r + (4 * db + a4) * 256 + 4 * lane);
        }
        float mn = M;
#pragma unroll
        for (int i = 0; i < UP; ++i) {
            if (p0 + i >= tl.n) ml[i] = float2{-INFINITY, 0.f};
            mn = fmaxf(mn, ml[i].x);
        }
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float al = exp2_fast(M - ms);
        L *= al;
#pragma unroll
        for (int a4 = 0; a4 < 4; ++a4) acc[a4] *= al;
#pragma unroll
        for (int i = 0; i < UP; ++i) {
            const float w = exp2_fast(ml[i].x - ms);
            L = fmaf(w, ml[i].y, L);
            if (p0 + i < tl.n) {
#pragma unroll
                for (int a4 = 0; a4 < 4; ++a4)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[a4][e] = fmaf(w, v[i][a4][e], acc[a4][e]);
            }
        }
        M = mn;
    }
    const int qrow = r0 + nl;
    if (qrow >= nq) return;
    const int64_t row = (int64_t)(st.q0 + qrow) * a.hq + h;
    const float inv = (L == 0.f) ? 0.f : 1.0f / L;
#pragma unroll
    for (int a4 = 0; a4 < 4; ++a4) paged_store4(a, row * D + 32 * db + 8 * a4 + 4 * hh, acc[a4] * inv);
    if (a.lse && db == 0 && hh == 0) a.lse[row] = L == 0.f ? INFINITY : M + log2f(L);
}

template <int HD, int KVG, bool QF16, bool KV8>
static void launch_pc(const ChunkArgs& ca, unsigned nwg, hipStream_t st) {
    const dim3 grid(nwg), block(PC<HD, KVG>::NT);
    if (ca.a.capk != 0.f) hipLaunchKernelGGL((paged_chunk_kernel<HD, KVG, QF16, 3, KV8>), grid, block, 0, st, ca);
    else if (ca.a.cap != 0.f) hipLaunchKernelGGL((paged_chunk_kernel<HD, KVG, QF16, 2, KV8>), grid, block, 0, st, ca);
    else if (ca.a.n2 != 0) hipLaunchKernelGGL((paged_chunk_kernel<HD, KVG, QF16, 1, KV8>), grid, block, 0, st, ca);
    else hipLaunchKernelGGL((paged_chunk_kernel<HD, KVG, QF16, 0, KV8>), grid, block, 0, st, ca);
}

// sc: of pages of 8 bits (null: F16)
template <int HD, bool KV8>
static hipError_t launch_chunk(const PagedAttn& a, const PagedScales* sc, hipStream_t st) {
    using P = PC<HD>;
    ChunkArgs ca;
    ca.a = a;
    ca.sc = KV8 ? *sc : PagedScales{};
    uint32_t l2 = 0;
    while ((2 << l2) <= P::NW && (a.hq / a.hkv) % (2 << l2) == 0) ++l2;
    const int hpw = 1 << l2;
    ca.nhg = a.hq / hpw;
    ca.p.pieces = a.pieces;
    const ChunkBounds cb = chunk_plan(a.b, HD, ca.nhg, 32 * (P::NW >> l2), a.window, (size_t)P::NW * P::REC * sizeof(float), a.ws_bytes, ca.p);
    ca.p.hpw_log2 = l2;
    if (cb.table > a.ws_bytes) return hipErrorOutOfMemory;    // (16 bytes a tile: 2.5 million of them fit)
    ca.tiles = reinterpret_cast<ChunkTile*>(a.ws);
    ca.rec = reinterpret_cast<float*>(a.ws + cb.table);
    const int64_t nwg = (int64_t)ca.p.items * ca.nhg;
    if (nwg > 0xffffffffll / 512) return hipErrorNotSupported;
    if constexpr (HD == 64) {
        if (ca.p.kvg == 2) {
            if (a.q_f16) launch_pc<HD, 2, true, KV8>(ca, (unsigned)nwg, st);
            else launch_pc<HD, 2, false, KV8>(ca, (unsigned)nwg, st);
        }
    }
    if (ca.p.kvg == 1) {
        if (a.q_f16) launch_pc<HD, 1, true, KV8>(ca, (unsigned)nwg, st);
        else launch_pc<HD, 1, false, KV8>(ca, (unsigned)nwg, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !ca.p.cuts) return e;
    hipLaunchKernelGGL((paged_chunk_combine<HD>), dim3((unsigned)(cb.tiles * ca.nhg * P::NW)), dim3(64 * P::DB), 0, st, ca);
    return hipGetLastError();
}

}  // namespace vxfa
