// fa_paged_weights.hip — the attention weight that each row of a paged cache
// gathers from the tokens of a call, for gfx950.
//
// A row's weight is the sum, over tokens i and the kv head's query heads, of
// P_ij = 2^(x_ij - lse_i), where lse_i (the logarithm of the row sum) is only
// known when the attention is done: the scores are formed again, from K alone,
// half the attention's products. (Single tokens: paged_rows_kernel has left its
// scores, and paged_rows_weights sums them; see there.)
//   Workgroup = 128 rows of a stream and kv head, 4 wavefronts: 32 rows each, or two
//   halves of 64 rows by two halves of the query rows (NB below). S^T = K Q^T by
//   v_mfma_f32_32x32x16_f16: a lane has the scores of 16 rows for one query row,
//   so lse, position and slope are one register each, and the sums over query rows
//   stay in 16 registers a block until the end. K stays in registers; 64 query
//   rows (tokens x heads, packed) a step go through LDS, loaded a step ahead, of
//   those tokens only that see some of the 128 rows.
// One workgroup owns a row's sum: no atomics, the same bits every time.
// Bound by its VALU work (three instructions a score, and the masks of the blocks
// on the diagonal and at a window's edge) and each workgroup's chain of loads: 8
// streams of 250 tokens, window 750, 20 heads of 64, 22 us (a thread per row and
// head, which this replaced, 331). Query rows are not split over workgroups: one stream's
// 2000 tokens on as many rows are 128 workgroups, the first of which walks all 8000 query
// rows, 125 steps, and the call takes 196 us (without weights 67).
// Spills: F32 queries at hd 128 14 or 15 VGPRs (60 or 64 bytes of scratch a lane), F16
// ones at hd 64 with a cap or slopes 3 (16 bytes).
#include "fa_paged.h"

namespace vxfa {

constexpr int PW_ROWS = kPagedWeightRows;

struct WeightsArgs {
    PagedAttn a;
    DivMod grp;               // query heads per kv head
    int32_t ntiles;           // row tiles of a stream at most
};

// MOD: 1 the scores have a cap or a distance term, 2 a wide cap (as a test at run time it
// cost the narrow one 6 to 15 % of this kernel).
// NB blocks of 32 rows a wavefront, NB wavefronts share a step's 64 query rows: 2 at
// hd 128, whose products wait for the query rows from LDS (2000 tokens on as many rows
// 195 us of a call, with one block 208; 600 on 3000 with slopes 123, 129), 1 at hd 64
// for the registers, four workgroups a CU in place of three (the window case's call 58
// against 67, 16 streams of 100 tokens and up to 8000 rows 297 against 395).
template <int D, bool QF16, int MOD>
__global__ __launch_bounds__(256, (D == 128 ? 2 : QF16 ? 4 : 3)) void paged_weights_kernel(WeightsArgs wa) {
    constexpr int KS = D / 16, ROW = 2 * D, CH = D / 8;
    constexpr int STEP = 64 * ROW;                  // bytes of 64 query rows
    constexpr int NB = D == 128 ? 2 : 1, QB = 2 / NB;   // blocks of rows, of query rows a wavefront
    __shared__ __attribute__((aligned(16))) char smem[2 * STEP];
    __shared__ float part[NB == 2 ? PW_ROWS : 1];
    const PagedAttn& a = wa.a;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nl = lane & 31, hh = lane >> 5;
    const int ph = wave / NB, rh = wave % NB;       // part of the rows, of the query rows
    const int s = (int)blockIdx.y, hk = (int)blockIdx.x % a.hkv, kv0 = (int)blockIdx.x / a.hkv * PW_ROWS;
    const PagedStream st = paged_stream(a.b, s);
    if (kv0 >= st.n) return;
    const int lg = a.b.ps_log2, pmask = (1 << lg) - 1;
    const int G = (int)wa.grp.d, nq = min(st.t, a.b.max_nq), past = st.n - st.t;

    // ---- query rows (token G + head) that see some of the rows -----------------
    const int t0 = min(max(kv0 - past, 0), nq);
    int t1 = nq;
    if (a.window > 0) t1 = min((int)min((int64_t)kv0 + PW_ROWS - 1 + a.window - past, (int64_t)nq), nq);
    const int r_begin = t0 * G, r_end = max(t1, t0) * G;

    // (the table's entries first, then the query rows, then K: the entries' latency is
    // hidden behind the second)
    int pos[NB], pages[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        pos[b] = kv0 + 32 * (NB * ph + b);
        const int j = pos[b] + nl;
        pages[b] = j < st.n ? paged_page(a.b, s, j >> lg) : -1;
    }

    constexpr int QN = QF16 ? 64 * CH / 256 : 2 * 64 * CH / 256;   // 16-byte loads of a thread
    constexpr int QC = QF16 ? CH : 2 * CH;                          // of a row
    floatx4 qraw[QN];
    auto load_q = [&](int r0) {
#pragma unroll
        for (int u = 0; u < QN; ++u) {
            const int e = tid + 256 * u, r = min(r0 + e / QC, r_end - 1);
            const int tk = (int)wa.grp.div((uint32_t)r), h = hk * G + r - tk * G;
            qraw[u] = *((const floatx4*)((const char*)a.q + (int64_t)(st.q0 + tk) * a.q_nb1 + (int64_t)h * a.q_nb2) + e % QC);
        }
    };
    // 16-byte chunk j of row r at j ^ (r % CH)
    auto put_q = [&](int buf) {
#pragma unroll
        for (int u = 0; u < QN; ++u) {
            const int e = tid + 256 * u, r = e / QC, j = e % QC;
            char* row = smem + buf * STEP + r * ROW;
            if constexpr (QF16) {
                *(floatx4*)(row + ((j ^ (r % CH)) * 16)) = qraw[u];
            } else {
                half4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (_Float16)qraw[u][i];
                *(half4*)(row + (((j >> 1) ^ (r % CH)) * 16) + (j & 1) * 8) = y;
            }
        }
    };
    // the lane's query row of each block of a step: its token, head and lse
    int tk[QB], h[QB];
    float lse[QB];
    auto rows_of = [&](int r0) {
#pragma unroll
        for (int c = 0; c < QB; ++c) {
            const int r = r0 + 32 * (QB * rh + c) + nl, rc = min(r, r_end - 1);
            tk[c] = (int)wa.grp.div((uint32_t)rc);
            h[c] = hk * G + rc - tk[c] * G;
            const float y = a.lse[(int64_t)(st.q0 + tk[c]) * a.hq + h[c]];
            lse[c] = r < r_end ? y : INFINITY;      // (weight 0)
        }
    };
    if (r_begin < r_end) {
        load_q(r_begin);
        rows_of(r_begin);
    }

    // ---- K: A operand, row nl of a block, dims 16 ks + 8 hh .. (rows that are not
    // there: zeros) ------------------------------------------------------------------
    half8 kr[NB][KS];
    float old[NB];                                  // what the lane's rows have gathered so far
    const bool writes = rh == 0 && ((nl >> 2) & 1) == hh;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int j = pos[b] + nl, page = pages[b];
        old[b] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kr[b][ks] = half8{};
        if (page >= 0 && r_begin < r_end) {
            const char* p = a.kv.k + a.kv.at(page, hk, j & pmask) + 16 * hh;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kr[b][ks] = *(const half8*)(p + 32 * ks);
        }
        if (page >= 0 && writes && a.w_in)
            old[b] = *(const float*)((const char*)a.w_in + page * a.wi_nb3 + hk * a.wi_nb2 + 4 * (int64_t)(j & pmask));
    }

    float sum[NB][16];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[b][j] = 0.f;

    for (int r0 = r_begin, buf = 0; r0 < r_end; r0 += 64, buf ^= 1) {
        put_q(buf);
        int p[QB];
        float slope[QB], lse_now[QB];
#pragma unroll
        for (int c = 0; c < QB; ++c) {
            p[c] = past + tk[c];
            slope[c] = MOD ? paged_slope(a, h[c]) : 0.f;
            lse_now[c] = lse[c];
        }
        if (r0 + 64 < r_end) {
            load_q(r0 + 64);
            rows_of(r0 + 64);
        }
        __syncthreads();                            // (the other buffer is read until the next one)
#pragma unroll
        for (int c = 0; c < QB; ++c) {
            const int first = a.window > 0 ? p[c] - a.window + 1 : INT32_MIN;
            half8 qb[KS];
            const char* row = smem + buf * STEP + (32 * (QB * rh + c) + nl) * ROW;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qb[ks] = *(const half8*)(row + (((2 * ks + hh) ^ (nl % CH)) * 16));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                floatx16 x = {};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(kr[b][ks], qb[ks], x, 0, 0, 0);
                // element j: row pos + 8 (j / 4) + 4 hh + j % 4
                const int j0 = pos[b] + 4 * hh;
                if constexpr (MOD != 0) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float y = MOD == 2 ? paged_wide_cap(a.c * x[j], a.cap, a.capk) : paged_score(a, x[j]);
                        x[j] = fmaf(slope[c], (float)(j0 + 8 * (j >> 2) + (j & 3) - p[c]), y) - lse_now[c];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[j] = fmaf(a.c, x[j], -lse_now[c]);
                }
                // (a block that all the wavefront's query rows see whole needs no mask)
                if (__any(pos[b] + 31 > p[c] || pos[b] < first)) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int k = j0 + 8 * (j >> 2) + (j & 3);
                        x[j] = k > p[c] || k < first ? -INFINITY : x[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) sum[b][j] += exp2_fast(x[j]);
                if constexpr (NB == 2) __builtin_amdgcn_sched_barrier(0);   // (one block's scores at a time: registers)
            }
        }
    }
    // ---- over the lanes of a half, then the wavefronts ----------------------------
    float mine[NB];                                 // lane nl: block b's row nl (both halves of lanes alike)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        mine[b] = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float y = row16_sum(sum[b][j]);
            const int yi = __builtin_bit_cast(int, y);
            const auto sw = __builtin_amdgcn_permlane16_swap(yi, yi, false, false);
            y = __builtin_bit_cast(float, (int)sw[0]) + __builtin_bit_cast(float, (int)sw[1]);
            // (lanes of half hh now hold row 8 (j / 4) + 4 hh + j % 4)
            if (nl == 8 * (j >> 2) + 4 * hh + (j & 3)) mine[b] = y;
        }
    }
    if constexpr (NB == 2) {
        if (rh == 1) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
                if (((nl >> 2) & 1) == hh) part[pos[b] - kv0 + nl] = mine[b];
        }
        __syncthreads();
    }
    if (writes) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if constexpr (NB == 2) mine[b] += part[pos[b] - kv0 + nl];
            if (pages[b] >= 0)
                *(float*)((char*)a.w_out + pages[b] * a.wo_nb3 + hk * a.wo_nb2 + 4 * (int64_t)((pos[b] + nl) & pmask)) =
                    old[b] + mine[b];
        }
    }
}

template <int D, bool QF16>
static void launch_pw_q(const WeightsArgs& wa, const dim3& grid, hipStream_t st) {
    if (wa.a.capk != 0.f) hipLaunchKernelGGL((paged_weights_kernel<D, QF16, 2>), grid, dim3(256), 0, st, wa);
    else if (wa.a.cap != 0.f || wa.a.n2 != 0) hipLaunchKernelGGL((paged_weights_kernel<D, QF16, 1>), grid, dim3(256), 0, st, wa);
    else hipLaunchKernelGGL((paged_weights_kernel<D, QF16, 0>), grid, dim3(256), 0, st, wa);
}
template <int D>
static void launch_pw(const WeightsArgs& wa, const dim3& grid, hipStream_t st) {
    if (wa.a.q_f16) launch_pw_q<D, true>(wa, grid, st);
    else launch_pw_q<D, false>(wa, grid, st);
}

hipError_t launch_paged_weights(const PagedAttn& a, int head_dim, hipStream_t st) {
    if (a.b.max_nkv <= 0 || a.b.n_streams <= 0) return hipSuccess;
    WeightsArgs wa;
    wa.a = a;
    wa.grp = DivMod::make((uint32_t)(a.hq / a.hkv > 0 ? a.hq / a.hkv : 1));
    wa.ntiles = (int32_t)(((int64_t)a.b.max_nkv + PW_ROWS - 1) / PW_ROWS);
    if (!paged_weights_fit(a)) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(wa.ntiles * a.hkv), (unsigned)a.b.n_streams);
    if (head_dim == 128) launch_pw<128>(wa, grid, st);
    else if (head_dim == 64) launch_pw<64>(wa, grid, st);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace vxfa
