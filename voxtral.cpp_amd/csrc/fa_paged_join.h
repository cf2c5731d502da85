// fa_paged_join.h — what fa_paged_rows.hip and fa_paged_walk.hip share: the parts that the
// rows of a stream's few tokens are cut into, their records, the launch that joins them;
// loads to LDS.
#pragma once

#include "fa_paged.h"
#include "fa_paged_plan.h"
#include "fa_paged_q8.h"

namespace vxfa {

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

// Joins the parts of a stream: a wavefront per (token, query head, 32 dims), 8
// lanes of 4 dims for every eighth part, all loads of 8 parts a lane at once.
// TOKENS: each packed token has `parts` of its own.
template <int D, bool TOKENS>
static __global__ __launch_bounds__(64) void paged_rows_combine(RowsArgs ra, int parts) {
    const PagedAttn& a = ra.a;
    const int lane = (int)threadIdx.x, f = lane & 7, grp = lane >> 3;
    // kv head fastest, as in the kernel that wrote the records
    const int hk = (int)blockIdx.x % a.hkv, rest = (int)blockIdx.x / a.hkv;
    const int g = rest / (D / 32), sl = rest % (D / 32);
    const int i = TOKENS ? 0 : (int)blockIdx.y, s = (int)blockIdx.z;
    PagedStream st;
    int2 cut;
    // (One stream's parts begin at 0: its records are on their way before their number is known, as
    // far as a round of the lanes takes them. Of a bound far above the rows there are up to 513: read
    // ahead -> not, 32/8 heads of 128, bound 131072: 8 bits 8192 rows 11.6 -> 9.8 us, four heads a workgroup 15.3
    // -> 11.1 and 300 rows 14.2 -> 9.4; F16 pages, 8192 rows 13.6 -> 11.9. Up to 128 records the two are even.)
    bool one = a.b.n_streams == 1 && ra.items <= 64;
    if constexpr (TOKENS) {
        const int t = (int)blockIdx.y;
        st = PagedStream{t, paged_token(a.b, t).s >= 0 ? 1 : 0, 0};
        cut = int2{t * parts, parts};
        one = false;
    } else {
        st = paged_stream(a.b, s);
        cut = ra.cut[s];
    }
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

}  // namespace vxfa
