// fa_paged_attn.hip — attention of ragged chunks over a paged cache, and the
// weights that its rows gather.
#include "fa_paged.h"

namespace vxfa {

// One wavefront per (token, query head): 64 rows at a time, a row per lane for
// the scores, dims per lane for P V.
template <int D>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttn a) {
    const int lane = (int)threadIdx.x, tok = (int)blockIdx.x, h = (int)blockIdx.y;
    int lo = 0, hi = a.b.n_streams;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.b.q_start[mid] <= tok) lo = mid;
        else hi = mid;
    }
    const PagedStream s = paged_stream(a.b, lo);
    const int i = tok - s.q0;
    if (i < 0 || i >= min(s.t, a.b.max_nq)) return;
    const int hk = h / (a.hq / a.hkv);
    const int p = s.n - s.t + i;
    const int first = a.window > 0 ? max(p - a.window + 1, 0) : 0;
    const float slope = paged_slope(a, h);
    __shared__ _Float16 q[D];
    for (int d = 8 * lane; d < D; d += 512)
        *(half8*)(q + d) = load_q8(a.q, (int64_t)tok * a.q_nb1 + (int64_t)h * a.q_nb2 + d * (a.q_f16 ? 2 : 4), a.q_f16);
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[D / 64];
    for (int u = 0; u < D / 64; ++u) o[u] = 0.f;
    for (int j0 = first; j0 <= p; j0 += 64) {
        const int j = j0 + lane;
        const int page = j <= p ? paged_page(a.b, lo, j >> a.b.ps_log2) : -1;
        const int64_t at = page < 0 ? -1 : page * a.k.nb3 + hk * a.k.nb2 + (j & ((1 << a.b.ps_log2) - 1)) * a.k.nb1;
        float x = -INFINITY;
        if (at >= 0) {
            float dot = 0.f;
            for (int d = 0; d < D; d += 8) {
                const half8 k8 = *(const half8*)(a.k.base + at + 2 * d);
                for (int e = 0; e < 8; ++e) dot = fmaf((float)k8[e], (float)q[d + e], dot);
            }
            x = paged_score(dot, a.c, a.cap) + slope * (float)(j - p);
        }
        float mx = x;
        for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, shfl_xor(mx, w));
        const float mn = fmaxf(m, mx), ms = mn == -INFINITY ? 0.f : mn;
        const float al = exp2_fast(m - ms), pj = exp2_fast(x - ms);
        l = l * al + pj;
        m = mn;
        for (int u = 0; u < D / 64; ++u) o[u] *= al;
        for (int r = 0; r < 64; ++r) {
            const float pr = __shfl(pj, r, 64);
            const int pg = __shfl(page, r, 64);
            if (pg < 0) continue;
            const char* vr = a.v.base + pg * a.v.nb3 + hk * a.v.nb2 + ((j0 + r) & ((1 << a.b.ps_log2) - 1)) * a.v.nb1;
            for (int u = 0; u < D / 64; ++u) o[u] = fmaf(pr, (float)((const _Float16*)vr)[64 * u + lane], o[u]);
        }
    }
    for (int w = 1; w < 64; w <<= 1) l += shfl_xor(l, w);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t at = ((int64_t)tok * a.hq + h) * D;
    for (int u = 0; u < D / 64; ++u) {
        if (a.dst_f16) ((_Float16*)a.dst)[at + 64 * u + lane] = (_Float16)(o[u] * inv);
        else ((float*)a.dst)[at + 64 * u + lane] = o[u] * inv;
    }
    if (a.lse && lane == 0) a.lse[(int64_t)tok * a.hq + h] = l == 0.f ? INFINITY : m + log2f(l);
}

// One thread per (row of a stream, kv head): the scores again, now that the
// tokens' sums are known.
template <int D>
__global__ __launch_bounds__(64) void paged_weights_kernel(PagedAttn a) {
    const int s = (int)blockIdx.y, hk = (int)blockIdx.z, j = (int)blockIdx.x * 64 + (int)threadIdx.x;
    const PagedStream st = paged_stream(a.b, s);
    if (j >= st.n) return;
    const int page = paged_page(a.b, s, j >> a.b.ps_log2), r = j & ((1 << a.b.ps_log2) - 1);
    if (page < 0) return;
    half8 k[D / 8];
    for (int d = 0; d < D / 8; ++d) k[d] = ((const half8*)(a.k.base + page * a.k.nb3 + hk * a.k.nb2 + r * a.k.nb1))[d];
    float sum = 0.f;
    const int G = a.hq / a.hkv;
    for (int i = 0; i < min(st.t, a.b.max_nq); ++i) {
        const int p = st.n - st.t + i;
        if (j > p || (a.window > 0 && j <= p - a.window)) continue;
        for (int h = hk * G; h < (hk + 1) * G; ++h) {
            float dot = 0.f;
            for (int d = 0; d < D / 8; ++d) {
                const half8 q = load_q8(a.q, (int64_t)(st.q0 + i) * a.q_nb1 + (int64_t)h * a.q_nb2 + 8 * d * (a.q_f16 ? 2 : 4), a.q_f16);
                for (int e = 0; e < 8; ++e) dot = fmaf((float)k[d][e], (float)q[e], dot);
            }
            sum += exp2_fast(paged_score(dot, a.c, a.cap) + paged_slope(a, h) * (float)(j - p) - a.lse[(int64_t)(st.q0 + i) * a.hq + h]);
        }
    }
    const float old = a.w_in ? *(const float*)((const char*)a.w_in + page * a.wi_nb3 + hk * a.wi_nb2 + 4 * r) : 0.f;
    *(float*)((char*)a.w_out + page * a.wo_nb3 + hk * a.wo_nb2 + 4 * r) = old + sum;
}

hipError_t launch_paged_attn(const PagedAttn& a, int head_dim, hipStream_t st) {
    if (a.b.tokens <= 0 || a.b.n_streams <= 0) return hipSuccess;
    if (paged_rows_takes(a)) return launch_paged_rows(a, head_dim, st);
    const dim3 grid((unsigned)a.b.tokens, (unsigned)a.hq);
    if (head_dim == 128) hipLaunchKernelGGL((paged_attn_kernel<128>), grid, dim3(64), 0, st, a);
    else if (head_dim == 64) hipLaunchKernelGGL((paged_attn_kernel<64>), grid, dim3(64), 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_paged_weights(const PagedAttn& a, int head_dim, hipStream_t st) {
    if (a.b.max_nkv <= 0 || a.b.n_streams <= 0) return hipSuccess;
    const dim3 grid((unsigned)((a.b.max_nkv + 63) / 64), (unsigned)a.b.n_streams, (unsigned)a.hkv);
    if (head_dim == 128) hipLaunchKernelGGL((paged_weights_kernel<128>), grid, dim3(64), 0, st, a);
    else if (head_dim == 64) hipLaunchKernelGGL((paged_weights_kernel<64>), grid, dim3(64), 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace vxfa
