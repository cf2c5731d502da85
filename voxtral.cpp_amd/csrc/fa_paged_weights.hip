// fa_paged_weights.hip — the weights that the rows of a paged cache gather.
#include "fa_paged.h"

namespace vxfa {

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

hipError_t launch_paged_weights(const PagedAttn& a, int head_dim, hipStream_t st) {
    if (a.b.max_nkv <= 0 || a.b.n_streams <= 0) return hipSuccess;
    const dim3 grid((unsigned)((a.b.max_nkv + 63) / 64), (unsigned)a.b.n_streams, (unsigned)a.hkv);
    if (head_dim == 128) hipLaunchKernelGGL((paged_weights_kernel<128>), grid, dim3(64), 0, st, a);
    else if (head_dim == 64) hipLaunchKernelGGL((paged_weights_kernel<64>), grid, dim3(64), 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace vxfa
