// fa_paged_append.hip — new K and V rows of a ragged batch of chunks into the
// pages of an f16 cache.
//
// The paged form of fa_kv_append.hip, for the two ggml_cpy nodes and the two
// rope nodes of a decoder layer (src/voxtral.cpp:1746-1770). Each element
// is rounded once, F32 -> f16 to nearest even. One workgroup per packed token:
// it looks its stream up in q_start (by bisection), its page in the table,
// forms the cos / sin of its position once for all heads, and converts 8
// elements per thread and step (two 16-byte loads, one 16-byte store). Bound by
// HBM: 8192 tokens of 32 + 8 + 8 heads of 128 53.5 us, 5.6 TB/s read and
// written (the sources' nontemporal hint: 58.3 -> 53.5; one at the stores: 54.3);
// 32 tokens 4.4 us in a graph (launch cadence and three dependent loads).
#include "fa_paged.h"

namespace vxfa {

__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppend a) {
    __shared__ float2 cs[64];
    const int t = (int)blockIdx.x;
    // the stream: the last one that starts at or before the token
    int lo = 0, hi = a.b.n_streams;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.b.q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const PagedStream s = paged_stream(a.b, lo);
    const int i = t - s.q0;
    if (i < 0 || i >= min(s.t, a.b.max_nq)) return;        // a token of no stream
    if (a.rope_pos) {
        if (threadIdx.x < a.d / 2) cs[threadIdx.x] = rope_cs_chain<64>(a.rope_pos[t], (int)threadIdx.x, a.rope_ts);
        __syncthreads();
    }
    const int row = s.n - s.t + i;
    const int page = row >= 0 ? paged_page(a.b, lo, row >> a.b.ps_log2) : -1;
    const int r = row & ((1 << a.b.ps_log2) - 1);
    const int per = a.hkv * a.d / 8, perq = a.q ? a.hq * a.d / 8 : 0;
    for (int c = (int)threadIdx.x; c < 2 * per + perq; c += 256) {
        const int m = c < per ? 0 : (c < 2 * per ? 1 : 2);   // K, V, Q
        const int e = 8 * (c - m * per);
        const int h = e / a.d, d = e - h * a.d;
        if (m < 2 && page < 0) continue;
        const char* src = m == 0 ? (const char*)a.k_new + (int64_t)t * a.kn_nb1 + 4 * (int64_t)e
                        : m == 1 ? (const char*)a.v_new + (int64_t)t * a.vn_nb1 + 4 * (int64_t)e
                                 : (const char*)a.q + (int64_t)t * a.q_nb1 + (int64_t)h * a.q_nb2 + 4 * d;
        const floatx4 x0 = __builtin_nontemporal_load((const floatx4*)src), x1 = __builtin_nontemporal_load((const floatx4*)src + 1);
        float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
        if (m != 1 && a.rope_pos) rope8_tab(x, d, cs, a.rope_dims);
        half8 y;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (_Float16)x[j];
        char* dst = m == 2 ? (char*)a.q_out + (int64_t)t * a.qo_nb1 + (int64_t)h * a.qo_nb2
                           : (m == 0 ? a.kv.k : a.kv.v) + a.kv.at(page, h, r);
        *(half8*)(dst + 2 * d) = y;
    }
}

hipError_t launch_paged_append(const PagedAppend& a, hipStream_t st) {
    if (a.b.tokens <= 0 || a.b.n_streams <= 0) return hipSuccess;
    if (a.d > 128 || a.d % 8) return hipErrorInvalidValue;
    hipLaunchKernelGGL(paged_append_kernel, dim3((unsigned)a.b.tokens), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace vxfa
