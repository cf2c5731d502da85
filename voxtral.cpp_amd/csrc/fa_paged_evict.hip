// fa_paged_evict.hip — the rows of each stream and kv head with the largest
// accumulated weights, moved to other pages.
//
// Two launches. paged_select_kernel, a workgroup per (stream, kv head), finds
// the smallest key that is kept by a radix selection over the weights (four
// digits of 8 bits of an unsigned key that orders as the floats do, a
// histogram in LDS each; counts do not depend on the order of the atomics),
// then lists the kept rows in order: of the rows whose key is that very one the
// first are taken, as many as are still wanted. paged_move_kernel copies the
// listed rows, 16 bytes a lane.
#include "fa_paged.h"

namespace vxfa {

constexpr int SEL_NT = 1024;

// orders as the floats do, -0 as +0, NaN below all
__device__ __forceinline__ uint32_t sel_key(float x) {
    if (x != x) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__global__ __launch_bounds__(SEL_NT) void paged_select_kernel(PagedEvict a) {
    const int s = (int)blockIdx.x, h = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const int n = min(max(a.b.n_kv[s], 0), a.b.max_nkv);
    int32_t* kept = a.kept + ((int64_t)s * a.hkv + h) * a.kept_row;
    if (h == 0 && tid == 0 && a.n_out) a.n_out[s] = min(n, a.budget);
    if (n <= a.budget) {
        for (int r = tid; r < a.kept_row; r += SEL_NT) kept[r] = r < n ? r : -1;
        return;
    }
    const int end = n - a.n_recent;   // rows [n_sink, end) compete
    auto key_of = [&](int j) -> uint32_t {
        const int page = paged_page(a.b, s, j >> a.b.ps_log2);
        if (page < 0) return 0;
        return sel_key(*(const float*)(a.w + page * a.w_nb3 + h * a.w_nb2 + 4 * (int64_t)(j & ((1 << a.b.ps_log2) - 1))));
    };
    __shared__ uint32_t hist[256];
    __shared__ uint32_t pick[2];
    uint32_t want = (uint32_t)(a.budget - a.n_sink - a.n_recent), prefix = 0;
    // want > 0: the want-th largest key
    if (want > 0) {
        for (int sh = 24; sh >= 0; sh -= 8) {
            for (int i = tid; i < 256; i += SEL_NT) hist[i] = 0;
            __syncthreads();
            for (int j = a.n_sink + tid; j < end; j += SEL_NT) {
                const uint32_t k = key_of(j);
                if (sh == 24 || (k >> (sh + 8)) == (prefix >> (sh + 8))) atomicAdd(&hist[(k >> sh) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t left = want;
                int d = 255;
                while (d > 0 && hist[d] < left) left -= hist[d--];
                pick[0] = (uint32_t)d;
                pick[1] = left;
            }
            __syncthreads();
            prefix |= pick[0] << sh;
            want = pick[1];
            __syncthreads();
        }
    }
    // rows in order; `want` of the equal ones
    __shared__ int wsum[SEL_NT / 64][2];
    int done = 0, eq_done = 0;   // kept and equal rows before this step
    const bool any = a.budget - a.n_sink - a.n_recent > 0;
    for (int j0 = 0; j0 < n; j0 += SEL_NT) {
        const int j = j0 + tid;
        const bool in = j < n, always = in && (j < a.n_sink || j >= end);
        const uint32_t k = in && !always && any ? key_of(j) : 0;
        const bool eq = in && !always && any && k == prefix, gt = in && !always && any && k > prefix;
        const uint64_t below = ((uint64_t)1 << lane) - 1, em = __ballot(eq);
        if (lane == 0) wsum[wave][0] = __popcll(em);
        __syncthreads();
        int eb = eq_done + __popcll(em & below), et = 0;
        for (int w = 0; w < SEL_NT / 64; ++w) {
            if (w < wave) eb += wsum[w][0];
            et += wsum[w][0];
        }
        const bool keep = always || gt || (eq && eb < (int)want);
        const uint64_t km = __ballot(keep);
        if (lane == 0) wsum[wave][1] = __popcll(km);
        __syncthreads();
        int kb = done + __popcll(km & below), kt = 0;
        for (int w = 0; w < SEL_NT / 64; ++w) {
            if (w < wave) kb += wsum[w][1];
            kt += wsum[w][1];
        }
        if (keep && kb < a.kept_row) kept[kb] = j;
        done += kt;
        eq_done += et;
        __syncthreads();
    }
    for (int r = done + tid; r < a.kept_row; r += SEL_NT) kept[r] = -1;
}

// a wavefront per kept row: K, V and the weight
__global__ __launch_bounds__(256) void paged_move_kernel(PagedEvict a) {
    const int lane = (int)threadIdx.x & 63, r = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
    const int h = (int)blockIdx.y, s = (int)blockIdx.z;
    if (r >= a.kept_row) return;
    const int j = a.kept[((int64_t)s * a.hkv + h) * a.kept_row + r];
    if (j < 0) return;
    const int lg = a.b.ps_log2, mask = (1 << lg) - 1;
    if ((r >> lg) >= a.max_to) return;
    const int to = a.to[(int64_t)s * a.max_to + (r >> lg)];
    if ((uint32_t)to >= (uint32_t)a.b.n_pages) return;
    const int from = paged_page(a.b, s, j >> lg);
    const int ch = a.d / 8;
    if (lane < 2 * ch) {
        const PagedPool& p = lane < ch ? a.k : a.v;
        const int64_t o = 16 * (lane % ch) + h * p.nb2;
        u32x4 x = {0, 0, 0, 0};
        if (from >= 0) x = *(const u32x4*)(p.base + from * p.nb3 + (j & mask) * p.nb1 + o);
        *(u32x4*)(p.base + to * p.nb3 + (r & mask) * p.nb1 + o) = x;
    }
    if (lane == 63) {
        float x = __builtin_nanf("");
        if (from >= 0) x = *(const float*)(a.w + from * a.w_nb3 + h * a.w_nb2 + 4 * (j & mask));
        *(float*)(a.w + to * a.w_nb3 + h * a.w_nb2 + 4 * (r & mask)) = x;
    }
}

hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t st) {
    if (a.b.n_streams <= 0 || a.kept_row <= 0) return hipSuccess;
    hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)a.b.n_streams, (unsigned)a.hkv), dim3(SEL_NT), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(paged_move_kernel, dim3((unsigned)((a.kept_row + 3) / 4), (unsigned)a.hkv, (unsigned)a.b.n_streams), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace vxfa
