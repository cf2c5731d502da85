// fa_paged_evict.hip — the rows of each stream and kv head with the largest
// accumulated weights, moved to other pages.
//
// Two launches.
//   paged_select_kernel, a workgroup per (stream, kv head): a radix selection
//   over the weights, as unsigned keys that order as the floats do. Digits of
//   11, 11 and 10 bits: a histogram in LDS (counts do not depend on the order
//   of the atomics), a scan of it from the top, and the digit that holds the
//   last key to be kept. Then the kept rows are listed in order: those of larger
//   keys, and of those with that very key the first, as many as are still
//   wanted. A thread has 8 neighbouring rows, whose keys stay in registers from
//   pass to pass (up to 8192 rows; a longer stream is read again, a segment at
//   a time).
//   paged_move_kernel: 8 kept rows a wavefront, K and V at once, 16 bytes a lane,
//   the four loads of a lane in flight together.
// Measured, 8 kv heads of 128: 32 streams of up to 8192 rows to 1000 74 us (the move
// 52: 5.1 TB/s read and written, what a large copy reaches), one stream of 8192 to
// 4096 22 us: 14 the selection, whose 8 workgroups are a chain of loads, three
// passes of about 2 us and the list, 8 the move.
#include "fa_paged.h"

namespace vxfa {

constexpr int SEL_NT = 1024, SEL_PER = 8, SEL_SEG = SEL_NT * SEL_PER, SEL_BINS = 2048;

// orders as the floats do, -0 as +0, NaN below all
__device__ __forceinline__ uint32_t sel_key(float x) {
    if (x != x) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Sum over the wavefronts before this one, and over all, of each one's `total` (all
// its lanes alike); w: 16 ints of LDS, not read by a slower wavefront any more.
__device__ __forceinline__ int2 sel_before(int total, int* w, int wave, int lane) {
    if (lane == 0) w[wave] = total;
    __syncthreads();
    const int incl = wave_scan(lane < SEL_NT / 64 ? w[lane] : 0);
    const int all = __builtin_amdgcn_readlane(incl, SEL_NT / 64 - 1);
    return int2{wave > 0 ? __builtin_amdgcn_readlane(incl, wave > 0 ? wave - 1 : 0) : 0, all};
}

__global__ __launch_bounds__(SEL_NT) void paged_select_kernel(PagedEvict a) {
    const int s = (int)blockIdx.x, h = (int)blockIdx.y, tid = (int)threadIdx.x;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int32_t* kept = a.kept + ((int64_t)s * a.hkv + h) * a.kept_row;
    const int lg = a.b.ps_log2;
    uint32_t key[SEL_PER];
    // the keys of 8 rows, which are half a page at most (of rows that the table has;
    // those from n on are not looked at, so the first loads need not wait for n)
    auto load = [&](int j0) {
        const int j = j0 + SEL_PER * tid;
        const int page = j < a.b.max_nkv ? paged_page(a.b, s, j >> lg) : -1;
        const float* w = (const float*)(a.w + max(page, 0) * a.w_nb3 + h * a.w_nb2 + 4 * (int64_t)(j & ((1 << lg) - 1)));
        float x[SEL_PER];
#pragma unroll
        for (int i = 0; i < SEL_PER; ++i) x[i] = page >= 0 ? w[i] : 0.f;
#pragma unroll
        for (int i = 0; i < SEL_PER; ++i) key[i] = page >= 0 ? sel_key(x[i]) : 0;
    };
    load(0);
    const int n = min(max(a.b.n_kv[s], 0), a.b.max_nkv);
    if (h == 0 && tid == 0 && a.n_out) a.n_out[s] = min(n, a.budget);
    if (n <= a.budget) {
        for (int r = tid; r < a.kept_row; r += SEL_NT) kept[r] = r < n ? r : -1;
        return;
    }
    const int end = n - a.n_recent;   // rows [n_sink, end) compete
    __shared__ uint32_t hists[3][SEL_BINS];
    __shared__ int list[SEL_SEG];
    __shared__ int wsum[2][SEL_NT / 64];
    __shared__ uint32_t pick[2];
    // (a histogram for each pass)
    for (int i = tid; i < 3 * SEL_BINS; i += SEL_NT) (&hists[0][0])[i] = 0;
    const bool one = n <= SEL_SEG;
    __syncthreads();
    int want = a.budget - a.n_sink - a.n_recent;   // of the competing rows
    const bool any = want > 0;
    uint32_t prefix = 0;
    if (any) {
        for (int pass = 0; pass < 3; ++pass) {
            const int sh = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = pass == 2 ? 10 : 11;
            uint32_t* const hist = hists[pass];
            for (int j0 = 0; j0 < n; j0 += SEL_SEG) {
                if (!one) load(j0);
#pragma unroll
                for (int i = 0; i < SEL_PER; ++i) {
                    const int j = j0 + SEL_PER * tid + i;
                    if (j >= a.n_sink && j < end && (pass == 0 || (key[i] >> (sh + bits)) == (prefix >> (sh + bits))))
                        atomicAdd(&hist[(key[i] >> sh) & ((1 << bits) - 1)], 1u);
                }
            }
            __syncthreads();
            // thread t: bins 2047 - 2 t and the one below, from the top
            const int b1 = SEL_BINS - 1 - 2 * tid;
            const int c1 = (int)hist[b1], c2 = (int)hist[b1 - 1];
            const int incl = wave_scan(c1 + c2);
            const int above = sel_before(__builtin_amdgcn_readlane(incl, 63), wsum[0], wave, lane).x + incl - c1 - c2;
            if (above < want && above + c1 >= want) {
                pick[0] = (uint32_t)b1;
                pick[1] = (uint32_t)(want - above);
            } else if (above + c1 < want && above + c1 + c2 >= want) {
                pick[0] = (uint32_t)(b1 - 1);
                pick[1] = (uint32_t)(want - above - c1);
            }
            __syncthreads();
            prefix |= pick[0] << sh;
            want = (int)pick[1];
            // (pick is written again only after the next barrier but one)
        }
    }
    // rows in order; `want` of those with the key `prefix`
    int done = 0, eq_done = 0;   // kept and equal rows of the segments before
    for (int j0 = 0; j0 < n; j0 += SEL_SEG) {
        if (!one) load(j0);
        const int jt = j0 + SEL_PER * tid;
        int eq = 0;
#pragma unroll
        for (int i = 0; i < SEL_PER; ++i) eq += any && jt + i >= a.n_sink && jt + i < end && key[i] == prefix;
        __syncthreads();
        const int ei = wave_scan(eq);
        const int2 es = sel_before(__builtin_amdgcn_readlane(ei, 63), wsum[0], wave, lane);
        int eb = eq_done + es.x + ei - eq;
        eq_done += es.y;
        uint32_t keep = 0;
#pragma unroll
        for (int i = 0; i < SEL_PER; ++i) {
            const int j = jt + i;
            if (j >= n) continue;
            if (j < a.n_sink || j >= end) keep |= 1u << i;
            else if (any && key[i] > prefix) keep |= 1u << i;
            else if (any && key[i] == prefix && eb++ < want) keep |= 1u << i;
        }
        const int c = __popc(keep), ki = wave_scan(c);
        const int2 ks = sel_before(__builtin_amdgcn_readlane(ki, 63), wsum[1], wave, lane);
        // through LDS, so that the list is written in whole lines
        int kb = ks.x + ki - c;
#pragma unroll
        for (int i = 0; i < SEL_PER; ++i)
            if ((keep >> i) & 1) list[kb++] = jt + i;
        __syncthreads();
        for (int r = tid; r < ks.y; r += SEL_NT)
            if (done + r < a.kept_row) kept[done + r] = list[r];
        done += ks.y;
    }
    for (int r = done + tid; r < a.kept_row; r += SEL_NT) kept[r] = -1;
}

static_assert(kPagedMoveRows == 4 * 8, "four wavefronts");
template <int D>
__global__ __launch_bounds__(256) void paged_move_kernel(PagedEvict a) {
    constexpr int CH = D / 8, RPW = 64 / (2 * CH);   // rows of one step: CH lanes of K, CH of V each
    constexpr int U = 8 / RPW;
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    const int h = (int)blockIdx.x % a.hkv, r0 = (int)blockIdx.x / a.hkv * kPagedMoveRows + 8 * wave, s = (int)blockIdx.y;
    const int lg = a.b.ps_log2, mask = (1 << lg) - 1;
    const int32_t* kept = a.kept + ((int64_t)s * a.hkv + h) * a.kept_row;
    char* const pool = ((lane / CH) & 1 ? a.kv.v : a.kv.k) + 16 * (lane % CH);
    int j[U], to[U], from[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = r0 + RPW * u + lane / (2 * CH);
        j[u] = r < a.kept_row ? kept[r] : -1;
        to[u] = (r >> lg) < a.max_to && r < a.kept_row ? a.to[(int64_t)s * a.max_to + (r >> lg)] : -1;
        if ((uint32_t)to[u] >= (uint32_t)a.b.n_pages) to[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) from[u] = j[u] >= 0 && to[u] >= 0 ? paged_page(a.b, s, j[u] >> lg) : -1;
    u32x4 x[U];
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        x[u] = u32x4{0, 0, 0, 0};
        w[u] = __builtin_nanf("");
        if (from[u] >= 0) {
            x[u] = __builtin_nontemporal_load((const u32x4*)(pool + a.kv.at(from[u], h, j[u] & mask)));
            if (lane % (2 * CH) == 0) w[u] = *(const float*)(a.w + from[u] * a.w_nb3 + h * a.w_nb2 + 4 * (j[u] & mask));
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = r0 + RPW * u + lane / (2 * CH);
        if (j[u] < 0 || to[u] < 0) continue;
        *(u32x4*)(pool + a.kv.at(to[u], h, r & mask)) = x[u];
        if (lane % (2 * CH) == 0) *(float*)(a.w + to[u] * a.w_nb3 + h * a.w_nb2 + 4 * (r & mask)) = w[u];
    }
}

hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t st) {
    if (a.b.n_streams <= 0 || a.kept_row <= 0) return hipSuccess;
    if (!paged_evict_fits(a) || (a.d != 64 && a.d != 128)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(paged_select_kernel, dim3((unsigned)a.b.n_streams, (unsigned)a.hkv), dim3(SEL_NT), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 grid((unsigned)paged_move_grid(a), (unsigned)a.b.n_streams);
    if (grid.x == 0) return e;
    if (a.d == 128) hipLaunchKernelGGL((paged_move_kernel<128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((paged_move_kernel<64>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace vxfa
