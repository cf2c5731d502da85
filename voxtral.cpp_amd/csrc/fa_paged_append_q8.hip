// fa_paged_append_q8.hip — new K and V rows of a ragged batch of chunks into the
// pages of a cache of 8 bits, for gfx950.
//
// The form of fa_paged_append.hip in which 16 rows of a page and head share a scale 2^e:
// e the least with max |x| <= 127 2^e over the new rows, or that of the rows ahead of
// them if it is larger; x / 2^e rounded to nearest even (exact but for that rounding:
// e and the division are exponents), rows ahead rounded again where e grows.
// Work: a workgroup per 16 rows that new rows lie in, one for K and one for V, a
// wavefront per head: it holds the new rows in registers (16 x D floats, 16 bytes a
// lane and load, all in flight together), takes their maximum by DPP and
// stores 4 bytes a lane. So each element is read once, and rows of one block are in one
// wavefront, whatever order they came in. Queries, which have no scales, have workgroups of
// their own, a wavefront per token. The angles' cos / sin are formed once for
// all heads. Bound by HBM: 8192 tokens of 32 + 8 + 8 heads of 128 53 us, 5.4 TB/s read and
// written (four wavefronts a SIMD: 55.8 -> 53.1; eight of a token's query loads in flight: 61 -> 55.8); 32
// tokens 5.4 us in a graph.
#include "fa_paged_q8.h"

namespace vxfa {

// |x| of four, NaN passed over
__device__ __forceinline__ float amax4(floatx4 x) { return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))); }

// x as a whole number from -127 to 127, NaN as 0
__device__ __forceinline__ uint32_t byte_of(float x) {
    const float r = fminf(fmaxf(rintf(x), -127.f), 127.f);
    return (uint32_t)(x == x ? (int)r : 0) & 255u;
}
__device__ __forceinline__ uint32_t bytes_of(floatx4 x, float f) {
    return byte_of(x[0] * f) | byte_of(x[1] * f) << 8 | byte_of(x[2] * f) << 16 | byte_of(x[3] * f) << 24;
}

// cos / sin of pair j < 64 at position p, the angle p ts^j in 64 bits: as a running product in F32
// (which f16 values hide) it is off by up to 1e-3 at position 8192, and as many whole numbers by one.
__device__ __forceinline__ float2 rope_cs_far(int p, int j, double ts) {
    double th = (double)p;
#pragma unroll
    for (int b = 0; b < 6; ++b) {
        th *= (j >> b) & 1 ? ts : 1.0;
        ts *= ts;
    }
    return rope_cs_of_angle(th);
}

template <int D>
__global__ __launch_bounds__(256, 4) void paged_append_q8_kernel(PagedAppend8 p, int units) {
    constexpr int PER = D / 4, RPI = 64 / PER, NI = kScaleRows / RPI;   // lanes of a row, rows of a load, loads
    const PagedAppend& a = p.a;
    __shared__ float2 cs[kScaleRows][D / 2];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if ((int)blockIdx.x >= 2 * units) {
        // ---- queries: four tokens, a wavefront each -----------------------------------
        const int t = 4 * ((int)blockIdx.x - 2 * units) + wave;
        if (t >= a.b.tokens) return;
        const PagedUnit u = paged_token(a.b, t);
        if (u.s < 0) return;
        if (lane < D / 2) cs[wave][lane] = rope_cs_far(a.rope_pos[t], lane, p.rope_ts);
        __builtin_amdgcn_wave_barrier();   // (a wavefront's LDS accesses run in order)
        constexpr int U = 4;                           // 16-byte pairs in flight
        const int n = a.hq * (D / 8);
        for (int c0 = lane; c0 < n; c0 += 64 * U) {
            floatx4 x0[U], x1[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int c = min(c0 + 64 * j, n - 1), h = c / (D / 8), d = 8 * (c % (D / 8));
                const char* src = (const char*)a.q + (int64_t)t * a.q_nb1 + (int64_t)h * a.q_nb2 + 4 * d;
                x0[j] = __builtin_nontemporal_load((const floatx4*)src);
                x1[j] = __builtin_nontemporal_load((const floatx4*)src + 1);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int c = c0 + 64 * j, h = c / (D / 8), d = 8 * (c % (D / 8));
                if (c >= n) continue;
                float x[8] = {x0[j][0], x0[j][1], x0[j][2], x0[j][3], x1[j][0], x1[j][1], x1[j][2], x1[j][3]};
                rope8_tab(x, d, cs[wave], a.rope_dims);
                half8 y;
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = (_Float16)x[i];
                *(half8*)((char*)a.q_out + (int64_t)t * a.qo_nb1 + (int64_t)h * a.qo_nb2 + 2 * d) = y;
            }
        }
        return;
    }
    // ---- 16 rows of K or V -----------------------------------------------------------
    const bool isv = blockIdx.x & 1;
    const PagedUnit u = paged_unit(a.b, (int)blockIdx.x >> 1, [&](const PagedStream& s) { return blocks_count(s, a.b.max_nq, 4); });
    if (u.s < 0) return;
    const int past = u.st.n - u.st.t, nq = min(u.st.t, a.b.max_nq);
    const int row0 = kScaleRows * (blocks_first(u.st, 4) + u.i);
    const int r0 = max(past - row0, 0), r1 = min(past + nq - row0, kScaleRows);   // new rows [r0, r1)
    const int page = paged_page(a.b, u.s, row0 >> a.b.ps_log2);
    const int tok0 = u.st.q0 + row0 - past;                                       // token of row 0
    if (page < 0) return;
    const bool turn = !isv && a.rope_pos;
    if (turn) {
        for (int i = tid; i < kScaleRows * 64; i += 256) {
            const int r = i >> 6, j = i & 63;
            if (j < D / 2 && r >= r0 && r < r1) cs[r][j] = rope_cs_far(a.rope_pos[tok0 + r], j, p.rope_ts);
        }
        __syncthreads();
    }
    const int at = row0 & ((1 << a.b.ps_log2) - 1), d = 4 * (lane % PER), rl = lane / PER;
    const char* const src = isv ? (const char*)a.v_new : (const char*)a.k_new;
    const int64_t snb = isv ? a.vn_nb1 : a.kn_nb1;
    for (int h = wave; h < a.hkv; h += 4) {
        floatx4 x[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = RPI * i + rl;
            x[i] = floatx4{0.f, 0.f, 0.f, 0.f};
            if (r >= r0 && r < r1) x[i] = __builtin_nontemporal_load((const floatx4*)(src + (int64_t)(tok0 + r) * snb + 4 * (int64_t)(h * D + d)));
        }
        float* const sp = (float*)((isv ? p.sc.v : p.sc.k) + p.sc.at(page, h, at));
        // (the exponent of what rows ahead have; of garbage, any in the range)
        const int eo = r0 > 0 ? min(max((int)((__builtin_bit_cast(uint32_t, *sp) >> 23) & 255u) - 127, kMinExp), kMaxExp) : kMinExp;
        if (turn) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = RPI * i + rl;
                if (r < r0 || r >= r1) continue;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (d + 2 * k < a.rope_dims) {
                        const float2 t = cs[r][d / 2 + k];
                        const float y0 = x[i][2 * k], y1 = x[i][2 * k + 1];
                        x[i][2 * k] = y0 * t.x - y1 * t.y;
                        x[i][2 * k + 1] = y0 * t.y + y1 * t.x;
                    }
            }
        }
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) m = fmaxf(m, amax4(x[i]));
        // (positive floats order as their bits do)
        const int e = max(exp_for(__builtin_bit_cast(float, wave_max(__builtin_bit_cast(int, m)))), eo);
        const float f = two_to(-e);
        char* const dst = (isv ? a.kv.v : a.kv.k) + a.kv.at(page, h, at) + d;
        if (e > eo && r0 > 0) {
            const float g = two_to(max(eo - e, -126));
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = RPI * i + rl;
                if (r >= r0) continue;
                uint32_t* const w = (uint32_t*)(dst + r * a.kv.nb1);
                const int b = (int)*w;
                const floatx4 y = {(float)(b << 24 >> 24), (float)(b << 16 >> 24), (float)(b << 8 >> 24), (float)(b >> 24)};
                *w = bytes_of(y, g);
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = RPI * i + rl;
            if (r >= r0 && r < r1) *(uint32_t*)(dst + r * a.kv.nb1) = bytes_of(x[i], f);
        }
        if (lane == 0) *sp = two_to(e);
    }
}

hipError_t launch_paged_append_q8(const PagedAppend8& p, hipStream_t st) {
    const PagedAppend& a = p.a;
    if (a.b.tokens <= 0 || a.b.n_streams <= 0) return hipSuccess;
    const int64_t units = blocks_bound(a.b, 4), qs = a.q && a.hq > 0 ? ((int64_t)a.b.tokens + 3) / 4 : 0;
    const int64_t grid = 2 * units + qs;
    if (grid > kMaxGridX) return hipErrorNotSupported;
    if (a.d == 128) hipLaunchKernelGGL((paged_append_q8_kernel<128>), dim3((unsigned)grid), dim3(256), 0, st, p, (int)units);
    else if (a.d == 64) hipLaunchKernelGGL((paged_append_q8_kernel<64>), dim3((unsigned)grid), dim3(256), 0, st, p, (int)units);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace vxfa
