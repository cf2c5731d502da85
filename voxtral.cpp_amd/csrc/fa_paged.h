// fa_paged.h — what the kernels over a paged K/V cache share: the launch
// descriptors, a stream's sizes and pages as the kernels read them, scores.
//
// Tables and sizes lie on the device and may hold anything: every number
// read there is brought into its range before it is used as an index.
#pragma once

#include "fa_common.h"

#include <type_traits>

namespace vxfa {

constexpr int kPagedMinLog2 = 4, kPagedMaxLog2 = 16;   // page sizes 16 .. 65536

// The batch: streams, their tables, the pool's pages.
struct PagedBatch {
    const int32_t* pages;     // [n_streams][max_pages]
    const int32_t* n_kv;      // [n_streams]
    const int32_t* q_start;   // [n_streams + 1]
    int32_t n_streams, max_pages, n_pages;
    int32_t ps_log2;          // log2 of a page's rows
    int32_t tokens;           // packed tokens of the call
    int32_t max_nq;           // tokens of a stream that are looked at
    int32_t max_nkv;          // rows of a stream at most (within max_pages pages)
};

// A stream's sizes: t tokens from packed token q0 on, the last of n rows.
struct PagedStream {
    int q0, t, n;
};
__device__ __forceinline__ PagedStream paged_stream(const PagedBatch& b, int s) {
    PagedStream r;
    r.q0 = min(max(b.q_start[s], 0), b.tokens);
    r.t = min(max(b.q_start[s + 1], r.q0), b.tokens) - r.q0;
    r.n = min(max(b.n_kv[s], 0), b.max_nkv);
    return r;
}

// Inclusive sums over the lanes of a wavefront, by DPP shifts within a row of 16
// lanes and broadcasts of a row's last lane (no LDS round trips).
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);   // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);   // row_bcast 31 into rows 2 and 3
    return x;
}
// (x >= 0)
__device__ __forceinline__ float wave_sum(float x) {
    auto add = [&](auto ctl, auto rows) {
        x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctl)::value, decltype(rows)::value, 0xF, false));
    };
    add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ int wave_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xF, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xA, 0xF, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// The page of entry i of stream s, or -1 (absent).
__device__ __forceinline__ int paged_page(const PagedBatch& b, int s, int i) {
    const int p = b.pages[(int64_t)s * b.max_pages + i];
    return (uint32_t)p < (uint32_t)b.n_pages ? p : -1;
}

// The pool: row r of head h in page p lies at (of K) or (of V) + at(p, h, r).
struct PagedPool {
    char *k, *v;
    int64_t nb1, nb2, nb3;
    __device__ __forceinline__ int64_t at(int page, int h, int r) const { return page * nb3 + h * nb2 + r * nb1; }
};

struct PagedAttn {
    PagedBatch b;
    const void* q;            // [token][head][D], F16 or F32
    int64_t q_nb1, q_nb2;     // bytes between tokens, heads
    PagedPool kv;
    void* dst;                // [token][head][D], F16 or F32
    uint8_t q_f16, dst_f16;
    int32_t hq, hkv, window;
    // scores in log2 units: c s; with a cap, cap tanh of it: up to kNarrowCap as
    // cap - 2 cap / (1 + 2^(c s)) with c = 2 log2(e) scale / softcap, beyond by
    // paged_wide_cap
    float c;                  // scale * log2(e), or the factor above
    float cap;                // softcap * log2(e); 0: none
    float capk;               // a wide cap's 2 / softcap; 0: a narrow one, or none
    // distance slopes (n2 != 0): head h of hq, n2 the largest power of two
    // in hq: 2^(bias1 (h + 1)) for h < n2, else 2^(bias1 (h - n2 + 1/2))
    float bias1;              // -max_bias / n2 (which may be 0: slopes of 1)
    int32_t n2;
    // accumulated weights
    const float* w_in;        // null: zeros
    float* w_out;             // null: none
    int64_t wi_nb2, wi_nb3, wo_nb2, wo_nb3;
    float* lse;               // [token][head] log2 of the sum of the row's 2^x (+inf: no row seen); null: not wanted
    char* ws;                 // scratch
    size_t ws_bytes;
    int32_t pieces;           // chunks: pieces of the longest walk (0: the plan's choice)
};

// slope_h * log2(e)
__device__ __forceinline__ float paged_slope(const PagedAttn& a, int h) {
    if (a.n2 == 0) return 0.f;
    return kLog2e * exp2f(a.bias1 * (h < a.n2 ? (float)(h + 1) : (float)(h - a.n2) + 0.5f));
}
// A cap on scores w = c s in log2 units, to the digits of w whatever the cap:
// cap tanh(w / cap) with u = 2 w / softcap (so that 2^u = e^(2 w / cap)). Below a
// fifth of the cap (y = w / cap = u ln(2) / 2 < 0.2) by tanh's series,
// w (1 - y^2/3 + 2 y^4/15 - 17 y^6/315), off by 62/2835 y^8 < 2^-24 of w; from there on
// by cap (1 - 2 / (1 + 2^u)), whose subtraction leaves 2^-22 of the cap (E, 1 + E,
// reciprocal and difference rounded), 2^-18.6 of w at most. That second form alone, at
// all scores, is what narrow caps take (kNarrowCap): 2^-22 of 64 is 1.5e-5 in an
// exponent, a thirtieth of the step that P is rounded by. (With the wide form for all
// caps: 16 streams of up to 512 tokens and 4096 rows, cap and slopes, 193 -> 278 us, with
// weights 354 -> 486; 8192 tokens with a cap 760 -> 1060; single tokens, which wait for
// HBM, 113.3 -> 113.9.)
constexpr float kNarrowCap = 64.f;
__device__ __forceinline__ float paged_wide_cap(float w, float cap, float k) {
    constexpr float h = 0.34657359028f * 0.34657359028f;   // (ln(2) / 2)^2
    const float u = k * w, z = u * u;
    const float p = fmaf(fmaf(-17.f / 315.f * h * h * h, z, 2.f / 15.f * h * h), z, -h / 3.f) * z;
    const float far = cap * fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + exp2_fast(u)), 1.f);   // (2 cap may be infinite)
    return fabsf(u) < 0.57707802f ? fmaf(w, p, w) : far;   // (0.4 / ln(2))
}
// log2-domain score of a product s, without the distance term (no cap or a narrow one)
__device__ __forceinline__ float paged_score(const PagedAttn& a, float s) {
    if (a.cap == 0.f) return a.c * s;
    return fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(1.f + exp2_fast(a.c * s)), a.cap);
}

// four output values at element `at`, 16-byte (F16: 8-byte) aligned
__device__ __forceinline__ void paged_store4(const PagedAttn& a, int64_t at, floatx4 x) {
    if (a.dst_f16) {
        half4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (_Float16)x[i];
        *(half4*)((_Float16*)a.dst + at) = y;
    } else {
        *(floatx4*)((float*)a.dst + at) = x;
    }
}

struct PagedAppend {
    PagedBatch b;
    const float* k_new;       // [token][Hkv D]
    const float* v_new;
    int64_t kn_nb1, vn_nb1;
    PagedPool kv;
    int32_t d, hq, hkv;
    const int32_t* rope_pos;  // [token]; null: no rotation
    float rope_ts;
    int32_t rope_dims;
    const float* q;           // null: keys and values only
    int64_t q_nb1, q_nb2;
    _Float16* q_out;
    int64_t qo_nb1, qo_nb2;
};

struct PagedEvict {
    PagedBatch b;
    PagedPool kv;
    char* w;                  // weights [row of the page] at w + page nb3 + head nb2
    int64_t w_nb2, w_nb3;
    int32_t d, hkv;
    const int32_t* to;        // [n_streams][max_to]
    int32_t max_to;
    int32_t budget, n_sink, n_recent;
    int32_t* kept;            // [n_streams][hkv][kept_row]
    int32_t kept_row;         // entries of a row (>= min(budget, max_nkv))
    int32_t* n_out;           // null: not wanted
};

hipError_t launch_paged_append(const PagedAppend& a, hipStream_t st);
// single tokens, and a few at once (paged_rows_takes)
bool paged_rows_takes(const PagedAttn& a);
// weighed: the accumulated weights are done, too (else launch_paged_weights)
hipError_t launch_paged_rows(const PagedAttn& a, int head_dim, hipStream_t st, bool& weighed);
// any chunks (as from launch_paged_rows, before any launch: hipErrorOutOfMemory where the
// workspace does not hold the work's tables, hipErrorNotSupported beyond the grid's limit)
hipError_t launch_paged_chunk(const PagedAttn& a, int head_dim, hipStream_t st);
hipError_t launch_paged_chunk64(const PagedAttn& a, hipStream_t st);
// what the launches below take: workgroups along x
constexpr int kPagedWeightRows = 128;        // rows of a workgroup of the weights
constexpr int kPagedMoveRows = 32;           // of the eviction's move
inline bool paged_weights_fit(const PagedAttn& a) {
    return ((int64_t)a.b.max_nkv + kPagedWeightRows - 1) / kPagedWeightRows * a.hkv <= kMaxGridX;
}
inline int64_t paged_move_grid(const PagedEvict& a) {
    const int64_t rows = a.kept_row < a.b.max_nkv ? a.kept_row : a.b.max_nkv;   // kept of a stream at most
    return (rows + kPagedMoveRows - 1) / kPagedMoveRows * a.hkv;
}
inline bool paged_evict_fits(const PagedEvict& a) { return paged_move_grid(a) <= kMaxGridX; }

hipError_t launch_paged_weights(const PagedAttn& a, int head_dim, hipStream_t st);
hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t st);

}  // namespace vxfa
