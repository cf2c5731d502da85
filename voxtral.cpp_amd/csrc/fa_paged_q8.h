// fa_paged_q8.h — what the kernels over pages of 8 bits and over chosen blocks
// share: launch descriptors, scales, whole numbers of 8 bits as f16, units of work.
#pragma once

#include "fa_paged.h"

namespace vxfa {

constexpr int kScaleRows = 16;                        // rows that share a scale
constexpr int kSelectSeg = 4096, kSelectMost = 262144; // blocks of a segment of the choice at most, of a stream
constexpr int kMaxTop = 1024;                         // blocks chosen
constexpr int kMinExp = -64, kMaxExp = 64;            // of a scale

// Scales of a pool: F32 of rows 16 i .. of head h in page p at base + p nb3 + h nb2 + 4 i.
struct PagedScales {
    char *k, *v;
    int64_t nb2, nb3;
    __device__ __forceinline__ int64_t at(int page, int h, int r) const { return page * nb3 + h * nb2 + 4 * (int64_t)(r / kScaleRows); }
};

struct PagedAppend8 {
    PagedAppend a;
    PagedScales sc;
    double rope_ts;                                   // a.rope_ts in 64 bits
};

// Bounds of blocks: rows [block of the page] of 2 D bytes at b + page nb3 + head nb2 +
// block nb1, their scales at s + page s_nb3 + head s_nb2 + 4 block.
struct PagedBoundRows {
    char *b, *s;
    int64_t nb1, nb2, nb3, s_nb2, s_nb3;
    int32_t lg;                                       // log2 of a block's rows
};

struct PagedBounds {
    PagedBatch b;
    PagedPool kv;                                     // (v: null)
    PagedScales sc;                                   // k null: an F16 pool
    PagedBoundRows out;
    int32_t d, hkv;
};

struct PagedSelect {
    PagedBatch b;
    const void* q;
    int64_t q_nb1, q_nb2;
    uint8_t q_f16;
    int32_t d, hq, hkv, window;
    PagedBoundRows in;
    int32_t* list;                                    // [token][hkv][top]
    int32_t top, n_sink, n_recent;
    char* ws;
    size_t ws_bytes;
};

// Attention over chosen blocks (list null: all rows)
struct PagedBlocks {
    PagedAttn a;
    PagedScales sc;                                   // k null: an F16 pool
    const int32_t* list;                              // [token][hkv][top]
    int32_t top;
    int32_t lg;                                       // log2 of a block's rows
};

hipError_t launch_paged_append_q8(const PagedAppend8& a, hipStream_t st);
hipError_t launch_paged_bounds(const PagedBounds& a, hipStream_t st);
hipError_t launch_paged_select(const PagedSelect& a, hipStream_t st);
// single tokens and a few at once over pages of 8 bits (paged_rows_takes)
hipError_t launch_paged_rows_q8(const PagedBlocks& a, int head_dim, hipStream_t st);
// any tokens over chosen blocks
hipError_t launch_paged_blocks(const PagedBlocks& a, int head_dim, hipStream_t st);
// chunks over pages of 8 bits
hipError_t launch_paged_chunk_q8(const PagedAttn& a, const PagedScales& sc, int head_dim, hipStream_t st);
hipError_t launch_paged_chunk64_q8(const PagedAttn& a, const PagedScales& sc, hipStream_t st);

// 2^e as F32
__host__ __device__ __forceinline__ float two_to(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// The least e from kMinExp to kMaxExp with x <= 127 2^e (x >= 0; NaN as infinity). 127 2^e is
// (2 - 2^-6) 2^(e + 6): a mantissa up to 0x7E0000 leaves x's own exponent less 6, a larger one
// adds one, which the carry of the addition does.
__host__ __device__ __forceinline__ int exp_for(float x) {
    const int e = (int)((__builtin_bit_cast(uint32_t, x) + 0x1FFFFu) >> 23) - 133;
    return e < kMinExp ? kMinExp : (e > kMaxExp ? kMaxExp : e);
}

#ifdef __HIPCC__
// A scale as attention takes it: NaN and what lies outside brought into the range, so
// that rows which no token sees (whose scales may be anything) take part as zeros.
__device__ __forceinline__ float scale_in_range(float s) { return fminf(fmaxf(s, two_to(kMinExp)), two_to(kMaxExp)); }

// The four bytes of w, in order, as f16: with the sign bit turned over (b + 128) and 0x64 above
// it a byte is the f16 number 1024 + (b + 128), exact, from which 1152 leaves b.
__device__ __forceinline__ half4 half4_of_bytes(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const half2 off = {(_Float16)1152.f, (_Float16)1152.f};
    const half2 lo = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    const half2 hi = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    return half4{lo[0], lo[1], hi[0], hi[1]};
}
// Two bytes b + 128 in the low halves' bits (the high bytes 0) as f16 numbers b / 512: as f16 the bits are
// (b + 128) 2^-24, subnormal and exact; one multiply-add.
__device__ __forceinline__ half2 halves_over_512(uint32_t w) {
    const half2 f = {(_Float16)32768.f, (_Float16)32768.f}, off = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_elementwise_fma(__builtin_bit_cast(half2, w), f, off);
}
__device__ __forceinline__ half8 half8_of_bytes(uint32_t w0, uint32_t w1) {
    const half4 lo = half4_of_bytes(w0), hi = half4_of_bytes(w1);
    return half8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Unit `item` of a batch whose streams have count(stream) units each, in order: its
// stream (-1: none) and its number there.
struct PagedUnit {
    int s, i;
    PagedStream st;
};
template <class F>
__device__ __forceinline__ PagedUnit paged_unit(const PagedBatch& b, int item, F count) {
    const int lane = (int)threadIdx.x & 63;
    PagedUnit r;
    r.s = -1;
    int before = 0;
    for (int s0 = 0; s0 < b.n_streams; s0 += 64) {
        PagedStream s{0, 0, 0};
        if (s0 + lane < b.n_streams) s = paged_stream(b, s0 + lane);
        // (no grid has more: sizes that break the bounds do not overflow the sums)
        const int n = s.t > 0 ? min(count(s), 1 << 24) : 0;
        const int incl = wave_scan(n);
        const uint64_t hit = __ballot(before + incl > item);
        if (hit) {
            const int w = (int)__builtin_ctzll(hit);
            r.s = s0 + w;
            r.i = item - before - __builtin_amdgcn_readlane(incl - n, w);
            r.st.q0 = __builtin_amdgcn_readlane(s.q0, w);
            r.st.t = __builtin_amdgcn_readlane(s.t, w);
            r.st.n = __builtin_amdgcn_readlane(s.n, w);
            return r;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return r;
}
// The stream of packed token t (-1: none, or past max_nq of it; the first where chunks overlap).
__device__ __forceinline__ PagedUnit paged_token(const PagedBatch& b, int t) {
    const int lane = (int)threadIdx.x & 63;
    PagedUnit r;
    r.s = -1;
    for (int s0 = 0; s0 < b.n_streams; s0 += 64) {
        PagedStream s{0, 0, 0};
        if (s0 + lane < b.n_streams) s = paged_stream(b, s0 + lane);
        const uint64_t hit = __ballot(t >= s.q0 && t - s.q0 < min(s.t, b.max_nq));
        if (hit) {
            const int w = (int)__builtin_ctzll(hit);
            r.s = s0 + w;
            r.st.q0 = __builtin_amdgcn_readlane(s.q0, w);
            r.st.t = __builtin_amdgcn_readlane(s.t, w);
            r.st.n = __builtin_amdgcn_readlane(s.n, w);
            r.i = t - r.st.q0;
            return r;
        }
    }
    return r;
}

// Blocks of 2^lg rows that a stream's new tokens (those looked at) lie in: the first, and how many.
__device__ __forceinline__ int blocks_first(const PagedStream& s, int lg) { return max(s.n - s.t, 0) >> lg; }
__device__ __forceinline__ int blocks_count(const PagedStream& s, int max_nq, int lg) {
    const int end = s.n - s.t + min(s.t, max_nq);       // rows up to the last token's
    return end > 0 && max_nq > 0 ? ((end - 1) >> lg) - blocks_first(s, lg) + 1 : 0;
}
#endif
// of all streams, at most
inline int64_t blocks_bound(const PagedBatch& b, int lg) {
    const int64_t n = ((int64_t)b.tokens >> lg) + 2 * (int64_t)b.n_streams;
    return n < b.tokens ? n : b.tokens;
}

}  // namespace vxfa
