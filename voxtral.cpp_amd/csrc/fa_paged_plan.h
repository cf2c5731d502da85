// fa_paged_plan.h — how the rows of a batch's streams are cut into parts, one
// workgroup (per head group) each. The sizes are known on the device only, so
// the host fixes the grid from their bounds and every workgroup finds its part
// by a scan over the streams, a lane each.
#pragma once

#include "fa_paged.h"

namespace vxfa {

// Query heads that share a workgroup of 16 query rows: the group's heads, in
// equal shares where they are more than 16.
inline int rows_heads(int group) {
    const int n = (group + 15) / 16;
    return n > 0 ? (group + n - 1) / n : 1;
}

struct RowsPlan {
    int32_t small, large;     // parts (per head group) that all streams' rows are cut into
    int32_t limit;            // rows of a part from which `large` holds
    int32_t cuts;             // 0: a part per stream
};

// The grid of a call: `items` parts per head group.
inline RowsPlan rows_plan(const PagedBatch& b, int nhg, int64_t room, int32_t& items) {
    RowsPlan p;
    p.small = 512 / nhg > 0 ? 512 / nhg : 1;
    p.large = 2048 / nhg > 0 ? 2048 / nhg : 1;
    p.limit = 512;
    // with n parts' worth of rows, streams of their own rounding: n + streams at most
    const int64_t all = (int64_t)b.n_streams * b.max_nkv;
    if (all <= (int64_t)p.small * p.limit) p.large = p.small;
    p.cuts = 1;
    while (p.cuts && (int64_t)p.large + b.n_streams > room) {
        if (p.large > 64) p.large /= 2;
        else p.cuts = 0;
    }
    if (p.small > p.large) p.small = p.large;
    if (b.max_nkv <= 64) p.cuts = 0;
    items = b.n_streams;
    if (p.cuts) {
        const int64_t by_rows = (int64_t)b.n_streams * ((b.max_nkv + 63) / 64);
        const int64_t by_parts = (int64_t)p.large + b.n_streams;
        items = (int32_t)(by_rows < by_parts ? by_rows : by_parts);
    }
    return p;
}

// A part: piece of n of stream s (-1: none), whose rows from lo on count (a
// multiple of 16), and the number of the stream's first part.
struct Part {
    int s, piece, n, first, lo;
    PagedStream st;
};

#ifdef __HIPCC__
__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) x += __shfl_xor(x, w, 64);
    return x;
}

// the first row that any of a stream's tokens sees, down to a whole tile
__device__ __forceinline__ int rows_first(const PagedStream& s, int window) {
    return window > 0 ? max(s.n - s.t - window + 1, 0) & ~15 : 0;
}

// rows of a part, given all streams' rows: whole rounds of four tiles
__device__ __forceinline__ int rows_chunk(const RowsPlan& p, int64_t total) {
    int64_t c = (total + p.small - 1) / p.small;
    if (c > p.limit) {
        c = (total + p.large - 1) / p.large;
        if (c < p.limit) c = p.limit;
    }
    c = (c + 63) & ~(int64_t)63;
    return c < 64 ? 64 : (c > 0x40000000 ? 0x40000000 : (int)c);
}

__device__ __forceinline__ Part rows_locate(const PagedBatch& b, const RowsPlan& p, int window, int item) {
    Part r;
    const int lane = (int)threadIdx.x & 63;
    auto parts = [&](const PagedStream& s, int chunk) -> int {
        if (s.t <= 0) return 0;
        const int len = s.n - rows_first(s, window);
        return p.cuts && len > chunk ? (len + chunk - 1) / chunk : 1;
    };
    if (b.n_streams == 1) {
        r.st = paged_stream(b, 0);
        r.lo = rows_first(r.st, window);
        r.n = parts(r.st, rows_chunk(p, max(r.st.n - r.lo, 0)));
        r.first = 0;
        r.piece = item;
        r.s = item < r.n ? 0 : -1;
        return r;
    }
    // all streams' rows; the first 64 streams stay in registers
    PagedStream mine{0, 0, 0};
    int64_t total = 0;
    for (int s0 = 0; s0 < b.n_streams; s0 += 64) {
        PagedStream s{0, 0, 0};
        if (s0 + lane < b.n_streams) s = paged_stream(b, s0 + lane);
        if (s0 == 0) mine = s;
        if (p.cuts) total += wave_sum(s.t > 0 ? max(s.n - rows_first(s, window), 0) >> 4 : 0);
    }
    const int chunk = rows_chunk(p, 16 * total + 15 * (int64_t)b.n_streams);
    int before = 0;
    r.s = -1;
    for (int s0 = 0; s0 < b.n_streams; s0 += 64) {
        PagedStream s = mine;
        if (s0 > 0) {
            s = PagedStream{0, 0, 0};
            if (s0 + lane < b.n_streams) s = paged_stream(b, s0 + lane);
        }
        const int n = parts(s, chunk);
        int incl = n;
#pragma unroll
        for (int w = 1; w < 64; w <<= 1) {
            const int y = __shfl_up(incl, w, 64);
            if (lane >= w) incl += y;
        }
        const uint64_t hit = __ballot(before + incl > item);
        if (hit) {
            const int w = (int)__builtin_ctzll(hit);
            r.s = s0 + w;
            r.n = __builtin_amdgcn_readlane(n, w);
            r.first = before + __builtin_amdgcn_readlane(incl, w) - r.n;
            r.piece = item - r.first;
            r.st.q0 = __builtin_amdgcn_readlane(s.q0, w);
            r.st.t = __builtin_amdgcn_readlane(s.t, w);
            r.st.n = __builtin_amdgcn_readlane(s.n, w);
            r.lo = rows_first(r.st, window);
            return r;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return r;
}
#endif

}  // namespace vxfa
