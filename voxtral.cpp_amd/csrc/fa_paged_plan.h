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

// All streams' rows are cut into `small` parts per head group (512 workgroups), two
// a CU at once; where these would hold more than `limit` rows, into parts of that
// many, up to `large` (2048 workgroups), so that streams of uneven lengths leave no
// long last round. (Parts of 1024 rows: 16 equal streams of 8192 107.9 -> 103.7 us,
// 32 uneven ones with weights 151.6 -> 155.3; of 2048: uneven ones +3 to 7 %.)
struct RowsPlan {
    int32_t small, large;
    int32_t limit;
    int32_t cuts;             // 0: a part per stream
    int32_t empty;            // 1: one, too, for a stream without tokens
};

// Whether streams are left whole: what a cut costs (its join, a launch of its own)
// against what it gains, by the bounds. In us: a workgroup alone takes about 10.5 ns
// a row (hd 64: 6.5), all together move 5.6 TB/s; the streams are taken for seven
// tenths of the bound on average, and for too uneven beyond 2048 rows. Measured, cut
// -> whole, 8 kv heads of 128: 1 stream of 256 rows 8.5 -> 7.1, of 512 8.6 -> 9.8; 4
// uneven ones of up to 256 8.8 -> 6.9, 1024 9.5 -> 12.7; 16 of up to 512 12.1 -> 10.3,
// 2048 22.1 -> 27.5; 32 of up to 1024 24.2 -> 18.3, 2048 35.7 -> 32.4, 8192 102.8 ->
// 117.4. Over 196 mixes of heads, streams and rows (half of them even, half uneven)
// the rule is 0.5 % off the better choice on average, 15 % at worst: 1 stream
// that is shorter than its bound of 512.
// i8: pages of 8 bits, by another kernel, which gains more by a cut: a workgroup alone
// 7.5 ns a row (hd 64: 5), and none whole beyond 1024 rows. Cut -> whole, 8 kv heads of
// 128: 1 stream of 256 rows 7.7 -> 6.0, of 512 7.5 -> 8.2; 4 uneven ones of 1024 8.8 ->
// 12.5; 16 of 512 12.1 -> 10.4; 32 uneven ones of 512 12.8 -> 10.4, of 2048 24.6 -> 31.5;
// 20 heads of 64: 8 of 512 10.8 -> 9.4, of 1024 13.5 -> 15.9, 32 of 2048 44.9 -> 56.8. Over
// 195 mixes 0.5 % off the better choice, 31 % at worst (2 streams that are shorter than
// their bound of 512); by the rule for F16 3.3 %, 52 %.
inline bool rows_whole(const PagedBatch& b, int nhg, int head_dim, bool i8) {
    if (i8) {
        const double n = 1e-3 * b.max_nkv, alone = head_dim == 128 ? 7.5 : 5.0;
        const double together = (double)b.n_streams * nhg * 2 * head_dim / 5600;
        return b.max_nkv <= 1024 && n * (alone > 0.7 * together ? alone : 0.7 * together) < 2.5 + 0.6 * n * together;
    }
    const double n = 1e-3 * b.max_nkv, alone = head_dim == 128 ? 10.5 : 6.5;
    const double together = 0.7 * (double)b.n_streams * nhg * 4 * head_dim / 5600;
    return b.max_nkv <= 2048 && 4.5 + n * (alone > together ? alone : together) < 7.5 + 1.05 * n * together;
}

// The grid of a call: `items` parts per head group.
inline RowsPlan rows_plan(const PagedBatch& b, int nhg, int head_dim, int64_t room, int32_t& items, bool i8 = false) {
    RowsPlan p;
    p.empty = 0;
    p.small = 512 / nhg > 0 ? 512 / nhg : 1;
    p.large = 2048 / nhg > 0 ? 2048 / nhg : 1;
    p.limit = 512;
    // n parts' worth of rows are at most n parts of one stream, n + streams of more
    const int64_t more = b.n_streams > 1 ? b.n_streams : 0;
    const int64_t all = (int64_t)b.n_streams * b.max_nkv;
    if (all <= (int64_t)p.small * p.limit) p.large = p.small;
    p.cuts = 1;
    while (p.cuts && (int64_t)p.large + more > room) {
        if (p.large > 64) p.large /= 2;
        else p.cuts = 0;
    }
    if (p.small > p.large) p.small = p.large;
    if (rows_whole(b, nhg, head_dim, i8)) p.cuts = 0;
    items = b.n_streams;
    if (p.cuts) {
        const int64_t by_rows = (int64_t)b.n_streams * ((b.max_nkv + 63) / 64);
        const int64_t by_parts = (int64_t)p.large + more;
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
// the first row that any of a stream's tokens sees, down to a whole tile
__device__ __forceinline__ int rows_first(const PagedStream& s, int window) {
    return window > 0 ? max(s.n - s.t - window + 1, 0) & ~15 : 0;
}

#endif

// rows of a part, given all streams' rows: whole rounds of four tiles
__host__ __device__ __forceinline__ int rows_chunk(const RowsPlan& p, int64_t total) {
    // (a division of 64 bits takes a hundred instructions: only where it has to be one)
    auto parts_of = [&](int32_t n) -> int64_t {
        if (total <= 0x40000000) return (int64_t)(((uint32_t)total + (uint32_t)n - 1) / (uint32_t)n);
        return (total + n - 1) / n;
    };
    int64_t c = parts_of(p.small);
    if (c > p.limit) {
        c = parts_of(p.large);
        if (c < p.limit) c = p.limit;
    }
    c = (c + 63) & ~(int64_t)63;
    return c < 64 ? 64 : (c > 0x40000000 ? 0x40000000 : (int)c);
}
// all streams' rows as rows_chunk takes them: `tiles` whole tiles, and what is left of
// each stream counted as a tile less one row
__host__ __device__ __forceinline__ int64_t rows_total(int64_t tiles, int n_streams) { return 16 * tiles + 15 * (int64_t)n_streams; }
// parts of a stream of len rows
__host__ __device__ __forceinline__ int rows_parts(const RowsPlan& p, int len, int chunk) {
    // (both at most 2^30)
    return p.cuts && len > chunk ? (int)(((uint32_t)len + (uint32_t)chunk - 1) / (uint32_t)chunk) : 1;
}

#ifdef __HIPCC__
__device__ __forceinline__ Part rows_locate(const PagedBatch& b, const RowsPlan& p, int window, int item) {
    Part r;
    const int lane = (int)threadIdx.x & 63;
    auto parts = [&](const PagedStream& s, int chunk) -> int {
        if (s.t <= 0) return s.t == 0 ? p.empty : 0;   // (-1: no such stream)
        return rows_parts(p, s.n - rows_first(s, window), chunk);
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
        PagedStream s{0, -1, 0};
        if (s0 + lane < b.n_streams) s = paged_stream(b, s0 + lane);
        if (s0 == 0) mine = s;
        if (p.cuts) total += wave_sum(s.t > 0 ? max(s.n - rows_first(s, window), 0) >> 4 : 0);
    }
    const int chunk = rows_chunk(p, rows_total(total, b.n_streams));
    int before = 0;
    r.s = -1;
    for (int s0 = 0; s0 < b.n_streams; s0 += 64) {
        PagedStream s = mine;
        if (s0 > 0) {
            s = PagedStream{0, -1, 0};
            if (s0 + lane < b.n_streams) s = paged_stream(b, s0 + lane);
        }
        const int n = parts(s, chunk);
        const int incl = wave_scan(n);
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

// ---- chunks -------------------------------------------------------------------
// A stream's tokens in tiles (bm positions), the rows that a tile walks in
// pieces; all tiles of a stream have as many pieces. The pieces' length `lp`
// (blocks of 32 rows) is one of 64 that the lanes weigh.

struct ChunkPlan {
    uint32_t hpw_log2;        // log2 of the query heads per workgroup
    int32_t kvg;              // groups of wavefronts that share a piece's blocks
    int32_t cuts;             // 0: a piece per tile
    int32_t pieces;           // > 0: pieces of the longest walk (else chunk_choose's)
    int32_t items;            // pieces in the grid per head group
    int32_t tiles;            // tiles of all streams at most (sizes that break the bounds: the rest is left out)
    int32_t room;             // records (of a workgroup's piece) per head group
    int32_t nhg;
};
struct ChunkTile {
    int32_t s, tile, n, slot; // stream, tile, its pieces, its first record
};
struct ChunkBounds {
    int64_t tiles;            // tiles of all streams at most
    size_t table;             // bytes of their ChunkTiles
};
constexpr int kChunkStreams = 64;   // more streams are not cut

// A cut's time in blocks of 32 rows: `total` blocks of a head group, in `items`
// workgroups (of each head group) of `lp` at most. A workgroup costs its blocks
// (shared among kvg groups of wavefronts) and kWg, 256 run at once; a record costs
// its traffic, and the joining of a walk's pieces goes one after another. Measured,
// pieces as chosen by it -> the best of 1 to 16 that were forced (VXFA_PAGED_PIECES), us:
// 600 tokens on 3000 rows 61.4 -> 61.4 (3 pieces; 2 69.6, uncut 104), 300 on 7892 68.9 ->
// 68.3, 100 on 8092 45.3 -> 44.9, 1200 on 1200 42.0 -> 42.4, 2 streams of 256 on 4000 57.6 ->
// 56.8, 4 uneven ones of up to 500 on 4000 53.7 -> 56.0 (of one count for all); 20 heads of
// 64: 600 on 3000 35.2 -> 33.9, 100 on 8092 29.3 -> 29.1.
__host__ __device__ inline float chunk_cost(float total, int items, int recs, int lp, int nhg, int pieces, int kvg) {
    constexpr float kWg = 4.f, kRecord = 0.05f, kPiece = 0.3f;
    const float count = (float)(items * nhg), rounds = ceilf(count * (1.f / 256.f));
    const float share = 1.f / (float)kvg;
    return fmaxf(rounds * (share * total * (float)nhg / fmaxf(count, 1.f) + kWg), share * (float)lp + kWg) + kRecord * (float)(recs * nhg) +
           (recs ? kPiece * (float)pieces : 0.f);
}
// length of the pieces of a walk of nb blocks in n pieces: whole steps
__host__ __device__ inline int chunk_length(int nb, int n) {
    const int l = ((nb + n - 1) / n + 1) & ~1;
    return l > 4 ? l : 4;
}
// all blocks of a stream's tiles, the last of which walks nb: one before it walks
// bm / 32 less, but for a window
__host__ __device__ inline float chunk_blocks(int tiles, int nb, int bm, int window) {
    const float all = (float)tiles * (float)nb;
    if (window > 0) return all;
    const float less = all - (float)(bm / 32) * 0.5f * (float)tiles * (float)(tiles - 1);
    return less > (float)tiles ? less : (float)tiles;
}

inline ChunkBounds chunk_plan(const PagedBatch& b, int head_dim, int nhg, int bm, int window, size_t record, size_t ws_bytes, ChunkPlan& p) {
    ChunkBounds r;
    // sum of ceil(t / bm) over streams of `tokens` tokens in all, max_nq at most each
    const int64_t per = ((int64_t)b.max_nq + bm - 1) / bm;
    r.tiles = (int64_t)b.tokens / bm + b.n_streams;
    if (b.n_streams == 1) r.tiles = ((int64_t)b.tokens + bm - 1) / bm;
    if (r.tiles > per * b.n_streams) r.tiles = per * b.n_streams;
    if (r.tiles > b.tokens) r.tiles = b.tokens;
    r.table = ((size_t)(1 + r.tiles) * sizeof(ChunkTile) + 255) & ~(size_t)255;
    p.nhg = nhg;
    p.kvg = head_dim == 64 && r.tiles * nhg <= 256 ? 2 : 1;
    p.tiles = (int32_t)r.tiles;
    const int64_t room = r.table < ws_bytes ? (int64_t)((ws_bytes - r.table) / (record * (size_t)nhg)) : 0;
    p.room = (int32_t)(room < 4096 ? room : 4096);
    int64_t nb = ((int64_t)b.max_nkv + 31) / 32;          // blocks of the longest walk
    if (window > 0 && nb > ((int64_t)window + bm) / 32 + 1) nb = ((int64_t)window + bm) / 32 + 1;
    // Not cut: tiles for two rounds of the chip's 256 CUs (16 streams of up to 512
    // tokens on up to 4096 rows, 600 workgroups: uncut 169 us, in halves 172), or for
    // one round and more where the longest walk is short, so that a cut gains less than
    // its join's launch takes (cut -> uncut, 320 workgroups: 8 streams of 250 tokens,
    // 20 heads of 64, window 750 37.9 -> 35.2 us, 1500 rows 43.8 -> 41.1; 4 of 634, 32/8
    // heads of 128, 1500 rows 92.6 -> 89.0; but uneven ones, 4 streams of up to 890 tokens
    // of 20 heads, 2000 rows 37.3 -> 35.4, 4000 56.5 -> 61.7, 8192 79.9 -> 113.4; 16 of
    // up to 512, a cap, 2048 rows 136.8 -> 142.1), or too few rows.
    p.cuts = r.tiles * nhg < (nb > 48 ? 512 : 257) && b.max_nkv >= 128 && b.n_streams <= kChunkStreams && p.room >= 2;
    int64_t items = r.tiles;
    if (p.cuts) items = r.tiles > 512 / nhg ? r.tiles : (512 / nhg > 1 ? 512 / nhg : 1);
    if (p.cuts && items < 2) items = 2;
    if (p.cuts && p.pieces == 0 && b.n_streams == 1) {
        // one stream, whose sizes are near the bounds: the pieces are chosen here,
        // and the grid holds no more
        const int tiles = (int)r.tiles;
        float best = 3.0e38f;
        p.pieces = 1;
        for (int n = 1; n <= 64; ++n) {
            const int lp = chunk_length((int)nb, n), k = n == 1 ? 1 : (int)((nb + lp - 1) / lp), all = k * tiles;
            if (k > 1 && all > p.room) break;
            const float cost = chunk_cost(chunk_blocks(tiles, (int)nb, bm, window), all, k > 1 ? all : 0, lp, nhg, k, p.kvg);
            if (cost < best) {
                best = cost;
                p.pieces = k;
            }
        }
    }
    if (p.pieces > 64) p.pieces = 64;
    if (p.pieces > 0) items = r.tiles * p.pieces;
    if (p.pieces == 1) p.cuts = 0;
    p.items = (int32_t)items;
    return r;
}

// piece `piece` of the n of tile `tile` of stream s (-1: none); slot: the tile's
// first record; tile_no: its number among all tiles, of which there are `tiles`
struct ChunkItem {
    int s, tile, piece, n, slot, tile_no, tiles;
    PagedStream st;
};

#ifdef __HIPCC__
// pieces of at most 1 / inv blocks of a walk of nb, nb > 0: ceil(nb / lp) (exact
// for fewer than 2^20 blocks, the half keeping clear of the steps; beyond, one
// more or less does no harm)
__device__ __forceinline__ int chunk_pieces(int nb, int lp, float inv) { return (int)(((float)(nb + lp - 1) + 0.5f) * inv); }

// Up to 64 streams, a lane each: their tiles (none past the last stream), blocks
// that the longest tile walks, and pieces per tile.
__device__ __forceinline__ int chunk_choose(const PagedBatch& b, const ChunkPlan& p, int window, int bm, int lane,
                                            const PagedStream& st, int tiles, int& nb) {
    // blocks that the last tile walks, which is the longest
    int lo = 0;
    if (window > 0) lo = max(st.n - st.t + (tiles - 1) * bm - window + 1, 0) / 32;
    nb = tiles > 0 ? max((st.n + 31) / 32 - lo, 1) : 0;
    if (!p.cuts) return 1;
    // all blocks: a tile before it walks bm / 32 less
    float total = tiles > 0 ? chunk_blocks(tiles, nb, bm, window) : 0.f;
    int longest = nb;
    if (b.n_streams > 1) {
        longest = wave_max(longest);
        total = wave_sum(total);
    } else {
        longest = __builtin_amdgcn_readfirstlane(longest);
    }
    if (p.pieces > 0) {
        // (those of the longest walk, where their records fit)
        const int lp = chunk_length(longest, p.pieces), n = max((nb + lp - 1) / lp, 1);
        int recs = n > 1 ? n * tiles : 0;
        if (b.n_streams > 1) recs = wave_sum(recs);
        else recs = __builtin_amdgcn_readfirstlane(recs);
        return recs <= p.room ? n : 1;
    }
    // this lane's length, from the longest walk down to a 64th of it
    const int lp = lane == 0 ? longest : max((int)((uint32_t)longest * (uint32_t)(64 - lane) >> 6) & ~1, 4);
    const float inv = __builtin_amdgcn_rcpf((float)max(lp, 1));
    int items = 0, recs = 0;
    for (int s = 0; s < b.n_streams; ++s) {
        const int n = chunk_pieces(__builtin_amdgcn_readlane(nb, s), lp, inv), ts = __builtin_amdgcn_readlane(tiles, s);
        items += n * ts;
        recs += n > 1 ? n * ts : 0;
    }
    float cost = chunk_cost(total, items, recs, lp, p.nhg, chunk_pieces(longest, lp, inv), p.kvg);
    if (items > p.items || recs > p.room) cost = 3.0e38f;
    if (lane == 0) cost = fminf(cost, 1.0e38f);   // (one piece a tile always fits)
    // (costs are positive: they order as integers)
    const float best = __builtin_bit_cast(float, -wave_max(-__builtin_bit_cast(int, cost)));
    const int pick = (int)__builtin_ctzll(__ballot(cost == best));
    const float inv_pick = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, inv), pick));
    return pick == 0 ? 1 : max(chunk_pieces(nb, __builtin_amdgcn_readlane(lp, pick), inv_pick), 1);
}

__device__ __forceinline__ ChunkItem chunk_locate(const PagedBatch& b, const ChunkPlan& p, int window, int bm, int item) {
    const int lane = (int)threadIdx.x & 63;
    ChunkItem r;
    r.s = -1;
    r.tiles = 0;
    int before = 0;
    for (int s0 = 0; s0 < b.n_streams; s0 += 64) {
        PagedStream st{0, 0, 0};
        if (s0 + lane < b.n_streams) st = paged_stream(b, s0 + lane);
        const int tiles = (min(st.t, b.max_nq) + bm - 1) / bm;
        int nb, np;
        np = chunk_choose(b, p, window, bm, lane, st, tiles, nb);
        // pieces, tiles and records of the streams ahead of the lane's: those of longer
        // walks (and, of equal ones, the earlier)
        const int n = tiles * np, rec = np > 1 ? n : 0;
        int ahead = 0, tahead = 0, rahead = 0, all = 0, tall = 0;
        for (int s = 0; s < min(b.n_streams - s0, 64); ++s) {
            const int nbs = __builtin_amdgcn_readlane(nb, s), ns = __builtin_amdgcn_readlane(n, s);
            const int ts = __builtin_amdgcn_readlane(tiles, s), rs = __builtin_amdgcn_readlane(rec, s);
            const bool first = nbs > nb || (nbs == nb && s < lane);
            ahead += first ? ns : 0;
            tahead += first ? ts : 0;
            rahead += first ? rs : 0;
            all += ns;
            tall += ts;
        }
        const int mine = item - before - ahead;
        const uint64_t hit = r.s < 0 ? __ballot(mine >= 0 && mine < n) : 0;
        if (hit) {
            const int w = (int)__builtin_ctzll(hit);
            r.s = s0 + w;
            r.n = __builtin_amdgcn_readlane(np, w);
            const int ts = __builtin_amdgcn_readlane(tiles, w), i = __builtin_amdgcn_readlane(mine, w);
            r.tile = ts - 1 - i / r.n;              // the longest first
            r.piece = i % r.n;
            r.slot = r.n > 1 ? __builtin_amdgcn_readlane(rahead, w) + (i - r.piece) : 0;
            r.tile_no = r.tiles + __builtin_amdgcn_readlane(tahead, w) + r.tile;
            r.st.q0 = __builtin_amdgcn_readlane(st.q0, w);
            r.st.t = __builtin_amdgcn_readlane(st.t, w);
            r.st.n = __builtin_amdgcn_readlane(st.n, w);
            if (r.tile_no >= p.tiles) r.s = -1;
        }
        before += all;
        r.tiles += tall;
        if (hit && item > 0) return r;              // (the first one goes on to count the tiles)
    }
    // (sizes that break the bounds: tiles of which no workgroup knows are not joined)
    r.tiles = before > p.items ? 0 : min(r.tiles, p.tiles);
    return r;
}
#endif

}  // namespace vxfa
