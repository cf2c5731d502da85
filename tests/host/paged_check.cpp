// Host check of the paged entry points (vxfa_paged.cpp, linked in, no GPU): the
// HIP calls are stand-ins and the launchers note their arguments. Valid calls
// reach the right launcher with the sizes as documented; every violation comes
// back as its status and launches nothing; and the grids that the host fixes from
// the bounds hold the parts that random batches within the bounds are cut into.
// Built and run by tests/test_paged_checks.py.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <random>
#include <string>
#include <vector>

#include "../../include/vxfa.h"
#include "../../voxtral.cpp_amd/csrc/fa_paged.h"
#include "../../voxtral.cpp_amd/csrc/fa_paged_plan.h"
#include "../../voxtral.cpp_amd/csrc/vxfa_ctx.h"

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
}

static int g_launches = 0, g_bad = 0;
static std::string g_last;
static vxfa::PagedAttn g_attn;
static vxfa::PagedEvict g_evict;
static vxfa::PagedAppend g_append;
namespace vxfa {
hipError_t launch_paged_append(const PagedAppend& a, hipStream_t) { ++g_launches; g_last = "append"; g_append = a; return hipSuccess; }
bool paged_rows_takes(const PagedAttn& a) { return (int64_t)a.b.max_nq * rows_heads(a.hq / a.hkv) <= 16; }
hipError_t launch_paged_rows(const PagedAttn& a, int, hipStream_t, bool& w) { ++g_launches; g_last = "rows"; g_attn = a; w = true; return hipSuccess; }
hipError_t launch_paged_chunk(const PagedAttn& a, int, hipStream_t) { ++g_launches; g_last = "chunk"; g_attn = a; return hipSuccess; }
hipError_t launch_paged_weights(const PagedAttn& a, int, hipStream_t) { ++g_launches; g_last += "+weights"; g_attn = a; return hipSuccess; }
hipError_t launch_paged_evict(const PagedEvict& a, hipStream_t) { ++g_launches; g_last = "evict"; g_evict = a; return hipSuccess; }
}  // namespace vxfa

#define CHECK(x) do { if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); ++g_bad; } } while (0)

static void* const kAddr = reinterpret_cast<void*>(0x7e0000000000ull);   // (never dereferenced)

static vxfa_tensor tensor(int type, int64_t n0, int64_t n1, int64_t n2, int64_t n3) {
    vxfa_tensor t;
    std::memset(&t, 0, sizeof(t));
    t.data = kAddr;
    t.type = type;
    const int64_t ne[4] = {n0, n1, n2, n3};
    size_t nb = type == VXFA_TYPE_F16 ? 2 : 4;
    for (int d = 0; d < 4; ++d) { t.ne[d] = ne[d]; t.nb[d] = nb; nb *= (size_t)(ne[d] > 0 ? ne[d] : 1); }
    return t;
}

struct Call {
    vxfa_tensor k, v, q, dst, w, w_in, kn, vn, qf, qo;
    vxfa_paged b;
    vxfa_evict e;
    vxfa_rope r;
    float scale = 0.1f, bias = 0.f, cap = 0.f;
    Call() {
        // a pool [page][head][row][D] of 100 pages of 16 rows, 2 heads of 128
        k = v = tensor(VXFA_TYPE_F16, 128, 16, 2, 100);
        q = tensor(VXFA_TYPE_F16, 128, 7, 8, 1);
        q.nb[1] = 128 * 8 * 2; q.nb[2] = 256;
        dst = tensor(VXFA_TYPE_F16, 128, 8, 7, 1);
        w = w_in = tensor(VXFA_TYPE_F32, 16, 2, 100, 1);
        kn = vn = tensor(VXFA_TYPE_F32, 256, 7, 1, 1);
        qf = tensor(VXFA_TYPE_F32, 128, 7, 8, 1);
        qo = tensor(VXFA_TYPE_F16, 128, 7, 8, 1);
        const int32_t* p = static_cast<const int32_t*>(kAddr);
        b = vxfa_paged{p, p + 1, p + 2, 3, 10, 5, 0, 0, 0};
        e = vxfa_evict{p, 4, 50, 4, 10, const_cast<int32_t*>(p), nullptr};
        r = vxfa_rope{p, 128, 0, 1e6f, 1.0f};
    }
};

static vxfa_ctx g_ctx;
static int attend(Call& c, bool w = true, bool wi = true) {
    return vxfa_flash_attn_ext_paged(&g_ctx, &c.q, &c.k, &c.v, &c.b, &c.dst, c.scale, c.bias, c.cap, wi ? &c.w_in : nullptr,
                                     w ? &c.w : nullptr, nullptr);
}
static int append(Call& c, bool rope = true, bool q = true) {
    return vxfa_paged_append(&g_ctx, &c.kn, &c.vn, &c.b, &c.k, &c.v, rope ? &c.r : nullptr, q ? &c.qf : nullptr,
                             q ? &c.qo : nullptr, nullptr);
}
static int evict(Call& c) { return vxfa_paged_evict(&g_ctx, &c.k, &c.v, &c.w, &c.b, &c.e, nullptr); }

// a changed call gives `want`, a message, and no launch
static void refuses(int line, int (*run)(Call&), int want, std::function<void(Call&)> change) {
    Call c;
    change(c);
    const int before = g_launches;
    const int rc = run(c);
    if (rc != want || g_launches != before || !vxfa_last_error(&g_ctx)[0]) {
        std::printf("line %d: status %d for %d, %d launches, \"%s\"\n", line, rc, want, g_launches - before, g_ctx.last_error);
        ++g_bad;
    }
}
extern "C" const char* vxfa_last_error(const vxfa_ctx* c) { return c->last_error; }
#define REFUSES(run, want, change) refuses(__LINE__, [](Call& c) { return run(c); }, want, [](Call& c) { change; })

static void grids() {
    std::mt19937_64 g(7);
    auto pick = [&](int lo, int hi) { return lo + (int)(g() % (uint64_t)(hi - lo + 1)); };
    for (int it = 0; it < 200000; ++it) {
        vxfa::PagedBatch b;
        std::memset(&b, 0, sizeof(b));
        b.n_streams = pick(1, it % 3 ? 8 : 400);
        b.max_nkv = it % 5 ? pick(1, 9000) : pick(1, 300000);
        b.max_nq = pick(1, 3);
        const int nhg = pick(1, 64);
        int32_t items = 0;
        const int64_t room = it % 4 ? 100000 : pick(0, 500);
        const vxfa::RowsPlan p = vxfa::rows_plan(b, nhg, it % 7 ? 128 : 64, room, items);
        int64_t tiles = 0, parts = 0;
        std::vector<int> len((size_t)b.n_streams);
        for (int& l : len) {
            l = it % 2 ? b.max_nkv : pick(0, b.max_nkv);
            tiles += l >> 4;
        }
        // (one stream's rows are taken as they are)
        const int chunk = vxfa::rows_chunk(p, b.n_streams == 1 ? len[0] : vxfa::rows_total(tiles, b.n_streams));
        for (int l : len) parts += vxfa::rows_parts(p, l, chunk);
        if (parts > items || (p.cuts && items > room)) {
            std::printf("rows: %d streams of up to %d rows: %lld parts, %d in the grid, room %lld\n", b.n_streams, b.max_nkv,
                        (long long)parts, items, (long long)room);
            ++g_bad;
            return;
        }
    }
    for (int it = 0; it < 100000; ++it) {
        vxfa::PagedBatch b;
        std::memset(&b, 0, sizeof(b));
        b.n_streams = pick(1, it % 3 ? 6 : 100);
        b.max_nq = pick(1, it % 2 ? 300 : 3000);
        b.max_nkv = pick(1, 9000);
        const int bm = 32 << pick(0, 3), nhg = pick(1, 40);
        int64_t tiles = 0;
        for (int s = 0; s < b.n_streams; ++s) {
            const int t = pick(0, b.max_nq);
            b.tokens += t;
            tiles += (t + bm - 1) / bm;
        }
        if (!b.tokens) continue;
        vxfa::ChunkPlan p;
        std::memset(&p, 0, sizeof(p));
        const size_t ws = (size_t)pick(1, 40) << 20, record = 133120;
        const vxfa::ChunkBounds r = vxfa::chunk_plan(b, it % 2 ? 128 : 64, nhg, bm, it % 3 ? 0 : pick(1, 5000), record, ws, p);
        const bool ok = tiles <= r.tiles && tiles <= p.items && (b.n_streams > 1 || p.pieces <= 1 || !p.cuts || p.items <= p.room) &&
                        (!p.cuts || r.table + (size_t)p.room * record * nhg <= ws) && p.items >= 1;
        if (!ok) {
            std::printf("chunk: %d streams, %d tokens, tiles %lld of %lld, items %d, room %d\n", b.n_streams, b.tokens, (long long)tiles,
                        (long long)r.tiles, p.items, p.room);
            ++g_bad;
            return;
        }
    }
}

int main() {
    g_ctx.ws = reinterpret_cast<char*>(0x7d0000000000ull);
    {
        Call c;
        CHECK(attend(c) == VXFA_OK && g_last == "chunk+weights");
        CHECK(g_attn.b.max_nkv == 160 && g_attn.b.ps_log2 == 4 && g_attn.b.tokens == 7 && g_attn.lse && g_attn.ws > (char*)g_attn.lse);
        c.b.max_nq = 4;   // 4 tokens of 4 heads: 16 rows
        CHECK(attend(c) == VXFA_OK && g_last == "rows");
        c.b.max_nkv = 33;
        c.b.window = 33;   // as wide as the bound: no window
        CHECK(attend(c, false, false) == VXFA_OK && g_attn.b.max_nkv == 33 && g_attn.window == 0 && !g_attn.lse && !g_attn.w_out);
        c.b.window = 32;
        c.cap = 20.f;
        c.bias = 8.f;
        CHECK(attend(c, true, false) == VXFA_OK && g_attn.window == 32 && !g_attn.w_in && g_attn.cap > 28.f && g_attn.n2 == 8 && g_attn.bias1 == -1.f);
        const size_t nb2 = c.dst.nb[2];
        c.q.ne[2] = c.dst.ne[1] = 0;   // no heads: nothing of q is read, the weights are taken over
        c.dst.nb[2] = 0;
        CHECK(attend(c) == VXFA_OK && g_attn.b.max_nq == 0);
        c.q.ne[2] = c.dst.ne[1] = 8;
        c.dst.nb[2] = nb2;
        const int before = g_launches;
        c.b.max_nq = 0;
        CHECK(attend(c, false, false) == VXFA_OK && g_launches == before);
        c.q.ne[1] = c.dst.ne[2] = 0;
        CHECK(attend(c, false, false) == VXFA_OK && g_launches == before);
    }
    {
        Call c;
        c.k.ne[3] = c.v.ne[3] = c.w.ne[2] = c.w_in.ne[2] = 0;   // no pages: no rows are looked at
        CHECK(attend(c) == VXFA_OK && g_attn.b.max_nkv == 0);
    }
    { Call c; CHECK(append(c) == VXFA_OK && g_last == "append" && g_append.q_out && g_append.rope_dims == 128); }
    { Call c; CHECK(append(c, false, false) == VXFA_OK && !g_append.rope_pos && !g_append.q); }
    { Call c; CHECK(evict(c) == VXFA_OK && g_last == "evict" && g_evict.kept_row == 50 && g_evict.kept == c.e.kept); }
    { Call c; c.e.kept = nullptr; c.e.budget = 1000; CHECK(evict(c) == VXFA_OK && g_evict.kept_row == 160 && (char*)g_evict.kept == g_ctx.ws); }
    { Call c; c.b.max_pages = 0x7fffffff; c.e.budget = 1 << 20; CHECK(evict(c) == VXFA_OK && g_evict.b.max_nkv == 1 << 30); }
    { Call c; c.b.q_start = nullptr; c.b.n_streams = 0; CHECK(evict(c) == VXFA_OK); }
    CHECK(vxfa_flash_attn_ext_paged(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, nullptr, nullptr, nullptr) == VXFA_INVALID_ARG);
    CHECK(vxfa_paged_append(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == VXFA_INVALID_ARG);
    CHECK(vxfa_paged_evict(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) == VXFA_INVALID_ARG);

    // the pool and the batch, by each entry point
#define ALL(want, change) REFUSES(attend, want, change); REFUSES(append, want, change); REFUSES(evict, want, change)
    ALL(VXFA_INVALID_ARG, c.v.ne[3] = 99);
    ALL(VXFA_INVALID_ARG, c.k.ne[2] = c.v.ne[2] = 0);
    ALL(VXFA_INVALID_ARG, c.k.ne[3] = c.v.ne[3] = -1);
    ALL(VXFA_INVALID_ARG, c.k.nb[3] = (size_t)1 << 61);
    ALL(VXFA_INVALID_ARG, c.k.type = 7);
    ALL(VXFA_INVALID_ARG, c.b.n_streams = -1);
    ALL(VXFA_INVALID_ARG, c.b.max_pages = -1);
    ALL(VXFA_INVALID_ARG, c.b.max_nq = -1);
    ALL(VXFA_INVALID_ARG, c.b.max_nkv = -1);
    ALL(VXFA_INVALID_ARG, c.b.window = -1);
    ALL(VXFA_INVALID_ARG, c.b.pad_ = 1);
    ALL(VXFA_INVALID_ARG, c.b.pages = nullptr);
    ALL(VXFA_INVALID_ARG, c.b.n_kv = nullptr);
    ALL(VXFA_INVALID_ARG, c.b.n_kv = (const int32_t*)((const char*)c.b.n_kv + 2));
    REFUSES(attend, VXFA_INVALID_ARG, c.b.q_start = nullptr);
    REFUSES(append, VXFA_INVALID_ARG, c.b.q_start = nullptr);
    ALL(VXFA_UNSUPPORTED, c.k.ne[1] = c.v.ne[1] = 24);
    ALL(VXFA_UNSUPPORTED, c.k.ne[1] = c.v.ne[1] = 8);
    ALL(VXFA_UNSUPPORTED, c.k.ne[1] = c.v.ne[1] = 1 << 17);
    ALL(VXFA_UNSUPPORTED, c.k.type = c.v.type = VXFA_TYPE_F32);
    ALL(VXFA_UNSUPPORTED, c.k.ne[0] = c.v.ne[0] = 96);
    ALL(VXFA_UNSUPPORTED, c.k.nb[1] = c.v.nb[1] = 264);
    ALL(VXFA_UNSUPPORTED, c.k.nb[1] = c.v.nb[1] = 1 << 23);
    ALL(VXFA_UNSUPPORTED, c.v.nb[3] += 16);
    ALL(VXFA_UNSUPPORTED, c.k.data = (char*)c.k.data + 8);
    ALL(VXFA_UNSUPPORTED, c.b.n_streams = 65536);
    // attention
    REFUSES(attend, VXFA_INVALID_ARG, c.q.ne[0] = 64);
    REFUSES(attend, VXFA_INVALID_ARG, c.q.ne[2] = 7);
    REFUSES(attend, VXFA_INVALID_ARG, c.q.ne[3] = 2);
    REFUSES(attend, VXFA_INVALID_ARG, c.dst.ne[2] = 6);
    REFUSES(attend, VXFA_UNSUPPORTED, c.dst.nb[2] += 16);
    REFUSES(attend, VXFA_UNSUPPORTED, c.q.nb[1] += 8);
    REFUSES(attend, VXFA_UNSUPPORTED, c.scale = __builtin_nanf(""));
    REFUSES(attend, VXFA_UNSUPPORTED, c.cap = -1.f);
    REFUSES(attend, VXFA_UNSUPPORTED, c.bias = -1.f);
    REFUSES(attend, VXFA_UNSUPPORTED, c.bias = __builtin_inff());
    REFUSES(attend, VXFA_INVALID_ARG, c.w.ne[2] = 99);
    REFUSES(attend, VXFA_UNSUPPORTED, c.w.type = VXFA_TYPE_F16);
    REFUSES(attend, VXFA_UNSUPPORTED, c.w_in.nb[1] += 2);
    REFUSES(attend, VXFA_UNSUPPORTED, c.scale = 1.f; c.cap = 1e-39f);
    REFUSES(attend, VXFA_UNSUPPORTED, c.scale = 3e38f);
    REFUSES(attend, VXFA_UNSUPPORTED, c.b.max_pages = 0x7fffffff; c.k.ne[2] = c.v.ne[2] = c.w.ne[1] = c.w_in.ne[1] = 8);
    REFUSES(attend, VXFA_NO_WORKSPACE, c.q.ne[1] = c.dst.ne[2] = 2000000);
    { Call c; CHECK(attend(c, false, true) == VXFA_INVALID_ARG); }
    // append
    REFUSES(append, VXFA_INVALID_ARG, c.kn.ne[0] = 128);
    REFUSES(append, VXFA_INVALID_ARG, c.vn.ne[1] = 6);
    REFUSES(append, VXFA_UNSUPPORTED, c.vn.type = VXFA_TYPE_F16);
    REFUSES(append, VXFA_UNSUPPORTED, c.kn.nb[1] += 4);
    REFUSES(append, VXFA_INVALID_ARG, c.r.positions = nullptr);
    REFUSES(append, VXFA_INVALID_ARG, c.r.n_dims = 130);
    REFUSES(append, VXFA_INVALID_ARG, c.r.n_dims = 31);
    REFUSES(append, VXFA_UNSUPPORTED, c.r.mode = 2);
    REFUSES(append, VXFA_UNSUPPORTED, c.r.freq_scale = 0.5f);
    REFUSES(append, VXFA_UNSUPPORTED, c.r.freq_base = 0.f);
    REFUSES(append, VXFA_INVALID_ARG, c.qo.ne[2] = 4);
    REFUSES(append, VXFA_UNSUPPORTED, c.qo.type = VXFA_TYPE_F32);
    { Call c; CHECK(append(c, false, true) == VXFA_INVALID_ARG); }
    // eviction
    REFUSES(evict, VXFA_INVALID_ARG, c.e.budget = 0);
    REFUSES(evict, VXFA_UNSUPPORTED, c.e.budget = (1 << 30) + 1);
    REFUSES(evict, VXFA_INVALID_ARG, c.e.n_sink = 45);
    REFUSES(evict, VXFA_INVALID_ARG, c.e.n_recent = -1);
    REFUSES(evict, VXFA_INVALID_ARG, c.e.pages = nullptr);
    REFUSES(evict, VXFA_INVALID_ARG, c.e.n_kv = const_cast<int32_t*>(c.b.n_kv));
    REFUSES(evict, VXFA_NO_WORKSPACE, c.e.kept = nullptr; c.e.budget = 1 << 21; c.b.max_pages = 1 << 20);

    grids();
    std::printf(g_bad ? "%d wrong\n" : "ok\n", g_bad);
    return g_bad != 0;
}
