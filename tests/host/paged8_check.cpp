// Host check of the entry points over pages of 8 bits and over chosen blocks as libvxfa.so has
// them, launchers and all, without a GPU: the HIP calls are stand-ins of this program,
// which the library's references bind to, and count the launches. Every violation comes back as its
// status, with a message and no launch; calls at the documented limits are taken. Built and run by
// tests/test_paged8_checks.py.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstring>
#include <functional>

#include "../../include/vxfa.h"
#include "../../voxtral.cpp_amd/csrc/vxfa_ctx.h"

static int g_launches = 0, g_bad = 0;

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
static dim3 g_grid, g_block;
static size_t g_lds;
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t) { g_grid = g; g_block = b; g_lds = lds; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) { *g = g_grid; *b = g_block; *lds = g_lds; *s = nullptr; return hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t lds, hipStream_t) {
    ++g_launches;
    // what the hardware takes: 2^32 threads along x, 65535 workgroups along y and z, 64 KiB asked for at a launch
    if ((uint64_t)grid.x * block.x >= (1ull << 32) || !grid.x || grid.y > 65535 || grid.z > 65535 || lds > 65536 || block.x > 1024) {
        std::printf("launch of %u x %u x %u workgroups of %u, %zu bytes\n", grid.x, grid.y, grid.z, block.x, lds);
        ++g_bad;
    }
    return hipSuccess;
}
}

static void* const kAddr = reinterpret_cast<void*>(0x7e0000000000ull);   // (never dereferenced)

static vxfa_tensor tensor(int type, int64_t n0, int64_t n1, int64_t n2, int64_t n3) {
    vxfa_tensor t;
    std::memset(&t, 0, sizeof(t));
    t.data = kAddr;
    t.type = type;
    const int64_t ne[4] = {n0, n1, n2, n3};
    size_t nb = type == VXFA_TYPE_F16 ? 2 : (type == VXFA_TYPE_I8 ? 1 : 4);
    for (int d = 0; d < 4; ++d) { t.ne[d] = ne[d]; t.nb[d] = nb; nb *= (size_t)(ne[d] > 0 ? ne[d] : 1); }
    return t;
}

// pages of 64 rows, blocks of 32; T tokens of hq heads over hkv, at most max_nq of a stream
struct Call {
    vxfa_tensor k, v, ks, vs, k16, v16, q, dst, b, bs, kn, vn, qf, qo;
    vxfa_paged p;
    vxfa_blocks l;
    vxfa_rope r;
    float scale = 0.1f, bias = 0, cap = 0;
    Call(int64_t T = 7, int64_t hq = 8, int64_t hkv = 2, int streams = 3, int max_nq = 5, int64_t D = 128, int top = 4) {
        k = v = tensor(VXFA_TYPE_I8, D, 64, hkv, 100);
        ks = vs = tensor(VXFA_TYPE_F32, 4, hkv, 100, 1);
        k16 = v16 = tensor(VXFA_TYPE_F16, D, 64, hkv, 100);
        q = tensor(VXFA_TYPE_F16, D, T, hq, 1);
        dst = tensor(VXFA_TYPE_F16, D, hq, T, 1);
        b = tensor(VXFA_TYPE_I8, 2 * D, 2, hkv, 100);
        bs = tensor(VXFA_TYPE_F32, 2, hkv, 100, 1);
        kn = vn = tensor(VXFA_TYPE_F32, hkv * D, T, 1, 1);
        qf = tensor(VXFA_TYPE_F32, D, T, hq, 1);
        qo = tensor(VXFA_TYPE_F16, D, T, hq, 1);
        int32_t* x = static_cast<int32_t*>(kAddr);
        p = vxfa_paged{x, x + 1, x + 2, streams, 10, max_nq, 0, 0, 0};
        l = vxfa_blocks{x, 32, top, 1, 2};
        r = vxfa_rope{x, (int32_t)D, 0, 1e6f, 1.0f};
    }
};

static vxfa_ctx g_ctx;
static int append(Call& c) { return vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, &c.p, &c.k, &c.ks, &c.v, &c.vs, &c.r, &c.qf, &c.qo, nullptr); }
static int append_only(Call& c) { return vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, &c.p, &c.k, &c.ks, &c.v, &c.vs, nullptr, nullptr, nullptr, nullptr); }
static int attend(Call& c) { return vxfa_flash_attn_ext_paged_q8(&g_ctx, &c.q, &c.k, &c.ks, &c.v, &c.vs, &c.p, &c.dst, c.scale, c.bias, c.cap, nullptr); }
static int bounds(Call& c) { return vxfa_paged_bounds(&g_ctx, &c.k, &c.ks, &c.p, &c.b, &c.bs, nullptr); }
static int bounds16(Call& c) { return vxfa_paged_bounds(&g_ctx, &c.k16, nullptr, &c.p, &c.b, &c.bs, nullptr); }
static int choose(Call& c) { return vxfa_paged_select(&g_ctx, &c.q, &c.b, &c.bs, &c.p, &c.l, nullptr); }
static int blocks(Call& c) {
    return vxfa_flash_attn_ext_paged_blocks(&g_ctx, &c.q, &c.k, &c.ks, &c.v, &c.vs, &c.p, &c.l, &c.dst, c.scale, c.bias, c.cap, nullptr);
}
static int blocks16(Call& c) {
    return vxfa_flash_attn_ext_paged_blocks(&g_ctx, &c.q, &c.k16, nullptr, &c.v16, nullptr, &c.p, &c.l, &c.dst, c.scale, c.bias, c.cap, nullptr);
}

// the call gives `want`, and launches just where that is VXFA_OK and `work`
static void gives(int line, int want, bool work, int (*run)(Call&), Call c) {
    const int before = g_launches, rc = run(c);
    const bool launched = g_launches != before, said = vxfa_last_error(&g_ctx)[0] != 0;
    if (rc != want || launched != (want == VXFA_OK && work) || said != (want != VXFA_OK)) {
        std::printf("line %d: status %d for %d, %d launches, \"%s\"\n", line, rc, want, g_launches - before, g_ctx.last_error);
        ++g_bad;
    }
}
static Call with(Call c, std::function<void(Call&)> change) { change(c); return c; }
#define GIVES(want, run, call) gives(__LINE__, want, true, run, call)
#define NOTHING(run, call) gives(__LINE__, VXFA_OK, false, run, call)
#define CHANGED(change) with(Call(), [](Call& c) { change; })
#define INVALID(run, change) GIVES(VXFA_INVALID_ARG, run, CHANGED(change))
#define UNSUPPORTED(run, change) GIVES(VXFA_UNSUPPORTED, run, CHANGED(change))

static void pools() {
    for (auto run : {append, attend, bounds, blocks}) {
        GIVES(VXFA_OK, run, Call());
        INVALID(run, c.k.data = nullptr);
        INVALID(run, c.ks.data = nullptr);
        INVALID(run, c.k.type = 7);
        INVALID(run, c.k.ne[0] = -1);
        INVALID(run, c.ks.type = 24);
        INVALID(run, c.ks.ne[0] = 64);
        INVALID(run, c.ks.ne[1] = 3);
        INVALID(run, c.ks.ne[2] = 99);
        INVALID(run, c.ks.ne[3] = 2);
        UNSUPPORTED(run, c.ks.type = VXFA_TYPE_F16);
        UNSUPPORTED(run, c.ks.nb[0] = 8);
        UNSUPPORTED(run, c.ks.nb[1] = 18);
        UNSUPPORTED(run, c.ks.nb[2] = 2);
        UNSUPPORTED(run, c.ks.data = (char*)kAddr + 2);
        UNSUPPORTED(run, c.k.type = c.v.type = VXFA_TYPE_F16);
        UNSUPPORTED(run, c.k.type = c.v.type = VXFA_TYPE_F32);
        UNSUPPORTED(run, c.k.nb[1] = c.v.nb[1] = 136);
        UNSUPPORTED(run, c.k.nb[1] = c.v.nb[1] = 1 << 23);
        UNSUPPORTED(run, c.k.nb[0] = c.v.nb[0] = 2);
        UNSUPPORTED(run, c.k.data = (char*)kAddr + 8);
        UNSUPPORTED(run, c.k.ne[0] = c.v.ne[0] = 96);
        UNSUPPORTED(run, c.k.ne[1] = c.v.ne[1] = 48);
        UNSUPPORTED(run, c.p.n_streams = 65536);
        INVALID(run, c.p.n_streams = -1);
        INVALID(run, c.p.max_nq = -1);
        INVALID(run, c.p.window = -1);
        INVALID(run, c.p.pad_ = 1);
        INVALID(run, c.p.pages = nullptr);
        INVALID(run, c.p.n_kv = nullptr);
        INVALID(run, c.p.q_start = nullptr);
        INVALID(run, c.p.n_kv = (const int32_t*)((char*)kAddr + 2));
    }
    for (auto run : {append, attend, blocks}) {
        INVALID(run, c.v.data = nullptr);
        INVALID(run, c.vs.data = nullptr);
        INVALID(run, c.v.ne[3] = 99);
        UNSUPPORTED(run, c.v.nb[3] *= 2);
        UNSUPPORTED(run, c.vs.nb[2] *= 2);
    }
    // no pages: none are looked at
    for (auto run : {attend, blocks}) GIVES(VXFA_OK, run, CHANGED(c.k.data = c.v.data = c.ks.data = c.vs.data = nullptr; c.k.ne[3] = c.v.ne[3] = c.ks.ne[2] = c.vs.ne[2] = 0));
    NOTHING(bounds, CHANGED(c.k.data = c.ks.data = c.b.data = c.bs.data = nullptr; c.k.ne[3] = c.v.ne[3] = c.ks.ne[2] = c.b.ne[3] = c.bs.ne[2] = 0));
    for (auto run : {append, attend, bounds, bounds16, choose, blocks, blocks16}) NOTHING(run, CHANGED(c.p.n_streams = 0; c.p.pages = c.p.n_kv = c.p.q_start = nullptr));
}

static void tokens() {
    GIVES(VXFA_OK, append_only, Call());
    INVALID(append, c.kn.data = nullptr);
    INVALID(append, c.vn.ne[1] = 6);
    INVALID(append, c.kn.ne[0] = 128);
    UNSUPPORTED(append, c.kn.type = c.vn.type = VXFA_TYPE_F16);
    INVALID(append, c.r.n_dims = 130);
    INVALID(append, c.r.n_dims = 3);
    INVALID(append, c.r.positions = nullptr);
    UNSUPPORTED(append, c.r.mode = 2);
    UNSUPPORTED(append, c.r.freq_base = 0);
    INVALID(append, c.qf.ne[1] = c.qo.ne[1] = 6);
    UNSUPPORTED(append, c.qo.type = VXFA_TYPE_F32);
    GIVES(VXFA_UNSUPPORTED, append, Call(1 << 24));
    NOTHING(append_only, CHANGED(c.kn.ne[1] = c.vn.ne[1] = 0; c.kn.data = c.vn.data = nullptr));
    for (auto run : {attend, blocks, blocks16}) {
        GIVES(VXFA_OK, run, Call());
        INVALID(run, c.q.data = nullptr);
        INVALID(run, c.dst.data = nullptr);
        INVALID(run, c.q.ne[0] = 64);
        INVALID(run, c.q.ne[2] = 7);
        INVALID(run, c.q.type = VXFA_TYPE_I8);
        INVALID(run, c.dst.ne[1] = 4);
        UNSUPPORTED(run, c.dst.nb[1] = 512);
        UNSUPPORTED(run, c.scale = INFINITY);
        UNSUPPORTED(run, c.cap = -1);
        UNSUPPORTED(run, c.bias = -1);
        GIVES(VXFA_UNSUPPORTED, run, Call(1 << 24));
        GIVES(VXFA_UNSUPPORTED, run, Call(7, 65536));
        NOTHING(run, CHANGED(c.p.max_nq = 0));
        NOTHING(run, CHANGED(c.q.ne[1] = c.dst.ne[2] = 0; c.q.data = c.dst.data = nullptr));
    }
}

static void chosen() {
    for (auto run : {choose, blocks, blocks16}) {
        INVALID(run, c.l.list = nullptr);
        INVALID(run, c.l.list = (int32_t*)((char*)kAddr + 2));
        INVALID(run, c.l.block = 8);
        INVALID(run, c.l.block = 48);
        INVALID(run, c.l.top = 0);
        GIVES(VXFA_OK, run, CHANGED(c.l.top = 1024));
        UNSUPPORTED(run, c.l.top = 1025);
    }
    for (auto run : {blocks, blocks16}) INVALID(run, c.l.block = 128);
    GIVES(VXFA_OK, choose, CHANGED(c.l.block = 128));   // (of pages of 256 rows, two blocks each)
    for (auto run : {blocks, blocks16}) GIVES(VXFA_OK, run, CHANGED(c.l.n_sink = -5; c.l.n_recent = 100));   // (not looked at)
    // half a pool of 8 bits is none
    { Call c; const int rc = vxfa_flash_attn_ext_paged_blocks(&g_ctx, &c.q, &c.k, &c.ks, &c.v, nullptr, &c.p, &c.l, &c.dst, 1, 0, 0, nullptr);
      if (rc != VXFA_INVALID_ARG) { std::printf("line %d: %d\n", __LINE__, rc); ++g_bad; } }
    { Call c; const int rc = vxfa_flash_attn_ext_paged_blocks(&g_ctx, &c.q, &c.k, nullptr, &c.v, nullptr, &c.p, &c.l, &c.dst, 1, 0, 0, nullptr);
      if (rc != VXFA_INVALID_ARG) { std::printf("line %d: %d\n", __LINE__, rc); ++g_bad; } }
    GIVES(VXFA_OK, choose, Call());
    INVALID(choose, c.l.n_sink = -1);
    INVALID(choose, c.l.n_recent = 4);
    GIVES(VXFA_OK, choose, CHANGED(c.l.n_recent = 3));
    INVALID(choose, c.q.data = nullptr);
    INVALID(choose, c.q.ne[2] = 7);
    INVALID(choose, c.q.ne[0] = 64);
    UNSUPPORTED(choose, c.q.nb[1] = 8);
    GIVES(VXFA_UNSUPPORTED, choose, Call(1 << 24));
    // 262144 blocks of a stream
    GIVES(VXFA_OK, choose, CHANGED(c.p.max_pages = 131072));
    UNSUPPORTED(choose, c.p.max_pages = 131073);
    GIVES(VXFA_OK, choose, CHANGED(c.p.max_pages = 131073; c.p.max_nkv = 262144 * 32));
    // pairs of 5000 tokens, 8 heads and 16 segments: 8 bytes each for 8 blocks 41 MB, for 9 more than there is
    GIVES(VXFA_OK, choose, with(Call(5000, 32, 8, 1, 5000, 128, 8), [](Call& c) { c.p.max_pages = 32768; }));
    GIVES(VXFA_NO_WORKSPACE, choose, with(Call(5000, 32, 8, 1, 5000, 128, 9), [](Call& c) { c.p.max_pages = 32768; }));
    for (auto run : {bounds, bounds16, choose}) {
        INVALID(run, c.b.data = nullptr);
        INVALID(run, c.bs.data = nullptr);
        INVALID(run, c.b.ne[0] = 255);
        INVALID(run, c.b.ne[1] = 3);
        INVALID(run, c.b.ne[2] = 3);
        INVALID(run, c.bs.ne[0] = 4);
        INVALID(run, c.b.type = 9);
        UNSUPPORTED(run, c.b.type = VXFA_TYPE_F16);
        UNSUPPORTED(run, c.b.nb[1] = 264);
        UNSUPPORTED(run, c.bs.type = VXFA_TYPE_F16);
    }
    for (auto run : {bounds, bounds16}) {
        INVALID(run, c.b.ne[1] = c.bs.ne[0] = 8);      // blocks of 8 rows
        INVALID(run, c.b.ne[3] = 99);
        GIVES(VXFA_OK, run, CHANGED(c.b.ne[1] = c.bs.ne[0] = 4));
        NOTHING(run, CHANGED(c.p.max_nq = 0));
    }
}

// grids at and past their limits
static void grids() {
    for (int64_t D : {64, 128}) {
        GIVES(VXFA_OK, attend, Call(65535, 128, 128, 65535, 1, D));
        GIVES(VXFA_UNSUPPORTED, attend, Call(65535, 65535, 65535, 65535, 1, D));
        const int64_t bm = 2 * D;
        GIVES(VXFA_OK, attend, Call(65535 * bm / 2, 255, 255, 1, 1 << 24, D));
        GIVES(VXFA_UNSUPPORTED, attend, Call(65535 * bm / 2, 257, 257, 1, 1 << 24, D));
        for (auto run : {blocks, blocks16}) {
            GIVES(VXFA_OK, run, Call(65535, 256, 256, 1, 1 << 24, D));
            GIVES(VXFA_UNSUPPORTED, run, Call(65537, 256, 256, 1, 1 << 24, D));
        }
        GIVES(VXFA_OK, append, Call((1 << 24) / 2 - 1, 8, 2, 1, 1 << 24, D));
        for (auto run : {bounds, bounds16}) {
            GIVES(VXFA_OK, run, Call(7, 8, 2, 65535, 1000, D));
            GIVES(VXFA_UNSUPPORTED, run, Call(7, 4000, 4000, 65535, 1000, D));
        }
        GIVES(VXFA_OK, choose, Call(65535, 60, 60, 65535, 1, D));
        GIVES(VXFA_UNSUPPORTED, choose, Call(65535, 70, 70, 65535, 1, D));
    }
}

int main() {
    g_ctx.ws = reinterpret_cast<char*>(0x7d0000000000ull);
    pools();
    tokens();
    chosen();
    grids();
    if (vxfa_paged_append_q8(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) != VXFA_INVALID_ARG ||
        vxfa_flash_attn_ext_paged_q8(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, nullptr) != VXFA_INVALID_ARG ||
        vxfa_paged_bounds(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) != VXFA_INVALID_ARG ||
        vxfa_paged_select(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr) != VXFA_INVALID_ARG ||
        vxfa_flash_attn_ext_paged_blocks(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, nullptr) != VXFA_INVALID_ARG) {
        std::printf("no context\n");
        ++g_bad;
    }
    // null arguments, each in its place
    {
        Call c;
        const vxfa_tensor* n = nullptr;
        const int got[] = {
            vxfa_paged_append_q8(&g_ctx, n, &c.vn, &c.p, &c.k, &c.ks, &c.v, &c.vs, nullptr, n, nullptr, nullptr),
            vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, nullptr, &c.k, &c.ks, &c.v, &c.vs, nullptr, n, nullptr, nullptr),
            vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, &c.p, nullptr, &c.ks, &c.v, &c.vs, nullptr, n, nullptr, nullptr),
            vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, &c.p, &c.k, nullptr, &c.v, &c.vs, nullptr, n, nullptr, nullptr),
            vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, &c.p, &c.k, &c.ks, &c.v, nullptr, nullptr, n, nullptr, nullptr),
            vxfa_paged_append_q8(&g_ctx, &c.kn, &c.vn, &c.p, &c.k, &c.ks, &c.v, &c.vs, nullptr, &c.qf, &c.qo, nullptr),
            vxfa_flash_attn_ext_paged_q8(&g_ctx, n, &c.k, &c.ks, &c.v, &c.vs, &c.p, &c.dst, 1, 0, 0, nullptr),
            vxfa_flash_attn_ext_paged_q8(&g_ctx, &c.q, &c.k, n, &c.v, &c.vs, &c.p, &c.dst, 1, 0, 0, nullptr),
            vxfa_flash_attn_ext_paged_q8(&g_ctx, &c.q, &c.k, &c.ks, &c.v, &c.vs, &c.p, nullptr, 1, 0, 0, nullptr),
            vxfa_paged_bounds(&g_ctx, n, &c.ks, &c.p, &c.b, &c.bs, nullptr),
            vxfa_paged_bounds(&g_ctx, &c.k, &c.ks, &c.p, nullptr, &c.bs, nullptr),
            vxfa_paged_bounds(&g_ctx, &c.k, &c.ks, &c.p, &c.b, nullptr, nullptr),
            vxfa_paged_select(&g_ctx, n, &c.b, &c.bs, &c.p, &c.l, nullptr),
            vxfa_paged_select(&g_ctx, &c.q, n, &c.bs, &c.p, &c.l, nullptr),
            vxfa_paged_select(&g_ctx, &c.q, &c.b, &c.bs, nullptr, &c.l, nullptr),
            vxfa_paged_select(&g_ctx, &c.q, &c.b, &c.bs, &c.p, nullptr, nullptr),
            vxfa_flash_attn_ext_paged_blocks(&g_ctx, &c.q, &c.k, &c.ks, &c.v, &c.vs, &c.p, nullptr, &c.dst, 1, 0, 0, nullptr),
        };
        for (size_t i = 0; i < sizeof(got) / sizeof(got[0]); ++i)
            if (got[i] != VXFA_INVALID_ARG) { std::printf("null %zu: %d\n", i, got[i]); ++g_bad; }
    }
    std::printf(g_bad ? "%d wrong\n" : "ok\n", g_bad);
    return g_bad != 0;
}
