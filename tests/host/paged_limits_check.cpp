// Host check of the paged entry points as libvxfa.so has them, launchers and all,
// without a GPU: the HIP calls are stand-ins of this program, which the library's
// references bind to, and count the launches. Descriptors without data, grids beyond
// the launch limits and sizes beyond the documented ones are refused before any launch. Built and run by tests/test_paged_limits.py.
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
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3*, dim3*, size_t*, hipStream_t*) { return hipSuccess; }
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { ++g_launches; return hipSuccess; }
}

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

// pages of 16 rows; T tokens of hq heads over hkv, at most max_nq of a stream
struct Call {
    vxfa_tensor k, v, q, dst, w, w_in, kn, vn, qf, qo;
    vxfa_paged b;
    vxfa_evict e;
    vxfa_rope r;
    Call(int64_t T = 7, int64_t hq = 8, int64_t hkv = 2, int streams = 3, int max_nq = 5, int64_t D = 128) {
        k = v = tensor(VXFA_TYPE_F16, D, 16, hkv, 100);
        q = tensor(VXFA_TYPE_F16, D, T, hq, 1);
        dst = tensor(VXFA_TYPE_F16, D, hq, T, 1);
        w = w_in = tensor(VXFA_TYPE_F32, 16, hkv, 100, 1);
        kn = vn = tensor(VXFA_TYPE_F32, hkv * D, T, 1, 1);
        qf = tensor(VXFA_TYPE_F32, D, T, hq, 1);
        qo = tensor(VXFA_TYPE_F16, D, T, hq, 1);
        const int32_t* p = static_cast<const int32_t*>(kAddr);
        b = vxfa_paged{p, p + 1, p + 2, streams, 10, max_nq, 0, 0, 0};
        e = vxfa_evict{p, 4, 50, 4, 10, const_cast<int32_t*>(p), nullptr};
        r = vxfa_rope{p, (int32_t)D, 0, 1e6f, 1.0f};
    }
};

static vxfa_ctx g_ctx;
static int attend(Call& c) {
    return vxfa_flash_attn_ext_paged(&g_ctx, &c.q, &c.k, &c.v, &c.b, &c.dst, 0.1f, 0, 0, &c.w_in, &c.w, nullptr);
}
static int attend_only(Call& c) {
    return vxfa_flash_attn_ext_paged(&g_ctx, &c.q, &c.k, &c.v, &c.b, &c.dst, 0.1f, 0, 0, nullptr, nullptr, nullptr);
}
static int append(Call& c) { return vxfa_paged_append(&g_ctx, &c.kn, &c.vn, &c.b, &c.k, &c.v, &c.r, &c.qf, &c.qo, nullptr); }
static int evict(Call& c) { return vxfa_paged_evict(&g_ctx, &c.k, &c.v, &c.w, &c.b, &c.e, nullptr); }

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
#define CHANGED(change) with(Call(), [](Call& c) { change; })

static void data() {
    GIVES(VXFA_OK, attend, Call());
    GIVES(VXFA_OK, append, Call());
    GIVES(VXFA_OK, evict, Call());
    for (auto run : {attend, append, evict}) {
        GIVES(VXFA_INVALID_ARG, run, CHANGED(c.k.data = nullptr));
        GIVES(VXFA_INVALID_ARG, run, CHANGED(c.v.data = nullptr));
    }
    GIVES(VXFA_INVALID_ARG, attend, CHANGED(c.q.data = nullptr));
    GIVES(VXFA_INVALID_ARG, attend, CHANGED(c.dst.data = nullptr));
    GIVES(VXFA_INVALID_ARG, attend, CHANGED(c.w.data = nullptr));
    GIVES(VXFA_INVALID_ARG, attend, CHANGED(c.w_in.data = nullptr));
    GIVES(VXFA_INVALID_ARG, append, CHANGED(c.kn.data = nullptr));
    GIVES(VXFA_INVALID_ARG, append, CHANGED(c.vn.data = nullptr));
    GIVES(VXFA_INVALID_ARG, append, CHANGED(c.qf.data = nullptr));
    GIVES(VXFA_INVALID_ARG, append, CHANGED(c.qo.data = nullptr));
    GIVES(VXFA_INVALID_ARG, evict, CHANGED(c.w.data = nullptr));
    // where there are no elements, or no streams, there need be no data
    GIVES(VXFA_OK, attend, CHANGED(c.k.data = c.v.data = c.w.data = c.w_in.data = nullptr; c.k.ne[3] = c.v.ne[3] = c.w.ne[2] = c.w_in.ne[2] = 0));
    gives(__LINE__, VXFA_OK, false, attend_only, CHANGED(c.q.data = c.dst.data = nullptr; c.q.ne[1] = c.dst.ne[2] = 0));
    gives(__LINE__, VXFA_OK, false, append, CHANGED(c.kn.data = c.vn.data = c.qf.data = c.qo.data = nullptr; c.kn.ne[1] = c.vn.ne[1] = c.qf.ne[1] = c.qo.ne[1] = 0));
    gives(__LINE__, VXFA_OK, false, attend, CHANGED(c.k.data = c.v.data = c.w.data = nullptr; c.b.n_streams = 0));
    gives(__LINE__, VXFA_OK, false, evict, CHANGED(c.k.data = c.v.data = c.w.data = nullptr; c.b.n_streams = 0));
}

// workgroups of an attention call: parts of streams (or tiles) by head groups, 2^23 - 1 at most
static void grids() {
    for (int64_t D : {64, 128}) {
        // single tokens of 65535 streams, 128 and 129 kv heads: 8388480 and 8454015
        GIVES(VXFA_OK, attend_only, Call(65535, 128, 128, 65535, 1, D));
        GIVES(VXFA_UNSUPPORTED, attend_only, Call(65535, 129, 129, 65535, 1, D));
        GIVES(VXFA_UNSUPPORTED, attend_only, Call(65535, 65535, 65535, 65535, 1, D));
        // chunks: tiles of 256 (128) tokens, a head each
        const int64_t bm = 2 * D;
        GIVES(VXFA_OK, attend_only, Call(65535 * bm / 2, 255, 255, 1, 1 << 24, D));
        GIVES(VXFA_UNSUPPORTED, attend_only, Call(65535 * bm / 2, 257, 257, 1, 1 << 24, D));
        GIVES(VXFA_UNSUPPORTED, attend_only, Call(1 << 23, 60000, 60000, 1, 1 << 24, D));
    }
}

// the sizes that the header names
static void sizes() {
    GIVES(VXFA_OK, append, Call(7, 65535));
    GIVES(VXFA_UNSUPPORTED, append, Call(7, 65536));
    GIVES(VXFA_UNSUPPORTED, attend_only, Call(7, 65536));
    GIVES(VXFA_UNSUPPORTED, append, Call(1 << 24));
    GIVES(VXFA_UNSUPPORTED, attend_only, Call(1 << 24));
    for (auto run : {attend, append, evict}) {
        GIVES(VXFA_UNSUPPORTED, run, Call(7, 65536, 65536));
        GIVES(VXFA_UNSUPPORTED, run, Call(7, 8, 2, 65536));
        // K and V pools share their strides, rows less than 8 MiB apart
        GIVES(VXFA_UNSUPPORTED, run, CHANGED(c.v.nb[3] *= 2));
        GIVES(VXFA_OK, run, CHANGED(c.k.nb[1] = c.v.nb[1] = (1 << 23) - 16));
        GIVES(VXFA_UNSUPPORTED, run, CHANGED(c.k.nb[1] = c.v.nb[1] = 1 << 23));
    }
}

int main() {
    g_ctx.ws = reinterpret_cast<char*>(0x7d0000000000ull);
    data();
    grids();
    sizes();
    std::printf(g_bad ? "%d wrong\n" : "ok\n", g_bad);
    return g_bad != 0;
}
