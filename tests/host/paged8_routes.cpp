// Which kernels the entry points over pages of 8 bits and over chosen blocks launch for a call of given sizes, as libvxfa.so
// has them, without a GPU: the HIP calls are stand-ins of this program, which the library's references bind
// to. One line a launch: kernel|workgroups|threads|bytes of LDS asked for. Built and run by tests/test_paged8_routes.py.
#include <hip/hip_runtime.h>

#include <cxxabi.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <string>

#include "../../include/vxfa.h"
#include "../../voxtral.cpp_amd/csrc/vxfa_ctx.h"

static std::map<const void*, std::string>& names() {
    static std::map<const void*, std::string> m;
    return m;
}

extern "C" {
hipError_t hipGetDevice(int* d) { *d = 0; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError(void) { return hipSuccess; }
void __hipRegisterFunction(void**, const void* host, char*, const char* device, unsigned, void*, void*, void*, void*, int*) { names()[host] = device; }
static dim3 g_grid, g_block;
static size_t g_lds;
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t) { g_grid = g; g_block = b; g_lds = lds; return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* s) { *g = g_grid; *b = g_block; *lds = g_lds; *s = nullptr; return hipSuccess; }
hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void**, size_t lds, hipStream_t) {
    int status = 0;
    std::string mangled = names()[f];
    mangled = mangled.substr(0, mangled.find('.'));      // (a static kernel's name has its file's hash behind it)
    char* s = abi::__cxa_demangle(mangled.c_str(), nullptr, nullptr, &status);
    std::printf("%s|%u|%u|%zu\n", status == 0 ? s : mangled.c_str(), grid.x, block.x, lds);
    std::free(s);
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
    for (int d = 0; d < 4; ++d) { t.ne[d] = ne[d]; t.nb[d] = nb; nb *= (size_t)ne[d]; }
    return t;
}

int main(int argc, char** argv) {
    if (argc < 2) return 2;
    std::map<std::string, long> a = {{"hq", 8}, {"hkv", 8}, {"hd", 128}, {"streams", 1}, {"nq", 1}, {"tokens", 0}, {"page", 64}, {"max_pages", 1},
                                     {"max_nkv", 0}, {"window", 0}, {"block", 16}, {"top", 8}, {"bits", 8}, {"cap", 0}};
    for (int i = 2; i < argc; ++i) {
        const std::string arg = argv[i], key = arg.substr(0, arg.find('='));
        if (key == arg || !a.count(key)) return 2;
        a[key] = std::atol(arg.c_str() + key.size() + 1);
    }
    const long T = a["tokens"] ? a["tokens"] : a["streams"] * a["nq"], D = a["hd"], hkv = a["hkv"], page = a["page"], N = 100;
    vxfa_ctx ctx;
    ctx.ws = reinterpret_cast<char*>(0x7d0000000000ull);
    vxfa_tensor k = tensor(a["bits"] == 8 ? VXFA_TYPE_I8 : VXFA_TYPE_F16, D, page, hkv, N), v = k;
    vxfa_tensor ks = tensor(VXFA_TYPE_F32, page / 16, hkv, N, 1), vs = ks;
    vxfa_tensor q = tensor(VXFA_TYPE_F16, D, T, a["hq"], 1), dst = tensor(VXFA_TYPE_F16, D, a["hq"], T, 1);
    vxfa_tensor b = tensor(VXFA_TYPE_I8, 2 * D, page / a["block"], hkv, N), bs = tensor(VXFA_TYPE_F32, page / a["block"], hkv, N, 1);
    int32_t* x = static_cast<int32_t*>(kAddr);
    vxfa_paged p{x, x + 1, x + 2, (int32_t)a["streams"], (int32_t)a["max_pages"], (int32_t)a["nq"], (int32_t)a["max_nkv"], (int32_t)a["window"], 0};
    vxfa_blocks l{x, (int32_t)a["block"], (int32_t)a["top"], 0, 0};
    const bool i8 = a["bits"] == 8;
    int rc = -1;
    if (!std::strcmp(argv[1], "attend")) rc = vxfa_flash_attn_ext_paged_q8(&ctx, &q, &k, &ks, &v, &vs, &p, &dst, 0.1f, 0, (float)a["cap"], nullptr);
    if (!std::strcmp(argv[1], "choose")) rc = vxfa_paged_select(&ctx, &q, &b, &bs, &p, &l, nullptr);
    if (!std::strcmp(argv[1], "blocks"))
        rc = vxfa_flash_attn_ext_paged_blocks(&ctx, &q, &k, i8 ? &ks : nullptr, &v, i8 ? &vs : nullptr, &p, &l, &dst, 0.1f, 0, (float)a["cap"], nullptr);
    if (rc != VXFA_OK) std::printf("status %d: %s\n", rc, vxfa_last_error(&ctx));
    return rc != VXFA_OK;
}
