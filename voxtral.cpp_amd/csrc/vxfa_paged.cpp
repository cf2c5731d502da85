// vxfa_paged.cpp — the paged entry points of include/vxfa.h: checks of their
// arguments, workspace layout, dispatch.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include "../../include/vxfa.h"
#include "fa_paged.h"
#include "vxfa_ctx.h"

namespace {

using vxfa::PagedBatch;
using vxfa::PagedPool;

int fail(vxfa_ctx* c, int rc, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(c->last_error, sizeof(c->last_error), fmt, ap);
    va_end(ap);
    return rc;
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool sane(const vxfa_tensor* t) {
    if (t->type != VXFA_TYPE_F32 && t->type != VXFA_TYPE_F16) return false;
    for (int d = 0; d < 4; ++d)   // (offsets have to fit 64 bits)
        if (t->ne[d] < 0 || t->nb[d] > ((size_t)1 << 60) / (size_t)(t->ne[d] > 0 ? t->ne[d] : 1)) return false;
    return true;
}

// elements that a call over streams would touch, but no data
bool missing(const vxfa_paged* b, const vxfa_tensor* t) {
    if (t->data || b->n_streams == 0) return false;
    for (int d = 0; d < 4; ++d)
        if (t->ne[d] == 0) return false;
    return true;
}

// 16-byte loads of rows of `elt`-sized elements
bool vector_rows(const vxfa_tensor* t, size_t elt, int dims) {
    if (t->nb[0] != elt || !aligned(t->data, 16)) return false;
    for (int d = 1; d < dims; ++d)
        if (t->nb[d] & 15) return false;
    return true;
}

// The pool and the batch over it. need_q: q_start and max_nq are looked at.
int check_pool(const vxfa_tensor* k, const vxfa_tensor* v, const vxfa_paged* b, bool need_q, const char** why) {
    if (!k || !v || !b) { *why = "k, v and batch are required"; return VXFA_INVALID_ARG; }
    if (!sane(k) || !sane(v)) { *why = "k and v: unknown type, negative ne or absurd nb"; return VXFA_INVALID_ARG; }
    for (int d = 0; d < 4; ++d)
        if (k->ne[d] != v->ne[d]) { *why = "k and v pools differ"; return VXFA_INVALID_ARG; }
    if (b->n_streams < 0 || b->max_pages < 0 || b->max_nq < 0 || b->max_nkv < 0 || b->window < 0 || b->pad_ != 0) {
        *why = "batch: negative sizes, or pad_ not 0";
        return VXFA_INVALID_ARG;
    }
    if (b->n_streams > 0 && (!b->n_kv || (need_q && !b->q_start) || (b->max_pages > 0 && !b->pages))) {
        *why = "batch: pages, n_kv and q_start are required";
        return VXFA_INVALID_ARG;
    }
    if (!aligned(b->pages, 4) || !aligned(b->n_kv, 4) || (need_q && !aligned(b->q_start, 4))) {
        *why = "batch: misaligned arrays";
        return VXFA_INVALID_ARG;
    }
    if (missing(b, k) || missing(b, v)) { *why = "k and v: data is required"; return VXFA_INVALID_ARG; }
    const int64_t ps = k->ne[1];
    if (ps < (1 << vxfa::kPagedMinLog2) || ps > (1 << vxfa::kPagedMaxLog2) || (ps & (ps - 1))) {
        *why = "page size must be a power of two from 16 to 65536";
        return VXFA_UNSUPPORTED;
    }
    if (k->ne[2] < 1) { *why = "no kv heads"; return VXFA_INVALID_ARG; }
    if (k->type != VXFA_TYPE_F16 || v->type != VXFA_TYPE_F16) { *why = "pages must be F16"; return VXFA_UNSUPPORTED; }
    if (k->ne[0] != 64 && k->ne[0] != 128) { *why = "head dim must be 64 or 128"; return VXFA_UNSUPPORTED; }
    if (k->ne[2] > 65535 || k->ne[3] > 0x7fffffff || b->n_streams > 65535) {
        *why = "sizes beyond the launch limits";
        return VXFA_UNSUPPORTED;
    }
    if (k->nb[1] >= ((size_t)1 << 23) || v->nb[1] >= ((size_t)1 << 23)) {
        *why = "k/v row stride must be below 8 MiB";
        return VXFA_UNSUPPORTED;
    }
    for (int d = 1; d < 4; ++d)
        if (k->nb[d] != v->nb[d]) { *why = "k and v pools must have the same strides"; return VXFA_UNSUPPORTED; }
    if (!vector_rows(k, 2, 4) || !vector_rows(v, 2, 4)) {
        *why = "pool rows must be contiguous, data and strides 16-byte aligned";
        return VXFA_UNSUPPORTED;
    }
    return VXFA_OK;
}

constexpr int64_t kMaxRows = (int64_t)1 << 30;

PagedBatch batch_of(const vxfa_paged* b, const vxfa_tensor* k, int64_t tokens) {
    PagedBatch r;
    r.pages = b->pages; r.n_kv = b->n_kv; r.q_start = b->q_start;
    r.n_streams = b->n_streams;
    r.max_pages = b->max_pages;
    r.n_pages = (int32_t)k->ne[3];
    r.ps_log2 = 0;
    while (((int64_t)1 << r.ps_log2) < k->ne[1]) ++r.ps_log2;
    r.tokens = (int32_t)tokens;
    r.max_nq = b->max_nq;
    // (rows, and sums and differences of two of their numbers, fit 32 bits)
    int64_t rows = (int64_t)b->max_pages << r.ps_log2;
    if (rows > kMaxRows) rows = kMaxRows;
    r.max_nkv = (int32_t)(b->max_nkv > 0 && b->max_nkv < rows ? b->max_nkv : rows);
    if (r.n_pages == 0) r.max_nkv = 0;   // (an absent page's rows may be loaded from page 0)
    return r;
}

PagedPool pool_of(const vxfa_tensor* k, const vxfa_tensor* v) {
    return PagedPool{static_cast<char*>(k->data), static_cast<char*>(v->data), (int64_t)k->nb[1], (int64_t)k->nb[2],
                     (int64_t)k->nb[3]};
}

// F32 [Hkv * D, T, 1, 1]
int check_new(const vxfa_tensor* t, const vxfa_tensor* pool, const char** why) {
    if (t->ne[0] != pool->ne[0] * pool->ne[2] || t->ne[2] != 1 || t->ne[3] != 1) {
        *why = "new rows must be [Hkv * D, T, 1, 1]";
        return VXFA_INVALID_ARG;
    }
    if (t->type != VXFA_TYPE_F32) { *why = "new rows must be F32"; return VXFA_UNSUPPORTED; }
    if (!vector_rows(t, 4, 2)) { *why = "new rows must be contiguous and 16-byte aligned"; return VXFA_UNSUPPORTED; }
    return VXFA_OK;
}

// [page_size, Hkv, n_pages, 1] F32
int check_weights(const vxfa_tensor* w, const vxfa_tensor* k, const char** why) {
    if (!sane(w) || w->ne[0] != k->ne[1] || w->ne[1] != k->ne[2] || w->ne[2] != k->ne[3] || w->ne[3] != 1) {
        *why = "weights must be [page_size, Hkv, n_pages, 1]";
        return VXFA_INVALID_ARG;
    }
    if (w->type != VXFA_TYPE_F32 || w->nb[0] != 4 || !aligned(w->data, 4) || (w->nb[1] & 3) || (w->nb[2] & 3)) {
        *why = "weights must be F32, contiguous within a page and 4-byte aligned";
        return VXFA_UNSUPPORTED;
    }
    return VXFA_OK;
}

constexpr int64_t kMaxTokens = vxfa::kMaxGridX;

// The context's device for the time of a call.
struct OnDevice {
    int prev = -1;
    hipError_t e;
    explicit OnDevice(int device) {
        int cur = -1;
        e = hipGetDevice(&cur);
        if (e == hipSuccess && cur != device) {
            e = hipSetDevice(device);
            prev = cur;
        }
    }
    ~OnDevice() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

}  // namespace

extern "C" {

int vxfa_paged_append(vxfa_ctx* c, const vxfa_tensor* k_new, const vxfa_tensor* v_new, const vxfa_paged* batch,
                      vxfa_tensor* k, vxfa_tensor* v, const vxfa_rope* rope, const vxfa_tensor* q, vxfa_tensor* q_out,
                      void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    int rc = check_pool(k, v, batch, true, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if (!k_new || !v_new) return fail(c, VXFA_INVALID_ARG, "k_new and v_new are required");
    if (!sane(k_new) || !sane(v_new)) return fail(c, VXFA_INVALID_ARG, "new rows: unknown type, negative ne or absurd nb");
    if ((rc = check_new(k_new, k, &why)) != VXFA_OK || (rc = check_new(v_new, v, &why)) != VXFA_OK)
        return fail(c, rc, "%s", why);
    if (missing(batch, k_new) || missing(batch, v_new)) return fail(c, VXFA_INVALID_ARG, "new rows: data is required");
    const int64_t T = k_new->ne[1], D = k->ne[0];
    if (v_new->ne[1] != T) return fail(c, VXFA_INVALID_ARG, "k_new and v_new row counts differ");
    if ((q == nullptr) != (q_out == nullptr) || (q && !rope))
        return fail(c, VXFA_INVALID_ARG, "q and q_out come together, with rope");
    if (rope) {
        if (!rope->positions || !aligned(rope->positions, 4) || rope->n_dims <= 0 || rope->n_dims % 2 || rope->n_dims > D)
            return fail(c, VXFA_INVALID_ARG, "rope: positions are required; n_dims must be even and at most the head dim");
        if (rope->mode != 0 || rope->freq_scale != 1.0f || !(rope->freq_base > 0.0f) || !isfinite(rope->freq_base))
            return fail(c, VXFA_UNSUPPORTED, "rope: mode 0, freq_scale 1 and freq_base > 0 only");
    }
    if (q) {
        if (!sane(q) || !sane(q_out)) return fail(c, VXFA_INVALID_ARG, "q and q_out: unknown type, negative ne or absurd nb");
        for (int d = 0; d < 4; ++d)
            if (q->ne[d] != q_out->ne[d]) return fail(c, VXFA_INVALID_ARG, "q and q_out shapes differ");
        if (missing(batch, q) || missing(batch, q_out)) return fail(c, VXFA_INVALID_ARG, "q and q_out: data is required");
        if (q->ne[0] != D || q->ne[1] != T || q->ne[3] != 1)
            return fail(c, VXFA_INVALID_ARG, "q must be [D, T, Hq, 1]");
        if (q->type != VXFA_TYPE_F32 || q_out->type != VXFA_TYPE_F16)
            return fail(c, VXFA_UNSUPPORTED, "q must be F32, q_out F16");
        if (!vector_rows(q, 4, 3) || !vector_rows(q_out, 2, 3))
            return fail(c, VXFA_UNSUPPORTED, "q and q_out rows must be contiguous and 16-byte aligned");
    }
    if (T > kMaxTokens || (q && q->ne[2] > 65535)) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    vxfa::PagedAppend a;
    memset(&a, 0, sizeof(a));
    a.b = batch_of(batch, k, T);
    a.k_new = static_cast<const float*>(k_new->data);
    a.v_new = static_cast<const float*>(v_new->data);
    a.kn_nb1 = (int64_t)k_new->nb[1];
    a.vn_nb1 = (int64_t)v_new->nb[1];
    a.kv = pool_of(k, v);
    a.d = (int32_t)D;
    a.hkv = (int32_t)k->ne[2];
    if (rope) {
        a.rope_pos = rope->positions;
        a.rope_ts = powf(rope->freq_base, -2.0f / (float)rope->n_dims);
        a.rope_dims = rope->n_dims;
    }
    if (q) {
        a.q = static_cast<const float*>(q->data);
        a.q_nb1 = (int64_t)q->nb[1]; a.q_nb2 = (int64_t)q->nb[2];
        a.q_out = static_cast<_Float16*>(q_out->data);
        a.qo_nb1 = (int64_t)q_out->nb[1]; a.qo_nb2 = (int64_t)q_out->nb[2];
        a.hq = (int32_t)q->ne[2];
    }
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    const hipError_t e = vxfa::launch_paged_append(a, reinterpret_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "paged append: %s", hipGetErrorString(e));
    return VXFA_OK;
}

int vxfa_flash_attn_ext_paged(vxfa_ctx* c, const vxfa_tensor* q, const vxfa_tensor* k, const vxfa_tensor* v,
                              const vxfa_paged* batch, vxfa_tensor* dst, float scale, float max_bias,
                              float logit_softcap, const vxfa_tensor* weights_in, vxfa_tensor* weights, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    int rc = check_pool(k, v, batch, true, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if (!q || !dst) return fail(c, VXFA_INVALID_ARG, "q and dst are required");
    if (!sane(q) || !sane(dst)) return fail(c, VXFA_INVALID_ARG, "q and dst: unknown type, negative ne or absurd nb");
    if (missing(batch, q) || missing(batch, dst)) return fail(c, VXFA_INVALID_ARG, "q and dst: data is required");
    const int64_t D = k->ne[0], T = q->ne[1], Hq = q->ne[2], Hkv = k->ne[2];
    if (q->ne[0] != D || q->ne[3] != 1 || Hq % Hkv) return fail(c, VXFA_INVALID_ARG, "q must be [D, T, Hq, 1], Hq a multiple of Hkv");
    if (dst->ne[0] != D || dst->ne[1] != Hq || dst->ne[2] != T || dst->ne[3] != 1)
        return fail(c, VXFA_INVALID_ARG, "dst must be [D, Hq, T, 1]");
    const size_t ds = dst->type == VXFA_TYPE_F16 ? 2 : 4;
    if (dst->nb[0] != ds || dst->nb[1] != ds * (size_t)D || dst->nb[2] != ds * (size_t)(D * Hq) || !aligned(dst->data, 16))
        return fail(c, VXFA_UNSUPPORTED, "dst must be contiguous and 16-byte aligned");
    if (!vector_rows(q, q->type == VXFA_TYPE_F16 ? 2 : 4, 3))
        return fail(c, VXFA_UNSUPPORTED, "q rows must be contiguous and 16-byte aligned");
    if (!isfinite(scale) || !isfinite(max_bias) || !isfinite(logit_softcap) || max_bias < 0 || logit_softcap < 0)
        return fail(c, VXFA_UNSUPPORTED, "scale, max_bias and logit_softcap must be finite, the latter two not negative");
    const bool wide_cap = logit_softcap > vxfa::kNarrowCap;
    const float c_score = logit_softcap > 0 && !wide_cap ? 2.0f * vxfa::kLog2e * (scale / logit_softcap) : scale * vxfa::kLog2e;
    if (!isfinite(c_score) || !isfinite(logit_softcap * vxfa::kLog2e))
        return fail(c, VXFA_UNSUPPORTED, "scale and logit_softcap: their ratio is out of range");
    if (T > kMaxTokens || Hq > 65535) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    if (weights_in && !weights) return fail(c, VXFA_INVALID_ARG, "weights_in without weights");
    if (weights && (rc = check_weights(weights, k, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if (weights_in && (rc = check_weights(weights_in, k, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if ((weights && missing(batch, weights)) || (weights_in && missing(batch, weights_in)))
        return fail(c, VXFA_INVALID_ARG, "weights: data is required");

    vxfa::PagedAttn a;
    memset(&a, 0, sizeof(a));
    a.b = batch_of(batch, k, T);
    if (Hq == 0) a.b.max_nq = 0;   // (nothing of q is read)
    a.q = q->data;
    a.q_nb1 = (int64_t)q->nb[1]; a.q_nb2 = (int64_t)q->nb[2];
    a.kv = pool_of(k, v);
    a.dst = dst->data;
    a.q_f16 = q->type == VXFA_TYPE_F16;
    a.dst_f16 = dst->type == VXFA_TYPE_F16;
    a.hq = (int32_t)Hq;
    a.hkv = (int32_t)Hkv;
    a.window = batch->window < a.b.max_nkv ? batch->window : 0;   // (a window of all rows is none)
    a.c = c_score;
    if (logit_softcap > 0) a.cap = logit_softcap * vxfa::kLog2e;
    if (wide_cap) a.capk = 2.0f / logit_softcap;
    if (max_bias > 0 && Hq > 0) {
        int64_t n2 = 1;
        while (2 * n2 <= Hq) n2 *= 2;
        a.n2 = (int32_t)n2;
        a.bias1 = -max_bias / (float)n2;
    }
    a.pieces = c->tune.paged_pieces;
    a.ws = c->ws;
    a.ws_bytes = kWorkspaceBytes;
    if (weights) {
        if (!vxfa::paged_weights_fit(a)) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
        const size_t lse = ((size_t)T * (size_t)Hq * sizeof(float) + 255) & ~(size_t)255;
        if (lse > a.ws_bytes)
            return fail(c, VXFA_NO_WORKSPACE, "weights need %zu bytes; the workspace holds %zu", lse, a.ws_bytes);
        a.lse = reinterpret_cast<float*>(a.ws);
        a.ws += lse;
        a.ws_bytes -= lse;
        if (weights_in) {
            a.w_in = static_cast<const float*>(weights_in->data);
            a.wi_nb2 = (int64_t)weights_in->nb[1]; a.wi_nb3 = (int64_t)weights_in->nb[2];
        }
        a.w_out = static_cast<float*>(weights->data);
        a.wo_nb2 = (int64_t)weights->nb[1]; a.wo_nb3 = (int64_t)weights->nb[2];
    }
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    // few tokens: every row's K and V read by the workgroup of all its query rows
    // (up to 16); else tiles of 32 query rows
    hipError_t e = hipSuccess;
    bool weighed = false;
    if (T * Hq > 0 && a.b.n_streams > 0 && a.b.max_nq > 0)
        e = vxfa::paged_rows_takes(a) ? vxfa::launch_paged_rows(a, (int)D, st, weighed) : vxfa::launch_paged_chunk(a, (int)D, st);
    if (e == hipSuccess && weights && !weighed) e = vxfa::launch_paged_weights(a, (int)D, st);
    if (e == hipErrorNotSupported) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    if (e == hipErrorOutOfMemory) return fail(c, VXFA_NO_WORKSPACE, "the tables of the call's work do not fit the workspace");
    if (e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "paged attention: %s", hipGetErrorString(e));
    return VXFA_OK;
}

int vxfa_paged_evict(vxfa_ctx* c, vxfa_tensor* k, vxfa_tensor* v, vxfa_tensor* weights, const vxfa_paged* batch,
                     const vxfa_evict* ev, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    int rc = check_pool(k, v, batch, false, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if (!weights || !ev) return fail(c, VXFA_INVALID_ARG, "weights and evict are required");
    if ((rc = check_weights(weights, k, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if (missing(batch, weights)) return fail(c, VXFA_INVALID_ARG, "weights: data is required");
    if (ev->budget <= 0 || ev->n_sink < 0 || ev->n_recent < 0 || (int64_t)ev->n_sink + ev->n_recent > ev->budget)
        return fail(c, VXFA_INVALID_ARG, "evict: budget > 0, n_sink >= 0, n_recent >= 0 and their sum within the budget");
    if (ev->max_pages < 0 || (ev->max_pages > 0 && !ev->pages) || !aligned(ev->pages, 4) || !aligned(ev->kept, 4) || !aligned(ev->n_kv, 4))
        return fail(c, VXFA_INVALID_ARG, "evict: pages are required, arrays 4-byte aligned");
    if (ev->n_kv && ev->n_kv == batch->n_kv) return fail(c, VXFA_INVALID_ARG, "evict: n_kv must not be the batch's");
    if (ev->budget > kMaxRows) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    vxfa::PagedEvict a;
    memset(&a, 0, sizeof(a));
    a.b = batch_of(batch, k, 0);
    a.kv = pool_of(k, v);
    a.w = static_cast<char*>(weights->data);
    a.w_nb2 = (int64_t)weights->nb[1]; a.w_nb3 = (int64_t)weights->nb[2];
    a.d = (int32_t)k->ne[0];
    a.hkv = (int32_t)k->ne[2];
    a.to = ev->pages;
    a.max_to = ev->max_pages;
    a.budget = ev->budget;
    a.n_sink = ev->n_sink;
    a.n_recent = ev->n_recent;
    a.n_out = ev->n_kv;
    a.kept = ev->kept;
    a.kept_row = ev->budget;
    if (!a.kept) {
        a.kept_row = ev->budget < a.b.max_nkv ? ev->budget : (a.b.max_nkv > 0 ? a.b.max_nkv : 1);
        const size_t need = (size_t)a.kept_row * (size_t)a.hkv * (size_t)a.b.n_streams * sizeof(int32_t);
        if (need > kWorkspaceBytes)
            return fail(c, VXFA_NO_WORKSPACE, "the kept rows' numbers need %zu bytes; the workspace holds %zu", need, kWorkspaceBytes);
        a.kept = reinterpret_cast<int32_t*>(c->ws);
    }
    if (!vxfa::paged_evict_fits(a)) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    const hipError_t e = vxfa::launch_paged_evict(a, reinterpret_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "paged evict: %s", hipGetErrorString(e));
    return VXFA_OK;
}

}  // extern "C"
