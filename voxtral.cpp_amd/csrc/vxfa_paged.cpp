// vxfa_paged.cpp — the paged entry points of include/vxfa.h over F16 pages: workspace
// layout, dispatch. (Checks of arguments: vxfa_paged_checks.h.)
#include "vxfa_paged_checks.h"

extern "C" {

int vxfa_paged_append(vxfa_ctx* c, const vxfa_tensor* k_new, const vxfa_tensor* v_new, const vxfa_paged* batch,
                      vxfa_tensor* k, vxfa_tensor* v, const vxfa_rope* rope, const vxfa_tensor* q, vxfa_tensor* q_out,
                      void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    int rc = check_pool(k, v, batch, true, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    vxfa::PagedAppend a;
    if ((rc = append_of(c, k_new, v_new, batch, k, v, rope, q, q_out, a)) != VXFA_OK) return rc;
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
    vxfa::PagedAttn a;
    if ((rc = attn_of(c, q, k, v, batch, dst, scale, max_bias, logit_softcap, a)) != VXFA_OK) return rc;
    const int64_t D = k->ne[0], T = q->ne[1], Hq = q->ne[2];
    if (weights_in && !weights) return fail(c, VXFA_INVALID_ARG, "weights_in without weights");
    if (weights && (rc = check_weights(weights, k, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if (weights_in && (rc = check_weights(weights_in, k, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if ((weights && missing(batch, weights)) || (weights_in && missing(batch, weights_in)))
        return fail(c, VXFA_INVALID_ARG, "weights: data is required");
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
