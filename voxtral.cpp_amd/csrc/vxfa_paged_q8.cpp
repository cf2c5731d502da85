// vxfa_paged_q8.cpp — the entry points of include/vxfa.h over pages of 8 bits and over
// chosen blocks: checks of their arguments, dispatch.
#include "fa_paged_q8.h"
#include "vxfa_paged_checks.h"

namespace {

using vxfa::PagedScales;

// F32 [page_size / rows, Hkv, n_pages, 1] beside a pool k
int check_scales(const vxfa_tensor* s, const vxfa_tensor* k, int64_t per_page, const char** why) {
    if (!sane(s) || s->ne[0] != per_page || s->ne[1] != k->ne[2] || s->ne[2] != k->ne[3] || s->ne[3] != 1) {
        *why = "scales must be [page_size / rows, Hkv, n_pages, 1]";
        return VXFA_INVALID_ARG;
    }
    if (s->type != VXFA_TYPE_F32 || s->nb[0] != 4 || !aligned(s->data, 4) || (s->nb[1] & 3) || (s->nb[2] & 3)) {
        *why = "scales must be F32, contiguous within a page and 4-byte aligned";
        return VXFA_UNSUPPORTED;
    }
    return VXFA_OK;
}

// A pool of 8 bits with its scales and the batch over it.
int check_pool8(const vxfa_tensor* k, const vxfa_tensor* ks, const vxfa_tensor* v, const vxfa_tensor* vs, const vxfa_paged* b, PagedScales& sc,
                const char** why) {
    int rc = check_pool(k, v, b, true, why, VXFA_TYPE_I8);
    if (rc != VXFA_OK) return rc;
    if (!ks || !vs) { *why = "k_scale and v_scale are required"; return VXFA_INVALID_ARG; }
    const int64_t per = k->ne[1] / vxfa::kScaleRows;
    if ((rc = check_scales(ks, k, per, why)) != VXFA_OK || (rc = check_scales(vs, k, per, why)) != VXFA_OK) return rc;
    if (missing(b, ks) || missing(b, vs)) { *why = "k_scale and v_scale: data is required"; return VXFA_INVALID_ARG; }
    if (ks->nb[1] != vs->nb[1] || ks->nb[2] != vs->nb[2]) { *why = "k_scale and v_scale must have the same strides"; return VXFA_UNSUPPORTED; }
    sc = PagedScales{static_cast<char*>(ks->data), static_cast<char*>(vs->data), (int64_t)ks->nb[1], (int64_t)ks->nb[2]};
    return VXFA_OK;
}

// Bounds I8 [2 D, page_size / block, Hkv, n_pages] and their scales; k: a pool, or what stands for one
int check_bounds(const vxfa_tensor* b, const vxfa_tensor* bs, const vxfa_tensor* k, const vxfa_paged* batch, vxfa::PagedBoundRows& r, const char** why) {
    if (b->ne[0] != 2 * k->ne[0] || b->ne[2] != k->ne[2] || b->ne[3] != k->ne[3] || b->ne[1] < 1 || (b->ne[1] & (b->ne[1] - 1)) ||
        b->ne[1] > k->ne[1] / 16) {
        *why = "bounds must be [2 D, page_size / block, Hkv, n_pages], blocks of 16 rows at least";
        return VXFA_INVALID_ARG;
    }
    if (b->type != VXFA_TYPE_I8 || !vector_rows(b, 1, 4)) {
        *why = "bounds must be I8, rows contiguous, data and strides 16-byte aligned";
        return VXFA_UNSUPPORTED;
    }
    const int rc = check_scales(bs, k, b->ne[1], why);
    if (rc != VXFA_OK) return rc;
    if (missing(batch, b) || missing(batch, bs)) { *why = "bounds and their scales: data is required"; return VXFA_INVALID_ARG; }
    r = vxfa::PagedBoundRows{static_cast<char*>(b->data), static_cast<char*>(bs->data), (int64_t)b->nb[1], (int64_t)b->nb[2], (int64_t)b->nb[3],
                             (int64_t)bs->nb[1], (int64_t)bs->nb[2], 0};
    while ((b->ne[1] << r.lg) < k->ne[1]) ++r.lg;
    return VXFA_OK;
}

// T tokens' lists of blocks of a pool with pages of `page` rows
int check_blocks(const vxfa_blocks* l, const vxfa_paged* batch, int64_t page, int64_t tokens, bool choose, const char** why) {
    if (!l) { *why = "blocks are required"; return VXFA_INVALID_ARG; }
    if (l->block < 16 || l->block > page || (l->block & (l->block - 1))) {
        *why = "blocks: a power of two from 16 to the page size";
        return VXFA_INVALID_ARG;
    }
    if (l->top < 1 || (choose && (l->n_sink < 0 || l->n_recent < 0 || (int64_t)l->n_sink + l->n_recent > l->top))) {
        *why = "blocks: top > 0, n_sink >= 0, n_recent >= 0 and their sum at most top";
        return VXFA_INVALID_ARG;
    }
    if ((!l->list && tokens > 0 && batch->n_streams > 0) || !aligned(l->list, 4)) {
        *why = "blocks: the list is required, 4-byte aligned";
        return VXFA_INVALID_ARG;
    }
    if (l->top > vxfa::kMaxTop) { *why = "blocks: 1024 of a token at most"; return VXFA_UNSUPPORTED; }
    return VXFA_OK;
}

int log2_of(int64_t x) {
    int r = 0;
    while (((int64_t)1 << r) < x) ++r;
    return r;
}

int launched(vxfa_ctx* c, hipError_t e, const char* what) {
    if (e == hipErrorNotSupported) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    if (e == hipErrorOutOfMemory) return fail(c, VXFA_NO_WORKSPACE, "the tables of the call's work do not fit the workspace");
    if (e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "%s: %s", what, hipGetErrorString(e));
    return VXFA_OK;
}

}  // namespace

extern "C" {

int vxfa_paged_append_q8(vxfa_ctx* c, const vxfa_tensor* k_new, const vxfa_tensor* v_new, const vxfa_paged* batch, vxfa_tensor* k,
                         vxfa_tensor* k_scale, vxfa_tensor* v, vxfa_tensor* v_scale, const vxfa_rope* rope, const vxfa_tensor* q,
                         vxfa_tensor* q_out, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    vxfa::PagedAppend8 a;
    int rc = check_pool8(k, k_scale, v, v_scale, batch, a.sc, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if ((rc = append_of(c, k_new, v_new, batch, k, v, rope, q, q_out, a.a)) != VXFA_OK) return rc;
    a.rope_ts = rope ? pow((double)rope->freq_base, -2.0 / (double)rope->n_dims) : 1.0;
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    return launched(c, vxfa::launch_paged_append_q8(a, reinterpret_cast<hipStream_t>(stream)), "paged append");
}

int vxfa_flash_attn_ext_paged_q8(vxfa_ctx* c, const vxfa_tensor* q, const vxfa_tensor* k, const vxfa_tensor* k_scale, const vxfa_tensor* v,
                                 const vxfa_tensor* v_scale, const vxfa_paged* batch, vxfa_tensor* dst, float scale, float max_bias,
                                 float logit_softcap, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    vxfa::PagedBlocks a;
    memset(&a, 0, sizeof(a));
    int rc = check_pool8(k, k_scale, v, v_scale, batch, a.sc, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if ((rc = attn_of(c, q, k, v, batch, dst, scale, max_bias, logit_softcap, a.a)) != VXFA_OK) return rc;
    a.a.pieces = c->tune.paged_pieces;
    a.a.ws = c->ws;
    a.a.ws_bytes = kWorkspaceBytes;
    if (a.a.b.tokens == 0 || a.a.hq == 0 || a.a.b.n_streams == 0 || a.a.b.max_nq == 0) return VXFA_OK;
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const int D = (int)k->ne[0];
    return launched(c, vxfa::paged_rows_takes(a.a) ? vxfa::launch_paged_rows_q8(a, D, st) : vxfa::launch_paged_chunk_q8(a.a, a.sc, D, st),
                    "paged attention");
}

int vxfa_paged_bounds(vxfa_ctx* c, const vxfa_tensor* k, const vxfa_tensor* k_scale, const vxfa_paged* batch, vxfa_tensor* bounds,
                      vxfa_tensor* bounds_scale, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    vxfa::PagedBounds a;
    memset(&a, 0, sizeof(a));
    int rc = k_scale ? check_pool8(k, k_scale, k, k_scale, batch, a.sc, &why) : check_pool(k, k, batch, true, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if (!bounds || !bounds_scale) return fail(c, VXFA_INVALID_ARG, "bounds and their scales are required");
    if (!sane(bounds, true)) return fail(c, VXFA_INVALID_ARG, "bounds: unknown type, negative ne or absurd nb");
    if ((rc = check_bounds(bounds, bounds_scale, k, batch, a.out, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    // (how many tokens there are is on the device alone: chunks are as long as q_start has it)
    a.b = batch_of(batch, k, 0x7fffffff);
    a.kv = pool_of(k, k);
    a.d = (int32_t)k->ne[0];
    a.hkv = (int32_t)k->ne[2];
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    return launched(c, vxfa::launch_paged_bounds(a, reinterpret_cast<hipStream_t>(stream)), "paged bounds");
}

int vxfa_paged_select(vxfa_ctx* c, const vxfa_tensor* q, const vxfa_tensor* bounds, const vxfa_tensor* bounds_scale, const vxfa_paged* batch,
                      const vxfa_blocks* blocks, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    if (!bounds || !bounds_scale || !batch || !blocks) return fail(c, VXFA_INVALID_ARG, "bounds, their scales, batch and blocks are required");
    if (!sane(bounds, true)) return fail(c, VXFA_INVALID_ARG, "bounds: unknown type, negative ne or absurd nb");
    if (bounds->ne[0] % 2 || blocks->block < 16 || bounds->ne[1] < 1 || bounds->ne[1] > (1 << 16) || (bounds->ne[1] & (bounds->ne[1] - 1)))
        return fail(c, VXFA_INVALID_ARG, "bounds must be [2 D, page_size / block, Hkv, n_pages], blocks of 16 rows at least");
    if (blocks->block & (blocks->block - 1)) return fail(c, VXFA_INVALID_ARG, "blocks: a power of two from 16 to the page size");
    // (the pool itself is not looked at: its page size is the blocks of a page times their rows)
    vxfa_tensor k = *bounds;
    k.type = VXFA_TYPE_I8;
    k.ne[0] = bounds->ne[0] / 2;
    k.ne[1] = bounds->ne[1] * blocks->block;
    for (int d = 0; d < 4; ++d) k.nb[d] = d == 0 ? 1 : 16;
    int rc = check_pool(&k, &k, batch, true, &why, VXFA_TYPE_I8);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    vxfa::PagedSelect a;
    memset(&a, 0, sizeof(a));
    if ((rc = check_bounds(bounds, bounds_scale, &k, batch, a.in, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if (!q || !sane(q)) return fail(c, VXFA_INVALID_ARG, "q: required; unknown type, negative ne or absurd nb");
    if (missing(batch, q)) return fail(c, VXFA_INVALID_ARG, "q: data is required");
    const int64_t D = k.ne[0], T = q->ne[1], Hq = q->ne[2], Hkv = k.ne[2];
    if (q->ne[0] != D || q->ne[3] != 1 || Hq % Hkv) return fail(c, VXFA_INVALID_ARG, "q must be [D, T, Hq, 1], Hq a multiple of Hkv");
    if (!vector_rows(q, q->type == VXFA_TYPE_F16 ? 2 : 4, 3)) return fail(c, VXFA_UNSUPPORTED, "q rows must be contiguous and 16-byte aligned");
    if ((rc = check_blocks(blocks, batch, k.ne[1], T, true, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    if (T > kMaxTokens || Hq > 65535) return fail(c, VXFA_UNSUPPORTED, "sizes beyond the launch limits");
    a.b = batch_of(batch, &k, T);
    if (((int64_t)a.b.max_nkv + blocks->block - 1) / blocks->block > vxfa::kSelectMost)
        return fail(c, VXFA_UNSUPPORTED, "more than %d blocks of a stream (max_nkv)", vxfa::kSelectMost);
    a.q = q->data;
    a.q_nb1 = (int64_t)q->nb[1]; a.q_nb2 = (int64_t)q->nb[2];
    a.q_f16 = q->type == VXFA_TYPE_F16;
    a.d = (int32_t)D;
    a.hq = (int32_t)Hq;
    a.hkv = (int32_t)Hkv;
    a.window = batch->window < a.b.max_nkv ? batch->window : 0;
    a.list = blocks->list;
    a.top = blocks->top;
    a.n_sink = blocks->n_sink;
    a.n_recent = blocks->n_recent;
    a.ws = c->ws;
    a.ws_bytes = kWorkspaceBytes;
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    return launched(c, vxfa::launch_paged_select(a, reinterpret_cast<hipStream_t>(stream)), "paged select");
}

int vxfa_flash_attn_ext_paged_blocks(vxfa_ctx* c, const vxfa_tensor* q, const vxfa_tensor* k, const vxfa_tensor* k_scale, const vxfa_tensor* v,
                                     const vxfa_tensor* v_scale, const vxfa_paged* batch, const vxfa_blocks* blocks, vxfa_tensor* dst, float scale,
                                     float max_bias, float logit_softcap, void* stream) {
    if (!c) return VXFA_INVALID_ARG;
    c->last_error[0] = 0;
    const char* why = "";
    vxfa::PagedBlocks a;
    memset(&a, 0, sizeof(a));
    int rc = k_scale || v_scale ? check_pool8(k, k_scale, v, v_scale, batch, a.sc, &why) : check_pool(k, v, batch, true, &why);
    if (rc != VXFA_OK) return fail(c, rc, "%s", why);
    if ((rc = attn_of(c, q, k, v, batch, dst, scale, max_bias, logit_softcap, a.a)) != VXFA_OK) return rc;
    if ((rc = check_blocks(blocks, batch, k->ne[1], q->ne[1], false, &why)) != VXFA_OK) return fail(c, rc, "%s", why);
    a.list = blocks->list;
    a.top = blocks->top;
    a.lg = log2_of(blocks->block);
    a.a.ws = c->ws;
    a.a.ws_bytes = kWorkspaceBytes;
    if (a.a.b.tokens == 0 || a.a.hq == 0 || a.a.b.n_streams == 0 || a.a.b.max_nq == 0) return VXFA_OK;
    OnDevice on(c->device);
    if (on.e != hipSuccess) return fail(c, VXFA_HIP_ERROR, "hipSetDevice: %s", hipGetErrorString(on.e));
    return launched(c, vxfa::launch_paged_blocks(a, (int)k->ne[0], reinterpret_cast<hipStream_t>(stream)), "paged attention over blocks");
}

}  // extern "C"
