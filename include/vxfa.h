/*
 * vxfa.h — C ABI of the MI355X (gfx950) attention path for voxtral.cpp.
 *
 * One operation: GGML_OP_FLASH_ATTN_EXT, with ggml's tensor contract.
 *
 *   dst = softmax(scale * Q K^T + mask) V, per query head, GQA-broadcast K/V.
 *
 * voxtral.cpp emits this op at two sites:
 *   src/voxtral.cpp:1611  encoder self-attention   (hd 64, no mask offline)
 *   src/voxtral.cpp:1802  decoder GQA attention    (32 q / 8 kv heads, hd 128,
 *                                                  causal mask or none)
 * Both pass max_bias = 0 and logit_softcap = 0.
 * The op constructor is ggml_flash_attn_ext(ctx, q, k, v, mask, scale,
 * max_bias, logit_softcap). It lives in ggml (external, pinned in
 * CMakeLists.txt:36-39). It is executed by a ggml backend's graph_compute,
 * which the scheduler calls from src/voxtral.cpp:2097, 2193, 2382.
 *
 * Tensor contract (ggml order, ne[0] fastest, nb in bytes):
 *   q    [D,  Nq,  Hq,  B ]  F32 or F16, rows contiguous (nb[0] = elt size)
 *   k    [D,  Nkv, Hkv, Bk]  F16 or F32, rows contiguous
 *   v    [D,  Nkv, Hkv, Bk]  same type as k, rows contiguous (not transposed)
 *   mask [Nkv, >=Nq, Hm, Bm] F16 additive (0 / -inf in voxtral), nullable,
 *                            elements contiguous along ne[0]
 *   dst  [D,  Hq,  Nq,  B ]  F32, contiguous (permuted relative to q)
 * with Hq % Hkv == 0, B % Bk == 0, Hq % Hm == 0, B % Bm == 0.
 * Query head h reads kv head h / (Hq / Hkv) and mask plane h % Hm.
 *
 * Semantics follow ggml's CPU kernel: a mask entry of -inf removes that kv
 * position; a query row with every position removed produces zeros. K and V
 * at removed positions are not skipped one by one: they may be read and
 * multiplied by zero where a block of 32 positions (128 in the offline and
 * realtime encoder's kernel, hd 64) holds a position that one of the tile's
 * rows attends, so they have to be finite there. Blocks that all of a tile's
 * rows remove, and rows past n_kv, may hold anything.
 *
 * Everything here is plain C: pointers, sizes and status codes. No HIP or
 * torch types cross the boundary. The stream argument is a hipStream_t
 * passed as void* (NULL = the null stream).
 */
#ifndef VXFA_H
#define VXFA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. The numeric values equal ggml's GGML_TYPE_F32 / GGML_TYPE_F16 /
 * GGML_TYPE_I8, so a ggml backend can pass tensor->type through unchanged. I8 is for
 * the pools of 8 bits below. */
enum vxfa_type {
    VXFA_TYPE_F32 = 0,
    VXFA_TYPE_F16 = 1,
    VXFA_TYPE_I8  = 24,
};

/* Status codes. Nothing aborts and no C++ exception crosses the ABI.
 * VXFA_UNSUPPORTED plays the role of ggml's supports_op() == false: the
 * caller runs the op elsewhere (ggml's scheduler falls back to the CPU
 * backend, which voxtral lists last at src/voxtral.cpp:1167-1170). */
enum vxfa_status {
    VXFA_OK           = 0,
    VXFA_UNSUPPORTED  = 1,  /* valid op, but this path does not implement it  */
    VXFA_INVALID_ARG  = 2,  /* violates the ggml contract (shapes, strides)   */
    VXFA_NO_WORKSPACE = 3,  /* the context's fixed workspace is too small     */
    VXFA_HIP_ERROR    = 4,  /* a HIP call failed; see vxfa_last_error()       */
};

/* A ggml tensor view: exactly the fields of struct ggml_tensor that the op
 * reads (type, ne, nb, data). data is a device pointer. */
typedef struct vxfa_tensor {
    void*   data;
    int32_t type;   /* enum vxfa_type */
    int32_t pad_;   /* keep ne[] 8-byte aligned; ignored */
    int64_t ne[4];
    size_t  nb[4];
} vxfa_tensor;

/* Per-stream context (the analogue of a ggml backend context). Owns one
 * device workspace of fixed size, allocated by vxfa_ctx_create and freed by
 * vxfa_ctx_destroy: 40 MiB, which hold a decode call's split-KV partial
 * records (8 MiB at most: partial O, running max and sum per split), or a
 * prefill call's f16 copies of F32 K/V (32 MiB at most: K and V of up to 8192
 * rows of 8 x 128), mask row intervals, rotated queries and records of KV
 * pieces, or what a paged call needs (records, scores and row sums, numbers of
 * kept rows). No other call allocates, frees or synchronises, so every call
 * can be captured into a HIP graph; a call whose records would need more
 * runs with fewer splits or pieces, a
 * prefill call with F32 K/V beyond the 32 MiB returns VXFA_NO_WORKSPACE. The
 * caller's tensors are never allocated or freed here. One context per
 * stream; calls on one context must not overlap. */
typedef struct vxfa_ctx vxfa_ctx;

/* Create a context bound to HIP device `device` and allocate its workspace
 * (40 MiB). Returns NULL on failure. */
vxfa_ctx* vxfa_ctx_create(int device);

/* Destroy a context and free its workspace. NULL is accepted. */
void vxfa_ctx_destroy(vxfa_ctx* ctx);

/* Capability check. Mirrors a ggml backend's supports_op() for
 * GGML_OP_FLASH_ATTN_EXT (the scheduler consults it when placing the node;
 * placement order is set at src/voxtral.cpp:1156-1175). Pure host code: it
 * only reads the descriptors, never dereferences data, and makes no HIP call,
 * so it runs on a machine without a GPU.
 * Returns VXFA_OK, VXFA_UNSUPPORTED or VXFA_INVALID_ARG. */
int vxfa_supports(const vxfa_tensor* q, const vxfa_tensor* k,
                  const vxfa_tensor* v, const vxfa_tensor* mask,
                  const vxfa_tensor* dst, float scale, float max_bias,
                  float logit_softcap);

/* Execute GGML_OP_FLASH_ATTN_EXT. Replaces the backend kernel behind
 * ggml_flash_attn_ext(ctx, q, k, v, mask, scale, max_bias, logit_softcap)
 * at src/voxtral.cpp:1611 and :1802. Asynchronous on `stream`: the call
 * returns after the launches are queued, with no host synchronisation and no
 * allocation. Output is deterministic for equal inputs (fixed split
 * boundaries and merge order). F32 K/V (the reference's own cache,
 * src/voxtral.cpp:1126-1136, and the encoder's K/V, :1581-1605): a decode
 * step reads them in place and keeps both products in F32 with Q unrounded,
 * as ggml's CPU kernel does for F32 K; a prefill call copies them to f16 in
 * the context's staging area first and rounds Q, K and V to f16 as for f16
 * K/V. */
int vxfa_flash_attn_ext(vxfa_ctx* ctx, const vxfa_tensor* q,
                        const vxfa_tensor* k, const vxfa_tensor* v,
                        const vxfa_tensor* mask, vxfa_tensor* dst, float scale,
                        float max_bias, float logit_softcap, void* stream);

/* Implicit masks. voxtral.cpp fills every mask it passes from a formula:
 *   decoder prefill   causal [n, n]           fill_causal_mask,
 *                                             src/voxtral.cpp:2104-2111
 *                                             (used at :2421 and :2493)
 *   realtime encoder  causal window of 750    src/voxtral.cpp:2179-2190
 * then uploads it and casts it to F16 inside every layer's graph (:1564,
 * :1801). A descriptor of the formula replaces the tensor: query row i
 * (0-based along q's ne[1]) attends kv position j iff
 *   j <= i + offset   and, when window > 0,   j >= i + offset - window + 1.
 * (Decoder prefill: offset 0, window 0. Realtime encoder: offset 0, window
 * 750. A decode step with a sliding window W over n_kv cached rows:
 * offset n_kv - 1, window W.) The result equals vxfa_flash_attn_ext with an
 * F16 mask [Nkv, Nq, 1, 1] holding 0 at those positions and -inf elsewhere,
 * within rounding: bit for bit where both forms take the same kernel, as hd
 * 128 prefill of Nkv <= 512 does; larger calls and decode steps take the
 * kernel or the splits that are faster for the form.
 * The kernels derive live ranges and tile classes from the formula instead
 * of reading a mask, so no mask is filled, copied or scanned. */
enum vxfa_mask_kind {
    VXFA_MASK_NONE   = 0,  /* no mask: same as passing mask = NULL */
    VXFA_MASK_CAUSAL = 1,  /* causal, optionally limited to a window */
};

typedef struct vxfa_mask_desc {
    int32_t kind;    /* enum vxfa_mask_kind                                  */
    int32_t window;  /* 0: unbounded; W > 0: the last W positions up to the
                        diagonal                                             */
    int64_t offset;  /* kv position on query row 0's diagonal                 */
} vxfa_mask_desc;

/* Validate a mask descriptor (pure host code). NULL is valid (no mask).
 * Returns VXFA_OK or VXFA_INVALID_ARG. */
int vxfa_check_mask_desc(const vxfa_mask_desc* mask);

/* GGML_OP_FLASH_ATTN_EXT with an implicit mask (see above) in place of the
 * mask tensor; otherwise the same contract, status codes and stream
 * behaviour as vxfa_flash_attn_ext. No counterpart in ggml's op: it is for a
 * caller that owns the mask's formula (voxtral.cpp's builders at
 * src/voxtral.cpp:1801 and :1564 would pass a descriptor instead of the
 * cast mask tensor). mask = NULL or kind VXFA_MASK_NONE means no mask. */
int vxfa_flash_attn_ext_implicit(vxfa_ctx* ctx, const vxfa_tensor* q,
                                 const vxfa_tensor* k, const vxfa_tensor* v,
                                 const vxfa_mask_desc* mask, vxfa_tensor* dst,
                                 float scale, float max_bias,
                                 float logit_softcap, void* stream);

/* F16 KV cache append. build_decoder_layer stores each layer's new keys and
 * values with two ggml_cpy nodes into cache views (src/voxtral.cpp:1758-1770);
 * with an F16 cache these are F32 -> F16 conversions (round to nearest even,
 * overflow to inf). k_new, v_new: F32 [Hkv * D, n_new, 1, Bk], rows
 * contiguous (kv head h at elements h * D .. h * D + D - 1, the layout of
 * the reshape at :1743); k, v: the F16 cache views [D, n_kv, Hkv, Bk] the
 * attention op reads (:1773-1794). Rows n_kv - n_new .. n_kv - 1 of k and v
 * receive the new rows (voxtral's n_kv = kv_offset + n_tokens).
 * One launch for K and V; asynchronous on `stream`. */
int vxfa_kv_append(vxfa_ctx* ctx, const vxfa_tensor* k_new,
                   const vxfa_tensor* v_new, vxfa_tensor* k, vxfa_tensor* v,
                   void* stream);

/* vxfa_kv_append(k_new, v_new, k, v) followed by vxfa_flash_attn_ext(q, k,
 * v, mask, dst, ...). For a single-token decode step (Nq = 1, n_new = 1) the
 * append is fused into the attention kernel: the new row is read once from
 * the F32 source, used, and written to the cache by the same launch, with the
 * same cache bytes and a result that differs in the order of the F32 sums
 * (the new row last; within 1e-5); otherwise the append kernel runs first on
 * the same stream, with the same result bits. No counterpart in ggml's op:
 * it replaces the two ggml_cpy nodes plus the attention node of each decoder
 * layer (:1758-1802). */
int vxfa_flash_attn_ext_append(vxfa_ctx* ctx, const vxfa_tensor* q,
                               vxfa_tensor* k, vxfa_tensor* v,
                               const vxfa_tensor* k_new,
                               const vxfa_tensor* v_new,
                               const vxfa_tensor* mask, vxfa_tensor* dst,
                               float scale, float max_bias,
                               float logit_softcap, void* stream);

/* KV cache as a ring buffer. Once its cache holds VOXTRAL_DEC_WINDOW rows,
 * voxtral.cpp moves every layer's K and V one row to the left before each
 * decode step (kv_cache_shift_left, src/voxtral.cpp:1237-1266, called at
 * :2446-2449): (window - 1) rows per layer, K and V, on every token. With a
 * ring the same step is O(1): logical position p (0 = oldest kept token)
 * lives in cache row (start + p) mod capacity, so dropping the oldest row is
 * start = (start + 1) mod capacity, and no row is moved or cleared (rows at
 * logical positions >= n_kv are never read, which also makes the full-cache
 * memset of clear_kv_cache, :1222-1235, unnecessary). */
typedef struct vxfa_ring {
    int64_t start;  /* cache row of logical position 0; 0 <= start < capacity */
    int64_t n_kv;   /* rows in use (logical 0 .. n_kv - 1); <= capacity        */
} vxfa_ring;

/* A decode step over a ring: q [D, 1, Hq, B]; k, v the whole cache
 * [D, capacity, Hkv, Bk] (F16); attention over logical positions
 * 0 .. n_kv - 1 with no mask (voxtral's decode steps pass none, :1961,
 * :2052). With k_new / v_new (F32 [Hkv * D, 1, 1, Bk], or both NULL) the
 * step's new row is logical position n_kv - 1: it is rounded to f16, used
 * and written to its ring row in the same launch (as
 * vxfa_flash_attn_ext_append). The result equals vxfa_flash_attn_ext on a
 * linear cache holding the same rows in logical order. Single-token decode
 * with GQA group 1, 2 or 4 only, capacity below 2^24 rows and capacity *
 * row stride below 2 GiB (else VXFA_UNSUPPORTED). No counterpart in
 * ggml's op: it replaces the host-side shift plus the attention node. */
int vxfa_flash_attn_ext_ring(vxfa_ctx* ctx, const vxfa_tensor* q,
                             vxfa_tensor* k, vxfa_tensor* v,
                             const vxfa_ring* ring, const vxfa_tensor* k_new,
                             const vxfa_tensor* v_new, vxfa_tensor* dst,
                             float scale, float max_bias, float logit_softcap,
                             void* stream);

/* Rotary embedding fused into the op. build_decoder_layer rotates Q and K
 * with ggml_rope_ext (src/voxtral.cpp:1746-1749: mode 0, n_dims = head dim,
 * freq_base = the decoder's rope theta, freq_scale 1, ext_factor 0,
 * attn_factor 1), copies them contiguous (:1752-1753), stores K and V in
 * the cache (:1758-1770) and attends (:1802); the realtime encoder rotates
 * Q and K the same way with its own theta (:1595-1598). Pair j = dims
 * (2j, 2j+1) of a head at position p turns by theta_j, theta_0 = p and
 * theta_{j+1} = theta_j * freq_base^(-2 / n_dims) (ggml's running product),
 * x0' = x0 cos - x1 sin, x1' = x0 sin + x1 cos; dims >= n_dims are not
 * rotated. */
typedef struct vxfa_rope {
    const int32_t* positions;  /* device; token i of batch b: positions[b * Nq + i] */
    int32_t n_dims;            /* rotated leading dims of each head (even, <= D)      */
    int32_t mode;              /* 0 (ggml's GGML_ROPE_TYPE_NORMAL: adjacent pairs)    */
    float   freq_base;         /* rope theta                                          */
    float   freq_scale;        /* 1                                                   */
} vxfa_rope;

/* The op on unrotated inputs: rotate q (F32 [D, Nq, Hq, B]) and the new K
 * rows, append the new rows (k_new, v_new F32 [Hkv * D, Nq, 1, B]: the new
 * rows are the query tokens, at the last Nq rows of the F16 views k, v),
 * then attend. Equals vxfa_flash_attn_ext_append(rope(q), k, v, rope(k_new),
 * v_new, mask, ...) within the rounding of cos / sin and, where a prefill
 * call takes another kernel, of its order of sums. A decode step is one
 * launch; otherwise the append (with K rotation) runs first. No counterpart
 * in ggml's op: it replaces the two rope nodes, their contiguous copies, the
 * two cache copies and the attention node of a layer. */
int vxfa_flash_attn_ext_rope(vxfa_ctx* ctx, const vxfa_tensor* q,
                             vxfa_tensor* k, vxfa_tensor* v,
                             const vxfa_tensor* k_new,
                             const vxfa_tensor* v_new, const vxfa_rope* rope,
                             const vxfa_tensor* mask, vxfa_tensor* dst,
                             float scale, float max_bias, float logit_softcap,
                             void* stream);

/* GGML_OP_FLASH_ATTN_EXT without a context and without any allocation. No
 * counterpart in the reference: it is for callers that cannot allocate
 * device memory or create a context at that point (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc). Same
 * contract, results (the same bits, unless staged F32 K/V leave a mask
 * tensor's row intervals no room) and status codes as vxfa_flash_attn_ext,
 * on the current HIP device and `stream`; the scratch it needs (what a
 * context's workspace holds, above) lives in static arrays in the library's
 * code object (8 MiB, and 40 MiB for the records of KV pieces), one of each per
 * GPU, kept until the process ends. Limits:
 * F32 K/V prefill calls whose f16 K and V exceed 8 MiB return
 * VXFA_NO_WORKSPACE; decode steps always run (with fewer splits if their
 * records would not fit, which the call shapes of voxtral never reach). Every call on one GPU shares the array, so calls that
 * overlap on one GPU race. Its messages are read with vxfa_last_error(NULL)
 * (per calling thread). */
int vxfa_flash_attn_ext_noalloc(const vxfa_tensor* q, const vxfa_tensor* k,
                                const vxfa_tensor* v, const vxfa_tensor* mask,
                                vxfa_tensor* dst, float scale, float max_bias,
                                float logit_softcap, void* stream);

/* ---- Paged K/V cache ---------------------------------------------------------
 *
 * Serving many streams from one pool of cache pages. No counterpart in the
 * reference, whose one stream owns a contiguous cache (src/voxtral.cpp:
 * 1126-1136) and drops its oldest row when that is full (:1237-1266).
 *
 * The pool is two descriptors, k and v [D, page_size, Hkv, n_pages] F16 (rows
 * contiguous; any 16-byte multiples as nb[1..3], so [page][row][head] and
 * [page][head][row] both do, but the same ones for k and v, and nb[1] below
 * 8 MiB), page_size a power of two from 16 to 65536. Pools of other strides, more
 * than 65535 streams, query or kv heads, or 2^24 - 1 tokens, and sizes beyond a
 * launch's grid give VXFA_UNSUPPORTED. Row r of stream s lies in row
 * r % page_size of the page that entry r / page_size of line s of the table
 * names. An entry outside [0, n_pages)
 * (-1, say) is an absent page: nothing is read there, its rows take no part,
 * and rows appended there are dropped. So pages that a window has left behind
 * can be freed at once.
 *
 * A call takes all streams of the batch with their chunks of new tokens, one
 * or many each, packed along q's ne[1]: stream s has the tokens q_start[s] ..
 * q_start[s + 1] - 1, and they are its last rows, n_kv[s] in all: token i of
 * t lies in row p = n_kv[s] - t + i. The tables and sizes are device memory,
 * read when the kernels run, so a captured call follows them from replay to
 * replay; the host gives bounds. Values out of range do no harm: n_kv is
 * taken as at most max_nkv (2^30 at most), q_start as within the call's tokens
 * and not decreasing, a row p below 0 takes no part, and tokens past max_nq of
 * a stream are left out; where chunks overlap, outputs and weights may be
 * anything. Rows of q and dst behind the last stream's are neither read nor
 * written. */
typedef struct vxfa_paged {
    const int32_t* pages;    /* device [n_streams][max_pages]                        */
    const int32_t* n_kv;     /* device [n_streams]: rows in use, the new ones included */
    const int32_t* q_start;  /* device [n_streams + 1], from 0 up                    */
    int32_t n_streams;
    int32_t max_pages;       /* entries of a line of the table                       */
    int32_t max_nq;          /* no stream has more new tokens                        */
    int32_t max_nkv;         /* no stream has more rows (0: max_pages * page_size)   */
    int32_t window;          /* W > 0: a token sees the last W rows up to its own    */
    int32_t pad_;            /* 0 */
} vxfa_paged;

/* Store the new rows of all streams in their pages: k_new, v_new F32
 * [Hkv * D, T, 1, 1] with contiguous rows, rounded to f16 as by
 * vxfa_kv_append. With rope (positions: one per packed token; they need not
 * be the rows' numbers) K is rotated first as by vxfa_flash_attn_ext_rope,
 * and, with q (F32 [D, T, Hq, 1]) and q_out (F16, same ne), so are the
 * queries, rounded to f16 into q_out; q and q_out come together and need rope.
 * Two tokens of one row (streams that share a page) leave either's values, 8
 * elements at a time.
 * One launch; asynchronous on `stream`. */
int vxfa_paged_append(vxfa_ctx* ctx, const vxfa_tensor* k_new,
                      const vxfa_tensor* v_new, const vxfa_paged* batch,
                      vxfa_tensor* k, vxfa_tensor* v, const vxfa_rope* rope,
                      const vxfa_tensor* q, vxfa_tensor* q_out, void* stream);

/* Attention of the new tokens over their streams' rows, a token in row p over
 * the rows j <= p (and j > p - window): q [D, T, Hq, 1] F16 or F32 (rounded
 * to f16), dst [D, Hq, T, 1] F16 or F32, contiguous, D 64 or 128, any
 * Hq % Hkv == 0. The score of query head h is
 *   x = scale q.k;  logit_softcap > 0: x = logit_softcap tanh(x / logit_softcap);
 *   x += slope_h (j - p), with ggml's slopes for max_bias > 0: n the largest
 *   power of two in Hq, slope_h = 2^(-max_bias (h + 1) / n) for h < n, else
 *   2^(-max_bias (2 (h - n) + 1) / (2 n)); 0 for max_bias = 0.
 * Sums and statistics are F32, the products f16 MFMA; a capped x is off by at
 * most 2^-22 of a cap of up to 64, by 2^-18 of itself with larger ones (which
 * take longer, chunks up to 1.5 times). A token that sees no row gets zeros.
 * Rows that a token does not see (those of later tokens, those that a window
 * removes) may still be read where a block of 32 rows holds one that it or
 * another token of its chunk sees, and have to be finite there.
 *
 * weights (nullable) collects what each row is worth to the tokens:
 * F32 [page_size, Hkv, n_pages, 1], elements contiguous along ne[0];
 * element (row, kv head, page) of every row of a stream becomes that of
 * weights_in plus the sum, over the tokens and the head's query heads, of the
 * softmax's weights. weights_in may be weights itself, another tensor of that
 * shape, or NULL (zeros). Of a page that the call's tables name more than once
 * (streams with a common prefix) the elements are left open: weights_in's plus
 * the sum of one of its streams or of some of them, and not the same ones from
 * call to call. Streams that share pages therefore take their weights in calls
 * of their own, one after another, in place (weights_in = weights): their sums
 * then add up in that order. Rows of no stream are left as they were. Needs
 * 4 * Hq * T bytes of the workspace beside the call's tables, 8 bytes a stream
 * or 16 a tile of at least 32 tokens (else VXFA_NO_WORKSPACE).
 *
 * dst is deterministic, and so are the weights of pages that are named once;
 * asynchronous on `stream`. */
int vxfa_flash_attn_ext_paged(vxfa_ctx* ctx, const vxfa_tensor* q,
                              const vxfa_tensor* k, const vxfa_tensor* v,
                              const vxfa_paged* batch, vxfa_tensor* dst,
                              float scale, float max_bias, float logit_softcap,
                              const vxfa_tensor* weights_in,
                              vxfa_tensor* weights, void* stream);

/* What an eviction keeps of every stream and kv head: all rows if there are no
 * more than `budget`; else the first n_sink, the last n_recent, and of the
 * others the budget - n_sink - n_recent with the largest weights (of equal
 * ones the first; a NaN counts as less than any number). */
typedef struct vxfa_evict {
    const int32_t* pages;   /* device [n_streams][max_pages]: where the kept rows go */
    int32_t max_pages;
    int32_t budget;         /* rows kept of a stream, 1 .. 2^30                       */
    int32_t n_sink;         /* >= 0; n_sink + n_recent <= budget                     */
    int32_t n_recent;
    int32_t* kept;          /* device [n_streams][Hkv][budget]: row numbers kept,
                               ascending, then -1; or NULL                           */
    int32_t* n_kv;          /* device [n_streams]: rows left, min(n_kv, budget); or
                               NULL; not batch->n_kv                                 */
} vxfa_evict;

/* Keep the best rows of every stream, for each kv head its own: the kept rows
 * of k, v and weights move, in their order, to rows 0, 1, .. of the pages that
 * evict->pages names, each at most once, pages of the same pool that no stream
 * of the call lies in (streams may share pages, which an eviction in place
 * would spoil for the others). The old pages are left as they were.
 * batch->q_start is not read; max_nq and window, which may not be negative here
 * either, have no effect. Rows that lie in absent pages count as rows of
 * weight NaN and of zeros. Afterwards row numbers are no longer token
 * positions: the distances and windows of further calls go by rows. Needs
 * 4 * Hkv * n_streams * min(budget, max_nkv) bytes of the workspace where kept
 * is NULL (else VXFA_NO_WORKSPACE). Asynchronous on `stream`. */
int vxfa_paged_evict(vxfa_ctx* ctx, vxfa_tensor* k, vxfa_tensor* v,
                     vxfa_tensor* weights, const vxfa_paged* batch,
                     const vxfa_evict* evict, void* stream);

/* ---- Paged K/V cache of 8 bits ------------------------------------------------
 *
 * The same pool with half the bytes: k, v [D, page_size, Hkv, n_pages] I8,
 * laid out as above (strides of 16-byte multiples, the same ones for k and v),
 * and beside each its scales, F32 [page_size / 16, Hkv, n_pages, 1], elements
 * contiguous along ne[0], the same strides for k_scale and v_scale. Row r of a
 * page and head holds the values scale[r / 16] * k[r]. No counterpart in the
 * reference, whose cache is F16 or F32 (src/voxtral.cpp:1126-1136).
 *
 * The scales that vxfa_paged_append_q8 writes are powers of two 2^e, -64 <= e
 * <= 64; the whole numbers go from -127 to 127. So the product with a scale is
 * exact, and the numbers of a block whose scale has to grow are shifted.
 * Attention takes any scales from 2^-64 to 2^64 (others count as the nearer
 * end, NaN as 2^-64). Rows under a scale of V that is less than 2^-96 of the
 * largest one that the token sees may be missing from the sum of its softmax
 * (rows of zeros have the least scale, 2^-64: so it takes elements of V beyond
 * 127 * 2^32). */

/* vxfa_paged_append into pages of 8 bits: arguments, rotation, queries and
 * absent pages as there, but for the angles: they are formed in 64 bits (a
 * running product in F32, as there and in ggml, is off by up to 1e-3 at
 * position 8192, which F16 hides less and less the further a position is). Of
 * every 16 rows (of a page) and head that new rows come into, K's scale and
 * V's become the least 2^e (-64 <= e <= 64) with max |x| <= 127 * 2^e over the
 * new rows, or stay what they are where rows ahead of the new ones have a
 * larger one (which has to be such a power). New rows are stored as x / 2^e
 * rounded to nearest even (NaN as 0; beyond 127 as 127); the rows ahead are
 * rounded again, to nearest even, where the scale grows: a value is off by at
 * most half a step of the final scale for its own rounding, and the same again
 * for every time that its block's scale has grown, by a factor of 2 at least,
 * since. Rows of the 16 behind the new ones keep their numbers and are worth
 * nothing until a later append. Streams whose new rows lie in the same 16 rows
 * of a page leave any values there. One launch; asynchronous on `stream`. */
int vxfa_paged_append_q8(vxfa_ctx* ctx, const vxfa_tensor* k_new,
                         const vxfa_tensor* v_new, const vxfa_paged* batch,
                         vxfa_tensor* k, vxfa_tensor* k_scale, vxfa_tensor* v,
                         vxfa_tensor* v_scale, const vxfa_rope* rope,
                         const vxfa_tensor* q, vxfa_tensor* q_out,
                         void* stream);

/* vxfa_flash_attn_ext_paged over pages of 8 bits, without accumulated weights.
 * The products are of f16 (in which the whole numbers are exact) and scales
 * are applied to the scores and sums in F32. A row's weight in the sum over V
 * is rounded to f16 times V's scale: by half a step (2^-11 of it), as over
 * pages of F16, or by 2^-25 of the largest such product that the token sees,
 * where there it is 2^-25 of the largest weight; times whole numbers of up to
 * 127. So of rows whose product lies more than 2^14 below the largest digits
 * are lost, and below 2^-25 of it they no longer count in the outputs (in the
 * sum of the softmax they do): this is felt where V's scales lie that far apart
 * and the elements under the large ones are 0. Rows that a token does not see
 * may hold anything. */
int vxfa_flash_attn_ext_paged_q8(vxfa_ctx* ctx, const vxfa_tensor* q,
                                 const vxfa_tensor* k, const vxfa_tensor* k_scale,
                                 const vxfa_tensor* v, const vxfa_tensor* v_scale,
                                 const vxfa_paged* batch, vxfa_tensor* dst,
                                 float scale, float max_bias,
                                 float logit_softcap, void* stream);

/* ---- Attention over chosen blocks ---------------------------------------------
 *
 * A token of a long stream looks at a few blocks of its rows only: those whose
 * keys may have the largest products with its queries. Bounds of every block's
 * keys are kept beside the pool (of F16 or 8 bits) and brought up to date
 * after each append; a call chooses blocks for every new token and kv head by
 * them; a call attends over the chosen ones. A block is 16, 32, .. rows, up to
 * a page: block b of a stream is its rows b * block .. (b + 1) * block - 1.
 *
 * Bounds: I8 [2 D, page_size / block, Hkv, n_pages], rows contiguous, strides
 * of 16-byte multiples, and their scales, F32 [page_size / block, Hkv,
 * n_pages, 1], contiguous along ne[0]. Of a block and head with keys k: 2^e
 * the least power (-64 <= e <= 64) with max |k| <= 127 * 2^e; element d < D
 * the largest k_d / 2^e, rounded up, element D + d the smallest, rounded down.
 * (NaN among keys is passed over, a dim without a number counts as 0; what
 * lies beyond 127 * 2^64, as infinities do, counts as that.) */

/* Bounds of the blocks that the batch's new tokens lie in, over the streams'
 * rows in them. k_scale: of a pool of 8 bits; NULL for F16. max_nq bounds the
 * new tokens as elsewhere; the window has no effect. Blocks of absent pages
 * are left out. The new tokens need not be new: a batch whose chunks are as
 * long as its streams brings all their bounds up to date, as after
 * vxfa_paged_evict, which moves rows and not their bounds. Streams with
 * different numbers of rows in one block of a page that they share leave any
 * values there (whole blocks of a common prefix may be written by all). One
 * launch; asynchronous on `stream`. */
int vxfa_paged_bounds(vxfa_ctx* ctx, const vxfa_tensor* k,
                      const vxfa_tensor* k_scale, const vxfa_paged* batch,
                      vxfa_tensor* bounds, vxfa_tensor* bounds_scale,
                      void* stream);

/* Blocks chosen for each token and kv head. */
typedef struct vxfa_blocks {
    int32_t* list;     /* device [T][Hkv][top]: numbers of a stream's blocks, then -1 */
    int32_t block;     /* rows of a block: a power of two from 16 to the page size    */
    int32_t top;       /* blocks of a token and head, 1 .. 1024                       */
    int32_t n_sink;    /* >= 0; n_sink + n_recent <= top                              */
    int32_t n_recent;
} vxfa_blocks;

/* Choose blocks for the batch's new tokens: blocks->list of token i and kv
 * head h becomes, of the blocks with rows that the token sees (within the
 * window), the first n_sink, the last n_recent, and of the others those of the
 * largest scores (of equal ones the first), `top` in all or as many as there
 * are; ascending, then -1. (Under a window the first are the window's, not the
 * stream's.) Blocks in absent pages are not chosen by score; the first and last
 * are listed wherever they lie and take their entries of `top`, also where their
 * pages are absent and they have no rows to attend. The score of a block is the
 * largest, over the kv head's query heads, of
 *   2^(e + f) sum_d (r_d > 0 ? r_d hi_d : r_d lo_d)
 * with the block's bounds hi, lo at scale 2^e and the head's query (as F16) in
 * 8 bits, r_d = q_d / 2^f rounded to nearest even, f as for bounds (infinities
 * as 127 * 2^64; with NaN in a query the choice is any). It is formed exactly
 * and the choice is the same everywhere. (No cap or slope changes it; a negative
 * scale of the attention turns its meaning around.) q [D, T, Hq, 1] F16 or F32.
 * Tokens of no stream leave the list as it was.
 * bounds_scale: powers of two from 2^-64 to 2^64 (what lies outside counts as
 * the nearer end, NaN as 2^-64; by others the choice may differ from the
 * formula's). At most 262144 blocks of a stream (max_nkv; else
 * VXFA_UNSUPPORTED). Where streams have more than 4096 blocks (with 16 / n
 * tokens of a stream at once for kv heads of n query heads, n rounded up to a
 * power of two, 16384 by that many), and with few tokens from 512 on, the call
 * leaves the best of segments of blocks in the workspace, 8 bytes times top
 * for each token, kv head and segment (else VXFA_NO_WORKSPACE). Up to 16384 of
 * these for a token and head are joined quickly: 65536 blocks of a stream with
 * top 1024 take 86 us, 69632 with 17 segments 1.3 ms. Asynchronous on
 * `stream`. */
int vxfa_paged_select(vxfa_ctx* ctx, const vxfa_tensor* q,
                      const vxfa_tensor* bounds, const vxfa_tensor* bounds_scale,
                      const vxfa_paged* batch, const vxfa_blocks* blocks,
                      void* stream);

/* vxfa_flash_attn_ext_paged, without accumulated weights, over the rows of
 * chosen blocks only: token i, kv head h over the rows of blocks->list[i][h],
 * as far as the token sees them (j <= p, the window). Numbers of blocks in any
 * order; those below 0, or of rows that the token does not see, count for
 * nothing, one that is listed twice counts twice. n_sink and n_recent are not
 * looked at. The pool is F16 (k_scale and v_scale NULL) or of 8 bits. A token
 * without a row gets zeros. Each token's list is walked by itself: for many
 * tokens of a stream the call over all rows is the faster one (32/8 heads of
 * 128, lists of 2048 rows: 64 tokens over 8192 rows take as long either way,
 * 256 tokens 145 us for 55, of 8 bits 91 for 55). In an F16 pool rows of a
 * token's blocks that it does not see have to be finite, within 16 rows of one
 * that it sees. */
int vxfa_flash_attn_ext_paged_blocks(vxfa_ctx* ctx, const vxfa_tensor* q,
                                     const vxfa_tensor* k, const vxfa_tensor* k_scale,
                                     const vxfa_tensor* v, const vxfa_tensor* v_scale,
                                     const vxfa_paged* batch,
                                     const vxfa_blocks* blocks, vxfa_tensor* dst,
                                     float scale, float max_bias,
                                     float logit_softcap, void* stream);

/* Human-readable name of a status code (static storage). */
const char* vxfa_status_str(int status);

/* Message for the last failing call on this context ("" if none); with
 * NULL, for the calling thread's last vxfa_flash_attn_ext_noalloc call. */
const char* vxfa_last_error(const vxfa_ctx* ctx);

/* Library version: major * 10000 + minor * 100 + patch. */
int vxfa_version(void);

#ifdef __cplusplus
}
#endif

#endif /* VXFA_H */
