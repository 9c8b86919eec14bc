/* vireo-b200: serving many requests from one paged key-value pool.
 *
 * The reference keeps its keys and values behind a store of its own
 * (vireo src/kvstore.h:48-71: append, attend; the dense store
 * src/kvstore_dense.c:39-49, the paged one src/kvstore_ooc.c with its pinned
 * first and last blocks and the mean-key block selection of
 * src/select/select_topk.c:18-44) and serves one sequence.  Here the pool is
 * device memory shared by any number of requests, each holding a list of
 * pages, and a decode step over all of them is four calls:
 *
 *   gguf_kv_plan       request lengths -> block tables, slots, positions
 *   gguf_kv_append     bias, QK norm, rotation; keys and values to their slots
 *   gguf_kv_attn       one token per request over all its cached positions
 *   gguf_kv_attn_topk  the same over the first, the last and the best pages
 *
 * All pointers are pointers to memory of the library's device (that of
 * vireo_device_init, or current at the first call).  Every call is stream-ordered (stream: a
 * cudaStream_t passed as void*, NULL = the library's own stream), allocates
 * nothing, synchronises nothing and may be captured into a CUDA graph, but
 * for the library's very first call in the process, which sets the device up:
 * make that (vireo_device_init, say) ahead of any capture.  A
 * bad value met on the device (a page or a slot outside the pool, a length
 * beyond the table) reads as stated at the call, never past a buffer, and
 * is reported by gguf_kv_sync as VIREO_ERR_ARG.  Arguments are checked
 * before anything is launched; types and shapes that are not supported
 * return VIREO_ERR_UNSUPPORTED.
 *
 * Types are GGML type ids: 0 F32, 1 F16, 30 BF16.  Activations and cache go
 * together as (F32, F32), (F32, F16), (F16, F16) and (BF16, BF16).  Sums,
 * softmax statistics and norms are held in fp32.  Over a 16-bit cache the
 * softmax weights, and fp32 queries, enter the products as two values of the
 * cache's type: 22 bits with F16 (of weights down to 2^-17 of the largest and
 * queries down to 2^-17 of their row's largest; 2^-39 of that below), 16 with
 * BF16.  A weight's power of two is good to 2^-22 of itself. */
#ifndef VIREO_GGUF_KV_H
#define VIREO_GGUF_KV_H
#include <stddef.h>
#include <stdint.h>

#include "vireo_status.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One layer's pool.  Element (page p, kv head g, position o, dimension d) of
 * k and of v is at p * page_stride + g * head_stride + o * pos_stride + d
 * (strides in elements), so heads may lie outside positions or inside them,
 * and k and v may share one buffer. */
typedef struct {
    int n_heads, n_kv_heads; /* n_heads a multiple of n_kv_heads */
    int head_size;           /* 64, 128 or 256 */
    int page_size;           /* positions per page: a power of two, 8 to 1024 */
    int n_pages;
    uint32_t kv_type, act_type;
    void *k, *v;             /* 16-byte aligned */
    int64_t page_stride, head_stride, pos_stride; /* multiples of 16 bytes; of a dimension of extent 1 unused */
    float eps;               /* of the QK norms */
    float rope_base;
    int rope_dim;            /* dimensions turned: 0 (none) or a multiple of 16 up to head_size */
} gguf_kv_desc;

typedef struct gguf_kv gguf_kv;

/* The handle holds the description and the tables made from it, no scratch:
 * calls on one handle may run on several streams at once (with workspaces of
 * their own).  The pool stays the caller's. */
int gguf_kv_create(const gguf_kv_desc *desc, gguf_kv **out);
void gguf_kv_destroy(gguf_kv *kv);
/* waits for the stream and returns the first device-side status recorded */
int gguf_kv_sync(gguf_kv *kv, void *stream);

/* ---- block tables and slot maps -------------------------------------------
 *
 * Request i has past[i] positions in the cache, on the pages
 * table[i * table_stride + 0 .. ceil(past[i] / page_size) - 1], and asks for
 * add[i] more (0: none; -1: the request ends and gives its pages back).
 * Free pages are in a ring of n_pages entries, state = {head, count}: the
 * free pages are ring[(head + j) % n_pages], j < count.
 *
 * A request is granted in order, first come first served: its new pages must
 * fit its table row (past + add <= max_pages * page_size), and unless it
 * needs none, the pages that it and every earlier request whose row holds
 * them asked for must be free; likewise, unless it asks for no tokens, the
 * tokens asked for so far must be at most n_slots.  Ends are always granted;
 * their pages go to the ring behind the last free one (in request order)
 * and are not handed out by the same call.  A request with past < 0,
 * add < -1 or more pages than its row has is refused.
 *
 * Written: the new pages' table entries (other entries stay); kv_len[i], the
 * cached positions after the call (past + add, 0 after an end, past when
 * refused and 0 where that is negative); granted[i] 1 or 0; cu[0 .. n_seqs],
 * the prefix sums of the tokens granted; per token, request after request, pos (its position) and
 * slots (page * page_size + offset); -1 and 0 in slots and pos behind the
 * last token, up to n_slots; the ring's new entries and state_out.  kv_len
 * may be past and state_out may be state; otherwise nothing written may
 * overlap anything read.  Page numbers are handed on as the table and the ring
 * hold them: the attention reports all that are not of the pool, and
 * gguf_kv_append skips the tokens of negative ones and reports the others; a
 * count outside 0 .. n_pages is cut to that.  n_seqs <= 8192, n_slots <= 2^30, max_pages *
 * page_size < 2^31.  With kv_len apart from past and state_out from state,
 * repeating a call repeats its results. */
typedef struct {
    int n_seqs, page_size, n_pages, max_pages, n_slots;
    int64_t table_stride;
    const int32_t *past, *add;
    int32_t *table, *ring;
    const int32_t *state;
    int64_t *slots;
    int32_t *pos, *cu, *kv_len, *granted, *state_out;
} gguf_kv_plan_args;
int gguf_kv_plan(const gguf_kv_plan_args *a, void *stream);

/* ---- append ------------------------------------------------------------------
 *
 * For every token t: q + bq, k + bk and v + bv (fp32 biases, any of them
 * NULL); RMSNorm of q and k with fp32 weights per head (norm_len =
 * head_size) or over the full width (norm_len = heads * head_size), or
 * without (NULL); the rotation of dimensions (j, j + rope_dim / 2) by
 * pos * rope_base^(-2j / rope_dim), the angle formed in 64 bits; q to q_out,
 * k and v to the pool at slots[t], each rounded once.  A token whose slot is
 * negative is skipped altogether (its q_out row too); a slot at or beyond
 * n_pages * page_size is skipped and reported.  Two tokens of a call may not
 * share a slot: which of them stays is not defined, value by value.
 *
 * means: NULL, or [n_pages][n_kv_heads][head_size] in the cache's type,
 * 16-byte aligned: for every page whose last position this call writes, the
 * mean over its page_size keys as the pool holds them then (summed in fp32,
 * rounded once).
 *
 * q, k, v, q_out, biases and norm weights are 16-byte aligned, token strides
 * (in elements) multiples of 16 bytes; heads are contiguous in a token's row.
 * A token's results do not depend on the tokens beside it.  q_out may
 * be q (with its stride); nothing else may overlap. */
typedef struct {
    int n_tokens;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    void *q_out;
    int64_t q_out_stride;
    const int32_t *pos;
    const int64_t *slots;
    const float *bq, *bk, *bv;
    const float *q_norm, *k_norm;
    int q_norm_len, k_norm_len;
    void *means;
} gguf_kv_append_args;
int gguf_kv_append(gguf_kv *kv, const gguf_kv_append_args *a, void *stream);

/* ---- attention -------------------------------------------------------------
 *
 * out[i] = softmax(scale * q[i] . K) V over positions 0 .. kv_len[i] - 1 of
 * request i, head h reading kv head h / (n_heads / n_kv_heads).  kv_len 0
 * (or below) gives zeros, as does a row whose scores are all -inf.  A length
 * beyond max_pages * page_size is cut to it and reported; a table entry outside the
 * pool reads as a page of zero keys and values and is reported.  Entries
 * behind a request's last page are not read, nor do positions behind its
 * length reach the result, whatever they hold.
 *
 * max_pages * page_size is at most 2^31 - 1024.  An infinite or NaN value of a
 * position within the length makes what it makes in fp32 (a value of inf
 * may come out as NaN), in its own heads' and request's rows only.
 *
 * scale * log2(e) is finite in fp32; scale 0 stands for 1 / sqrt(head_size).  q and out have the
 * activations' type, [n_seqs][n_heads][head_size] with a request stride in
 * elements (16-byte aligned, as in gguf_kv_append); out may be q (with its
 * stride).
 *
 * ws: gguf_kv_workspace bytes, 256-byte aligned; its content need not be
 * set and does not outlive the call.  Calls that may run at the same time
 * (also as replays of captured graphs) need a workspace each. */
typedef struct {
    int n_seqs, max_pages;
    const void *q;
    int64_t q_stride;
    void *out;
    int64_t out_stride;
    const int32_t *table;
    int64_t table_stride;
    const int32_t *kv_len;
    float scale;
    void *ws;
    size_t ws_bytes;
} gguf_kv_attn_args;
int gguf_kv_attn(gguf_kv *kv, const gguf_kv_attn_args *a, void *stream);

/* Attention over selected pages.  Of a request's n = ceil(kv_len / page_size)
 * pages each kv head attends to the first n_sink, the last n_window (the
 * unfinished one among them) and, of the rest, the n_top with the highest
 * score max over the kv head's q heads of q . means[page]; to all when n is
 * at most n_sink + n_window + n_top.  Scores are formed in 64 bits: products
 * are exact, and a sum is off by at most head_size * 2^-53 of the sum of its
 * products' magnitudes, so that pages with scores that near may come in either
 * order.  Scores that come out equal (those of equal means always) go to the
 * lower page, a NaN loses to every number.
 *
 * means: as gguf_kv_append keeps them.  sel: NULL, or
 * [n_seqs][n_kv_heads][n_sink + n_window + n_top], the chosen pages'
 * indices in the request in rising order, -1 behind the last.  n_window >= 1;
 * n_sink + n_window + n_top < 2^21; n_seqs <= 65535. */
typedef struct {
    const void *means;
    int n_sink, n_window, n_top;
    int32_t *sel;
} gguf_kv_select_args;
int gguf_kv_attn_topk(gguf_kv *kv, const gguf_kv_attn_args *a, const gguf_kv_select_args *s, void *stream);

/* workspace bytes of gguf_kv_attn (n_select 0) and of gguf_kv_attn_topk
 * (n_select = n_sink + n_window + n_top); 0 on a bad argument */
size_t gguf_kv_workspace(const gguf_kv *kv, int n_seqs, int max_pages, int n_select);

#ifdef __cplusplus
}
#endif
#endif
