/* vireo-b200: the choice of a beam search's continuations.
 *
 * The reference takes the most probable token (vireo src/gguf_run.c:254-259,
 * gguf_decoder_step here).  A beam search keeps n_beams continuations of a
 * request with the sum of their tokens' log-probabilities, and from all of
 * their next tokens takes the best; the rows of the block tables then follow
 * with gguf_kv_fork (include/gguf_kv.h), to which `parent` goes as it is.
 *
 * For row r = i * n_beams + b (beam b of request i) and token t
 *
 *   total(r, t) = score[r] + logits[r][t] - log sum_u exp(logits[r][u])
 *
 * and request i gets its n_out largest totals in falling order; equal ones in
 * the order of b * vocab + t.  Totals are compared as if they were formed in
 * 64 bits: two of them nearer than 2^-40 of their terms may come in either
 * order, none further apart.  A row with a non-zero done[r] has one
 * continuation, end_token, with total score[r].  What has no finite total is
 * none: tokens of logit -inf, rows of score -inf (a search begins with one
 * beam: 0, -inf, -inf, ...), rows whose logits hold a NaN or +inf or nothing
 * but -inf.
 *
 * Written, [n_seqs][n_out]: score_out, the total with a log sum exp that is off
 * by at most 2^-19 (beside 64 bits' own steps), rounded to fp32 (-inf beyond its
 * range), or a finished beam's score as it is; token; parent, the row r that it
 * continues; done_out (or NULL), 1 where token is end_token, else 0.  Where fewer
 * continuations are left than n_out: -inf, -1, -1 and 1.  The same call gives the
 * same bits; between calls score_out's last digits go by how a row is cut, that is
 * by the call's sizes and the row's alignment, and by whether it was summed again
 * in 64 bits because its totals lie near another row's.
 *
 * logits: [n_seqs * n_beams][vocab] of GGML type 0 (F32), 1 (F16) or 30
 * (BF16), aligned to their type, rows `stride` elements apart.  n_beams and
 * n_out are 1 to 32, n_beams * vocab >= n_out, vocab <= 2^20.  done may be
 * NULL; end_token is needed with it and may be -1 (no such token) without.
 * ws: gguf_beam_workspace bytes, 256-byte aligned; its content need not be
 * set.  The call is stream-ordered like gguf_kv_attn: it allocates nothing,
 * may be captured, and calls that may run at the same time need a workspace
 * each.  Nothing written may overlap anything read. */
#ifndef VIREO_GGUF_BEAM_H
#define VIREO_GGUF_BEAM_H
#include <stddef.h>
#include <stdint.h>

#include "vireo_status.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    int n_seqs, n_beams, n_out, vocab;
    uint32_t type;
    int end_token;
    const void *logits;
    int64_t stride;
    const float *score;
    const int32_t *done;
    float *score_out;
    int32_t *token, *parent, *done_out;
    void *ws;
    size_t ws_bytes;
} gguf_beam_args;
int gguf_beam_select(const gguf_beam_args *a, void *stream);

/* workspace bytes; 0 on a bad argument */
size_t gguf_beam_workspace(int n_seqs, int n_beams, int n_out, int vocab);

#ifdef __cplusplus
}
#endif
#endif
