/*
 * spiky_lm_tokens.h -- C ABI of the operators at the two ends of a language model:
 * the lookup of token embeddings with its gradient, the selection of a beam search
 * over beams and vocabulary, and the reordering of states that follows it.  They
 * have no counterpart in the reference, which leaves the lookup to a torch module
 * and has no search.
 *
 * The conventions are those of spiky_lm.h: device pointers, `stream` a `hipStream_t`,
 * element types SPIKY_F32, SPIKY_BF16 and SPIKY_F16, messages in spiky_lm_last_error().
 * Calls launch on the stream, allocate nothing, keep nothing and never synchronise.
 * Outputs do not overlap inputs unless their comment allows it.
 */
#ifndef SPIKY_LM_TOKENS_H
#define SPIKY_LM_TOKENS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- embedding ---------------------------------------------------------------
 * out[i] = scale * weight[tokens[i]], each product rounded to 32 bits and then to
 * out's type; zeros where a token is outside [0, vocab). */
typedef struct {
    uint64_t n, vocab, cols;   /* tokens, rows and columns of the table: n < 2^31, vocab < 2^31, cols <= 2^23 */
    int tokens_i64;            /* tokens are int64; else int32 */
    int weight_dtype;          /* of the table and its gradient */
    int out_dtype;             /* of out and its gradient: weight_dtype, or one of the two is F32 */
    const void *tokens;        /* [n] */
    const void *weight;        /* [vocab][cols], rows weight_stride elements apart (not read by the gradient) */
    int64_t weight_stride;
    double scale;              /* as a float, finite */
} spiky_lm_embed_args;

/* out [n][cols] */
int spiky_lm_embed(const spiky_lm_embed_args *args, void *out, void *stream);

/* d_weight[v] = scale * the sum of d_out[i] over tokens[i] == v, in 32 bits and in an
 * order that the tokens alone decide, rounded once; zeros for other rows.  Writes all
 * of d_weight [vocab][cols].  d_out: [n][cols], rows d_out_stride elements apart.
 * Host: the workspace's bytes, 16 bytes aligned. */
uint64_t spiky_lm_embed_workspace(const spiky_lm_embed_args *args);
int spiky_lm_embed_backward(const spiky_lm_embed_args *args, const void *d_out, int64_t d_out_stride, void *d_weight,
                            void *workspace, uint64_t workspace_bytes, void *stream);

/* ---- selection of a beam search ------------------------------------------------
 * Beam k of search b has a score, the sum of its tokens' log-probabilities.  Each of
 * its tokens v is a candidate of score
 *   s = scores[b][k] + logits[b][k][v] - log(sum over u of exp(logits[b][k][u]))
 * in 64 bits, over exponentials and sums of a slice's in 32, but where s is -infinity.  A
 * finished beam has one candidate, token `pad` with the beam's own score.  The n candidates of
 * largest s / length^length_penalty go on, in this order; length is lengths[b][k], plus 1 where
 * the beam is not finished, and at least 1.  Of equal ones, the lower beam comes first, then the larger logit, then
 * the lower token.  Where there are fewer than n, the others are (-infinity, beam 0, pad).
 * A beam that is not finished and whose score or one of whose logits is NaN or
 * +infinity has candidates of score NaN, in the order of their tokens; NaN ranks as +infinity. */
typedef struct {
    uint64_t searches, beams, vocab;   /* beams: 1 to 64; vocab < 2^31; searches * beams < 2^24 */
    uint64_t n;                        /* 1 to 64 */
    int dtype;                         /* of the logits */
    int lengths_i64;                   /* lengths are int64; else int32 */
    const void *logits;                /* [searches][beams][vocab] */
    int64_t search_stride, beam_stride; /* elements from search to search, from beam to beam */
    const float *scores;               /* [searches][beams] */
    const uint8_t *finished;           /* [searches][beams], non-zero: finished; or null: none is */
    const void *lengths;               /* [searches][beams], or null: 1 for all */
    double length_penalty;             /* -8 to 8 */
    int64_t pad;
    float *out_scores;                 /* [searches][n]; s, without the length */
    int64_t *out_parents, *out_tokens; /* [searches][n] */
} spiky_lm_beams_args;

/* Host: bytes of the workspace, 8 bytes aligned. */
uint64_t spiky_lm_beam_select_workspace(const spiky_lm_beams_args *args);
int spiky_lm_beam_select(const spiky_lm_beams_args *args, void *workspace, uint64_t workspace_bytes, void *stream);

/* ---- reordering of states --------------------------------------------------------
 * out[b][j] = in[b][parents[b][j]] for `count` states; zeros where a parent is outside
 * [0, beams).  A beam's part of a state is `runs` runs of run_bytes bytes each.  Strides
 * are in bytes.  out may be in with the same strides where n == beams <= 64; a state is
 * else apart from every other, and from parents. */
typedef struct {
    const void *in;
    void *out;
    uint64_t runs, run_bytes;          /* run_bytes < 2^35 */
    int64_t in_search, in_beam, in_run, out_search, out_beam, out_run;
} spiky_lm_state;

/* states is host memory, read before the call returns.  parents: [searches][n], int64 or int32. */
int spiky_lm_reorder(const spiky_lm_state *states, uint64_t count, const void *parents, int parents_i64,
                     uint64_t searches, uint64_t beams, uint64_t n, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SPIKY_LM_TOKENS_H */
