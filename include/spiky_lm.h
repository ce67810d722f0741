/*
 * spiky_lm.h -- C ABI of the language-model operators around the LUT blocks:
 * counter-based dropout, the residual join of a block with its norms, and the
 * processing of logits before a token is chosen.  They have no counterpart in
 * the reference, which leaves these steps to torch modules.
 *
 * Every pointer is a device pointer unless its comment says host; `stream` is a
 * `hipStream_t`.  Outputs do not overlap inputs unless their comment allows it.
 * Calls launch on the stream, allocate nothing, keep nothing
 * and never synchronise, so they can be captured into a HIP graph.  The return
 * codes are those of spiky_lut.h; the message of the last failed call on the
 * calling thread is spiky_lm_last_error().
 */
#ifndef SPIKY_LM_H
#define SPIKY_LM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define SPIKY_F32 0
#define SPIKY_BF16 1
#define SPIKY_F16 2

/* Norms: rms x / sqrt(mean x^2 + eps), layer (x - mean) / sqrt(var + eps). */
#define SPIKY_NORM_NONE 0
#define SPIKY_NORM_RMS 1
#define SPIKY_NORM_LAYER 2

/* Message of the last failed call on this thread ("" if none). */
const char *spiky_lm_last_error(void);

/* ---- dropout ---------------------------------------------------------------
 * y[r][c] = x[r][c] / (1 - p) where the element is kept, else 0 (whatever x
 * holds there).  The element at row r, column c is kept when word c % 4 of
 * Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw 2011: the fewest that
 * pass BigCrush) under key `seed` and counter (c / 4, r, offset) is at least
 * floor(p * 2^32 + 1/2).  The same call on the output's gradient is the
 * backward pass.  rng, if given, points to {seed, offset} in device memory and
 * stands for the two arguments.  x_stride: elements from one row of x to the
 * next; y has contiguous rows.  rows < 2^32, cols <= 2^34 - 16. */
int spiky_lm_dropout(const void *x, int64_t x_stride, void *y, uint64_t rows, uint64_t cols,
                     int dtype, double p, uint64_t seed, uint64_t offset, const int64_t *rng,
                     void *stream);

/* ---- residual join ---------------------------------------------------------
 * For each of rows < 2^32 rows of cols <= 2^26 columns: v = post(branch) * post_weight + post_bias, d = dropout(v) as
 * above, z = residual_scale * residual + branch_scale * gate * d, and
 * normed = pre(z) * pre_weight + pre_bias, of the sum z before it is rounded to
 * the residual's type.  Each part is left out where its pointer is null or its
 * norm SPIKY_NORM_NONE. */
typedef struct {
    uint64_t rows, cols;
    int res_dtype;             /* of residual, out and their gradients */
    int act_dtype;             /* of branch, normed and their gradients: res_dtype, or any where that is F32 */
    int post_norm, pre_norm;   /* SPIKY_NORM_* */
    int par_f32, gate_f32;     /* the norms' parameters (the gate) are fp32; else act_dtype */
    const void *residual;      /* [rows][cols], rows residual_stride apart */
    const void *branch;        /* or null: then out is not written and z = residual */
    int64_t residual_stride, branch_stride;
    const void *post_weight, *post_bias, *pre_weight, *pre_bias; /* [cols] or null */
    const void *gate;          /* [rows / gate_rows][cols], or null */
    uint64_t gate_rows;        /* consecutive rows that share one row of the gate; divides rows */
    double post_eps, pre_eps, residual_scale, branch_scale, dropout_p;
    uint64_t seed, offset;
    const int64_t *rng;        /* {seed, offset} in device memory, or null */
    float *stats;              /* [rows][4]: means and reciprocal deviations for the backward pass, or null */
} spiky_lm_residual_args;

/* out [rows][cols] of res_dtype, normed [rows][cols] of act_dtype. */
int spiky_lm_residual_norm(const spiky_lm_residual_args *args, void *out, void *normed, void *stream);

/* Gradients of the join; `args` as in the forward call, stats as it wrote them.
 * d_out and d_normed may be null (no gradient).  Each output may be null. */
typedef struct {
    const void *d_out;         /* [rows][cols] of res_dtype */
    const void *d_normed;      /* [rows][cols] of act_dtype */
    int64_t d_out_stride, d_normed_stride;
    void *d_residual;          /* res_dtype */
    void *d_branch;            /* act_dtype */
    void *d_post_weight, *d_post_bias, *d_pre_weight, *d_pre_bias;
    void *d_gate;              /* [rows / gate_rows][cols] */
    void *workspace;           /* spiky_lm_residual_norm_workspace() bytes */
    uint64_t workspace_bytes;
} spiky_lm_residual_grads;

/* Host: workspace bytes of the backward call (its pointers are only tested for null). */
uint64_t spiky_lm_residual_norm_workspace(const spiky_lm_residual_args *args,
                                          const spiky_lm_residual_grads *grads);
int spiky_lm_residual_norm_backward(const spiky_lm_residual_args *args,
                                    const spiky_lm_residual_grads *grads, void *stream);

/* ---- logits ----------------------------------------------------------------
 * For each row b and entry v:
 *   x  = logits + bias + the sum of bias_values[k] over bias_ids[k] == v
 *   x  = x > 0 ? x / repetition : x * repetition   if v is among the first lengths[b] tokens
 *   x -= frequency * n + presence * (n > 0)        n: times v is among tokens prompt_lengths[b]..lengths[b]
 *   x /= temperature                               unless temperature <= 0
 *   x  = -infinity                                 where the mask leaves v out
 * Quotients are products with the divisor's reciprocal: one rounding of 32 bits more than a division.  That
 * of a divisor past 2^126 is subnormal and has two bits fewer; one that would overflow is not used.
 * Tokens and bias ids outside [0, vocab) count nowhere.  out may be logits. */
typedef struct {
    uint64_t rows, vocab;
    const void *logits;
    void *out;
    int64_t logits_stride, out_stride;  /* elements from row to row */
    int dtype, out_dtype;
    const void *tokens;                 /* [rows][history], or null */
    int64_t tokens_stride;
    uint64_t history;
    int tokens_i64;                     /* tokens are int64; else int32 */
    int lengths_i64;                    /* lengths and prompt_lengths are int64; else int32 */
    const void *lengths;                /* [rows], or null: history.  Clamped to 0..history */
    const void *prompt_lengths;         /* [rows], or null: 0.  Clamped to 0..lengths */
    float repetition, presence, frequency, temperature;
    const float *repetition_rows, *presence_rows, *frequency_rows, *temperature_rows; /* [rows], in place of the number */
    const void *bias;                   /* [vocab], rows bias_stride apart (0: one for all), or null */
    int64_t bias_stride;
    int bias_dtype;
    const void *bias_ids;               /* [n_bias], rows bias_ids_stride apart (0: one for all), or null */
    const float *bias_values;
    int64_t bias_ids_stride, bias_values_stride;
    uint64_t n_bias;
    int bias_ids_i64;
    const void *mask;                   /* bytes, non-zero: allowed, or 32 entries a word, lowest bit first; or null */
    int64_t mask_stride;                /* bytes or words from row to row (0: one for all) */
    int mask_bits;
} spiky_lm_logits_args;

int spiky_lm_process_logits(const spiky_lm_logits_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* SPIKY_LM_H */
