/*
 * tc_step.h -- C-ABI of the MI355X (gfx950) operators that lie around the products
 * of tc_qmatmul.h and the attention of tc_attention.h in a serving program's step
 * (same library, libtc_hip.so):
 *
 *   tc_kv_plan         the step's geometry from its sequences' lengths: rows, positions,
 *                      cache slots, pages given out and taken back
 *   tc_norm_add        residual stream plus a block's gated, normalised output, and the
 *                      norm in front of the next block
 *   tc_rope_kv_write   rotary positions of queries and keys (after norms of their heads,
 *                      where a model has these), keys and values into the paged cache
 *   tc_logits_adjust   penalties for repeated tokens, biases and masks on logits, before
 *                      tc_spec_verify or a sampler of the caller's
 *
 * Conventions as in tc_qmatmul.h and tc_attention.h: device pointers unless a comment
 * says otherwise, `stream` a hipStream_t, TC_OK or a negative TC_E_* code with
 * tc_last_error(), nothing written when a call is refused. None of these calls uses the
 * library's scratch: they may run at once on several streams, as long as they do not
 * write what another one reads or writes, and can be captured into a graph without any
 * preparation. Every number that decides about lengths and places is read on the device
 * when a call runs, so that a graph's replays may find other ones there. The same call
 * gives the same bits.
 */
#ifndef TC_STEP_H
#define TC_STEP_H

#include <stddef.h>
#include <stdint.h>

#include "tc_attention.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- geometry of a step ---------------------------------------------------------- */

/* Sequence s holds held[s] tokens in the pages table[s*table_pages] .. of pages[s] entries
 * (more than its tokens need, where drafted tokens were not taken), and brings
 * new_tokens[s] more; below 0: it has ended. Pages not in use stand in a ring of
 * ring_pages entries: free[1] of them from ring[free[0]] on, going round. Lengths are
 * taken for at least 0, free[0] for a place of the ring, and free[1] and pages[s] for at most
 * what the ring and the table have room for. */
typedef struct tc_plan {
    uint32_t n_seq, n_tokens;         /* n_tokens: rows of the step, those behind the last sequence's too */
    uint32_t page_tokens, table_pages, ring_pages;
    const int32_t *new_tokens;        /* [n_seq] */
    const int32_t *held, *pages;      /* [n_seq] */
    const int32_t *free;              /* [2] */
    int32_t *table;                   /* [n_seq][table_pages]: new pages are entered */
    int32_t *ring;                    /* [ring_pages]: pages of ended sequences are entered */
    int32_t *start;                   /* [n_seq + 1]: first row of each sequence, tc_kv_batch's */
    int32_t *len, *pages_out;         /* [n_seq]: tokens and pages behind the step; may be held and pages */
    int32_t *free_out;                /* [3]: free of the next step, and the pages that were missing; may be free,
                                       * if that has 3 entries */
    int32_t *sequence, *position;     /* [n_tokens] of each row, -1 for rows behind the last; may be NULL */
    int64_t *slot;                    /* [n_tokens]: page * page_tokens + place in it, -1: none; may be NULL */
} tc_plan;

/* Rows go to the sequences in their order: start[s] = min(n_tokens, sum of new_tokens[r]
 * over r < s), and len[s] = held[s] + the rows of s. A sequence that has ended gets no
 * rows, length 0 and no pages; the first pages[s] entries of its table's row go behind the free ones,
 * sequences in their order, before any is given out (those that the ring has no room for are lost: a ring has room
 * where ring_pages is the cache's number of pages and no page is in two tables). Then the
 * sequences in their order get, from the front of the free ones, what ceil(len[s] /
 * page_tokens) is more than pages[s]. Where none is left, the table's entry is -1, its
 * positions hold no token for the other calls, and free_out[2] counts the page, as it
 * counts those past table_pages, which no entry is there for: where it is not 0 the step
 * is not to be used. Other entries of the tables and the ring stay as they are. n_seq up to
 * 2^16, n_tokens to 2^24, ring_pages and the tables' entries to 2^30. free_out[2] says 2^30 at most.
 * Lengths past 2^31 - 65 are taken for that. */
int tc_kv_plan(const tc_plan *plan, void *stream);

/* ---- norms ----------------------------------------------------------------------- */

enum { TC_NORM_RMS = 0, TC_NORM_LAYER = 1 };

/* norm(x) = x / sqrt(mean(x^2) + eps) * (weight + offset) + bias; TC_NORM_LAYER takes the
 * row's mean off x before that. */
typedef struct tc_norm {
    int32_t kind;
    float eps;            /* finite, at least 0 */
    const float *weight;  /* fp32 [cols], NULL: 1 */
    const float *bias;    /* fp32 [cols], NULL: 0 */
    float offset;         /* of the weights: 1 where they are stored as distances from 1 (without weights: nothing) */
} tc_norm;

enum { TC_GATE_NONE = 0, TC_GATE_CHANNEL = 1, TC_GATE_ROW = 2, TC_GATE_FULL = 3 };

/* Rows of `cols` values; the strides count elements, types are TC_F32, TC_F16 or TC_BF16. */
typedef struct tc_norm_rows {
    uint32_t n_rows, cols;
    const void *h;                    /* the residual stream */
    const void *y;                    /* the block's output; NULL: there is none, and h_out is not written */
    void *h_out;                      /* h + scale * gate * post(y), of h's type; may be h, or NULL */
    void *x;                          /* pre(h_out): the next block's input; may be NULL */
    int32_t h_type, y_type, x_type;
    uint32_t h_stride, y_stride, h_out_stride, x_stride;
    const tc_norm *post, *pre;        /* host structs; NULL: no norm (a NULL `pre` writes no x and no act) */
    const void *gate;                 /* [cols], [n_rows] or [n_rows][cols] contiguous, after gate_kind */
    int32_t gate_kind, gate_type;
    int32_t gate_sigmoid;             /* not 0: sigmoid(gate) instead of gate */
    float scale;
    int32_t act_type;                 /* with `act`: */
    void *act;                        /* pre(h_out) quantized as tc_act_quantize does for weights of act_type (tc_act_bytes
                                       * bytes, 256-byte aligned), for tc_gemv_q8; NULL: none. cols % 256 = 0, up to 12288 */
} tc_norm_rows;

/* One launch for every 2^21 rows. Everything between the inputs and the outputs' rounding is held in fp32: x is
 * the norm of h + scale * gate * post(y) before that is rounded to h's type; act is formed
 * from the fp32 values that an F32 x has, and is tc_act_quantize's of them bit for bit.
 * cols up to 32768. Rows may have any stride that keeps them apart and any
 * alignment that fits their elements. Outputs do not overlap inputs, apart from h_out = h with the same stride. An
 * infinity or NaN stays in its row; squares that pass fp32's range (values past 1.8 10^19) give
 * an infinite mean, and rows whose root mean square is below 10^-16 lose bits of it where eps is below 10^-30. */
int tc_norm_add(const tc_norm_rows *rows, void *stream);

/* ---- rotary positions ------------------------------------------------------------ */

/* Pairs of a head's first n_rot dims: dims i and i + n_rot/2, or dims 2i and 2i + 1. */
enum { TC_ROPE_HALF = 0, TC_ROPE_PAIRS = 1 };

/* Pair i of a row at position p is turned by a = 2 pi * p * turns[i]: (u, v) ->
 * factor * (u cos a - v sin a, u sin a + v cos a). The dims behind n_rot stay as they
 * are. Angles are formed in fp64 and reduced there: cos and sin are off by 2^-23 at most, before
 * the factor, at positions up to 2^26 (by 2^-20 at 2^31). */
typedef struct tc_rope {
    uint32_t n_rot;       /* even, up to the head's size */
    int32_t layout;
    const double *turns;  /* [n_rot / 2] turns a position */
    float factor;
} tc_rope;

/* How frequencies f_i = theta^(-2i / n_rot) are changed for contexts longer than those of
 * the training (`original` tokens), s = factor:
 *   LINEAR  f_i / s
 *   NTK     theta * s^(n_rot / (n_rot - 2)) for theta (n_rot > 2)
 *   YARN    between f_i and f_i / s by a ramp over the pairs, from the one that turns `high`
 *           times in `original` positions to the one that turns `low` times (0 for either:
 *           32 and 1); the factor is 0.1 ln(s) + 1 (1 where s <= 1)
 *   BANDS   f_i where the pair turns `high` times or more in `original` positions, f_i / s
 *           where `low` times or less, and between these by the number of turns
 * and then divided by divisors[i], where there are any (a device array). */
enum { TC_ROPE_NONE = 0, TC_ROPE_LINEAR = 1, TC_ROPE_NTK = 2, TC_ROPE_YARN = 3, TC_ROPE_BANDS = 4 };
typedef struct tc_rope_scaling {
    int32_t kind;
    double factor, original, low, high;
    const float *divisors;
} tc_rope_scaling;

/* Fills turns (device, [n_rot / 2]) and *factor (host) for a tc_rope; scaling (a host
 * struct) may be NULL. */
int tc_rope_turns(const tc_rope_scaling *scaling, uint32_t n_rot, double theta, double *turns, float *factor, void *stream);

/* Rotates rows of `xtype`, [heads][head_dim] each, row t at x + t * x_stride elements, at
 * position[t], into out ([n_tokens] rows at out_stride); out may be x with the same
 * stride. Rows with a position below 0 are not touched. head_dim: a multiple of 16, up to
 * 256; bases and strides of 16 bytes' multiples. Up to 4096 heads and 2^24 rows; n_tokens * heads
 * below 2^31 - 256, and n_tokens * ceil(heads / 4) * (head_dim / 8, up to a power of two) at
 * most 2^32 - 256. */
int tc_rope_apply(const tc_rope *rope, int xtype, const void *x, uint32_t x_stride, void *out, uint32_t out_stride,
                  const int32_t *position, uint32_t n_tokens, uint32_t heads, uint32_t head_dim, void *stream);

/* What lies between the q/k/v product and tc_attn, in one launch. For each row of the
 * batch, at its position (tc_kv_batch): the queries' heads are normalised (RMS over
 * head_dim, times q_norm[head_dim], fp32; NULL: not), rotated, and written to q_out
 * ([n_tokens][heads][head_dim] contiguous, of `xtype`; or q itself: in place, at q's stride); the
 * keys' heads likewise with k_norm, and written to their slots of the cache, as tc_kv_write
 * writes k; the values are written as tc_kv_write writes v. Between loading and the one
 * rounding at the end values are fp32 (a norm's squares too: heads with values past 10^18 get an infinite
 * mean, and those whose root mean square is below 10^-18 lose bits of it where eps is below 10^-34). Rows are laid out as tc_kv_write's k and v, and q
 * as tc_attn's; parts of one fused product's rows are fine. q may be NULL (heads 0): keys and
 * values only. Rows past the last sequence are not touched; q_out is written also for rows
 * whose position has no slot. heads up to 4096; sizes as tc_rope_apply's, with keys' and values' heads
 * counted too. eps: finite, at least 0. */
int tc_rope_kv_write(const tc_kv_cache *cache, const tc_kv_batch *batch, const tc_rope *rope, int xtype, const void *q,
                     uint32_t q_stride, void *q_out, uint32_t heads, const void *k, uint32_t k_stride, const void *v,
                     uint32_t v_stride, const float *q_norm, const float *k_norm, float eps, void *stream);

/* ---- rules on logits --------------------------------------------------------------- */

/* Every array may be NULL, with what its comment says then. */
typedef struct tc_logit_rules {
    const float *repetition, *frequency, *presence;   /* [n_seq]; NULL: 1, 0, 0 */
    const int32_t *history;           /* [n_history] tokens, sequence s's from history_start[s] to history_start[s + 1] - 1; */
    const int32_t *history_start;     /* [n_seq + 1]; NULL: nothing has gone before the step's tokens */
    const int32_t *prompt;            /* [n_seq] how many of them were asked, not answered; -n: the first n of them and of
                                       * the step's tokens behind them (a sequence's prompt may be among its rows then);
                                       * NULL: none */
    uint32_t n_history;
    const int32_t *bias_start;        /* [n_seq + 1]; NULL: no biases */
    const int32_t *bias_token;        /* [n_bias], sequence s's from bias_start[s] to bias_start[s + 1] - 1 */
    const float *bias_value;          /* [n_bias] */
    uint32_t n_bias;
    const uint32_t *mask;             /* [n_masks][mask_words]: bit t % 32 of word t / 32 is 1 where token t may come */
    uint32_t n_masks, mask_words;     /* mask_words >= ceil(vocab / 32) */
    const int32_t *mask_of;           /* [n_tokens] each row's mask, none where it is outside [0, n_masks); NULL: row t's is t */
} tc_logit_rules;

/* out[row] of sequence s (rows start[s] .. start[s+1]-1, as in tc_spec_verify) and token t, from
 * l = logits[row][t]:
 *   l > 0 ? l / repetition : l * repetition,  where t is in the history or among the tokens below
 *   - frequency * c - presence * (c > 0),     c: how often t was answered
 *   + the biases for t, added up in their order
 *   -infinity,                                where the row's mask has a 0 for t, whatever l is
 * For row start[s]+i the tokens start[s] .. start[s]+i of `tokens` ([n_tokens], the step's tokens; NULL:
 * none are counted) have come after the history: answered, but for those that prompt[s] below 0 goes on
 * over. So a prompt of n tokens, given as -n from its first chunk to its sequence's last token, is never
 * taken for answers, while any number above 0 (or NULL) wants rows without prompts in them. Where a token's logit changes it is formed in
 * fp64 and rounded once (the sum of its biases is fp32). Tokens outside [0, vocab) are passed over.
 * logits: [n_tokens] rows of xtype at x_stride elements, aligned to their type; out: fp32 rows at
 * out_stride; out may be logits, if these are F32 with the same stride, and does not overlap them
 * otherwise. Rows past the last sequence are not touched. n_seq and n_tokens up to 65535,
 * vocab to 2^30, n_history to 2^31 - 2^16, n_bias to 2^31 - 1. */
int tc_logits_adjust(const tc_logit_rules *rules, int xtype, const void *logits, uint32_t x_stride, uint32_t vocab,
                     uint32_t n_seq, uint32_t n_tokens, const int32_t *start, const int32_t *tokens, float *out,
                     uint32_t out_stride, void *stream);

#ifdef __cplusplus
}
#endif
#endif
