/*
 * tc_attention.h -- C-ABI of the MI355X (gfx950) operators between and behind
 * the quantized products of tc_qmatmul.h (same library, libtc_hip.so): a paged
 * cache of keys and values that is quantized as it is written, attention of a
 * chunk of new tokens over it, and the verification of drafted tokens.
 *
 * A step of a serving program that decodes several tokens per sequence at once:
 * q/k/v products of the chunk (tc_gemv for up to 8 tokens, tc_gemm), tc_kv_write,
 * tc_attn, the other products, and, where all but the first of a chunk's tokens
 * were drafted, tc_spec_verify on the last product's logits. Rejected tokens need
 * no undoing: the next call's len[] is shorter, and their slots are written again.
 *
 * Conventions as in tc_qmatmul.h: device pointers, `stream` a hipStream_t, TC_OK
 * or a negative TC_E_* code with tc_last_error(), nothing written when a call is
 * refused, calls that share a device's scratch serialized (tc_attn and
 * tc_spec_verify use it; tc_kv_write and tc_kv_read do not). Every call works on
 * the current device, can be captured into a graph (tc_attn and tc_spec_verify
 * once their scratch is in place: after tc_attn_reserve, or a call that needed as
 * much), and reads start, len and table on the device when it runs, so that a
 * graph's replays may find other lengths there.
 */
#ifndef TC_ATTENTION_H
#define TC_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (GGML's ids where it has one). Rows of q, k, v and outputs:
 * F32, F16, BF16. Cache: F16, BF16, I8, E4M3 (8-bit float, 4 exponent and 3
 * mantissa bits, no infinities, largest 448). */
enum { TC_F32 = 0, TC_F16 = 1, TC_I8 = 24, TC_BF16 = 30, TC_E4M3 = 100 };

/* A paged cache of one layer, in buffers of the caller:
 *   k, v              [n_pages][kv_heads][page_tokens][head_dim] of `type`,
 *                     16-byte aligned
 *   k_scale, v_scale  fp32 [n_pages][kv_heads][page_tokens] for I8 and E4M3 (one
 *                     factor per token and head), NULL for F16 and BF16
 * page_tokens: a multiple of 16. head_dim: a multiple of 16, up to 256. Factors as
 * tc_kv_write forms them are above 0; tc_attn takes a v_scale below 2^-80 (0 and
 * negative ones too) for 2^-80. Less than 2^32 runs of 16 tokens (n_pages * kv_heads *
 * page_tokens / 16). */
typedef struct tc_kv_cache {
    int32_t type;
    uint32_t n_pages, kv_heads, page_tokens, head_dim;
    void *k, *v;
    float *k_scale, *v_scale;
} tc_kv_cache;

/* A batch of chunks (device arrays). Sequence s < n_seq has the token rows
 * start[s] .. start[s+1]-1 of the call's n_tokens packed rows (start[0] = 0,
 * ascending; none is fine). len[s] counts its tokens in the cache with these
 * rows in it, so row start[s]+i has position len[s] - (start[s+1]-start[s]) + i.
 * Position p lies in slot p % page_tokens of page table[s*table_pages + p /
 * page_tokens]. Positions below 0, at table_pages * page_tokens or above, or in
 * a page outside [0, n_pages) hold no token: not written, read as zeros, not
 * attended to. Rows past start[n_seq] are not touched. Pages may be shared
 * between sequences; one slot is to be written by one row of a call. At most 2^20
 * sequences, 2^24 rows, 2^31 - 65 tokens of a sequence. */
typedef struct tc_kv_batch {
    uint32_t n_seq, n_tokens, table_pages;
    const int32_t *start, *len, *table;
} tc_kv_batch;

/* Keys and values of the batch's rows into their slots. k and v: [n_tokens] rows
 * of `xtype`, [kv_heads][head_dim] each, row t at k + t * k_stride elements (so
 * that they may be parts of one fused product's rows); bases and strides of 16
 * bytes' multiples. F16 and BF16 round to nearest even. I8: scale = max|x| / 127
 * (1 for a row of zeros), value = rint(x / scale); E4M3: scale = max|x| / 448,
 * value = x / scale to the nearest, ties to even; both quotients rounded to fp32
 * once, the second held to the type's largest (which it passes where the scale is a
 * subnormal number). A row with an infinity or NaN reads back as NaNs. */
int tc_kv_write(const tc_kv_cache *cache, const tc_kv_batch *batch, int xtype, const void *k, const void *v,
                uint32_t k_stride, uint32_t v_stride, void *stream);

/* The batch's rows back out of the cache, as `xtype` (8-bit types: value * scale
 * rounded to fp32, then to xtype): k and v [n_tokens][kv_heads][head_dim],
 * contiguous. A batch whose chunks are whole sequences (start[s+1]-start[s] =
 * len[s]) reads these whole. */
int tc_kv_read(const tc_kv_cache *cache, const tc_kv_batch *batch, int xtype, void *k, void *v, void *stream);

/* Causal attention of the batch's rows over the cache (which already holds their
 * keys and values): out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j over the
 * sequence's positions j <= p (p the row's own), and j > p - window where window is
 * not 0, with the keys and values of head h / (heads / kv_heads). A row that sees
 * no token gives zeros. q: [n_tokens] rows of `xtype`, [heads][head_dim] each, row
 * t at q + t * q_stride elements (base and stride of 16 bytes' multiples); out:
 * [n_tokens][heads][head_dim] of `xtype`, 16-byte aligned. Sums and the softmax are
 * held in fp32; q and the softmax's weights enter the matrix cores as F16 or BF16
 * (the 16-bit cache's own type; F16 for the 8-bit ones) in as many pieces as
 * `xtype` has bits for, so that fp32 rows keep fp32 results (as F16 a weight is held
 * to half a step or 2^-36 of its row's largest, whichever is more; over 8-bit caches
 * a weight here is the softmax's times the value's factor, rows of zeros left out).
 * Infinities and NaN in the cache reach only the rows that see them. The same call
 * gives the same bits. heads: a multiple of kv_heads, up to 4096; n_tokens * heads
 * < 2^31. scale: finite, not negative. start, len and table are not to change while
 * a call runs. */
int tc_attn(const tc_kv_cache *cache, const tc_kv_batch *batch, int xtype, const void *q, uint32_t q_stride, void *out,
            uint32_t heads, float scale, uint32_t window, void *stream);

/* Pre-size the scratch so that later tc_attn calls of at most `heads` query heads
 * and n_tokens rows of any head_dim, and tc_spec_verify calls of at most n_tokens
 * rows and as many sequences, allocate nothing (e.g. before a graph capture). */
int tc_attn_reserve(uint32_t heads, uint32_t n_tokens);

/* Verification of drafted tokens. Sequence s has the chunk tokens[start[s]] ..
 * tokens[start[s+1]-1], all but the first drafted; logits row start[s]+i (fp32,
 * [n_tokens][vocab]) is the target's for the token after the i-th. With
 * p_i = softmax(logits_i / temperature[s]) and q_i the distribution that draft i+1
 * was drawn from, the drafts x are taken in order while accept_u[start[s]+i] *
 * q_i(x) < p_i(x). At the first that is not, at row i, the next token is drawn from
 * max(p_i - q_i, 0) (from p_i where that is zero everywhere); where all are taken,
 * from the last row's p: the lowest token t whose sum of weights up to t exceeds
 * sample_u[s] times the sum of all (if none: the last of weight above 0; a sample_u
 * below 0 is taken for 0). draft_probs (fp32 [n_tokens][vocab], row start[s]+i for draft i+1; each
 * sequence's last row is not read) may be NULL: drafted without chance, q is 1 at
 * the draft. temperature[s] = 0 (or below, or NaN) takes the largest logit, lowest
 * token first, for p = 1 and needs no random numbers; an infinite one makes all
 * tokens above -infinity alike. Drafts outside [0, vocab) are rejected.
 * Probabilities and sums are formed in fp64. n_accepted[s] (drafts taken) and
 * next_token[s] are int32; a sequence without rows gives 0 and -1, one whose row
 * has a NaN or no finite largest logit the rejection of that draft and -1 as the token.
 * (Shares below 2^-900 of the largest count as 0.) 1 to 65535 rows, up to 65535
 * sequences, vocab up to 2^30. */
int tc_spec_verify(const float *logits, const float *draft_probs, uint32_t vocab, uint32_t n_seq, uint32_t n_tokens,
                   const int32_t *start, const int32_t *tokens, const float *temperature, const float *accept_u,
                   const float *sample_u, int32_t *n_accepted, int32_t *next_token, void *stream);

#ifdef __cplusplus
}
#endif
#endif
