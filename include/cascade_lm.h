/*
 * cascade_lm.h : C ABI of the language-model operators for MI355X (gfx950), libcascade_lm.so.
 *
 * They train and score a language model on the texts that cascade_hip.h sorts: uint16 tokens, a separator in front of every
 * document. No counterpart in the reference, whose suffix arrays serve the same corpora.
 *
 * Conventions are those of cascade_hip.h: every entry point returns 0 on success and a negative csa_status otherwise, nothing exits
 * the process, csa_lm_last_error() describes the calling thread's last failure, d_* are device addresses, `stream` is a hipStream_t
 * (NULL = the default stream). Every call only enqueues kernels on the stream, allocates nothing and keeps nothing; the stream's device
 * must be the current one. Scratch memory is the caller's: d_work, 256-byte aligned, of at least the bytes that the
 * operator's *_workspace function names for the same sizes; it is free again when the stream has passed the call.
 * Kernels only (no memset or copy nodes): every call may be recorded into a HIP graph. Results do not depend on the order in which workgroups run.
 */
#ifndef CASCADE_LM_H
#define CASCADE_LM_H

#include "cascade_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Sums, softmax statistics and norms are held in 32 bits or more, and results are rounded once at the end. The second products of attention, cross entropy and distillation also
 * take operands that are computed, rounded to the 16 bits of `type`, which is what the matrix units multiply at their rate: attention's probabilities (for out and d_v), its score
 * gradients (in two halves for d_q, once for d_k, in CSA_LM_F16 times a power of two for each row and key), and the gradients of the logits (cross entropy, distillation). D, the sum that score gradients are taken
 * relative to, is made of the rounded out and corrected for d_k. Against results that are rounded nowhere else, errors over short documents grow from 1.7e-3 to 1.9e-3 (out) and 2.4e-3
 * (gradients) in CSA_LM_BF16, from 2.1e-4 to 2.9e-4 in CSA_LM_F16, relative to the norm; those of the cross entropy's gradients stay at the result's rounding, those of distillation
 * grow from 1.7e-3 to 2.3e-3 and from 2.1e-4 to 2.9e-4 (up to 3.9e-3 and 4.9e-4 where a teacher weighs the words of all tokens alike), and stay at the result's rounding for up to 32
 * tokens (of 33 to 64, as far as entries above an eighth of their token's weight go: up to 1.18 times it where these make most of the sums). Few entries make most of a short text's gradients, so that errors spread: of 65 to some
 * hundred tokens up to 1.5 times the result's rounding, up to 1.7 where the tokens' weights differ by up to 2^10. Embeddings and norms round once, at the end. */

typedef enum csa_lm_type {
    CSA_LM_BF16 = 0,
    CSA_LM_F16 = 1,
    CSA_LM_F32 = 2 /* gradients to clip, embeddings and norms only: the matrix units multiply it at a sixteenth of the rate of the other two */
} csa_lm_type;

/* Flags of the *_workspace functions. */
enum {
    CSA_LM_BACKWARD = 1,  /* for the backward call; else for the forward one */
    CSA_LM_COPY_ROWS = 2, /* cross entropy: hidden or weight has rows that 16-byte loads cannot walk (below) */
};

/* ---- spans of documents ---- */

/* For position i of d_text[0, n): d_lo[i] = the last position j <= i with text[j] == separator, 0 if there is none;
 * d_hi[i] = i + 1; d_target[i] = text[i + 1], or -1 if i + 1 == n or text[i + 1] == separator. With the separators of a
 * corpus these are the keys [lo, hi) that a position of a causal model may see, and the token that it has to predict.
 * n <= 2^31 - 1. d_work: csa_lm_spans_workspace(n) bytes. */
uint64_t csa_lm_spans_workspace(uint64_t n);
int csa_lm_spans_u16_dev(const uint16_t* d_text, uint64_t n, uint32_t separator, int32_t* d_lo, int32_t* d_hi, int32_t* d_target,
                         void* d_work, uint64_t work_bytes, void* stream);

/* ---- attention over spans ---- */

/* One array of heads: value d of head h of token t at data[t * token_stride + h * head_stride + d]. 16-byte aligned data, strides
 * that are multiples of 8 values, token_stride >= head_dim and below 2^22. Inputs may overlap (slices of one array, heads in either order). */
typedef struct csa_lm_heads {
    void* data;
    int64_t token_stride;
    int64_t head_stride;
} csa_lm_heads;

typedef struct csa_lm_attention {
    int32_t type;          /* CSA_LM_BF16 or CSA_LM_F16: of all arrays of heads */
    uint32_t q_heads;      /* a multiple of kv_heads: head h of q reads head h / (q_heads / kv_heads) of k and v */
    uint32_t kv_heads;
    uint32_t head_dim;     /* 8 to 128, a multiple of 8 */
    uint64_t tokens;       /* up to 2^30, with fewer than 2^31 rows of q (tokens in 128s times q_heads); fewer than 2^29 for gradients */
    const int32_t* d_lo;   /* row i sees the keys [lo[i], hi[i]), cut to [0, tokens); none where that is empty. NULL: 0 */
    const int32_t* d_hi;   /* NULL: i + 1 */
    const float* d_slope;  /* NULL, or q_heads values: slope[h] * |i - j| is taken off the score of row i and key j */
    float scale;           /* of the products of q and k; positive */
    float cap;             /* > 0: scores become cap * tanh(score / cap), before the slope; 0: they stay. Up to 64 a score is off by 1.5e-7 of the cap, beyond by 5e-7 of itself */
    csa_lm_heads q, k, v;
} csa_lm_attention;

/* Infinities and NaN reach the rows that see them and the keys that such rows see, which may become infinite or NaN in all their values, and nothing else:
 * padding and other documents may hold anything. */

/* out = the softmax over each row's span times v (zeros for rows that see nothing), d_lse[h * tokens + i] = the
 * logarithm of the sum of exponentials of row i's scores (-infinity for rows that see nothing). */
uint64_t csa_lm_attention_workspace(uint64_t tokens, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t flags);
int csa_lm_attention_forward_dev(const csa_lm_attention* a, csa_lm_heads out, float* d_lse, void* d_work, uint64_t work_bytes, void* stream);

/* Gradients of q, k and v for the gradient d_out of out; out and d_lse as the forward call left them. Gradients of a head of k and v are summed
 * over the heads of q that share it. A key that no row sees gets zeros. */
int csa_lm_attention_backward_dev(const csa_lm_attention* a, csa_lm_heads out, const float* d_lse, csa_lm_heads d_out, csa_lm_heads d_q,
                                  csa_lm_heads d_k, csa_lm_heads d_v, void* d_work, uint64_t work_bytes, void* stream);

/* ---- embeddings ---- */

/* out[i] = scale * weight[token[i]], in `type` (any csa_lm_type), zeros where token[i] is no row of the weight, [0, rows). d_tokens: n tokens of token_bytes = 2 (uint16,
 * a text as it lies) or 4 (int32) bytes. weight: rows x dim, its rows weight_stride values apart (>= dim, below 2^22); out: n x dim, dense. dim >= 8; n, rows < 2^31. */
int csa_lm_embed_forward_dev(int type, const void* d_tokens, uint32_t token_bytes, uint64_t n, const void* d_weight, int64_t weight_stride, uint64_t rows, uint64_t dim,
                             float scale, void* d_out, void* stream);

/* weight_grad[v] = scale * the sum over the places i of word v, in a fixed order and in 32 bits, of out_grad[i]; zeros for words that are not there. rows x dim, dense.
 * Rows of out_grad whose token is no row may hold anything. */
uint64_t csa_lm_embed_backward_workspace(int type, uint64_t n, uint64_t rows, uint64_t dim);
int csa_lm_embed_backward_dev(int type, const void* d_tokens, uint32_t token_bytes, uint64_t n, const void* d_out_grad, int64_t out_grad_stride, uint64_t rows, uint64_t dim,
                              float scale, void* d_weight_grad, void* d_work, uint64_t work_bytes, void* stream);

/* ---- norm of a residual stream ---- */

/* total = x + residual, rounded to stream_type; rstd[i] = 1 / sqrt(mean of total[i]^2 + eps), of the rounded total, summed in 64 bits; out = total * rstd * gain.
 * x, gain, out: `type` (any csa_lm_type); residual, total: stream_type, which is `type` or CSA_LM_F32. Rows of x and residual are *_stride values apart (>= dim, below
 * 2^22), out and total are dense. d_residual NULL: total is x, d_total is not written and stream_type is `type`; d_gain NULL: ones. dim: 8 to 16384, eps > 0, fewer than 2^24
 * tokens, 2^22 of rows of more than 2048 values. */
int csa_lm_norm_forward_dev(int type, int stream_type, const void* d_x, int64_t x_stride, const void* d_residual, int64_t residual_stride, const void* d_gain, float eps,
                            uint64_t tokens, uint64_t dim, void* d_out, void* d_total, float* d_rstd, void* stream);

/* With g = out_grad * gain and u = total * rstd: the gradient of x and residual alike is rstd * (g - u * mean(g u)) + total_grad (stream_type; NULL: none flows into total
 * from elsewhere), and gain_grad = the sum over tokens of out_grad * u, in a fixed order, to which rows whose out_grad is zero add nothing, whatever they hold. x_grad (type), residual_grad (stream_type) and gain_grad (type) are dense; any of them may be
 * NULL. The workspace is for gain_grad and may be NULL without it. */
uint64_t csa_lm_norm_backward_workspace(uint64_t tokens, uint64_t dim);
int csa_lm_norm_backward_dev(int type, int stream_type, const void* d_out_grad, int64_t out_grad_stride, const void* d_total, int64_t total_stride, const float* d_rstd,
                             const void* d_gain, const void* d_total_grad, int64_t total_grad_stride, uint64_t tokens, uint64_t dim, void* d_x_grad, void* d_residual_grad,
                             void* d_gain_grad, void* d_work, uint64_t work_bytes, void* stream);

/* ---- softmax cross entropy over a vocabulary ---- */

/* logits[n][v] = sum_d hidden[n][d] weight[v][d] are never kept.
 * d_lse[n] = ln sum_v exp(logits[n][v]); d_loss[n] = d_lse[n] - logits[n][target[n]], 0 where target[n] lies outside [0, vocab).
 * hidden is tokens x dim, weight is vocab x dim, both of `type` (CSA_LM_BF16 or CSA_LM_F16) with their rows *_stride values
 * apart (>= dim, below 2^22). Rows that 16-byte loads cannot walk (an address, a stride or dim that is no multiple of 8 values)
 * are copied to the workspace first, for which it has to be sized with CSA_LM_COPY_ROWS; the rest is read where it lies.
 * tokens, vocab <= 2^30; 2^39 logits in a forward call (2^37 where tokens or words are few), 2^28 tokens in one, 2^42 values of a weight's
 * gradient or 2^35 values to copy are too many for its launches: CSA_ERR_TOO_LARGE, and a workspace of 0. Several calls then take some of the tokens each. */
uint64_t csa_lm_cross_entropy_workspace(uint64_t tokens, uint64_t dim, uint64_t vocab, uint32_t flags);
int csa_lm_cross_entropy_forward_dev(int type, const void* d_hidden, int64_t hidden_stride, const void* d_weight, int64_t weight_stride,
                                     const int32_t* d_target, uint64_t tokens, uint64_t dim, uint64_t vocab, float* d_loss, float* d_lse,
                                     void* d_work, uint64_t work_bytes, void* stream);

/* Gradients of hidden and weight for the gradient d_loss_grad[n] of every token's loss (the weight of token n in the sum that is
 * minimised); d_lse as the forward call left it. Tokens without a target add nothing, whatever their values are. Either gradient may be NULL. */
int csa_lm_cross_entropy_backward_dev(int type, const void* d_hidden, int64_t hidden_stride, const void* d_weight, int64_t weight_stride,
                                      const int32_t* d_target, const float* d_lse, const float* d_loss_grad, uint64_t tokens, uint64_t dim,
                                      uint64_t vocab, void* d_hidden_grad, int64_t hidden_grad_stride, void* d_weight_grad,
                                      int64_t weight_grad_stride, void* d_work, uint64_t work_bytes, void* stream);

/* ---- distillation from a teacher's top logits ---- */

/* Of every token a teacher has kept the logits of `kept` words (1 to 1024): d_ids and d_logits, tokens x kept, dense, in any order. An entry whose id lies outside [0, vocab), or whose
 * logit is -infinity, is none, whatever else it holds; a token without entries has no loss. With q = the softmax over a token's entries of logits / temperature, and z[n][v] = sum_d hidden[n][d]
 * weight[v][d] / temperature, which are never kept,
 *   d_lse[n] = ln sum_v exp(z[n][v]);   d_loss[n] = sum over its entries of q (ln q - z[n][id]) + d_lse[n], 0 without entries.
 * A word that is listed twice counts with both. Arguments, copies and limits are those of the cross entropy, with fewer than 2^24 tokens; temperature: 1e-4 to 1e4. */
uint64_t csa_lm_distill_workspace(uint64_t tokens, uint64_t dim, uint64_t vocab, uint32_t kept, uint32_t flags);
int csa_lm_distill_forward_dev(int type, const void* d_hidden, int64_t hidden_stride, const void* d_weight, int64_t weight_stride, const int32_t* d_ids, const float* d_logits,
                               uint32_t kept, float temperature, uint64_t tokens, uint64_t dim, uint64_t vocab, float* d_loss, float* d_lse, void* d_work, uint64_t work_bytes,
                               void* stream);

/* Gradients of hidden and weight for the gradient d_loss_grad[n] of every token's loss; d_lse as the forward call left it. Tokens without entries add nothing, whatever their values are. Either
 * gradient may be NULL. The teacher has none. */
int csa_lm_distill_backward_dev(int type, const void* d_hidden, int64_t hidden_stride, const void* d_weight, int64_t weight_stride, const int32_t* d_ids, const float* d_logits,
                                uint32_t kept, float temperature, const float* d_lse, const float* d_loss_grad, uint64_t tokens, uint64_t dim, uint64_t vocab,
                                void* d_hidden_grad, int64_t hidden_grad_stride, void* d_weight_grad, int64_t weight_grad_stride, void* d_work, uint64_t work_bytes, void* stream);

/* ---- clipping ---- */

typedef struct csa_lm_values {
    const void* in;
    void* out; /* may be `in` */
    uint64_t n;
    int32_t type; /* csa_lm_type */
} csa_lm_values;

/* *d_norm = the square root of the sum of the squares of all values of the `count` arrays of the host list (summed in 64 bits);
 * out = in * min(1, max_norm / norm), rounded to the type. Where the norm is no finite number of 32 bits the values stay as they are.
 * Arrays are aligned to their type's size. No array's out may overlap another's in or out, nor its own in but for the same address: one that is
 * named twice would be scaled twice, or not, and is refused (CSA_ERR_ARG). The list is read before the call returns. */
uint64_t csa_lm_clip_workspace(uint32_t count);
int csa_lm_clip_dev(const csa_lm_values* list, uint32_t count, float max_norm, float* d_norm, void* d_work, uint64_t work_bytes, void* stream);

/* Message of the calling thread's last failed call of this library ("" if none). */
const char* csa_lm_last_error(void);

#ifdef __cplusplus
}
#endif
#endif
