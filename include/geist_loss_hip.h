/*
 * geist_loss_hip.h -- losses over logit rows, with the gradient of the logits (gfx950).
 *
 * What a model is trained on after it answered: the rows it sampled from, under the same
 * temperature, soft-cap and allowed-token mask as the sampling entry points of
 * geist_sampler_hip.h. Three losses: distillation from a teacher's top logits, the clipped policy
 * loss with a KL term over sampled tokens, and the preference loss over pairs of sequences.
 * The reference (geistlib 0.9.0) does inference only and has no counterpart of these.
 *
 * As in geist_sampler_hip.h: plain C, device pointers, every call enqueues kernels on the
 * sampler's stream and returns; failures by status code with their text in
 * geist_hip_sampler_last_error. The sampler object gives device, stream and error text only; its
 * max_rows and max_vocab do not bound these calls. Nothing is allocated, so the calls may be
 * recorded into a HIP graph: scratch memory is the caller's (geist_hip_loss_workspace_bytes).
 */
#ifndef GEIST_LOSS_HIP_H
#define GEIST_LOSS_HIP_H

#include "geist_sampler_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of logits and gradients. */
#define GEIST_HIP_TYPE_F32 0
#define GEIST_HIP_TYPE_F16 1
#define GEIST_HIP_TYPE_BF16 2

/* Rows of logits and where their gradient goes. Row r starts at element r * ld of d_logits (any ld
 * >= n_vocab, any alignment of the type). What a row stands for is
 *   v_i = softcap(x_i) / temperature,  softcap(x) = c * tanh(x / c) for c > 0, else x,
 *   p = softmax(v) over the tokens that d_allowed allows (bit e % 32 of word
 *       d_allowed[r * allowed_ld + e / 32], allowed_ld = 0: one mask for all rows; NULL: all).
 * A forbidden token's logit is not looked at (it may be NaN) and its gradient is 0 (0 or NaN in a row whose
 * results are NaN).
 *
 * d_grad, if given, receives the gradient of the SUM of the call's losses by the logits, in the
 * type of the logits, rounded once; a training step that weighs the losses (a mean, an upstream
 * gradient) puts the weights into the call. NULL: loss only. It may be d_logits itself (with
 * grad_ld == ld): the rows are then replaced by their gradient. Otherwise the two must not overlap.
 * Sums over a row are formed in binary32 over a few groups of 16 bytes and in binary64 beyond them,
 * everything per row or per pair in binary64. How a row is added up follows from the call's sizes,
 * types and options: the same call gives the same bits.
 *
 * A row that has no token left (all forbidden, or every allowed v_i is -inf) has no distribution: its loss
 * and gradient are 0. NaN among a row's allowed logits, and without a soft-cap +inf, make that row's
 * results NaN, and no other row's (for the preference loss: no other pair's); where a row's or pair's
 * weight is 0, loss and gradient are 0 whatever its logits are. A soft-cap takes +inf to c and -inf to -c,
 * both with a gradient of 0: overflowed logits of a capped model do not show in its results.
 * Limits: temperature within 1e-4 .. 1e4, logit_softcap 0 or within 1e-3 .. 1e6, at most 2^22 - 1
 * rows; GEIST_HIP_E_UNSUPPORTED where rows x the parts a row is cut into exceeds that. */
struct geist_hip_loss_rows {
    const void     *d_logits;
    size_t          ld;
    size_t          rows;
    size_t          n_vocab;
    int             type;          /* GEIST_HIP_TYPE_* */
    const uint32_t *d_allowed;     /* NULL = every token allowed */
    size_t          allowed_ld;
    float           temperature;   /* > 0 */
    float           logit_softcap; /* 0 = off */
    void           *d_grad;        /* NULL = no gradient */
    size_t          grad_ld;
};

/* Bytes of scratch memory a call over `rows` rows of `n_vocab` logits needs (any of the losses, any
 * type). The contents mean nothing between calls; calls that can run at the same time (two
 * streams, two recorded graphs) need one workspace each. 16-byte aligned. */
size_t geist_hip_loss_workspace_bytes(size_t rows, size_t n_vocab);

/* Distillation from a teacher's top logits: row r lists k tokens d_ids[r * ld ..] with the teacher's
 * values d_values[r * ld ..]; d_count[r], if given, is how many of them count (0 .. k).
 *   tail = 0: values are the teacher's logits (or log-probabilities at temperature 1);
 *             q = softmax(values / temperature) over the list,
 *             loss_r = w_r * sum_j q_j (log q_j - log p_{id_j})
 *   tail = 1: values are the teacher's log-probabilities at the call's temperature, q = exp(values);
 *             the mass that is not listed is one more event, q_rest = max(0, 1 - sum q),
 *             p_rest = the student's mass of all tokens that are not listed:
 *             loss_r = w_r * (sum_j q_j (log q_j - log p_{id_j}) + q_rest (log q_rest - log p_rest))
 * An entry is left out (with tail = 1 its mass counts to the rest) when its id is outside
 * [0, n_vocab), forbidden by the mask, listed before in the same row, or when its value is -inf. A
 * row without entries has loss and gradient 0. A row that gives a listed token probability 0 has
 * loss +inf. (The usual factor temperature^2 goes into the weight.) */
#define GEIST_HIP_DISTILL_MAX_K 1024
struct geist_hip_teacher {
    const int32_t *d_ids;
    const float   *d_values;
    size_t         ld;       /* between the lists of consecutive rows, >= k */
    size_t         k;        /* 1 .. GEIST_HIP_DISTILL_MAX_K */
    const int32_t *d_count;  /* [rows], NULL = k everywhere */
    const float   *d_weight; /* [rows], NULL = 1 */
    int            tail;
};
int geist_hip_distill_rows(geist_hip_sampler *s, const struct geist_hip_loss_rows *rows,
                           const struct geist_hip_teacher *teacher, float *d_loss,
                           void *d_workspace, size_t workspace_bytes);

/* The clipped policy loss of sampled tokens with a KL term towards a reference policy:
 *   lp = log p_{token},  ratio = exp(lp - old),  H = -sum_i p_i log p_i,  d = ref - lp
 *   loss_r = w_r * ( -min(ratio * A, clip(ratio, 1 - clip_low, 1 + clip_high) * A)
 *                    + kl_coef * (exp(d) - d - 1) - entropy_coef * H )
 * d_old = NULL: the rows are those the tokens were drawn from (ratio 1, gradient -A (..)).
 * The gradient flows through the ratio where the first argument of min is not the larger one; an
 * advantage of 0 gives 0 whatever the ratio. Tokens outside [0, n_vocab) mark positions that are
 * not trained on (prompt, padding): loss, logprob and gradient 0, H is still reported. A token
 * with probability 0 (forbidden, or a logit of -inf) has logprob -inf and loss and gradient 0.
 * d_loss, d_logprob ([rows], lp), d_entropy ([rows], H) and d_grad may each be NULL, not all of them:
 * d_logprob alone scores the tokens. With d_ref = NULL, kl_coef must be 0; with kl_coef = 0, d_ref is
 * not looked at. */
struct geist_hip_policy {
    const int32_t *d_tokens;    /* [rows] */
    const float   *d_advantage; /* [rows] */
    const float   *d_old;       /* [rows] log-probabilities under the sampling policy, or NULL */
    const float   *d_ref;       /* [rows] log-probabilities under the reference policy, or NULL */
    const float   *d_weight;    /* [rows], NULL = 1 */
    float          clip_low;    /* 0 .. 1 */
    float          clip_high;   /* >= 0 */
    float          kl_coef;     /* >= 0 */
    float          entropy_coef;
};
int geist_hip_policy_loss_rows(geist_hip_sampler *s, const struct geist_hip_loss_rows *rows,
                               const struct geist_hip_policy *policy, float *d_loss,
                               float *d_logprob, float *d_entropy, void *d_workspace,
                               size_t workspace_bytes);

/* Preference loss over n_pairs pairs of token sequences laid end to end in the rows: sequence s is
 * the rows [d_seq_start[s], d_seq_start[s + 1]) (2 * n_pairs + 1 non-decreasing entries within
 * [0, rows]; the first and last are clamped to that range, the others to the range between those
 * two), pair i prefers sequence 2i to sequence 2i + 1.
 *   D_s = sum over the sequence's tokens of (log p_{token} - ref), ref = 0 when d_ref is NULL;
 *         length_normalised: divided by their number
 *   GEIST_HIP_PREFERENCE_SIGMOID  h = beta (D_2i - D_2i+1) - margin,
 *                 loss_i = w_i * (-(1 - label_smoothing) log sigma(h) - label_smoothing log sigma(-h))
 *   GEIST_HIP_PREFERENCE_HINGE    loss_i = w_i * max(0, 1 - h)
 *   GEIST_HIP_PREFERENCE_SQUARED  loss_i = w_i * (D_2i - D_2i+1 - 1 / (2 beta))^2
 * Rows whose token is outside [0, n_vocab) (prompt, padding) and rows that give their token
 * probability 0 are left out of the sums: logprob 0 or -inf, gradient 0. Rows in front of the first
 * sequence and behind the last are not read, and their logprob and gradient are not written.
 * d_loss [n_pairs], d_ratios [2 * n_pairs] (D_s), d_logprob [rows] and d_grad may each be NULL, not
 * all of them. */
#define GEIST_HIP_PREFERENCE_SIGMOID 0
#define GEIST_HIP_PREFERENCE_HINGE 1
#define GEIST_HIP_PREFERENCE_SQUARED 2
struct geist_hip_preference {
    const int32_t *d_tokens;    /* [rows] */
    const float   *d_ref;       /* [rows] or NULL */
    const int32_t *d_seq_start; /* [2 * n_pairs + 1] */
    size_t         n_pairs;
    const float   *d_weight;    /* [n_pairs], NULL = 1 */
    int            kind;
    float          beta;            /* > 0 */
    float          margin;          /* 0 for GEIST_HIP_PREFERENCE_SQUARED */
    float          label_smoothing; /* 0 .. 0.5, for GEIST_HIP_PREFERENCE_SIGMOID; else 0 */
    int            length_normalised;
};
int geist_hip_preference_loss(geist_hip_sampler *s, const struct geist_hip_loss_rows *rows,
                              const struct geist_hip_preference *preference, float *d_loss,
                              float *d_ratios, float *d_logprob, void *d_workspace,
                              size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* GEIST_LOSS_HIP_H */
