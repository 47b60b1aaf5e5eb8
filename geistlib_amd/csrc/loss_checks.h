/*
 * loss_checks.h -- what the losses over logit rows (include/geist_loss_hip.h) ask of their arguments,
 * and how a call is cut into workgroups. Plain C++: nothing here needs a device.
 */
#ifndef GEIST_LOSS_CHECKS_H
#define GEIST_LOSS_CHECKS_H

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstddef>
#include <cstdint>
#include <cstdio>

#include "../../include/geist_loss_hip.h"

namespace gs {

/* What one workgroup found out about its part of a row. Values w = softcap(x) log2(e) / T. */
struct LossPart {
    double s;       /* sum of 2^(w - c); with a teacher's tail without the listed tokens */
    double t;       /* sum of 2^u u, u = w - c (entropy only) */
    double c;       /* the reference, near the largest w; means nothing where s is 0 */
    double a;       /* chunk 0: sum of q_j (w_j - top) over the row's listed tokens; w of the sampled token */
    double listed;  /* chunk 0, tail only: sum of 2^(w_j - top) over the listed tokens */
    double top;     /* chunk 0: the largest listed w */
    float  m;       /* careful: c = m log2(e) / T */
    int    careful; /* the sums were made against a value m outside the range of plain references */
};

/* What the gradient of a row of the preference loss takes: 2^(w - ref) a, - q at the token. */
struct LossRowGrad {
    float a, ref, q;
    int   kind; /* 0: zeros; 1; 2: careful, the exponent is (y - ref) k */
};

struct LossPlan {
    int chunks;     /* parts a row is cut into; 1 and not a preference loss: one launch does the rows */
    int chunk_vecs; /* groups of 16 bytes each of them has */
};

constexpr size_t LOSS_MAP_MOST  = (size_t) 1 << 18; /* logits per workgroup its bit map has room for (32 KB) */
constexpr int    LOSS_WIDE_ROWS = 256;              /* up to a row per compute unit: wide workgroups */
constexpr size_t LOSS_GRID_MOST = 0x3fffff;         /* workgroups per launch (of up to 1024 threads) */

enum LossUse { LOSS_ALONE, LOSS_AND_GRADIENT, LOSS_PREFERENCE };

/* How a call over rows x n logits of `elem` bytes is cut. One launch with a workgroup per row reads every
 * logit once; two launches over parts of the rows read them twice and pay a launch more, but spread a few
 * long rows over the device. Measured, one launch against two (us):
 *   with a gradient  1 x 262 KB 15.3 / 8.4, 32 x 257 KB about equal, 16 x 524 KB 30.1 / 12.4,
 *                    64 x 513 KB 25.4 / 20.2 (with a list 26.3 / 32.4, which the rule does not look at: distillation of
 *                    33 to 64 such rows pays for it), 128 x 513 KB 35.5 / 43.1
 *   loss alone       1 x 257 KB 8.1 / 7.4, 64 x 257 KB 9.2 / 9.6, 16 x 524 KB 13.5 / 8.2, 128 x 524 KB 17.0 / 17.3
 * The preference loss has its sums and its gradient in two launches whatever the sizes; its parts of 64 KB
 * cost a large batch nothing (1760 x 257 KB: 264 us whole, 267 cut) and spread a small one
 * (16 x 257 KB 40.2 / 20.1). */
inline LossPlan loss_plan(size_t rows, size_t n, size_t elem, LossUse use) {
    const size_t vecs = n * elem / 16 + 1, row_bytes = n * elem;
    LossPlan     p    = {1, (int) vecs};
    size_t       chunks = 1;
    if (use == LOSS_PREFERENCE)
        chunks = rows < 64 ? (vecs + 2047) / 2048 : (vecs + 4095) / 4096;
    else if (row_bytes > 200000 && rows <= (use == LOSS_AND_GRADIENT && row_bytes > 400000 ? 64 : 32))
        chunks = std::min((vecs + 1023) / 1024, 2048 / rows);
    chunks = std::max(chunks, (n + LOSS_MAP_MOST - 1) / LOSS_MAP_MOST);
    if (chunks > 1) {
        p.chunk_vecs = (int) ((vecs + chunks - 1) / chunks);
        p.chunks     = (int) ((vecs + p.chunk_vecs - 1) / p.chunk_vecs);
    }
    return p;
}

inline size_t loss_chunks_most(size_t rows, size_t n, size_t elem) {
    int most = 1;
    for (LossUse use : {LOSS_ALONE, LOSS_AND_GRADIENT, LOSS_PREFERENCE})
        most = std::max(most, loss_plan(rows, n, elem, use).chunks);
    return (size_t) most;
}
inline size_t loss_workspace_bytes(size_t rows, size_t n_vocab) {
    if (rows == 0 || n_vocab == 0 || rows > LOSS_GRID_MOST || n_vocab > 0x7fffff00u)
        return 0;
    const size_t chunks = std::max(loss_chunks_most(rows, n_vocab, 2), loss_chunks_most(rows, n_vocab, 4));
    return (rows * (chunks * sizeof(LossPart) + sizeof(LossRowGrad)) + 15) / 16 * 16;
}

/* Each check returns a status code and leaves the reason of a refusal in `why`. */
struct Refusal {
    char text[256] = {0};
};
__attribute__((format(printf, 3, 4))) inline int refuse(Refusal &why, int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(why.text, sizeof why.text, fmt, ap);
    va_end(ap);
    return code;
}

/* result: one of the vectors that the call writes beside the gradient, if any */
inline int check_loss_rows(const geist_hip_loss_rows *r, const void *ws, size_t ws_bytes,
                           const float *result, Refusal &why) {
    if (!r || !r->d_logits)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "null rows or logits");
    if (r->type != GEIST_HIP_TYPE_F32 && r->type != GEIST_HIP_TYPE_F16 && r->type != GEIST_HIP_TYPE_BF16)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "unknown type %d", r->type);
    if (r->rows == 0 || r->n_vocab == 0)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "empty batch (rows=%zu, n_vocab=%zu)", r->rows,
                      r->n_vocab);
    if (r->n_vocab > 0x7fffff00u)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "n_vocab too large");
    const size_t elem = r->type == GEIST_HIP_TYPE_F32 ? 4 : 2;
    if (r->rows > LOSS_GRID_MOST ||
        loss_chunks_most(r->rows, r->n_vocab, elem) * r->rows > LOSS_GRID_MOST)
        return refuse(why, GEIST_HIP_E_UNSUPPORTED, "%zu rows of %zu logits in one call", r->rows,
                      r->n_vocab);
    if (r->ld < r->n_vocab || r->ld > ((size_t) 1 << 58) / r->rows)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "row stride %zu with n_vocab %zu", r->ld, r->n_vocab);
    if ((uintptr_t) r->d_logits % elem != 0 || (uintptr_t) r->d_grad % elem != 0)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "logits or gradient not aligned to their type");
    if (r->d_grad) {
        if (r->grad_ld < r->n_vocab || r->grad_ld > ((size_t) 1 << 58) / r->rows)
            return refuse(why, GEIST_HIP_E_INVALID_ARG, "gradient row stride %zu with n_vocab %zu",
                          r->grad_ld, r->n_vocab);
        const uintptr_t x = (uintptr_t) r->d_logits, g = (uintptr_t) r->d_grad;
        const size_t    x_bytes = ((r->rows - 1) * r->ld + r->n_vocab) * elem;
        const size_t    g_bytes = ((r->rows - 1) * r->grad_ld + r->n_vocab) * elem;
        if (x == g ? (r->rows > 1 && r->ld != r->grad_ld) : (x < g + g_bytes && g < x + x_bytes))
            return refuse(why, GEIST_HIP_E_INVALID_ARG,
                          "the gradient overlaps the logits without being in their place");
    }
    if (r->d_allowed && r->allowed_ld != 0 &&
        (r->allowed_ld < (r->n_vocab + 31) / 32 || r->allowed_ld > ((size_t) 1 << 58) / r->rows))
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "allowed_ld %zu with %zu mask words per row",
                      r->allowed_ld, (r->n_vocab + 31) / 32);
    if (!(r->temperature >= 1e-4f && r->temperature <= 1e4f))
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "temperature %g is not within 1e-4 .. 1e4",
                      (double) r->temperature);
    if (!(r->logit_softcap == 0.0f || (r->logit_softcap >= 1e-3f && r->logit_softcap <= 1e6f)))
        return refuse(why, GEIST_HIP_E_INVALID_ARG,
                      "logit_softcap %g is neither 0 nor within 1e-3 .. 1e6", (double) r->logit_softcap);
    const size_t need = loss_workspace_bytes(r->rows, r->n_vocab);
    if (!ws || (uintptr_t) ws % 16 != 0 || ws_bytes < need)
        return refuse(why, GEIST_HIP_E_INVALID_ARG,
                      "workspace: %zu bytes, 16-byte aligned, are needed (%zu given)", need,
                      ws ? ws_bytes : (size_t) 0);
    if (!result && !r->d_grad)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "neither a result nor a gradient is asked for");
    return GEIST_HIP_OK;
}

inline int check_teacher(const geist_hip_loss_rows &r, const geist_hip_teacher *t, Refusal &why) {
    if (!t || !t->d_ids || !t->d_values)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "null teacher, ids or values");
    if (t->k == 0 || t->k > GEIST_HIP_DISTILL_MAX_K || t->ld < t->k ||
        t->ld > ((size_t) 1 << 58) / r.rows)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "teacher lists of %zu entries (1 .. %d), stride %zu",
                      t->k, GEIST_HIP_DISTILL_MAX_K, t->ld);
    return GEIST_HIP_OK;
}

inline int check_policy(const geist_hip_policy *p, Refusal &why) {
    if (!p || !p->d_tokens || !p->d_advantage)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "null policy, tokens or advantages");
    if (!(p->clip_low >= 0.0f && p->clip_low <= 1.0f) ||
        !(p->clip_high >= 0.0f && std::isfinite(p->clip_high)))
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "clip range 1 - %g .. 1 + %g",
                      (double) p->clip_low, (double) p->clip_high);
    if (!(p->kl_coef >= 0.0f && std::isfinite(p->kl_coef)) || !std::isfinite(p->entropy_coef))
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "kl_coef %g, entropy_coef %g",
                      (double) p->kl_coef, (double) p->entropy_coef);
    if (p->kl_coef != 0.0f && !p->d_ref)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "a KL term without reference log-probabilities");
    return GEIST_HIP_OK;
}

inline int check_preference(const geist_hip_preference *p, Refusal &why) {
    if (!p || !p->d_tokens || !p->d_seq_start)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "null preference, tokens or sequence starts");
    if (p->n_pairs == 0 || p->n_pairs > LOSS_GRID_MOST)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "%zu pairs", p->n_pairs);
    if (p->kind != GEIST_HIP_PREFERENCE_SIGMOID && p->kind != GEIST_HIP_PREFERENCE_HINGE &&
        p->kind != GEIST_HIP_PREFERENCE_SQUARED)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "unknown preference loss %d", p->kind);
    if (!(p->beta > 0.0f && std::isfinite(p->beta)) || !std::isfinite(p->margin))
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "beta %g, margin %g", (double) p->beta,
                      (double) p->margin);
    if (p->kind == GEIST_HIP_PREFERENCE_SQUARED && p->margin != 0.0f)
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "the squared loss has no margin");
    if (!(p->label_smoothing >= 0.0f && p->label_smoothing <= 0.5f) ||
        (p->kind != GEIST_HIP_PREFERENCE_SIGMOID && p->label_smoothing != 0.0f))
        return refuse(why, GEIST_HIP_E_INVALID_ARG, "label_smoothing %g with loss %d",
                      (double) p->label_smoothing, p->kind);
    return GEIST_HIP_OK;
}

} // namespace gs
#endif /* GEIST_LOSS_CHECKS_H */
