/* Launchers of the losses over logit rows (loss_rows.hip, include/geist_loss_hip.h). */
#ifndef GEIST_LOSS_KERNELS_H
#define GEIST_LOSS_KERNELS_H

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "loss_checks.h"

namespace gs {

/* FEAT bits: what a kernel is compiled for beyond plain rows */
constexpr int F_ENTROPY = 1; /* sum 2^u u, and a term of p_i u_i in the gradient */
constexpr int F_CAP     = 2; /* a soft-cap */
constexpr int F_WIDE    = 8; /* 16-bit rows: a soft-cap above CAP_SMALL, whose tanh is formed more closely */
constexpr int F_BITS    = 4; /* an allowed-token mask or a teacher's tail: tokens that do not count */

constexpr float CAP_SMALL = 64.0f;

constexpr int OP_TOKEN      = 0; /* one token per row, policy loss */
constexpr int OP_DISTILL    = 1;
constexpr int OP_PREFERENCE = 2; /* one token per row, coefficient from the pair's margin */

struct LossArgs {
    const void     *x;
    void           *g;
    long            ld, gld;
    int             n, rows;
    const uint32_t *allowed;
    long            allowed_ld;
    float           k;       /* log2(e) / T */
    float           cap;     /* 0 = none */
    float           inv_cap;
    float           cap_k;   /* cap * k */
    float           tanh_k;  /* 2 log2(e) / cap */
    double          inv_t;
    int             chunks, chunk_vecs;
    int             stash, stash_at; /* k_loss_row: groups per thread that LDS keeps, and where */
    bool            streamed;      /* the rows are too many bytes to have come from the cache */
    int             streamed_rows; /* rows of the first pass over them that will not be in it later either */
    LossPart       *part;    /* [rows][chunks] */
    /* one token per row */
    const int32_t  *tokens;
    const float    *advantage, *old_lp, *ref_lp, *weight;
    float           clip_low, clip_high, kl_coef, entropy_coef;
    float          *loss, *logprob, *entropy;
    /* distillation */
    const int32_t  *ids, *count;
    const float    *values;
    long            list_ld;
    int             list_k, slots; /* slots: places of the table that finds repeated ids, a power of 2 */
    int             tail;
    /* preference */
    const int32_t  *seq_start;
    int             n_pairs;
    LossRowGrad    *row_grad; /* [rows] */
    float          *ratios;
    int             kind, length_normalised;
    float           beta, margin, smoothing;
};

enum LossStage { STAGE_ROW, STAGE_SUMS, STAGE_GRAD };
/* One kernel over all rows; chunks and chunk_vecs: how STAGE_GRAD cuts them. Instantiated per type. */
template <int TYPE>
void launch_loss(LossStage stage, int op, int feat, const LossArgs &a, size_t lds, int chunks,
                 int chunk_vecs, hipStream_t stream);

void launch_distill(const geist_hip_loss_rows &r, const geist_hip_teacher &t, float *loss, void *ws,
                    hipStream_t stream);
void launch_policy(const geist_hip_loss_rows &r, const geist_hip_policy &p, float *loss,
                   float *logprob, float *entropy, void *ws, hipStream_t stream);
void launch_preference(const geist_hip_loss_rows &r, const geist_hip_preference &p, float *loss,
                       float *ratios, float *logprob, void *ws, hipStream_t stream);

} // namespace gs
#endif /* GEIST_LOSS_KERNELS_H */
