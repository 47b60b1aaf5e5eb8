/*
 * loss_rows.hip -- how a call of the losses over logit rows (include/geist_loss_hip.h) becomes launches,
 * and the kernel between the two passes of the preference loss. The passes themselves:
 * loss_rows_kernels.h.
 */
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "loss_kernels.h"
#include "sampler_device.h"

namespace gs {
namespace {

constexpr double LN2   = 0.693147180559945309417232;
constexpr double LOG2E = 1.44269504088896340735992;

/* The pairs: log-probabilities of their rows, ratios, loss, and what each row's log-probability is
 * worth. */
constexpr int PAIR_THREADS = 512;
__global__ __launch_bounds__(PAIR_THREADS) void k_pair(LossArgs a) {
    __shared__ double slot[4][PAIR_THREADS / 64];
    const int         pair = blockIdx.x;
    /* the rows that were summed: nothing outside them is looked at, whatever the starts between say */
    const int first = max(0, min(a.rows, a.seq_start[0]));
    const int last  = max(first, min(a.rows, a.seq_start[2 * a.n_pairs]));
    int       edge[3];
    for (int i = 0; i < 3; ++i)
        edge[i] = max(i ? edge[i - 1] : first, min(last, a.seq_start[2 * pair + i]));
    double v[4] = {0.0, 0.0, 0.0, 0.0}; /* sums and numbers of tokens, of either side */
    for (int row = edge[0] + (int) threadIdx.x; row < edge[2]; row += PAIR_THREADS) {
        const LossPart *p    = a.part + (long) row * a.chunks;
        const int       id   = a.tokens[row];
        const bool      used = id >= 0 && id < a.n;
        double          lp   = 0.0;
        if (used) {
            /* the parts joined, as join_parts does it; four are asked for at a time */
            double top = -1e300, s = 0.0, w = 0.0;
            bool   plain = false;
            float  m = -FLT_MAX;
            for (int i = 0; i < a.chunks; i += 4) {
                LossPart four[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    four[k] = p[min(i + k, a.chunks - 1)];
                if (i == 0)
                    w = four[0].a;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k < a.chunks && four[k].s != 0.0) { /* (a part without a sum has no reference) */
                        const LossPart &q   = four[k];
                        const double    was = top;
                        top                 = fmax(top, q.c);
                        s = s * (double) __builtin_amdgcn_exp2f((float) fmax(was - top, -1e30)) +
                            q.s * (double) __builtin_amdgcn_exp2f((float) fmax(q.c - top, -1e30));
                        if (q.c == top) {
                            plain = (was == top && plain) || !q.careful;
                            m     = was == top ? m : -FLT_MAX;
                            if (q.careful)
                                m = fmaxf(m, q.m);
                        }
                    }
            }
            const bool   careful = !plain;
            float        at      = careful ? m : (float) top;
            const double ref = careful ? (double) at * (double) a.k : (double) at;
            s *= exp2(fmax(top - ref, -1e30));
            const double l2s = log2(s);
            lp               = s == 0.0 ? -INFINITY : (w - ref - l2s) * LN2;
            if (lp != -INFINITY) {
                const int side = row < edge[1] ? 0 : 1;
                v[side] += a.ref_lp ? lp - (double) a.ref_lp[row] : lp;
                v[2 + side] += 1.0;
            }
            if (a.row_grad) {
                /* against ref + log2(s) where that is a plain reference: the sum is then near 1 */
                if (!careful) {
                    at = (float) (ref + l2s);
                    s *= exp2(ref - (double) at);
                }
                a.row_grad[row] = {(float) (1.0 / s), at, 0.0f, lp == -INFINITY ? 0 : careful ? 2 : 1};
            }
        }
        if (a.logprob)
            a.logprob[row] = (float) lp;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = wave_sum_f64(v[i]);
    if ((threadIdx.x & 63) == 0)
        for (int i = 0; i < 4; ++i)
            slot[i][threadIdx.x >> 6] = v[i];
    lds_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = wave_sum_f64((threadIdx.x & 63) < PAIR_THREADS / 64 ? slot[i][threadIdx.x & 63] : 0.0);
    double ratio[2], share[2];
    for (int side = 0; side < 2; ++side) {
        share[side] = a.length_normalised ? 1.0 / fmax(v[2 + side], 1.0) : 1.0;
        ratio[side] = v[side] * share[side];
    }
    const double gap = ratio[0] - ratio[1], beta = (double) a.beta;
    const double w = a.weight ? (double) a.weight[pair] : 1.0;
    double       loss, d;
    if (a.kind == GEIST_HIP_PREFERENCE_SQUARED) {
        const double off = gap - 0.5 / beta;
        loss             = off * off;
        d                = 2.0 * off;
    } else {
        const double h = beta * gap - (double) a.margin;
        if (a.kind == GEIST_HIP_PREFERENCE_HINGE) {
            loss = h < 1.0 ? 1.0 - h : h >= 1.0 ? 0.0 : h;
            d    = h < 1.0 ? -beta : h >= 1.0 ? 0.0 : h;
        } else {
            /* -log sigma(h) = max(0, -h) + log(1 + e^-|h|) */
            const double s = (double) a.smoothing, e = exp(-fabs(h));
            loss = log1p(e) + (h < 0.0 ? -(1.0 - s) * h : s == 0.0 ? 0.0 : s * h);
            const double below = h >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e); /* sigma(-h) */
            d = beta * (s - below);
            if (h != h)
                loss = d = h;
        }
    }
    if (w == 0.0) /* a pair that is left out, whatever its rows hold */
        loss = d = 0.0;
    if (threadIdx.x == 0) {
        if (a.loss)
            a.loss[pair] = (float) (w * loss);
        if (a.ratios) {
            a.ratios[2 * pair]     = (float) ratio[0];
            a.ratios[2 * pair + 1] = (float) ratio[1];
        }
    }
    if (a.row_grad) {
        const double c0 = d * w * share[0] * a.inv_t, c1 = -d * w * share[1] * a.inv_t;
        for (int row = edge[0] + (int) threadIdx.x; row < edge[2]; row += PAIR_THREADS) {
            LossRowGrad g = a.row_grad[row];
            if (g.kind == 0)
                continue;
            const double dlp = row < edge[1] ? c0 : c1;
            g.a              = (float) (-dlp * (double) g.a);
            g.q              = (float) -dlp;
            if (dlp == 0.0)
                g.kind = 0;
            a.row_grad[row] = g;
        }
    }
}

/* ---- launches ------------------------------------------------------------------------------- */
/* The Infinity Cache holds 256 MB. Rows that cannot have come from it are read with non-temporal loads
 * (729 MB of sums 138 -> 121 us); where a second pass follows, all but the last of them, which that pass
 * reads first. */
constexpr size_t CACHE_BYTES = (size_t) 224 << 20, KEPT_BYTES = (size_t) 160 << 20;

constexpr size_t GRAD_VECS = 1024; /* groups of 16 bytes per workgroup of the second launch */

size_t elem_bytes(int type) { return type == GEIST_HIP_TYPE_F32 ? 4 : 2; }

LossArgs args_of(const geist_hip_loss_rows &r, void *ws, bool preference = false) {
    LossArgs       a    = {};
    const LossPlan plan = loss_plan(r.rows, r.n_vocab, elem_bytes(r.type),
                                          preference ? LOSS_PREFERENCE
                                          : r.d_grad ? LOSS_AND_GRADIENT
                                                     : LOSS_ALONE);
    a.x          = r.d_logits;
    a.g          = r.d_grad;
    a.ld         = (long) r.ld;
    a.gld        = (long) r.grad_ld;
    a.n          = (int) r.n_vocab;
    a.rows       = (int) r.rows;
    a.allowed    = r.d_allowed;
    a.allowed_ld = (long) r.allowed_ld;
    a.k          = (float) (LOG2E / (double) r.temperature);
    a.cap        = r.logit_softcap;
    if (a.cap > 0.0f) {
        a.inv_cap = 1.0f / a.cap;
        a.cap_k   = (float) ((double) a.cap * (double) a.k);
        a.tanh_k  = (float) (2.0 * LOG2E / (double) a.cap);
    }
    a.inv_t      = 1.0 / (double) r.temperature;
    a.chunks     = plan.chunks;
    a.chunk_vecs = plan.chunk_vecs;
    a.part       = static_cast<LossPart *>(ws);
    const size_t row_bytes = r.ld * elem_bytes(r.type);
    a.streamed      = r.rows * row_bytes > CACHE_BYTES;
    a.streamed_rows = a.streamed ? (int) (r.d_grad ? r.rows - KEPT_BYTES / row_bytes : r.rows) : 0;
    return a;
}
void launch_stage(int type, LossStage stage, int op, bool entropy, const LossArgs &a, size_t lds,
                  hipStream_t stream) {
    int rows = (a.cap > 0.0f ? F_CAP : 0) | (a.allowed || a.tail ? F_BITS : 0);
    if (a.cap > CAP_SMALL && type != GEIST_HIP_TYPE_F32) /* (not a soft-cap any model has: one kernel for all) */
        rows = F_CAP | F_WIDE | F_BITS;
    entropy        = entropy || (op == OP_TOKEN && (rows & F_CAP) && (rows & F_BITS));
    const int feat = rows | (entropy ? F_ENTROPY : 0);
    /* without a gradient the second launch only writes the rows' outputs */
    int c = 1, v = INT32_MAX / 64;
    if (stage == STAGE_GRAD && a.g) {
        const size_t vecs = (size_t) a.n * elem_bytes(type) / 16 + 1;
        size_t       per  = GRAD_VECS;
        while ((size_t) a.rows * ((vecs + per - 1) / per) > LOSS_GRID_MOST)
            per *= 2;
        c = (int) ((vecs + per - 1) / per);
        v = (int) per;
    }
    if (type == GEIST_HIP_TYPE_F32)
        launch_loss<GEIST_HIP_TYPE_F32>(stage, op, feat, a, lds, c, v, stream);
    else if (type == GEIST_HIP_TYPE_F16)
        launch_loss<GEIST_HIP_TYPE_F16>(stage, op, feat, a, lds, c, v, stream);
    else
        launch_loss<GEIST_HIP_TYPE_BF16>(stage, op, feat, a, lds, c, v, stream);
}

} // namespace

void launch_policy(const geist_hip_loss_rows &r, const geist_hip_policy &p, float *loss,
                   float *logprob, float *entropy, void *ws, hipStream_t stream) {
    LossArgs a     = args_of(r, ws);
    a.tokens       = p.d_tokens;
    a.advantage    = p.d_advantage;
    a.old_lp       = p.d_old;
    a.ref_lp       = p.d_ref;
    a.weight       = p.d_weight;
    a.clip_low     = p.clip_low;
    a.clip_high    = p.clip_high;
    a.kl_coef      = p.kl_coef;
    a.entropy_coef = p.entropy_coef;
    a.loss         = loss;
    a.logprob      = logprob;
    a.entropy      = entropy;
    const bool ent = entropy || p.entropy_coef != 0.0f;
    if (a.chunks == 1) {
        launch_stage(r.type, STAGE_ROW, OP_TOKEN, ent, a, 0, stream);
    } else {
        launch_stage(r.type, STAGE_SUMS, OP_TOKEN, ent, a, 0, stream);
        launch_stage(r.type, STAGE_GRAD, OP_TOKEN, ent, a, 0, stream);
    }
}

void launch_distill(const geist_hip_loss_rows &r, const geist_hip_teacher &t, float *loss, void *ws,
                    hipStream_t stream) {
    LossArgs a = args_of(r, ws);
    a.ids      = t.d_ids;
    a.values   = t.d_values;
    a.count    = t.d_count;
    a.list_ld  = (long) t.ld;
    a.list_k   = (int) t.k;
    a.slots    = 2;
    while (a.slots < 2 * a.list_k)
        a.slots *= 2;
    a.tail   = t.tail != 0;
    a.weight = t.d_weight;
    a.loss   = loss;
    /* ids, x, u, q of an entry, the table, and a bit per logit of a part with its head, tail and
     * alignment */
    const size_t list   = (size_t) a.list_k * 16 + (size_t) a.slots * 4;
    const size_t part_n = a.chunks == 1 ? r.n_vocab : (size_t) a.chunk_vecs * (16 / elem_bytes(r.type));
    const size_t map    = a.tail ? (part_n + 64) / 32 * 4 + 4 : 0;
    if (a.chunks == 1) {
        launch_stage(r.type, STAGE_ROW, OP_DISTILL, false, a, list + map, stream);
    } else {
        launch_stage(r.type, STAGE_SUMS, OP_DISTILL, false, a, list + map, stream);
        launch_stage(r.type, STAGE_GRAD, OP_DISTILL, false, a, list, stream);
    }
}

void launch_preference(const geist_hip_loss_rows &r, const geist_hip_preference &p, float *loss,
                       float *ratios, float *logprob, void *ws, hipStream_t stream) {
    LossArgs a  = args_of(r, ws, true);
    a.row_grad  = r.d_grad ? reinterpret_cast<LossRowGrad *>(a.part + r.rows * (size_t) a.chunks) : nullptr;
    a.tokens    = p.d_tokens;
    a.ref_lp    = p.d_ref;
    a.seq_start = p.d_seq_start;
    a.n_pairs   = (int) p.n_pairs;
    a.weight    = p.d_weight;
    a.kind      = p.kind;
    a.beta      = p.beta;
    a.margin    = p.margin;
    a.smoothing = p.label_smoothing;
    a.length_normalised = p.length_normalised;
    a.loss              = loss;
    a.ratios            = ratios;
    a.logprob           = logprob;
    launch_stage(r.type, STAGE_SUMS, OP_PREFERENCE, false, a, 0, stream);
    k_pair<<<dim3((unsigned) p.n_pairs), PAIR_THREADS, 0, stream>>>(a);
    if (r.d_grad)
        launch_stage(r.type, STAGE_GRAD, OP_PREFERENCE, false, a, 0, stream);
}

} // namespace gs
