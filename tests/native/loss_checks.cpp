/* The argument checks and the cutting of the losses over logit rows (loss_checks.h), without a device:
 * prints one line per failed expectation and ends with their number. */
#include "../../geistlib_amd/csrc/loss_checks.h"

#include <cstring>
#include <limits>
#include <vector>

using namespace gs;

static int bad = 0;
static void expect(int got, int want, const Refusal &why, const char *text, const char *what) {
    if (got != want || (want && !std::strstr(why.text, text))) {
        std::printf("%s: %d (%s), expected %d (%s)\n", what, got, why.text, want, text);
        ++bad;
    }
}

int main() {
    alignas(16) static char ws[1 << 16];
    alignas(16) static float x[1 << 12], g[1 << 12];
    uint32_t                 mask[8] = {0};
    float                    loss[8] = {0};
    const float              inf = std::numeric_limits<float>::infinity();
    const float              nan = std::numeric_limits<float>::quiet_NaN();
    geist_hip_loss_rows      ok  = {};
    ok.d_logits = x, ok.ld = 100, ok.rows = 8, ok.n_vocab = 100, ok.type = GEIST_HIP_TYPE_F32;
    ok.temperature = 1.0f, ok.d_grad = g, ok.grad_ld = 128;
#define ROWS(change, code, text)                                                    \
    {                                                                               \
        geist_hip_loss_rows r = ok;                                                 \
        const void         *w = ws;                                                 \
        size_t              n = sizeof ws;                                          \
        const float        *l = loss;                                               \
        Refusal             why;                                                    \
        change;                                                                     \
        expect(check_loss_rows(&r, w, n, l, why), code, why, text, #change);        \
        (void) w, (void) n, (void) l;                                               \
    }
    ROWS(, GEIST_HIP_OK, "")
    ROWS(l = nullptr, GEIST_HIP_OK, "")
    ROWS(r.d_grad = nullptr, GEIST_HIP_OK, "")
    ROWS(r.d_grad = x; r.grad_ld = 100, GEIST_HIP_OK, "")
    ROWS(r.d_grad = nullptr; l = nullptr, GEIST_HIP_E_INVALID_ARG, "neither")
    ROWS(r.d_logits = nullptr, GEIST_HIP_E_INVALID_ARG, "null")
    ROWS(r.type = 3, GEIST_HIP_E_INVALID_ARG, "type")
    ROWS(r.type = -1, GEIST_HIP_E_INVALID_ARG, "type")
    ROWS(r.rows = 0, GEIST_HIP_E_INVALID_ARG, "empty")
    ROWS(r.n_vocab = 0, GEIST_HIP_E_INVALID_ARG, "empty")
    ROWS(r.n_vocab = r.ld = (size_t) 1 << 31, GEIST_HIP_E_INVALID_ARG, "too large")
    ROWS(r.rows = (size_t) 1 << 22, GEIST_HIP_E_UNSUPPORTED, "rows")
    ROWS(r.n_vocab = r.ld = r.grad_ld = 0x7fffff00u; r.rows = 1024, GEIST_HIP_E_UNSUPPORTED, "rows")
    ROWS(r.ld = 99, GEIST_HIP_E_INVALID_ARG, "stride")
    ROWS(r.ld = (size_t) 1 << 60, GEIST_HIP_E_INVALID_ARG, "stride")
    ROWS(r.grad_ld = 99, GEIST_HIP_E_INVALID_ARG, "gradient row stride")
    ROWS(r.d_logits = (char *) x + 2, GEIST_HIP_E_INVALID_ARG, "aligned")
    ROWS(r.d_grad = (char *) g + 1; r.type = GEIST_HIP_TYPE_F16, GEIST_HIP_E_INVALID_ARG, "aligned")
    ROWS(r.d_logits = (char *) x + 2; r.type = GEIST_HIP_TYPE_BF16, GEIST_HIP_OK, "")
    ROWS(r.d_grad = x, GEIST_HIP_E_INVALID_ARG, "overlaps")
    ROWS(r.d_grad = x; r.rows = 1, GEIST_HIP_OK, "")
    ROWS(r.d_grad = x + 1; r.grad_ld = 100, GEIST_HIP_E_INVALID_ARG, "overlaps")
    ROWS(r.d_grad = x + 800; r.grad_ld = 100, GEIST_HIP_OK, "")
    ROWS(r.d_grad = x + 799; r.grad_ld = 100, GEIST_HIP_E_INVALID_ARG, "overlaps")
    ROWS(r.d_allowed = mask; r.allowed_ld = 3, GEIST_HIP_E_INVALID_ARG, "allowed_ld")
    ROWS(r.d_allowed = mask; r.allowed_ld = 4, GEIST_HIP_OK, "")
    ROWS(r.d_allowed = mask, GEIST_HIP_OK, "")
    ROWS(r.temperature = 0.0f, GEIST_HIP_E_INVALID_ARG, "temperature")
    ROWS(r.temperature = nan, GEIST_HIP_E_INVALID_ARG, "temperature")
    ROWS(r.temperature = inf, GEIST_HIP_E_INVALID_ARG, "temperature")
    ROWS(r.logit_softcap = -1.0f, GEIST_HIP_E_INVALID_ARG, "softcap")
    ROWS(r.logit_softcap = nan, GEIST_HIP_E_INVALID_ARG, "softcap")
    ROWS(w = nullptr, GEIST_HIP_E_INVALID_ARG, "workspace")
    ROWS(w = ws + 8, GEIST_HIP_E_INVALID_ARG, "workspace")
    ROWS(n = loss_workspace_bytes(8, 100) - 1, GEIST_HIP_E_INVALID_ARG, "workspace")
    ROWS(n = loss_workspace_bytes(8, 100), GEIST_HIP_OK, "")

    int32_t           ids[8] = {0};
    geist_hip_teacher t0     = {};
    t0.d_ids = ids, t0.d_values = loss, t0.ld = 4, t0.k = 4;
#define TEACHER(change, code, text)                                             \
    {                                                                           \
        geist_hip_teacher t = t0;                                               \
        Refusal           why;                                                  \
        change;                                                                 \
        expect(check_teacher(ok, &t, why), code, why, text, #change);           \
    }
    TEACHER(, GEIST_HIP_OK, "")
    TEACHER(t.k = t.ld = GEIST_HIP_DISTILL_MAX_K, GEIST_HIP_OK, "")
    TEACHER(t.k = t.ld = GEIST_HIP_DISTILL_MAX_K + 1, GEIST_HIP_E_INVALID_ARG, "entries")
    TEACHER(t.k = 0, GEIST_HIP_E_INVALID_ARG, "entries")
    TEACHER(t.ld = 3, GEIST_HIP_E_INVALID_ARG, "entries")
    TEACHER(t.d_ids = nullptr, GEIST_HIP_E_INVALID_ARG, "null")
    TEACHER(t.d_values = nullptr, GEIST_HIP_E_INVALID_ARG, "null")

    geist_hip_policy p0 = {};
    p0.d_tokens = ids, p0.d_advantage = loss, p0.clip_low = 0.2f, p0.clip_high = 0.2f;
#define POLICY(change, code, text)                                              \
    {                                                                           \
        geist_hip_policy p = p0;                                                \
        Refusal          why;                                                   \
        change;                                                                 \
        expect(check_policy(&p, why), code, why, text, #change);                \
    }
    POLICY(, GEIST_HIP_OK, "")
    POLICY(p.d_tokens = nullptr, GEIST_HIP_E_INVALID_ARG, "null")
    POLICY(p.d_advantage = nullptr, GEIST_HIP_E_INVALID_ARG, "null")
    POLICY(p.clip_low = 1.5f, GEIST_HIP_E_INVALID_ARG, "clip")
    POLICY(p.clip_low = nan, GEIST_HIP_E_INVALID_ARG, "clip")
    POLICY(p.clip_high = -0.1f, GEIST_HIP_E_INVALID_ARG, "clip")
    POLICY(p.clip_high = inf, GEIST_HIP_E_INVALID_ARG, "clip")
    POLICY(p.kl_coef = 0.1f, GEIST_HIP_E_INVALID_ARG, "KL term")
    POLICY(p.kl_coef = 0.1f; p.d_ref = loss, GEIST_HIP_OK, "")
    POLICY(p.kl_coef = -0.1f; p.d_ref = loss, GEIST_HIP_E_INVALID_ARG, "kl_coef")
    POLICY(p.entropy_coef = nan, GEIST_HIP_E_INVALID_ARG, "entropy_coef")
    POLICY(p.entropy_coef = -0.5f, GEIST_HIP_OK, "")

    geist_hip_preference q0 = {};
    q0.d_tokens = ids, q0.d_seq_start = ids, q0.n_pairs = 2, q0.beta = 0.1f;
#define PREFERENCE(change, code, text)                                          \
    {                                                                           \
        geist_hip_preference p = q0;                                            \
        Refusal              why;                                               \
        change;                                                                 \
        expect(check_preference(&p, why), code, why, text, #change);            \
    }
    PREFERENCE(, GEIST_HIP_OK, "")
    PREFERENCE(p.d_tokens = nullptr, GEIST_HIP_E_INVALID_ARG, "null")
    PREFERENCE(p.d_seq_start = nullptr, GEIST_HIP_E_INVALID_ARG, "null")
    PREFERENCE(p.n_pairs = 0, GEIST_HIP_E_INVALID_ARG, "pairs")
    PREFERENCE(p.kind = 3, GEIST_HIP_E_INVALID_ARG, "unknown")
    PREFERENCE(p.beta = 0.0f, GEIST_HIP_E_INVALID_ARG, "beta")
    PREFERENCE(p.margin = nan, GEIST_HIP_E_INVALID_ARG, "margin")
    PREFERENCE(p.kind = GEIST_HIP_PREFERENCE_SQUARED; p.margin = 1.0f, GEIST_HIP_E_INVALID_ARG, "margin")
    PREFERENCE(p.kind = GEIST_HIP_PREFERENCE_HINGE; p.margin = 1.0f, GEIST_HIP_OK, "")
    PREFERENCE(p.label_smoothing = 0.6f, GEIST_HIP_E_INVALID_ARG, "label_smoothing")
    PREFERENCE(p.kind = GEIST_HIP_PREFERENCE_HINGE; p.label_smoothing = 0.1f, GEIST_HIP_E_INVALID_ARG,
               "label_smoothing")

    /* every logit belongs to exactly one part, no part is empty by more than the last one's head, and
     * no part outgrows its bit map */
    for (size_t rows : {(size_t) 1, (size_t) 3, (size_t) 64, (size_t) 511, (size_t) 512, (size_t) 5000})
        for (size_t n : {(size_t) 1, (size_t) 7, (size_t) 4096, (size_t) 8191, (size_t) 50257,
                         (size_t) 262144, (size_t) 262145, (size_t) 1 << 24, (size_t) 0x7fffff00u})
            for (size_t elem : {(size_t) 2, (size_t) 4})
            for (LossUse use : {LOSS_ALONE, LOSS_AND_GRADIENT, LOSS_PREFERENCE}) {
                const LossPlan p    = loss_plan(rows, n, elem, use);
                const size_t   vecs = n * elem / 16, held = (size_t) p.chunks * p.chunk_vecs;
                if (p.chunks < 1 || p.chunk_vecs < 1 || held < vecs ||
                    (size_t) (p.chunks - 1) * p.chunk_vecs > vecs ||
                    (size_t) p.chunk_vecs * (16 / elem) > LOSS_MAP_MOST + 64) {
                    std::printf("plan of %zu x %zu, %zu bytes: %d x %d\n", rows, n, elem, p.chunks,
                                p.chunk_vecs);
                    ++bad;
                }
            }
    std::printf("%d failed\n", bad);
    return bad ? 1 : 0;
}
