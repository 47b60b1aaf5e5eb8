/*
 * loss_rows.hip -- losses over logit rows and their gradients (include/geist_loss_hip.h).
 *
 * Every loss here needs of a row x the numbers m = max y and S = sum 2^((y - m) k) with
 * y = softcap(x), k = log2(e) / T (and, for the entropy, sum 2^u u with u = (y - m) k), the values at
 * a few listed tokens, and its gradient by the logits has one form:
 *     g_i = (p_i (A + B u_i) - [i listed] q_i W) * softcap'(x_i) / T,     p_i = 2^u_i / S
 * with A, B, W of the row (A differs between listed and other tokens for a teacher with a tail).
 * So one streaming core serves all three: a pass that sums, a few scalars, a pass that writes.
 */
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "loss_kernels.h"

namespace gs {
namespace {

constexpr double LN2   = 0.693147180559945309417232;
constexpr double LOG2E = 1.44269504088896340735992;

/* FEAT bits: what a kernel is compiled for beyond plain rows */
constexpr int F_ENTROPY = 1; /* sum 2^u u, and B != 0 in the gradient */
constexpr int F_GENERAL = 2; /* soft-cap, allowed-token mask or a teacher's tail, looked at per group */

constexpr int OP_TOKEN      = 0; /* one token per row, policy loss */
constexpr int OP_DISTILL    = 1;
constexpr int OP_PREFERENCE = 2; /* one token per row, coefficient from the pair's margin */

/* ---- types ---------------------------------------------------------------------------------- */
typedef float    f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16   bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int TYPE> struct Elem;
template <> struct Elem<GEIST_HIP_TYPE_F32> {
    typedef float         mem;
    static constexpr int  N = 4;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = __float_as_uint(f[i]);
        return v;
    }
    static __device__ __forceinline__ float one(mem x) { return x; }
    static __device__ __forceinline__ mem   round(float x) { return x; }
};
template <> struct Elem<GEIST_HIP_TYPE_F16> {
    typedef _Float16      mem;
    static constexpr int  N = 8;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t) v[i]);
            f[2 * i]      = (float) h[0];
            f[2 * i + 1]  = (float) h[1];
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16x2 h = {(_Float16) f[2 * i], (_Float16) f[2 * i + 1]};
            v[i]          = __builtin_bit_cast(uint32_t, h);
        }
        return v;
    }
    static __device__ __forceinline__ float one(mem x) { return (float) x; }
    static __device__ __forceinline__ mem   round(float x) { return (_Float16) x; }
};
template <> struct Elem<GEIST_HIP_TYPE_BF16> {
    typedef __bf16        mem;
    static constexpr int  N = 8;
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i]     = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x2 p = {f[2 * i], f[2 * i + 1]};
            v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
        }
        return v;
    }
    static __device__ __forceinline__ float one(mem x) { return (float) x; }
    static __device__ __forceinline__ mem   round(float x) { return (__bf16) x; }
};

/* ---- arguments ------------------------------------------------------------------------------ */
struct LossArgs {
    const void     *x;
    void           *g;
    long            ld, gld;
    int             n, rows;
    const uint32_t *allowed;
    long            allowed_ld;
    float           k;      /* log2(e) / T */
    float           slack;  /* how far (in y) a value may exceed a thread's reference */
    float           cap;    /* 0 = none */
    float           tanh_k; /* 2 log2(e) / cap */
    double          inv_t;
    int             chunks, chunk_vecs;
    LossPart       *part;   /* [rows][chunks] */
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
    float          *coef; /* [rows] d loss / d logprob */
    float          *ratios;
    int             kind, length_normalised;
    float           beta, margin, smoothing;
};

/* ---- reductions ----------------------------------------------------------------------------- */
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1)
        v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1)
        v += __shfl_xor(v, d);
    return v;
}
/* over the workgroup, every thread gets the result; `slot`: 16 doubles of LDS */
template <int THREADS> __device__ __forceinline__ float block_max(float v, double *slot) {
    v = wave_max(v);
    float *f = reinterpret_cast<float *>(slot);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        f[threadIdx.x >> 6] = v;
    __syncthreads();
    v = f[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i)
        v = fmaxf(v, f[i]);
    return v;
}
template <int THREADS> __device__ __forceinline__ double block_sum(double v, double *slot) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i)
        v += slot[i];
    return v;
}

/* ---- a row ---------------------------------------------------------------------------------- */
/* c tanh(x / c) by t = (1 - e) / (1 + e), e = 2^(-2 |x| log2(e) / c); its slope is 4 e / (1 + e)^2 */
__device__ __forceinline__ float capped(float x, float cap, float tanh_k) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * tanh_k);
    return copysignf(cap * ((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e)), x);
}
__device__ __forceinline__ float capped_slope(float x, float tanh_k) {
    const float e = __builtin_amdgcn_exp2f(-fabsf(x) * tanh_k);
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    return 4.0f * e * (r * r);
}

template <int TYPE> struct Row {
    typedef typename Elem<TYPE>::mem mem;
    static constexpr int             N = Elem<TYPE>::N;
    const mem      *x;
    mem            *g;
    const uint32_t *allowed;
    int             n, head, nvec; /* elements in front of the first 16-byte boundary, groups behind it */
    bool            g_aligned;     /* the gradient's groups start on 16-byte boundaries too */
    int             v0, v1;        /* this workgroup's groups */
    bool            first, last;   /* it also takes the head / what is behind the last group */

    __device__ Row(const LossArgs &a, int row, int chunk) {
        x       = static_cast<const mem *>(a.x) + (long) row * a.ld;
        g       = a.g ? static_cast<mem *>(a.g) + (long) row * a.gld : nullptr;
        allowed = a.allowed ? a.allowed + (long) row * a.allowed_ld : nullptr;
        n       = a.n;
        head    = (int) ((16u - ((uintptr_t) x & 15u)) & 15u) / (int) sizeof(mem);
        if (head > n)
            head = n;
        nvec      = (n - head) / N;
        g_aligned = (((uintptr_t) (g + head)) & 15u) == 0;
        v0        = min(nvec, chunk * a.chunk_vecs);
        v1        = chunk == a.chunks - 1 ? nvec : min(nvec, v0 + a.chunk_vecs);
        first     = chunk == 0;
        last      = chunk == a.chunks - 1;
    }
    __device__ __forceinline__ int   elem0() const { return head + v0 * N; } /* of group v0 */
    __device__ __forceinline__ u32x4 load(int v) const {
        return *reinterpret_cast<const u32x4 *>(x + head + (long) v * N);
    }
    __device__ __forceinline__ void store(int v, u32x4 d) const {
        mem *p = g + head + (long) v * N;
        if (g_aligned) {
            *reinterpret_cast<u32x4 *>(p) = d;
        } else {
            const mem *e = reinterpret_cast<const mem *>(&d);
#pragma unroll
            for (int i = 0; i < N; ++i)
                p[i] = e[i];
        }
    }
    __device__ __forceinline__ bool may(int e) const {
        return !allowed || ((allowed[e >> 5] >> (e & 31)) & 1u);
    }
    /* mask bits of the group that starts at element e */
    __device__ __forceinline__ uint32_t bits(int e) const {
        const int sh = e & 31;
        uint32_t  w  = allowed[e >> 5] >> sh;
        if (sh > 32 - N)
            w |= allowed[(e >> 5) + 1] << (32 - sh);
        return w;
    }
    /* the i-th element that belongs to no group: the head, then the tail; -1 behind them */
    __device__ __forceinline__ int loose(int i) const {
        if (first && i < head)
            return i;
        if (first)
            i -= head;
        const int behind = head + nvec * N;
        return last && i < n - behind ? behind + i : -1;
    }
};

/* ---- the pass that sums --------------------------------------------------------------------- */
/* A thread sums 2^((y - m) k) against a reference m of its own that follows the largest value it has
 * seen at a distance: it moves only when a value exceeds it by more than 20 in the exponent, so the
 * usual batch costs no rescaling and no sum can overflow. The reference starts at the lowest finite
 * value: -inf then weighs 0, and a row whose values all are that lowest value is uniform.
 * A batch of U groups is added up in binary32 by halves, and the batches in binary64: a running
 * binary32 sum loses what is small beside a leading token, always downwards (2e-6 of the sum over
 * a whole row, 1e-7 over batches of 32). */
struct Acc {
    float  m = -FLT_MAX;
    double s = 0.0, t = 0.0;
};
template <int FEAT> __device__ __forceinline__ void acc_move(Acc &c, float m, float k) {
    const float  d  = fmaxf((c.m - m) * k, -1e30f);
    const double sc = (double) __builtin_amdgcn_exp2f(d);
    if (FEAT & F_ENTROPY)
        c.t = sc * (c.t + c.s * (double) d);
    c.s *= sc;
    c.m = m;
}
template <int COUNT, int FEAT>
__device__ __forceinline__ void acc_batch(Acc &c, const float (&y)[COUNT], float k, float slack) {
    float top = y[0];
#pragma unroll
    for (int i = 1; i < COUNT; ++i)
        top = fmaxf(top, y[i]);
    if (top > c.m + slack)
        acc_move<FEAT>(c, top, k);
    float e[COUNT], t = 0.0f;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
        const float u = (y[i] - c.m) * k;
        e[i]          = __builtin_amdgcn_exp2f(u);
        if (FEAT & F_ENTROPY)
            t = fmaf(e[i], fmaxf(u, -1e30f), t);
    }
#pragma unroll
    for (int half = COUNT / 2; half; half >>= 1)
#pragma unroll
        for (int i = 0; i < half; ++i)
            e[i] += e[i + half];
    c.s += (double) e[0];
    if (FEAT & F_ENTROPY)
        c.t += (double) t;
}

/* x -> y of a group; forbidden tokens become -inf */
template <int TYPE, int FEAT>
__device__ __forceinline__ void group_values(const LossArgs &a, const Row<TYPE> &r, int v,
                                             float (&y)[Elem<TYPE>::N]) {
    if (!(FEAT & F_GENERAL))
        return;
    if (a.cap > 0.0f) {
#pragma unroll
        for (int i = 0; i < Elem<TYPE>::N; ++i)
            y[i] = capped(y[i], a.cap, a.tanh_k);
    }
    if (r.allowed) {
        const uint32_t w = r.bits(r.head + v * Elem<TYPE>::N);
#pragma unroll
        for (int i = 0; i < Elem<TYPE>::N; ++i)
            y[i] = ((w >> i) & 1u) ? y[i] : -INFINITY;
    }
}
template <int TYPE, int FEAT>
__device__ __forceinline__ float one_value(const LossArgs &a, const Row<TYPE> &r, int e, float x) {
    if (!(FEAT & F_GENERAL))
        return x;
    if (!r.may(e))
        return -INFINITY;
    return a.cap > 0.0f ? capped(x, a.cap, a.tanh_k) : x;
}

/* Listed tokens of the workgroup's part of the row as bits (tail only): group v's start at bit
 * (v - v0 + 1) N, so that a group's bits lie in one byte; the head is in front of group v0. */
template <int N> __device__ __forceinline__ uint32_t listed_bits(const uint32_t *map, int group) {
    const int at = (group + 1) * N;
    return map[at >> 5] >> (at & 31);
}

template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ void sum_row(const LossArgs &a, const Row<TYPE> &r, const uint32_t *map,
                                        Acc &c) {
    constexpr int N = Elem<TYPE>::N, U = 4;
    for (int v = r.v0 + (int) threadIdx.x; v < r.v1; v += U * THREADS) {
        u32x4 raw[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (v + j * THREADS < r.v1)
                raw[j] = r.load(v + j * THREADS);
        float y[U * N];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int w = v + j * THREADS;
            float     z[N];
            if (w < r.v1) {
                Elem<TYPE>::unpack(raw[j], z);
                group_values<TYPE, FEAT>(a, r, w, z);
                if ((FEAT & F_GENERAL) && map) {
                    const uint32_t listed = listed_bits<N>(map, w - r.v0);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        z[i] = ((listed >> i) & 1u) ? -INFINITY : z[i];
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
                y[j * N + i] = w < r.v1 ? z[i] : -INFINITY;
        }
        acc_batch<U * N, FEAT>(c, y, a.k, a.slack);
    }
    if (threadIdx.x < 2 * N) {
        const int e = r.loose((int) threadIdx.x);
        if (e >= 0) {
            float     y  = one_value<TYPE, FEAT>(a, r, e, Elem<TYPE>::one(r.x[e]));
            const int at = e - r.elem0() + N;
            if ((FEAT & F_GENERAL) && map && ((map[at >> 5] >> (at & 31)) & 1u))
                y = -INFINITY;
            const float one[1] = {y};
            acc_batch<1, FEAT>(c, one, a.k, a.slack);
        }
    }
}

struct Sums {
    float  m;
    double s, t;
    float  m_listed; /* the largest listed y */
    double listed;   /* with a tail: the listed tokens' own sum against it */
};
/* the threads' sums, joined against the largest reference among them */
template <int FEAT, int THREADS>
__device__ __forceinline__ Sums join_threads(const Acc &c, float k, double *slot) {
    Sums j;
    j.m             = block_max<THREADS>(c.m, slot);
    const float  d  = fmaxf((c.m - j.m) * k, -1e30f);
    const float  d2 = c.m == j.m ? 0.0f : d; /* (+inf against itself: the sum is NaN already) */
    const double sc = (double) __builtin_amdgcn_exp2f(d2);
    j.s             = block_sum<THREADS>(sc * c.s, slot);
    j.t             = 0.0;
    if (FEAT & F_ENTROPY)
        j.t = block_sum<THREADS>(sc * (c.t + c.s * (double) d2), slot);
    j.m_listed = -FLT_MAX;
    j.listed   = 0.0;
    return j;
}
/* the parts of a row, joined by every wavefront for itself */
template <int FEAT> __device__ __forceinline__ Sums join_parts(const LossPart *p, int chunks, float k) {
    const int lane = threadIdx.x & 63;
    Sums      j;
    j.m = -FLT_MAX;
    for (int i = lane; i < chunks; i += 64)
        j.m = fmaxf(j.m, p[i].m);
    j.m = wave_max(j.m);
    double s = 0.0, t = 0.0;
    for (int i = lane; i < chunks; i += 64) {
        const float  d  = p[i].m == j.m ? 0.0f : fmaxf((p[i].m - j.m) * k, -1e30f);
        const double sc = (double) __builtin_amdgcn_exp2f(d);
        s += sc * p[i].s;
        if (FEAT & F_ENTROPY)
            t += sc * (p[i].t + p[i].s * (double) d);
    }
    j.s        = wave_sum(s);
    j.t        = (FEAT & F_ENTROPY) ? wave_sum(t) : 0.0;
    j.m_listed = p[0].m_listed;
    j.listed   = p[0].listed;
    return j;
}

/* ---- the gradient --------------------------------------------------------------------------- */
struct Coef {
    float a;        /* p_i (a + b u_i) ..., 1 / S and 1 / T are in them */
    float a_listed; /* ... of listed tokens */
    float b;
    float q;        /* ... - q_i q */
    float m_listed; /* the reference a_listed stands against */
    bool  zero;     /* the row is written as zeros */
};
template <int FEAT> __device__ __forceinline__ float grad_one(const Coef &c, float y, float m, float k) {
    const float u = (y - m) * k;
    const float e = __builtin_amdgcn_exp2f(u);
    if (FEAT & F_ENTROPY)
        return e * fmaf(c.b, fmaxf(u, -1e30f), c.a);
    return e * c.a;
}
template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ void write_row(const LossArgs &a, const Row<TYPE> &r, const Coef &c, float m) {
    constexpr int N = Elem<TYPE>::N, U = 4;
    for (int v = r.v0 + (int) threadIdx.x; v < r.v1; v += U * THREADS) {
        u32x4 raw[U];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (v + j * THREADS < r.v1)
                raw[j] = c.zero ? u32x4{0, 0, 0, 0} : r.load(v + j * THREADS);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int w = v + j * THREADS;
            if (w < r.v1) {
                float y[N], g[N];
                Elem<TYPE>::unpack(raw[j], y);
                float x[N];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    x[i] = y[i];
                group_values<TYPE, FEAT>(a, r, w, y);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    g[i] = grad_one<FEAT>(c, y[i], m, a.k);
                    if ((FEAT & F_GENERAL) && y[i] == -INFINITY)
                        g[i] = 0.0f; /* (a forbidden NaN has no slope either) */
                    else if ((FEAT & F_GENERAL) && a.cap > 0.0f)
                        g[i] *= capped_slope(x[i], a.tanh_k);
                    if (c.zero)
                        g[i] = 0.0f;
                }
                r.store(w, Elem<TYPE>::pack(g));
            }
        }
    }
    if (threadIdx.x < 2 * N) {
        const int e = r.loose((int) threadIdx.x);
        if (e >= 0) {
            const float x = Elem<TYPE>::one(r.x[e]);
            const float y = one_value<TYPE, FEAT>(a, r, e, x);
            float       g = grad_one<FEAT>(c, y, m, a.k);
            if ((FEAT & F_GENERAL) && y == -INFINITY)
                g = 0.0f;
            else if ((FEAT & F_GENERAL) && a.cap > 0.0f)
                g *= capped_slope(x, a.tanh_k);
            r.g[e] = Elem<TYPE>::round(c.zero ? 0.0f : g);
        }
    }
}

/* ---- one token per row ---------------------------------------------------------------------- */
struct Token {
    int   id; /* -1: none */
    float x, y;
};
template <int TYPE, int FEAT>
__device__ __forceinline__ Token load_token(const LossArgs &a, const Row<TYPE> &r, int row) {
    Token t;
    t.id = a.tokens[row];
    t.x = t.y = 0.0f;
    if (t.id < 0 || t.id >= r.n) {
        t.id = -1;
    } else {
        t.x = Elem<TYPE>::one(r.x[t.id]);
        t.y = one_value<TYPE, FEAT>(a, r, t.id, t.x);
    }
    return t;
}
/* log p of the token; -inf where the row gives it nothing or has no distribution */
__device__ __forceinline__ double token_logprob(const Sums &j, double y, float k) {
    if (j.s == 0.0)
        return -INFINITY;
    return ((y - (double) j.m) * (double) k - log2(j.s)) * LN2;
}

/* Policy loss of a row from its sums; `lead`: this thread writes the row's outputs. */
__device__ __forceinline__ Coef policy_coef(const LossArgs &a, int row, bool has_token, double y,
                                            const Sums &j, bool entropy, bool lead) {
    const bool   empty = j.s == 0.0;
    const double lp    = has_token ? token_logprob(j, y, a.k) : 0.0;
    const double l2s   = empty ? 0.0 : log2(j.s);
    const double H     = entropy && !empty ? LN2 * (l2s - j.t / j.s) : 0.0;
    const double w     = a.weight ? (double) a.weight[row] : 1.0;
    Coef         c     = {0.0f, 0.0f, 0.0f, 0.0f, j.m, true};
    double       loss  = 0.0;
    if (w != 0.0 && has_token && lp != -INFINITY) {
        const double A  = (double) a.advantage[row];
        double       d  = 0.0;
        const double ratio = a.old_lp ? exp(lp - (double) a.old_lp[row]) : 1.0;
        if (A != 0.0) {
            const double lo = 1.0 - (double) a.clip_low, hi = 1.0 + (double) a.clip_high;
            const double held = ratio < lo ? lo : ratio > hi ? hi : ratio; /* NaN stays */
            const double f = ratio * A, h = held * A;
            loss = h < f ? -h : -f;
            d    = h < f ? 0.0 : -f;
        }
        if (a.ref_lp) {
            const double far = (double) a.ref_lp[row] - lp;
            const double ex  = expm1(far);
            loss += (double) a.kl_coef * (ex - far);
            d -= (double) a.kl_coef * ex;
        }
        const double ec = (double) a.entropy_coef;
        if (ec != 0.0)
            loss -= ec * H;
        loss *= w;
        d *= w * a.inv_t;
        const double be = w * ec * a.inv_t;
        c.a = (float) ((be != 0.0 ? be * (H - l2s * LN2) - d : -d) / j.s);
        c.b = (float) (be * LN2 / j.s);
        c.a_listed = c.a;
        c.q    = (float) -d;
        c.zero = false;
    }
    if (lead) {
        if (a.loss)
            a.loss[row] = (float) loss;
        if (a.logprob)
            a.logprob[row] = (float) lp;
        if (a.entropy)
            a.entropy[row] = (float) H;
    }
    return c;
}
/* the token's own element, over what write_row left there */
template <int TYPE, int FEAT>
__device__ __forceinline__ void write_token(const LossArgs &a, const Row<TYPE> &r, const Token &t,
                                            const Coef &c, float m) {
    float g = grad_one<FEAT>(c, t.y, m, a.k) - c.q;
    if ((FEAT & F_GENERAL) && a.cap > 0.0f)
        g *= capped_slope(t.x, a.tanh_k);
    r.g[t.id] = Elem<TYPE>::round(g);
}
/* whether element e is in the workgroup's part of the row */
template <int TYPE> __device__ __forceinline__ bool mine(const Row<TYPE> &r, int e) {
    const int lo = r.first ? 0 : r.elem0();
    const int hi = r.last ? r.n : r.head + r.v1 * Elem<TYPE>::N;
    return e >= lo && e < hi;
}

/* ---- a teacher's list ----------------------------------------------------------------------- */
/* In LDS: ids (-1: left out), x and q of the entries; keys and owners find repeated ids; the bit map. */
struct List {
    int      *ids, *keys, *owner;
    float    *x, *q;
    uint32_t *map;
    double    q_log_q, q_sum; /* sum q_j log q_j, sum q_j */
    float     y_top;          /* max y_j */
    double    q_y;            /* sum q_j (y_j - y_top) */
    int       n;              /* entries that count */
};
__host__ __device__ __forceinline__ size_t list_lds(int k, int slots) {
    return (size_t) k * 12 + (size_t) slots * 8;
}
template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ List load_list(const LossArgs &a, const Row<TYPE> &r, int row, void *lds,
                                          double *slot, bool want_map) {
    List l;
    l.ids   = static_cast<int *>(lds);
    l.x     = reinterpret_cast<float *>(l.ids + a.list_k);
    l.q     = l.x + a.list_k;
    l.keys  = reinterpret_cast<int *>(l.q + a.list_k);
    l.owner = l.keys + a.slots;
    l.map   = reinterpret_cast<uint32_t *>(l.owner + a.slots);
    constexpr int N = Elem<TYPE>::N;
    int           k = a.list_k;
    if (a.count)
        k = max(0, min(k, a.count[row]));
    for (int i = threadIdx.x; i < a.slots; i += THREADS) {
        l.keys[i]  = -1;
        l.owner[i] = 0x7fffffff;
    }
    const int span  = (r.last ? r.n : r.head + r.v1 * N) - r.elem0() + N; /* bits of the map */
    const int words = want_map ? (span + 31) / 32 : 0;
    for (int i = threadIdx.x; i < words; i += THREADS)
        l.map[i] = 0u;
    __syncthreads();
    /* the table of ids keeps for each the first place that lists it */
    for (int j = threadIdx.x; j < k; j += THREADS) {
        const int   id = a.ids[(long) row * a.list_ld + j];
        const float v  = a.values[(long) row * a.list_ld + j];
        const bool  ok = id >= 0 && id < r.n && v != -INFINITY && r.may(id);
        l.ids[j]       = ok ? id : -1;
        l.q[j]         = v;
        if (ok) {
            uint32_t at = ((uint32_t) id * 2654435761u) & (uint32_t) (a.slots - 1);
            for (;;) { /* ends: there are twice as many places as entries */
                const int was = atomicCAS(&l.keys[at], -1, id);
                if (was == -1 || was == id)
                    break;
                at = (at + 1) & (uint32_t) (a.slots - 1);
            }
            atomicMin(&l.owner[at], j);
        }
    }
    __syncthreads();
    float top = -INFINITY;
    for (int j = threadIdx.x; j < k; j += THREADS) {
        const int id = l.ids[j];
        if (id < 0)
            continue;
        uint32_t at = ((uint32_t) id * 2654435761u) & (uint32_t) (a.slots - 1);
        while (l.keys[at] != id)
            at = (at + 1) & (uint32_t) (a.slots - 1);
        if (l.owner[at] != j) {
            l.ids[j] = -1;
            continue;
        }
        top    = fmaxf(top, l.q[j]);
        l.x[j] = Elem<TYPE>::one(r.x[id]);
        if (want_map && mine(r, id)) {
            const int bit = id - r.elem0() + N;
            atomicOr(&l.map[bit >> 5], 1u << (bit & 31));
        }
    }
    double scale = 1.0, log_sum = 0.0;
    if (!a.tail) {
        top        = block_max<THREADS>(top, slot);
        double sum = 0.0;
        for (int j = threadIdx.x; j < k; j += THREADS)
            if (l.ids[j] >= 0)
                sum += exp(((double) l.q[j] - (double) top) * a.inv_t);
        sum     = block_sum<THREADS>(sum, slot);
        log_sum = log(sum);
        scale   = 1.0 / sum;
    } else {
        top = 0.0f;
    }
    float y_top = -FLT_MAX;
    for (int j = threadIdx.x; j < k; j += THREADS)
        if (l.ids[j] >= 0)
            y_top = fmaxf(y_top, one_value<TYPE, FEAT>(a, r, l.ids[j], l.x[j]));
    l.y_top   = block_max<THREADS>(y_top, slot);
    double ql = 0.0, qs = 0.0, qy = 0.0;
    for (int j = threadIdx.x; j < k; j += THREADS)
        if (l.ids[j] >= 0) {
            const double v = a.tail ? (double) l.q[j] : ((double) l.q[j] - (double) top) * a.inv_t;
            const double q = exp(v) * scale;
            const float  y = one_value<TYPE, FEAT>(a, r, l.ids[j], l.x[j]);
            if (q != 0.0) {
                ql += q * (v - log_sum);
                qy += q * ((double) y - (double) l.y_top);
            }
            qs += q;
            l.q[j] = (float) q;
        }
    l.q_log_q = block_sum<THREADS>(ql, slot);
    l.q_sum   = block_sum<THREADS>(qs, slot);
    l.q_y     = block_sum<THREADS>(qy, slot);
    l.n       = k;
    __syncthreads();
    return l;
}
/* sum of 2^((y - y_top) k) of the listed tokens: apart from the others', so that neither mass is lost
 * beside the other however far the two lie apart */
template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ double listed_sum(const LossArgs &a, const Row<TYPE> &r, const List &l,
                                             double *slot) {
    double s = 0.0;
    for (int j = threadIdx.x; j < l.n; j += THREADS)
        if (l.ids[j] >= 0)
            s += (double) __builtin_amdgcn_exp2f(
                (one_value<TYPE, FEAT>(a, r, l.ids[j], l.x[j]) - l.y_top) * a.k);
    return block_sum<THREADS>(s, slot);
}
/* q_y and j.m_listed (sum of q_j (y_j - y_top) and y_top) are handed in: the rows may have been
 * replaced by their gradient since */
__device__ __forceinline__ Coef distill_coef(const LossArgs &a, int row, const List &l, double q_y,
                                             const Sums &j, bool lead) {
    const double w   = a.weight ? (double) a.weight[row] : 1.0;
    const double k   = (double) a.k;
    const float  top = a.tail ? fmaxf(j.m, j.m_listed) : j.m;
    /* everything against one reference: the listed tokens' sum and that of the rest */
    const double below = j.s == 0.0 ? 0.0 : ((double) j.m - (double) top) * k;
    double       rest = j.s, all = j.s;
    if (a.tail) {
        rest = j.m == top ? j.s : j.s * exp2(below);
        all  = rest + (j.m_listed == top ? j.listed
                                         : j.listed * exp2(((double) j.m_listed - (double) top) * k));
    }
    Coef   c    = {0.0f, 0.0f, 0.0f, 0.0f, top, true};
    double loss = 0.0;
    if (w != 0.0 && all != 0.0 && (a.tail || l.q_sum != 0.0)) {
        const double l2s = log2(all);
        /* sum q_j (log q_j - log p_j) */
        loss = l.q_log_q + LN2 * (l.q_sum * (l2s + ((double) top - (double) j.m_listed) * k) - q_y * k);
        const double ws = w * a.inv_t;
        c.a_listed      = (float) (ws / all);
        c.a             = c.a_listed;
        if (a.tail) {
            /* p_i (1 - q_rest / p_rest) = 2^((y_i - m) k) / s * (p_rest - q_rest) */
            const double q_rest = l.q_sum <= 1.0 ? 1.0 - l.q_sum : l.q_sum > 1.0 ? 0.0 : l.q_sum;
            if (q_rest != 0.0)
                loss += q_rest * (log(q_rest) -
                                  (j.s == 0.0 ? -INFINITY : LN2 * (log2(j.s) + below - l2s)));
            c.a = j.s == 0.0 ? 0.0f : (float) (ws * (rest / all - q_rest) / j.s);
        }
        loss *= w;
        c.q    = (float) ws;
        c.zero = false;
    }
    if (lead && a.loss)
        a.loss[row] = (float) loss;
    return c;
}
template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ void write_listed(const LossArgs &a, const Row<TYPE> &r, const List &l,
                                             const Coef &c) {
    for (int j = threadIdx.x; j < l.n; j += THREADS)
        if (l.ids[j] >= 0 && mine(r, l.ids[j])) {
            const float y = one_value<TYPE, FEAT>(a, r, l.ids[j], l.x[j]);
            float       g = __builtin_amdgcn_exp2f((y - c.m_listed) * a.k) * c.a_listed - l.q[j] * c.q;
            if ((FEAT & F_GENERAL) && a.cap > 0.0f)
                g *= capped_slope(l.x[j], a.tanh_k);
            r.g[l.ids[j]] = Elem<TYPE>::round(g);
        }
}

/* ---- kernels -------------------------------------------------------------------------------- */
/* A row per workgroup: sums, scalars, gradient. */
template <int TYPE, int OP, int FEAT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_loss_row(LossArgs a) {
    __shared__ double slot[16];
    extern __shared__ __align__(16) char lds[];
    const int       row = blockIdx.x;
    const Row<TYPE> r(a, row, 0);
    Acc             acc;
    if constexpr (OP == OP_DISTILL) {
        const bool tail = (FEAT & F_GENERAL) && a.tail;
        const List l    = load_list<TYPE, FEAT, THREADS>(a, r, row, lds, slot, tail);
        sum_row<TYPE, FEAT, THREADS>(a, r, tail ? l.map : nullptr, acc);
        Sums j = join_threads<FEAT, THREADS>(acc, a.k, slot);
        j.m_listed = l.y_top;
        if (tail)
            j.listed = listed_sum<TYPE, FEAT, THREADS>(a, r, l, slot);
        const Coef c = distill_coef(a, row, l, l.q_y, j, threadIdx.x == 0);
        if (r.g) {
            write_row<TYPE, FEAT, THREADS>(a, r, c, j.m);
            __syncthreads();
            if (!c.zero)
                write_listed<TYPE, FEAT, THREADS>(a, r, l, c);
        }
    } else {
        const Token t = load_token<TYPE, FEAT>(a, r, row);
        sum_row<TYPE, FEAT, THREADS>(a, r, nullptr, acc);
        const Sums j = join_threads<FEAT, THREADS>(acc, a.k, slot);
        const Coef c = policy_coef(a, row, t.id >= 0, (double) t.y, j, FEAT & F_ENTROPY,
                                   threadIdx.x == 0);
        if (r.g) {
            write_row<TYPE, FEAT, THREADS>(a, r, c, j.m);
            __syncthreads();
            if (!c.zero && threadIdx.x == 0)
                write_token<TYPE, FEAT>(a, r, t, c, j.m);
        }
    }
}

/* The sums of a part of a row. */
template <int TYPE, int OP, int FEAT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_loss_sums(LossArgs a) {
    __shared__ double slot[16];
    extern __shared__ __align__(16) char lds[];
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    if constexpr (OP == OP_PREFERENCE) {
        if (row < a.seq_start[0] || row >= a.seq_start[2 * a.n_pairs])
            return;
    }
    const Row<TYPE> r(a, row, chunk);
    Acc             acc;
    Sums            j;
    double          at = 0.0;
    if constexpr (OP == OP_DISTILL) {
        const bool tail = (FEAT & F_GENERAL) && a.tail;
        List       l    = {};
        if (tail || chunk == 0) {
            l  = load_list<TYPE, FEAT, THREADS>(a, r, row, lds, slot, tail);
            at = l.q_y;
        }
        sum_row<TYPE, FEAT, THREADS>(a, r, tail ? l.map : nullptr, acc);
        j = join_threads<FEAT, THREADS>(acc, a.k, slot);
        if (chunk == 0) {
            j.m_listed = l.y_top;
            if (tail)
                j.listed = listed_sum<TYPE, FEAT, THREADS>(a, r, l, slot);
        }
    } else {
        const Token t = load_token<TYPE, FEAT>(a, r, row);
        at            = (double) t.y;
        sum_row<TYPE, FEAT, THREADS>(a, r, nullptr, acc);
        j = join_threads<FEAT, THREADS>(acc, a.k, slot);
        if (OP == OP_PREFERENCE && chunk == 0 && threadIdx.x == 0 && a.coef)
            a.coef[row] = 0.0f;
    }
    if (threadIdx.x == 0)
        a.part[(long) row * a.chunks + chunk] = {j.s, j.t, at, j.listed, j.m_listed, j.m};
}

/* The gradient of a part of a row from the parts' sums; without one, a workgroup per row writes the
 * row's outputs. */
template <int TYPE, int OP, int FEAT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_loss_grad(LossArgs a, int chunks, int chunk_vecs) {
    __shared__ double slot[16];
    extern __shared__ __align__(16) char lds[];
    const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
    if constexpr (OP == OP_PREFERENCE) {
        if (row < a.seq_start[0] || row >= a.seq_start[2 * a.n_pairs])
            return;
    }
    const LossPart *p  = a.part + (long) row * a.chunks;
    const Sums      j  = join_parts<FEAT>(p, a.chunks, a.k);
    const double    at = p[0].a;
    a.chunks           = chunks;
    a.chunk_vecs       = chunk_vecs;
    const Row<TYPE> r(a, row, chunk);
    const bool      lead = chunk == 0 && threadIdx.x == 0;
    if constexpr (OP == OP_DISTILL) {
        const List l = load_list<TYPE, FEAT, THREADS>(a, r, row, lds, slot, false);
        const Coef c = distill_coef(a, row, l, at, j, lead);
        if (r.g) {
            write_row<TYPE, FEAT, THREADS>(a, r, c, j.m);
            __syncthreads();
            if (!c.zero)
                write_listed<TYPE, FEAT, THREADS>(a, r, l, c);
        }
    } else {
        const int id        = a.tokens[row];
        const bool has_token = id >= 0 && id < a.n;
        Token     t         = {-1, 0.0f, 0.0f};
        Coef      c;
        if (has_token && r.g && mine(r, id))
            t = load_token<TYPE, FEAT>(a, r, row);
        if constexpr (OP == OP_PREFERENCE) {
            const double d = (double) a.coef[row] * a.inv_t;
            c.a = c.a_listed = (float) (-d / j.s);
            c.b    = 0.0f;
            c.m_listed = j.m;
            c.q    = (float) -d;
            c.zero = d == 0.0;
        } else {
            c = policy_coef(a, row, has_token, at, j, FEAT & F_ENTROPY, lead);
        }
        if (r.g) {
            write_row<TYPE, FEAT, THREADS>(a, r, c, j.m);
            __syncthreads();
            if (!c.zero && threadIdx.x == 0 && t.id >= 0)
                write_token<TYPE, FEAT>(a, r, t, c, j.m);
        }
    }
}

/* The pairs: log-probabilities of their rows, ratios, loss, and what each row's log-probability is
 * worth. */
constexpr int PAIR_THREADS = 1024;
__global__ __launch_bounds__(PAIR_THREADS) void k_pair(LossArgs a) {
    __shared__ double slot[16];
    const int         pair = blockIdx.x;
    double            ratio[2], share[2];
    int               lo[2], hi[2];
    /* the rows that were summed: nothing outside them is looked at, whatever the starts between say */
    const int first = max(0, min(a.rows, a.seq_start[0]));
    const int last  = max(first, min(a.rows, a.seq_start[2 * a.n_pairs]));
    for (int side = 0; side < 2; ++side) {
        lo[side] = max(first, min(last, a.seq_start[2 * pair + side]));
        hi[side] = max(lo[side], min(last, a.seq_start[2 * pair + side + 1]));
        double sum = 0.0, n = 0.0;
        for (int row = lo[side] + (int) threadIdx.x; row < hi[side]; row += PAIR_THREADS) {
            const LossPart *p  = a.part + (long) row * a.chunks;
            const int       id = a.tokens[row];
            double          lp = 0.0;
            if (id >= 0 && id < a.n) {
                Sums j = {-FLT_MAX, 0.0, 0.0, -FLT_MAX, 0.0};
                for (int i = 0; i < a.chunks; ++i)
                    j.m = fmaxf(j.m, p[i].m);
                for (int i = 0; i < a.chunks; ++i)
                    j.s += p[i].s * (double) __builtin_amdgcn_exp2f(
                                        p[i].m == j.m ? 0.0f : fmaxf((p[i].m - j.m) * a.k, -1e30f));
                lp = token_logprob(j, p[0].a, a.k);
                if (lp != -INFINITY) {
                    sum += a.ref_lp ? lp - (double) a.ref_lp[row] : lp;
                    n += 1.0;
                }
            }
            if (a.logprob)
                a.logprob[row] = (float) lp;
            if (a.coef) /* marks the rows that count */
                a.coef[row] = (id >= 0 && id < a.n && lp != -INFINITY) ? 1.0f : 0.0f;
        }
        sum         = block_sum<PAIR_THREADS>(sum, slot);
        n           = block_sum<PAIR_THREADS>(n, slot);
        share[side] = a.length_normalised ? 1.0 / fmax(n, 1.0) : 1.0;
        ratio[side] = sum * share[side];
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
    if (a.coef)
        for (int side = 0; side < 2; ++side) {
            const float c = (float) ((side ? -d : d) * w * share[side]);
            for (int row = lo[side] + (int) threadIdx.x; row < hi[side]; row += PAIR_THREADS)
                a.coef[row] = a.coef[row] != 0.0f ? c : 0.0f;
        }
}

/* ---- launches ------------------------------------------------------------------------------- */
constexpr int ROW_THREADS  = 512;
constexpr int PART_THREADS = 256;

LossArgs args_of(const geist_hip_loss_rows &r) {
    LossArgs a   = {};
    a.x          = r.d_logits;
    a.g          = r.d_grad;
    a.ld         = (long) r.ld;
    a.gld        = (long) r.grad_ld;
    a.n          = (int) r.n_vocab;
    a.rows       = (int) r.rows;
    a.allowed    = r.d_allowed;
    a.allowed_ld = (long) r.allowed_ld;
    a.k          = (float) (LOG2E / (double) r.temperature);
    a.slack      = 20.0f / a.k;
    a.cap        = r.logit_softcap;
    a.tanh_k     = r.logit_softcap > 0.0f ? (float) (2.0 * LOG2E / (double) r.logit_softcap) : 0.0f;
    a.inv_t      = 1.0 / (double) r.temperature;
    return a;
}

enum Stage { STAGE_ROW, STAGE_SUMS, STAGE_GRAD };

template <int TYPE, int OP, int FEAT>
void launch_stage(Stage stage, LossArgs a, size_t lds, int chunks, int chunk_vecs, hipStream_t stream) {
    if (stage == STAGE_ROW) {
        if constexpr (OP != OP_PREFERENCE)
            k_loss_row<TYPE, OP, FEAT, ROW_THREADS><<<dim3(a.rows), ROW_THREADS, lds, stream>>>(a);
    } else if (stage == STAGE_SUMS) {
        k_loss_sums<TYPE, OP, FEAT, PART_THREADS>
            <<<dim3((unsigned) a.rows * a.chunks), PART_THREADS, lds, stream>>>(a);
    } else {
        k_loss_grad<TYPE, OP, FEAT, PART_THREADS>
            <<<dim3((unsigned) a.rows * chunks), PART_THREADS, lds, stream>>>(a, chunks, chunk_vecs);
    }
}
template <int OP, int FEAT>
void launch_typed(int type, Stage stage, const LossArgs &a, size_t lds, int chunks, int chunk_vecs,
                  hipStream_t stream) {
    if (type == GEIST_HIP_TYPE_F32)
        launch_stage<GEIST_HIP_TYPE_F32, OP, FEAT>(stage, a, lds, chunks, chunk_vecs, stream);
    else if (type == GEIST_HIP_TYPE_F16)
        launch_stage<GEIST_HIP_TYPE_F16, OP, FEAT>(stage, a, lds, chunks, chunk_vecs, stream);
    else
        launch_stage<GEIST_HIP_TYPE_BF16, OP, FEAT>(stage, a, lds, chunks, chunk_vecs, stream);
}

int elem_bytes(int type) { return type == GEIST_HIP_TYPE_F32 ? 4 : 2; }
bool general(const LossArgs &a) { return a.cap > 0.0f || a.allowed || a.tail; }

} // namespace

void launch_policy(const geist_hip_loss_rows &r, const geist_hip_policy &p, float *loss,
                   float *logprob, float *entropy, void *ws, hipStream_t stream) {
    LossArgs       a    = args_of(r);
    const LossPlan plan = loss_plan(r.rows, r.n_vocab, elem_bytes(r.type));
    a.chunks       = plan.chunks;
    a.chunk_vecs   = plan.chunk_vecs;
    a.part         = static_cast<LossPart *>(ws);
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
    auto       go  = [&](Stage s) {
        const int c = r.d_grad ? a.chunks : 1, v = r.d_grad ? a.chunk_vecs : INT32_MAX / 64;
        if (ent && general(a))
            launch_typed<OP_TOKEN, F_ENTROPY | F_GENERAL>(r.type, s, a, 0, c, v, stream);
        else if (ent)
            launch_typed<OP_TOKEN, F_ENTROPY>(r.type, s, a, 0, c, v, stream);
        else if (general(a))
            launch_typed<OP_TOKEN, F_GENERAL>(r.type, s, a, 0, c, v, stream);
        else
            launch_typed<OP_TOKEN, 0>(r.type, s, a, 0, c, v, stream);
    };
    if (a.chunks == 1) {
        go(STAGE_ROW);
    } else {
        go(STAGE_SUMS);
        go(STAGE_GRAD);
    }
}

void launch_distill(const geist_hip_loss_rows &r, const geist_hip_teacher &t, float *loss, void *ws,
                    hipStream_t stream) {
    LossArgs       a    = args_of(r);
    const LossPlan plan = loss_plan(r.rows, r.n_vocab, elem_bytes(r.type));
    a.chunks     = plan.chunks;
    a.chunk_vecs = plan.chunk_vecs;
    a.part       = static_cast<LossPart *>(ws);
    a.ids        = t.d_ids;
    a.values     = t.d_values;
    a.count      = t.d_count;
    a.list_ld    = (long) t.ld;
    a.list_k     = (int) t.k;
    a.slots      = 2;
    while (a.slots < 2 * a.list_k)
        a.slots *= 2;
    a.tail   = t.tail;
    a.weight = t.d_weight;
    a.loss   = loss;
    const size_t list = list_lds(a.list_k, a.slots);
    /* (the map: the part's logits, up to 16 bytes of head, tail and alignment) */
    const size_t part_n = a.chunks == 1 ? r.n_vocab : (size_t) a.chunk_vecs * (16 / elem_bytes(r.type));
    const size_t map    = t.tail ? (part_n + 64) / 32 * 4 + 4 : 0;
    auto         go     = [&](Stage s) {
        const size_t lds = list + (s == STAGE_GRAD ? 0 : map);
        const int    c = r.d_grad ? a.chunks : 1, v = r.d_grad ? a.chunk_vecs : INT32_MAX / 64;
        if (general(a))
            launch_typed<OP_DISTILL, F_GENERAL>(r.type, s, a, lds, c, v, stream);
        else
            launch_typed<OP_DISTILL, 0>(r.type, s, a, lds, c, v, stream);
    };
    if (a.chunks == 1) {
        go(STAGE_ROW);
    } else {
        go(STAGE_SUMS);
        go(STAGE_GRAD);
    }
}

void launch_preference(const geist_hip_loss_rows &r, const geist_hip_preference &p, float *loss,
                       float *ratios, float *logprob, void *ws, hipStream_t stream) {
    LossArgs       a    = args_of(r);
    const LossPlan plan = loss_plan(r.rows, r.n_vocab, elem_bytes(r.type));
    a.chunks            = plan.chunks;
    a.chunk_vecs        = plan.chunk_vecs;
    a.part              = static_cast<LossPart *>(ws);
    a.coef      = r.d_grad ? reinterpret_cast<float *>(a.part + r.rows * (size_t) plan.chunks) : nullptr;
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
    auto go = [&](Stage s) {
        if (general(a))
            launch_typed<OP_PREFERENCE, F_GENERAL>(r.type, s, a, 0, a.chunks, a.chunk_vecs, stream);
        else
            launch_typed<OP_PREFERENCE, 0>(r.type, s, a, 0, a.chunks, a.chunk_vecs, stream);
    };
    go(STAGE_SUMS);
    k_pair<<<dim3((unsigned) p.n_pairs), PAIR_THREADS, 0, stream>>>(a);
    if (r.d_grad)
        go(STAGE_GRAD);
}

} // namespace gs
