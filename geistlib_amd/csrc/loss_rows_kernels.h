/*
 * loss_rows_kernels.h -- the kernels of the losses over logit rows (include/geist_loss_hip.h), as
 * templates that loss_rows_f32.hip, loss_rows_f16.hip and loss_rows_bf16.hip instantiate.
 *
 * Every loss here needs of a row x the sum S = sum 2^(w_i - c) with w = softcap(x) k, k = log2(e) / T,
 * against some reference c near the largest w (and, for the entropy, sum 2^u u with u = w - c), the
 * values at a few listed tokens, and its gradient by the logits has one form:
 *     g_i = (p_i (A + B u_i) - [i listed] q_i W) * softcap'(x_i) / T,     p_i = 2^u_i / S
 * with A, B, W of the row (A differs between listed and other tokens for a teacher with a tail).
 * So one streaming core serves all three: a pass that sums, a few scalars, a pass that writes.
 *
 *   k_loss_row   a workgroup per row does all of it; where there is a gradient, what fits the registers
 *                of the row stays there between the passes and is read once
 *   k_loss_sums  the sums of a part of a row (few rows; preference loss)
 *   k_loss_grad  the gradient of a part of a row from the parts' sums
 *
 * A row's scalars (logarithms and exponentials in binary64) and its teacher's list are the first
 * wavefront's work alone: sixteen wavefronts that all form them cost the row 5 us of its 29.
 */
#ifndef GEIST_LOSS_ROWS_KERNELS_H
#define GEIST_LOSS_ROWS_KERNELS_H

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "loss_kernels.h"
#include "sampler_device.h"

namespace gs {
namespace {

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

/* ---- the workgroup -------------------------------------------------------------------------- */
/* LDS writes of the own wavefront before, LDS reads behind it */
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}
__device__ __forceinline__ float wave_max(float v) {
#define GS_STEP(ctrl, rows)                                                                        \
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), \
                                                            ctrl, rows, 0xf, false)));
    GS_STEP(0x111, 0xf) GS_STEP(0x112, 0xf) GS_STEP(0x114, 0xf) GS_STEP(0x118, 0xf)
    GS_STEP(0x142, 0xa) GS_STEP(0x143, 0xc)
#undef GS_STEP
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1)
        v = fmax(v, __shfl_xor(v, d));
    return v;
}
/* over the workgroup, every thread gets the results; rare paths only */
template <int THREADS, bool MAX> __device__ __forceinline__ double block_reduce(double v, double *slot) {
    v = MAX ? wave_max(v) : wave_sum_f64(v);
    lds_barrier();
    if ((threadIdx.x & 63) == 0)
        slot[threadIdx.x >> 6] = v;
    lds_barrier();
    v = slot[0];
    for (int w = 1; w < THREADS / 64; ++w)
        v = MAX ? fmax(v, slot[w]) : v + slot[w];
    return v;
}

/* ---- a row ---------------------------------------------------------------------------------- */
template <int TYPE> struct Row {
    typedef typename Elem<TYPE>::mem mem;
    static constexpr int             N = Elem<TYPE>::N;
    const mem      *x;
    mem            *g;
    const uint32_t *allowed;
    int             n, head, nvec; /* elements in front of the first 16-byte boundary, groups behind it */
    int             v0, v1;        /* this workgroup's groups */
    bool            first, last;   /* it also takes the head / what is behind the last group */

    __device__ Row(const LossArgs &a, int row, int chunk, int chunks, int chunk_vecs) {
        x       = static_cast<const mem *>(a.x) + (long) row * a.ld;
        g       = a.g ? static_cast<mem *>(a.g) + (long) row * a.gld : nullptr;
        allowed = a.allowed ? a.allowed + (long) row * a.allowed_ld : nullptr;
        n       = a.n;
        head    = (int) ((16u - ((uintptr_t) x & 15u)) & 15u) / (int) sizeof(mem);
        if (head > n)
            head = n;
        nvec      = (n - head) / N;
        v0        = min(nvec, chunk * chunk_vecs);
        v1        = chunk == chunks - 1 ? nvec : min(nvec, v0 + chunk_vecs);
        first     = chunk == 0;
        last      = chunk == chunks - 1;
    }
    __device__ __forceinline__ int   elem0() const { return head + v0 * N; } /* of group v0 */
    __device__ __forceinline__ u32x4 load(int v) const {
        return *reinterpret_cast<const u32x4 *>(x + head + (long) v * N);
    }
    /* for what is not read again and cannot have come from the cache */
    __device__ __forceinline__ u32x4 load_streamed(int v) const {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(x + head + (long) v * N));
    }
    /* to the place of lane 0 in `wave`, each lane's 16 bytes behind it */
    __device__ __forceinline__ void load_to_lds(int v, u32x4 *wave, bool streamed) const {
        typedef const __attribute__((address_space(1))) void *global_ptr;
        typedef __attribute__((address_space(3))) void       *lds_ptr;
        const global_ptr p = (global_ptr) (x + head + (long) v * N);
        const lds_ptr    l = (lds_ptr) wave;
        if (streamed)
            __builtin_amdgcn_global_load_lds(p, l, 16, 0, 2);
        else
            __builtin_amdgcn_global_load_lds(p, l, 16, 0, 0);
    }
    /* (the gradient's rows may start elsewhere within 16 bytes than the logits' do) */
    __device__ __forceinline__ void store(int v, u32x4 d, bool streamed) const {
        typedef u32x4 __attribute__((aligned(2))) loose_u32x4;
        loose_u32x4 *p = reinterpret_cast<loose_u32x4 *>(g + head + (long) v * N);
        if (streamed) {
            asm volatile("");
            __builtin_nontemporal_store(d, p);
            asm volatile("");
        } else {
            *p = d;
        }
    }
    __device__ __forceinline__ bool may(int e) const {
        return !allowed || ((allowed[e >> 5] >> (e & 31)) & 1u);
    }
    /* mask bits of the group that starts at element e: they lie in one byte or two */
    __device__ __forceinline__ uint32_t bits(int e) const {
        const uint8_t *p = reinterpret_cast<const uint8_t *>(allowed);
        return ((uint32_t) p[e >> 3] | (uint32_t) p[(e + N - 1) >> 3] << 8) >> (e & 7);
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
    /* whether element e is in the workgroup's part of the row */
    __device__ __forceinline__ bool mine(int e) const {
        const int lo = first ? 0 : elem0();
        const int hi = last ? n : head + v1 * N;
        return e >= lo && e < hi;
    }
};

/* ---- values --------------------------------------------------------------------------------- */
/* tanh(x / c) = 1 - 2 / (1 + E), E = 2^(2 x log2(e) / c): off by 1e-7 absolute, c 1e-7 in a capped
 * logit, which a 16-bit gradient does not show where c is what soft-caps are (up to 64). For f32 rows and
 * larger caps small arguments take the odd Taylor polynomial to z^13, relative error 2^-24 below 0.55. */
template <int TYPE, int FEAT> constexpr bool exact_cap = TYPE == GEIST_HIP_TYPE_F32 || (FEAT & F_WIDE) != 0;
__device__ __forceinline__ float cap_power(const LossArgs &a, float x) { /* E */
    return __builtin_amdgcn_exp2f(x * a.tanh_k);
}
__device__ __forceinline__ float cap_recip(const LossArgs &a, float x) { /* 1 / (1 + E) */
    return __builtin_amdgcn_rcpf(1.0f + cap_power(a, x));
}
/* E / (1 + E)^2; an E beyond binary32 gives 0 (its r is 0) */
__device__ __forceinline__ float cap_quarter(float E, float r) { return r * fminf(E * r, 1.0f); }
__device__ __forceinline__ float accurate_tanh(const LossArgs &a, float x, float r) {
    const float z = x * a.inv_cap, z2 = z * z;
    float       p = 21844.0f / 6081075.0f;
    p             = fmaf(p, z2, -1382.0f / 155925.0f);
    p             = fmaf(p, z2, 62.0f / 2835.0f);
    p             = fmaf(p, z2, -17.0f / 315.0f);
    p             = fmaf(p, z2, 2.0f / 15.0f);
    p             = fmaf(p, z2, -1.0f / 3.0f);
    p             = fmaf(p * z2, z, z);
    return fabsf(z) < 0.55f ? p : fmaf(-2.0f, r, 1.0f);
}
/* softcap(x) in binary32, as the degenerate rows' pass needs it */
template <int FEAT> __device__ __forceinline__ float capped(const LossArgs &a, float x) {
    return FEAT & F_CAP ? a.cap * accurate_tanh(a, x, cap_recip(a, x)) : x;
}
/* softcap(x) k in binary64, for the few values a row's scalars are made of */
template <int TYPE, int FEAT> __device__ __forceinline__ double value64(const LossArgs &a, float x) {
    if (FEAT & F_CAP) {
        if (exact_cap<TYPE, FEAT>)
            return (double) a.cap * (double) a.k * tanh((double) x / (double) a.cap);
        /* (by the rounded constants the 16-bit rows' sums are made with: their rounding cancels) */
        return (double) a.cap_k * tanh((double) x * (double) a.tanh_k * (0.5 * 0.693147180559945309417232));
    }
    return (double) x * (double) a.k;
}

__device__ __forceinline__ uint32_t bit_mask(uint32_t bits, int i) { /* all ones or none */
    return (uint32_t) __builtin_amdgcn_sbfe((int) bits, (unsigned) i, 1u);
}
/* Where the entropy multiplies by u, u stops here: 2^u is 0 in binary32 long before, and the product with a
 * coefficient of up to 10^35 (the weight is in it) is finite, so that 0 times it is 0. */
constexpr float U_LOW = -1024.0f;
/* A group's exponents u = w - c, and 2^u; `keep` (F_BITS): bits of the tokens that count. slope: a fourth of
 * the soft-cap's, (1 - tanh^2) / 4 = E / (1 + E)^2 (as a difference of tanh from 1 it would lose its digits
 * where it is small). */
template <int TYPE, int FEAT>
__device__ __forceinline__ void group_exps(const LossArgs &a, u32x4 raw, uint32_t keep, float c,
                                           float (&e)[Elem<TYPE>::N], float (&u)[Elem<TYPE>::N],
                                           float (&slope)[Elem<TYPE>::N]) {
    constexpr int N = Elem<TYPE>::N;
    float         x[N];
    Elem<TYPE>::unpack(raw, x);
    if (FEAT & F_CAP) {
        float r[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float E = cap_power(a, x[i]);
            r[i]          = __builtin_amdgcn_rcpf(1.0f + E);
            slope[i]      = cap_quarter(E, r[i]);
        }
        if (exact_cap<TYPE, FEAT>) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                u[i] = fmaf(a.cap * accurate_tanh(a, x[i], r[i]), a.k, -c);
        } else {
            const float at = a.cap_k - c;
#pragma unroll
            for (int i = 0; i < N; ++i)
                u[i] = fmaf(-2.0f * a.cap_k, r[i], at);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            u[i] = fmaf(x[i], a.k, -c);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        e[i] = __builtin_amdgcn_exp2f(u[i]);
    if (FEAT & F_BITS) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            e[i] = __uint_as_float(__float_as_uint(e[i]) & bit_mask(keep, i));
        }
    }
    if (FEAT & F_ENTROPY) { /* finite, whatever stands behind a mask: 0 * -inf is no term of an entropy */
#pragma unroll
        for (int i = 0; i < N; ++i)
            u[i] = FEAT & F_BITS ? __builtin_amdgcn_fmed3f(u[i], U_LOW, -U_LOW) : fmaxf(u[i], U_LOW);
    }
}
/* Listed tokens of the workgroup's part of the row as bits (tail only): group v's start at bit
 * (v - v0 + 1) N, so that a group's bits lie in one byte; the head is in front of group v0. */
template <int N> __device__ __forceinline__ uint32_t listed_bits(const uint32_t *map, int group) {
    const int at = (group + 1) * N;
    return map[at >> 5] >> (at & 31);
}
template <int TYPE, int FEAT>
__device__ __forceinline__ uint32_t keep_bits(const LossArgs &a, const Row<TYPE> &r, const uint32_t *map,
                                              int v) {
    uint32_t keep = ~0u;
    if (FEAT & F_BITS) {
        if (r.allowed)
            keep = r.bits(r.head + v * Elem<TYPE>::N);
        if (map)
            keep &= ~listed_bits<Elem<TYPE>::N>(map, v - r.v0);
    }
    return keep;
}
/* The allowed tokens of the groups that a thread holds, eight bits each, read once for both passes. */
template <int TYPE, int FEAT, int THREADS, int HELD> struct HeldBits {
    static constexpr int WORDS = FEAT & F_BITS ? (HELD + 3) / 4 : 1;
    uint32_t             w[WORDS];
    __device__ __forceinline__ void read(const LossArgs &a, const Row<TYPE> &r) {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            w[i] = ~0u;
        if constexpr (FEAT & F_BITS) {
            if (r.allowed) {
#pragma unroll
                for (int i = 0; i < WORDS; ++i)
                    w[i] = 0u;
#pragma unroll
                for (int h = 0; h < HELD; ++h) {
                    const int v = h * THREADS + (int) threadIdx.x;
                    if (v < r.nvec)
                        w[h >> 2] |= (r.bits(r.head + v * Elem<TYPE>::N) & 0xffu) << (8 * (h & 3));
                }
            }
        }
    }
    __device__ __forceinline__ uint32_t of(int h) const {
        return FEAT & F_BITS ? w[h >> 2] >> (8 * (h & 3)) : ~0u;
    }
};

/* ---- the pass that sums --------------------------------------------------------------------- */
/* A thread sums 2^(w - c) against a reference c of its own, the largest w of its first group: later
 * values that are larger only make larger terms, and a batch whose sum reaches 2^15 is done again
 * behind a reference moved to its largest value. So the usual element costs a fused multiply-add, an
 * exponential and an addition, and no maximum. A batch of U groups is added up in binary32 by halves,
 * the batches in binary64: a running binary32 sum loses what is small beside a leading token, always
 * downwards (2e-6 of the sum over a whole row, 1e-7 over batches of 32).
 * References stay above -2^20 and should stay below 2^26, where c's rounding is harmless; rows for
 * which that does not hold (nothing above -2^20, logits of 4e7 and more) are done again by
 * careful_sums. */
constexpr float C_LOW = -1048576.0f, C_HIGH = 67108864.0f, BATCH_HIGH = 0x1p15f;
struct Acc {
    float  c = C_LOW;
    double s = 0.0, t = 0.0;
};
/* the largest value of a group that counts */
template <int TYPE, int FEAT>
__device__ __forceinline__ float group_top(const LossArgs &a, u32x4 raw, uint32_t keep) {
    float x[Elem<TYPE>::N], top = -INFINITY;
    Elem<TYPE>::unpack(raw, x);
#pragma unroll
    for (int i = 0; i < Elem<TYPE>::N; ++i)
        if (!(FEAT & F_BITS) || ((keep >> i) & 1u))
            top = fmaxf(top, x[i]);
    return capped<FEAT>(a, top); /* (it is monotone) */
}
__device__ __forceinline__ void acc_move(Acc &c, float top, float k) {
    const float  w  = fmaxf(top * k, c.c);
    const float  d  = c.c - w;
    const double sc = (double) __builtin_amdgcn_exp2f(d);
    c.t = sc * (c.t + (c.s == 0.0 ? 0.0 : c.s * (double) d));
    c.s *= sc;
    c.c = w;
}
/* the sums of COUNT groups, of which the j-th counts if live has bit j, against c */
template <int TYPE, int FEAT, int COUNT>
__device__ __forceinline__ float batch_sum(const LossArgs &a, float c, const u32x4 (&raw)[COUNT],
                                           const uint32_t (&keep)[COUNT], uint32_t live, float &t) {
    constexpr int N = Elem<TYPE>::N;
    float         s[COUNT];
    t = 0.0f;
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        s[j] = 0.0f;
        if ((live >> j) & 1u) {
            float e[N], u[N], slope[N];
            group_exps<TYPE, FEAT>(a, raw[j], keep[j], c, e, u, slope);
            if (FEAT & F_ENTROPY) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    t = fmaf(e[i], u[i], t);
            }
#pragma unroll
            for (int half = N / 2; half; half >>= 1)
#pragma unroll
                for (int i = 0; i < half; ++i)
                    e[i] += e[i + half];
            s[j] = e[0];
        }
    }
#pragma unroll
    for (int half = COUNT / 2; half; half >>= 1)
#pragma unroll
        for (int j = 0; j < half; ++j)
            s[j] += s[j + half];
    return s[0];
}
template <int TYPE, int FEAT, int COUNT>
__device__ __forceinline__ void acc_batch(const LossArgs &a, Acc &c, u32x4 (&raw)[COUNT],
                                          const uint32_t (&keep)[COUNT], uint32_t live) {
    float t, s = batch_sum<TYPE, FEAT, COUNT>(a, c.c, raw, keep, live, t);
    if (__builtin_expect(!(s < BATCH_HIGH), 0)) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            asm volatile("" : "+v"(raw[j])); /* (nothing is kept in registers for this case) */
            if ((live >> j) & 1u)
                top = fmaxf(top, group_top<TYPE, FEAT>(a, raw[j], keep[j]));
        }
        acc_move(c, top, a.k);
        s = batch_sum<TYPE, FEAT, COUNT>(a, c.c, raw, keep, live, t);
    }
    c.s += (double) s;
    if (FEAT & F_ENTROPY)
        c.t += (double) t;
}
template <int TYPE, int FEAT>
__device__ __forceinline__ void acc_loose(const LossArgs &a, const Row<TYPE> &r, const uint32_t *map,
                                          Acc &c) {
    if (threadIdx.x < 2 * Elem<TYPE>::N) {
        const int e = r.loose((int) threadIdx.x);
        const int at = e - r.elem0() + Elem<TYPE>::N;
        if (e >= 0 && r.may(e) && !(map && ((map[at >> 5] >> (at & 31)) & 1u))) {
            const float y = capped<FEAT>(a, Elem<TYPE>::one(r.x[e]));
            if (y * a.k > c.c)
                acc_move(c, y, a.k);
            const float u = fmaf(y, a.k, -c.c), v = __builtin_amdgcn_exp2f(u);
            c.s += (double) v;
            if (FEAT & F_ENTROPY) /* (0 * -inf is no term, as in group_exps) */
                c.t += (double) v * (double) fmaxf(u, U_LOW);
        }
    }
}
/* the groups from v0 + `from` on, read as they come. (Loads stand under no condition of a lane's: behind
 * one, the compiler unpacks each group where it was loaded and so waits for every load by itself.) */
template <int TYPE, int FEAT, int THREADS, int U, bool STREAMED>
__device__ __forceinline__ void sum_groups(const LossArgs &a, const Row<TYPE> &r, const uint32_t *map,
                                           int from, Acc &c) {
    bool start = from == 0;
    for (int v = r.v0 + from + (int) threadIdx.x; v < r.v1; v += U * THREADS) {
        u32x4    raw[U];
        uint32_t keep[U], live = 0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int w = min(v + j * THREADS, r.v1 - 1);
            raw[j]      = STREAMED ? r.load_streamed(w) : r.load(w);
            live |= v + j * THREADS < r.v1 ? 1u << j : 0u;
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
            keep[j] = keep_bits<TYPE, FEAT>(a, r, map, min(v + j * THREADS, r.v1 - 1));
        if (start)
            acc_move(c, group_top<TYPE, FEAT>(a, raw[0], keep[0]), a.k);
        start = false;
        acc_batch<TYPE, FEAT, U>(a, c, raw, keep, live);
    }
}

/* A row's or a part's sums. Against c, or where `careful` against m k (which may be beyond binary32). */
struct Sums {
    double s, t;
    float  c, m;
    bool   careful;
    double top;    /* the largest listed value, in exponents */
    double listed; /* with a tail: the listed tokens' own sum against it */
    __device__ __forceinline__ double ref(float k) const {
        return careful ? (double) m * (double) k : (double) c;
    }
};
/* The sums against c = ref + log2(s) instead, rounded: s is then near 1 and the exponents of the tokens
 * that matter are small, so that they lose nothing to rounding when the gradient forms them again. */
__device__ __forceinline__ void rebase(Sums &j) {
    if (j.careful || j.s == 0.0)
        return;
    const float  c  = (float) ((double) j.c + log2(j.s));
    const double d  = (double) j.c - (double) c;
    const double sc = exp2(d);
    j.t = sc * (j.t + j.s * d);
    j.s *= sc;
    j.c = c;
}
/* Sums with the maximum known first and (y - m) k formed as a difference: any finite values. */
template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ Sums careful_sums(const LossArgs &a, const Row<TYPE> &r, const uint32_t *map,
                                          double *slot) {
    constexpr int N = Elem<TYPE>::N;
    const int     lo = r.first ? 0 : r.elem0(), hi = r.last ? r.n : r.head + r.v1 * N;
    auto counts = [&](int e) {
        const int at = e - r.elem0() + N;
        return r.may(e) && !(map && ((map[at >> 5] >> (at & 31)) & 1u));
    };
    double top = -FLT_MAX;
    for (int e = lo + (int) threadIdx.x; e < hi; e += THREADS)
        if (counts(e))
            top = fmax(top, (double) capped<FEAT>(a, Elem<TYPE>::one(r.x[e])));
    Sums j    = {};
    j.careful = true;
    j.m       = (float) block_reduce<THREADS, true>(top, slot);
    double s = 0.0, t = 0.0;
    for (int e = lo + (int) threadIdx.x; e < hi; e += THREADS)
        if (counts(e)) {
            const float u = (capped<FEAT>(a, Elem<TYPE>::one(r.x[e])) - j.m) * a.k;
            const float p = __builtin_amdgcn_exp2f(u);
            s += (double) p;
            t += (double) p * (double) fmaxf(u, U_LOW);
        }
    j.s = block_reduce<THREADS, false>(s, slot);
    j.t = block_reduce<THREADS, false>(t, slot);
    return j;
}
/* What the wavefronts of a workgroup tell one another. */
struct Shared {
    double s[16], t[16], slot[16];
    float  c[16];
    Sums   sums;
    struct Coef {
        float a;        /* 2^u_i (a + b u_i): 1 / S, 1 / T and the weight are in them */
        float b;
        float a_listed; /* 2^(w_j - top) a_listed - q_j q for listed tokens of a teacher */
        float q;
        bool  zero;     /* the row is written as zeros */
    } coef;
};
/* lanes' sums, joined against the largest reference among them */
template <int FEAT> __device__ __forceinline__ void join_lanes(float &c, double &s, double &t) {
    const float  top = wave_max(c);
    const float  d   = c - top; /* (NaN beside +inf: so is the row) */
    const double sc  = (double) __builtin_amdgcn_exp2f(d);
    if (FEAT & F_ENTROPY)
        t = wave_sum_f64(sc * (t + (s == 0.0 ? 0.0 : s * (double) d)));
    s = wave_sum_f64(sc * s);
    c = top;
}
template <int FEAT, int THREADS>
__device__ __forceinline__ Sums join_threads(Acc acc, Shared &sh) {
    join_lanes<FEAT>(acc.c, acc.s, acc.t);
    if constexpr (THREADS > 64) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane == 0) {
            sh.c[wave] = acc.c;
            sh.s[wave] = acc.s;
            sh.t[wave] = acc.t;
        }
        lds_barrier();
        const bool in = lane < THREADS / 64;
        acc.c         = in ? sh.c[lane] : C_LOW;
        acc.s         = in ? sh.s[lane] : 0.0;
        acc.t         = in ? sh.t[lane] : 0.0;
        join_lanes<FEAT>(acc.c, acc.s, acc.t);
    }
    Sums j = {};
    j.c    = acc.c;
    j.s    = acc.s;
    j.t    = acc.t;
    return j;
}
/* (a reference of a value's own has that value's 1 in its sum: less means that only C_LOW stands above the
 * row's values, whose terms may have lost bits) */
__device__ __forceinline__ bool needs_care(const Sums &j) { return !(j.c < C_HIGH) || j.s < 0.5; }
/* The parts of a row, joined by a wavefront. A part in which nothing counts (its sum is 0) has no reference: it
 * must not stand above parts whose values all lie below its own. A part that is careful beside a plain one with
 * a larger reference weighs next to nothing: the row is plain then. */
template <int FEAT> __device__ __forceinline__ Sums join_parts(const LossPart *p, int chunks, float k) {
    const int lane = threadIdx.x & 63;
    double    top  = -1e300;
    for (int i = lane; i < chunks; i += 64)
        if (p[i].s != 0.0)
            top = fmax(top, p[i].c);
    top         = wave_max(top);
    float m     = -FLT_MAX;
    bool  plain = false;
    for (int i = lane; i < chunks; i += 64)
        if (p[i].s != 0.0 && p[i].c == top) {
            plain |= p[i].careful == 0;
            if (p[i].careful)
                m = fmaxf(m, p[i].m);
        }
    Sums j    = {};
    j.careful = !__any(plain);
    j.m       = wave_max(m);
    j.c       = (float) top;
    const double ref = j.ref(k);
    double s = 0.0, t = 0.0;
    for (int i = lane; i < chunks; i += 64) {
        if (p[i].s == 0.0)
            continue;
        const double d  = fmax(p[i].c - ref, -1e30);
        const double sc = (double) __builtin_amdgcn_exp2f((float) d);
        s += sc * p[i].s;
        if (FEAT & F_ENTROPY)
            t += sc * (p[i].t + p[i].s * d);
    }
    j.s      = wave_sum_f64(s);
    j.t      = (FEAT & F_ENTROPY) ? wave_sum_f64(t) : 0.0;
    j.top    = p[0].top;
    j.listed = p[0].listed;
    return j;
}

/* ---- the gradient --------------------------------------------------------------------------- */
typedef Shared::Coef Coef;
template <int TYPE, int FEAT>
__device__ __forceinline__ u32x4 group_grad(const LossArgs &a, u32x4 raw, uint32_t keep, const Coef &c,
                                            float ref) {
    constexpr int N = Elem<TYPE>::N;
    float         e[N], u[N], slope[N], g[N];
    group_exps<TYPE, FEAT>(a, raw, keep, ref, e, u, slope);
    const float four = FEAT & F_CAP ? 4.0f : 1.0f, ca = four * c.a, cb = four * c.b;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        g[i] = e[i] * ((FEAT & F_ENTROPY) ? fmaf(cb, u[i], ca) : ca);
        if (FEAT & F_CAP)
            g[i] *= slope[i];
        if ((FEAT & F_BITS) && (FEAT & F_CAP)) /* (a forbidden NaN has no slope either) */
            g[i] = __uint_as_float(__float_as_uint(g[i]) & bit_mask(keep, i));
    }
    return Elem<TYPE>::pack(g);
}
template <int FEAT> __device__ __forceinline__ float cap_slope(const LossArgs &a, float x) {
    if (!(FEAT & F_CAP))
        return 1.0f;
    const float E = cap_power(a, x), r = __builtin_amdgcn_rcpf(1.0f + E);
    return 4.0f * cap_quarter(E, r);
}
/* one element by any row's reference */
template <int TYPE, int FEAT>
__device__ __forceinline__ float one_grad(const LossArgs &a, const Row<TYPE> &r, int e, float x,
                                          const Coef &c, const Sums &j) {
    if (!r.may(e))
        return 0.0f;
    const float y = capped<FEAT>(a, x);
    const float u = j.careful ? (y - j.m) * a.k : fmaf(y, a.k, -j.c);
    const float f = (FEAT & F_ENTROPY) ? fmaf(c.b, fmaxf(u, U_LOW), c.a) : c.a;
    return __builtin_amdgcn_exp2f(u) * f * cap_slope<FEAT>(a, x);
}
/* the groups from v0 + `from` on, read again */
template <int TYPE, int FEAT, int THREADS, int U>
__device__ __forceinline__ void write_groups(const LossArgs &a, const Row<TYPE> &r, const Coef &c,
                                             const Sums &j, int from) {
    for (int v = r.v0 + from + (int) threadIdx.x; v < r.v1; v += U * THREADS) {
        u32x4    raw[U];
        uint32_t keep[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            raw[i] = r.load(min(v + i * THREADS, r.v1 - 1));
#pragma unroll
        for (int i = 0; i < U; ++i)
            keep[i] = keep_bits<TYPE, FEAT>(a, r, nullptr, min(v + i * THREADS, r.v1 - 1));
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (v + i * THREADS < r.v1)
                r.store(v + i * THREADS, group_grad<TYPE, FEAT>(a, raw[i], keep[i], c, j.c), a.streamed);
    }
}
template <int TYPE, int FEAT>
__device__ __forceinline__ void write_loose(const LossArgs &a, const Row<TYPE> &r, const Coef &c,
                                            const Sums &j) {
    if (threadIdx.x < 2 * Elem<TYPE>::N) {
        const int e = r.loose((int) threadIdx.x);
        if (e >= 0)
            r.g[e] = Elem<TYPE>::round(one_grad<TYPE, FEAT>(a, r, e, Elem<TYPE>::one(r.x[e]), c, j));
    }
}
/* rows of zeros, and rows whose sums careful_sums made */
template <int TYPE, int FEAT, int THREADS>
__device__ __forceinline__ void write_rare(const LossArgs &a, const Row<TYPE> &r, const Coef &c, const Sums &j) {
    if (c.zero) {
        for (int v = r.v0 + (int) threadIdx.x; v < r.v1; v += THREADS)
            r.store(v, u32x4{0, 0, 0, 0}, a.streamed);
        const int e = threadIdx.x < 2 * Elem<TYPE>::N ? r.loose((int) threadIdx.x) : -1;
        if (e >= 0)
            r.g[e] = Elem<TYPE>::round(0.0f);
        return;
    }
    const int lo = r.first ? 0 : r.elem0(), hi = r.last ? r.n : r.head + r.v1 * Elem<TYPE>::N;
    for (int e = lo + (int) threadIdx.x; e < hi; e += THREADS)
        r.g[e] = Elem<TYPE>::round(one_grad<TYPE, FEAT>(a, r, e, Elem<TYPE>::one(r.x[e]), c, j));
}

/* ---- one token per row ---------------------------------------------------------------------- */
constexpr double LN2 = 0.693147180559945309417232;

template <int TYPE> struct Token {
    typename Elem<TYPE>::mem x;
    int                      id; /* -1: none */
    uint32_t                 may;
    /* softcap(x) k; -inf where the token is forbidden */
    template <int FEAT> __device__ __forceinline__ double w(const LossArgs &a) const {
        return !((may >> (max(id, 0) & 31)) & 1u) ? -INFINITY : value64<TYPE, FEAT>(a, Elem<TYPE>::one(x));
    }
};
/* (only asked for here: what was asked for before need not have arrived) */
template <int TYPE> __device__ __forceinline__ Token<TYPE> load_token(const LossArgs &a, const Row<TYPE> &r, int row) {
    Token<TYPE> t;
    t.id          = a.tokens[row];
    t.id          = t.id < 0 || t.id >= r.n ? -1 : t.id;
    const int at  = max(t.id, 0);
    t.x           = r.x[at];
    t.may         = r.allowed ? r.allowed[at >> 5] : ~0u;
    return t;
}
/* Policy loss of a row from its sums; `lead`: this thread writes the row's outputs. */
__device__ __forceinline__ Coef policy_coef(const LossArgs &a, int row, bool has_token, double tw,
                                            const Sums &j, bool entropy, bool lead) {
    const bool   empty = j.s == 0.0;
    const double l2s   = empty ? 0.0 : log2(j.s);
    const double lp    = !has_token ? 0.0 : empty ? -INFINITY : (tw - j.ref(a.k) - l2s) * LN2;
    const double H     = entropy && !empty ? LN2 * (l2s - j.t / j.s) : 0.0;
    const double w     = a.weight ? (double) a.weight[row] : 1.0;
    Coef         c     = {0.0f, 0.0f, 0.0f, 0.0f, true};
    double       loss  = 0.0;
    if (w != 0.0 && has_token && lp != -INFINITY) {
        const double A     = (double) a.advantage[row];
        double       d     = 0.0;
        const double ratio = a.old_lp ? exp(lp - (double) a.old_lp[row]) : 1.0;
        if (A != 0.0) {
            const double lo = 1.0 - (double) a.clip_low, hi = 1.0 + (double) a.clip_high;
            const double held = ratio < lo ? lo : ratio > hi ? hi : ratio; /* NaN stays */
            const double f = ratio * A, h = held * A;
            loss = h < f ? -h : -f;
            d    = h < f ? 0.0 : -f;
        }
        if (a.ref_lp && a.kl_coef != 0.0f) { /* (not 0 * inf) */
            const double far = (double) a.ref_lp[row] - lp;
            const double ex  = expm1(far);
            loss += (double) a.kl_coef * (ex - far);
            d -= (double) a.kl_coef * ex;
        }
        const double ec = (double) a.entropy_coef;
        if (ec != 0.0)
            loss -= ec * H;
        if (lp != lp) /* a spoilt row, also where no term above has seen it */
            loss = d = lp;
        loss *= w;
        d *= w * a.inv_t;
        const double be = w * ec * a.inv_t;
        c.a = (float) ((be != 0.0 ? be * (H - l2s * LN2) - d : -d) / j.s);
        c.b = (float) (be * LN2 / j.s);
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
/* the token's own element, over what stands there */
template <int TYPE, int FEAT>
__device__ __forceinline__ void write_token(const LossArgs &a, const Row<TYPE> &r, const Token<TYPE> &t,
                                            const Coef &c, const Sums &j) {
    const float u = (float) (t.template w<FEAT>(a) - j.ref(a.k)); /* (-inf below binary32's lowest) */
    const float f = (FEAT & F_ENTROPY) ? fmaf(c.b, fmaxf(u, U_LOW), c.a) : c.a;
    const float g = __builtin_amdgcn_exp2f(u) * f - c.q;
    r.g[t.id] = Elem<TYPE>::round(g * cap_slope<FEAT>(a, Elem<TYPE>::one(t.x)));
}

/* ---- a teacher's list ----------------------------------------------------------------------- */
/* In LDS, of each entry: its id (-1: left out), x, w - top (w = softcap(x) k, top the largest of them),
 * its value, then q. `first`: a table of entries by id that keeps the first of a repeated id. All of it is
 * one wavefront's. */
struct List {
    int   *ids, *first;
    float *x, *u, *q;
    __device__ List(const LossArgs &a, void *lds) {
        ids   = static_cast<int *>(lds);
        x     = reinterpret_cast<float *>(ids + a.list_k);
        u     = x + a.list_k;
        q     = u + a.list_k;
        first = reinterpret_cast<int *>(q + a.list_k);
    }
};
struct ListSums {
    double q_log_q, q_sum; /* sum q_j log q_j, sum q_j */
    double top;
    double q_u;            /* sum q_j (w_j - top) */
    double listed;         /* with a tail: sum 2^(w_j - top), apart from the other tokens' sum, so that
                            * neither mass is lost beside the other however far the two lie apart */
    int    n;
};
/* row_top: the rows may hold their gradient already outside the workgroup's part; then only entries of
 * that part are looked up, against this top. map, if given, is cleared and gets the listed tokens of the
 * workgroup's part. Called by one whole wavefront. */
template <int TYPE, int FEAT>
__device__ __forceinline__ ListSums read_list(const LossArgs &a, const Row<TYPE> &r, int row, const List &l,
                                              uint32_t *map, const double *row_top) {
    constexpr int N    = Elem<TYPE>::N;
    const int     lane = threadIdx.x & 63;
    int           k    = a.list_k;
    if (a.count)
        k = max(0, min(k, a.count[row]));
    for (int j = lane; j < k; j += 64) {
        const int   id = a.ids[(long) row * a.list_ld + j];
        const float v  = a.values[(long) row * a.list_ld + j];
        const bool  ok = id >= 0 && id < r.n && v != -INFINITY && r.may(id);
        l.ids[j]       = ok ? id : -1;
        l.q[j]         = v;
        l.x[j]         = ok && (!row_top || r.mine(id)) ? Elem<TYPE>::one(r.x[id]) : 0.0f;
    }
    for (int i = lane; i < a.slots; i += 64)
        l.first[i] = -1;
    if (map) {
        const int span = (r.last ? r.n : r.head + r.v1 * N) - r.elem0() + N; /* bits */
        for (int i = lane; i < (span + 31) / 32; i += 64)
            map[i] = 0u;
    }
    wave_fence();
    for (int j = lane; j < k; j += 64) {
        const int id = l.ids[j];
        if (id < 0)
            continue;
        uint32_t at = ((uint32_t) id * 2654435761u) & (uint32_t) (a.slots - 1);
        for (;;) { /* ends: there are twice as many places as entries */
            const int was = atomicCAS(&l.first[at], -1, j);
            if (was == -1)
                break;
            if (l.ids[was] == id) { /* (whoever holds this place, now or later, lists this id) */
                atomicMin(&l.first[at], j);
                break;
            }
            at = (at + 1) & (uint32_t) (a.slots - 1);
        }
    }
    wave_fence();
    float  v_top = -INFINITY;
    double top   = -1e300;
    for (int j = lane; j < k; j += 64) {
        const int id = l.ids[j];
        if (id < 0)
            continue;
        uint32_t at = ((uint32_t) id * 2654435761u) & (uint32_t) (a.slots - 1);
        int      f;
        while (l.ids[f = l.first[at]] != id)
            at = (at + 1) & (uint32_t) (a.slots - 1);
        l.u[j] = f == j ? 0.0f : 1.0f; /* (the id stays until every lane has looked its own up) */
        if (f == j) {
            top   = fmax(top, value64<TYPE, FEAT>(a, l.x[j]));
            v_top = fmaxf(v_top, l.q[j]);
            if (map && r.mine(id)) {
                const int bit = id - r.elem0() + N;
                atomicOr(&map[bit >> 5], 1u << (bit & 31));
            }
        }
    }
    wave_fence();
    v_top = wave_max(v_top);
    ListSums z;
    z.n   = k;
    z.top = row_top ? *row_top : wave_max(top);
    double e_sum = 0.0, ev = 0.0, eu = 0.0, listed = 0.0;
    for (int j = lane; j < k; j += 64) {
        if (l.ids[j] >= 0 && l.u[j] != 0.0f)
            l.ids[j] = -1;
        if (l.ids[j] >= 0) {
            const double v = a.tail ? (double) l.q[j] : ((double) l.q[j] - (double) v_top) * a.inv_t;
            const double e = exp(v), u = value64<TYPE, FEAT>(a, l.x[j]) - z.top;
            l.u[j]         = (float) u;
            e_sum += e;
            if (e != 0.0) {
                ev += e * v;
                eu += e * u;
            }
            if (a.tail)
                listed += (double) __builtin_amdgcn_exp2f((float) u);
        }
    }
    e_sum              = wave_sum_f64(e_sum);
    ev                 = wave_sum_f64(ev);
    eu                 = wave_sum_f64(eu);
    const bool   plain = a.tail || e_sum == 0.0;
    const double scale = plain ? 1.0 : 1.0 / e_sum;
    for (int j = lane; j < k; j += 64)
        if (l.ids[j] >= 0) {
            const double v = a.tail ? (double) l.q[j] : ((double) l.q[j] - (double) v_top) * a.inv_t;
            l.q[j]         = (float) (exp(v) * scale);
        }
    z.q_sum   = e_sum * scale;
    z.q_log_q = ev * scale - (plain ? 0.0 : log(e_sum));
    z.q_u     = eu * scale;
    z.listed  = a.tail ? wave_sum_f64(listed) : 0.0;
    wave_fence();
    return z;
}
/* q_u and j.top (sum of q_j (w_j - top) and top) are handed in: the rows may have been replaced by
 * their gradient since */
__device__ __forceinline__ Coef distill_coef(const LossArgs &a, int row, const ListSums &l, double q_u,
                                             const Sums &j, bool lead) {
    const double w   = a.weight ? (double) a.weight[row] : 1.0;
    const double ref = j.ref(a.k);
    /* everything against one reference: the listed tokens' sum and that of the rest */
    const double base = a.tail && (j.s == 0.0 || j.top > ref) ? j.top : ref;
    const double rest = j.s == 0.0 ? 0.0 : ref == base ? j.s : j.s * exp2(ref - base);
    const double all  = a.tail ? rest + (j.top == base ? j.listed : j.listed * exp2(j.top - base)) : rest;
    Coef   c    = {0.0f, 0.0f, 0.0f, 0.0f, true};
    double loss = 0.0;
    if (w != 0.0 && all != 0.0 && (a.tail || l.q_sum != 0.0)) {
        const double l2s = log2(all);
        /* sum q_j (log q_j - log p_j) */
        loss = l.q_log_q + LN2 * (l.q_sum * (l2s + (base - j.top)) - q_u);
        const double ws = w * a.inv_t;
        /* what log S is multiplied by, q_sum + q_rest: 1 unless the listed mass exceeds it */
        const double mass = a.tail && !(l.q_sum <= 1.0) ? l.q_sum : 1.0;
        c.a        = (float) (ws / all);
        c.a_listed = (float) (ws / all * mass * exp2(j.top - base));
        if (a.tail) {
            /* p_i (mass - q_rest / p_rest) = 2^(w_i - ref) / s * (p_rest mass - q_rest) */
            const double q_rest = l.q_sum <= 1.0 ? 1.0 - l.q_sum : l.q_sum > 1.0 ? 0.0 : l.q_sum;
            if (q_rest != 0.0)
                loss += q_rest * (log(q_rest) -
                                  (j.s == 0.0 ? -INFINITY : LN2 * (log2(j.s) + (ref - base) - l2s)));
            c.a = j.s == 0.0 ? 0.0f : (float) (ws * (rest / all * mass - q_rest) / j.s);
        }
        loss *= w;
        c.q    = (float) ws;
        c.zero = false;
    }
    if (lead && a.loss)
        a.loss[row] = (float) loss;
    return c;
}
/* by the wavefront that read the list */
template <int TYPE, int FEAT>
__device__ __forceinline__ void write_listed(const LossArgs &a, const Row<TYPE> &r, const List &l, int n,
                                             const Coef &c) {
    for (int j = threadIdx.x & 63; j < n; j += 64)
        if (l.ids[j] >= 0 && r.mine(l.ids[j])) {
            const float g = __builtin_amdgcn_exp2f(l.u[j]) * c.a_listed - l.q[j] * c.q;
            r.g[l.ids[j]] = Elem<TYPE>::round(g * cap_slope<FEAT>(a, l.x[j]));
        }
}

/* ---- kernels -------------------------------------------------------------------------------- */
/* A workgroup per row. HELD groups of 16 bytes per thread are kept between the passes: all of them are
 * asked for at the start, and the gradient goes out in one go (reading and writing in turn moves 5.8 TB/s
 * on this pattern, a next row's loads between the stores 5.2). Longer rows have further groups loaded
 * straight into LDS (a.stash per thread), and what is left is read twice. HELD = 0: no gradient is wanted, the row
 * is read as it comes by more wavefronts. */
template <int TYPE, int OP, int FEAT> struct Held { /* what 128 registers have room for */
    static constexpr int N = FEAT & (F_CAP | F_BITS) ? 12 : OP == OP_DISTILL ? 14 : 16;
};
constexpr int UH = 2;
template <int TYPE, int OP, int FEAT, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS, HELD ? 4 : 1) void k_loss_row(LossArgs a) {
    __shared__ Shared sh;
    extern __shared__ __align__(16) char lds[];
    const int       row = blockIdx.x, tid = (int) threadIdx.x;
    const bool      lead = tid < 64; /* the wavefront that forms the row's scalars */
    const bool      tail = OP == OP_DISTILL && (FEAT & F_BITS) && a.tail;
    const Row<TYPE> r(a, row, 0, 1, 0);
    uint32_t       *map = nullptr;
    ListSums        ls  = {};
    Token<TYPE>     t   = {};
    if constexpr (OP == OP_DISTILL) {
        if (tail)
            map = reinterpret_cast<uint32_t *>(lds + a.list_k * 16 + a.slots * 4);
        if (lead) /* (in front of its loads of the row: loads return in order) */
            ls = read_list<TYPE, FEAT>(a, r, row, List(a, lds), map, nullptr);
    }
    Acc   acc;
    u32x4 raw[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
        if (r.nvec > 0) {
            if (a.streamed) {
#pragma unroll
                for (int h = 0; h < HELD; ++h)
                    raw[h] = r.load_streamed(min(h * THREADS + tid, r.nvec - 1));
                asm volatile(""); /* (keeps the two kinds of loads from being made one) */
            } else {
#pragma unroll
                for (int h = 0; h < HELD; ++h)
                    raw[h] = r.load(min(h * THREADS + tid, r.nvec - 1));
            }
        }
    }
    /* [stash][THREADS] groups, each the own thread's */
    u32x4 *const stash = reinterpret_cast<u32x4 *>(lds + a.stash_at);
    if constexpr (HELD > 0)
        for (int h = 0; h < a.stash; ++h)
            if ((HELD + h) * THREADS + tid < r.nvec)
                r.load_to_lds((HELD + h) * THREADS + tid, stash + h * THREADS + (tid & ~63), a.streamed);
    HeldBits<TYPE, FEAT, THREADS, HELD ? HELD : 1> bits;
    if constexpr (OP != OP_DISTILL)
        t = load_token<TYPE>(a, r, row);
    if constexpr (HELD > 0)
        bits.read(a, r);
    if (tail)
        lds_barrier();
    if constexpr (HELD > 0) {
#pragma unroll
        for (int h = 0; h < HELD; h += UH) {
            uint32_t keep[UH], live = 0;
            u32x4    some[UH];
#pragma unroll
            for (int i = 0; i < UH; ++i) {
                const int v = (h + i) * THREADS + tid;
                keep[i]     = 0;
                some[i]     = raw[h + i];
                if (v < r.nvec) {
                    keep[i] = bits.of(h + i);
                    if ((FEAT & F_BITS) && map)
                        keep[i] &= ~listed_bits<Elem<TYPE>::N>(map, v);
                    live |= 1u << i;
                }
            }
            if (h == 0 && live)
                acc_move(acc, group_top<TYPE, FEAT>(a, raw[0], keep[0]), a.k);
            acc_batch<TYPE, FEAT, UH>(a, acc, some, keep, live);
            __builtin_amdgcn_sched_barrier(0); /* (interleaved, the batches would not fit the registers) */
        }
        if (a.stash) /* what this wavefront asked for has arrived in LDS */
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int h = 0; h < a.stash; ++h) {
            const int v = (HELD + h) * THREADS + tid;
            if (v < r.nvec) {
                u32x4          one[1]  = {stash[h * THREADS + tid]};
                const uint32_t keep[1] = {keep_bits<TYPE, FEAT>(a, r, map, v)};
                acc_batch<TYPE, FEAT, 1>(a, acc, one, keep, 1u);
            }
        }
        sum_groups<TYPE, FEAT, THREADS, UH, false>(a, r, map, (HELD + a.stash) * THREADS, acc);
    } else {
        if (a.streamed)
            sum_groups<TYPE, FEAT, THREADS, 4, true>(a, r, map, 0, acc);
        else
            sum_groups<TYPE, FEAT, THREADS, 4, false>(a, r, map, 0, acc);
    }
    acc_loose<TYPE, FEAT>(a, r, map, acc);
    Sums j = join_threads<FEAT, THREADS>(acc, sh);
    if (needs_care(j))
        j = careful_sums<TYPE, FEAT, THREADS>(a, r, map, sh.slot);
    if (lead) {
        rebase(j);
        Coef c;
        if constexpr (OP == OP_DISTILL) {
            j.top    = ls.top;
            j.listed = ls.listed;
            c        = distill_coef(a, row, ls, ls.q_u, j, tid == 0);
        } else {
            c = policy_coef(a, row, t.id >= 0, t.template w<FEAT>(a), j, FEAT & F_ENTROPY, tid == 0);
        }
        if (tid == 0) {
            sh.sums = j;
            sh.coef = c;
        }
    }
    if constexpr (HELD > 0) {
        __syncthreads(); /* every value of the row has been read before any is written */
        j            = sh.sums;
        const Coef c = sh.coef;
        if (c.zero || j.careful) {
            write_rare<TYPE, FEAT, THREADS>(a, r, c, j);
        } else {
#pragma unroll
            for (int h = 0; h < HELD; ++h) {
                const int v = h * THREADS + tid;
                /* (hides that this is what the sums were made of: the compiler would keep the unpacked
                 * values, twice the registers) */
                asm volatile("" : "+v"(raw[h]));
                if (v < r.nvec)
                    r.store(v, group_grad<TYPE, FEAT>(a, raw[h], bits.of(h), c, j.c), a.streamed);
                __builtin_amdgcn_sched_barrier(0);
            }
            for (int h = 0; h < a.stash; ++h) {
                const int v = (HELD + h) * THREADS + tid;
                if (v < r.nvec)
                    r.store(v, group_grad<TYPE, FEAT>(a, stash[h * THREADS + tid],
                                                      keep_bits<TYPE, FEAT>(a, r, nullptr, v), c, j.c),
                            a.streamed);
            }
            write_groups<TYPE, FEAT, THREADS, 2>(a, r, c, j, (HELD + a.stash) * THREADS);
            write_loose<TYPE, FEAT>(a, r, c, j);
        }
        __syncthreads();
        if (lead && !c.zero) {
            if constexpr (OP == OP_DISTILL)
                write_listed<TYPE, FEAT>(a, r, List(a, lds), ls.n, c);
            else if (tid == 0 && t.id >= 0)
                write_token<TYPE, FEAT>(a, r, t, c, j);
        }
    }
}

/* The sums of a part of a row. */
template <int TYPE, int OP, int FEAT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_loss_sums(LossArgs a) {
    __shared__ Shared sh;
    extern __shared__ __align__(16) char lds[];
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    if constexpr (OP == OP_PREFERENCE) {
        if (row < a.seq_start[0] || row >= a.seq_start[2 * a.n_pairs])
            return;
    }
    const Row<TYPE> r(a, row, chunk, a.chunks, a.chunk_vecs);
    const bool      tail = OP == OP_DISTILL && (FEAT & F_BITS) && a.tail;
    const bool      lead = threadIdx.x < 64;
    Acc             acc;
    ListSums        ls = {};
    Token<TYPE>     t  = {};
    uint32_t       *map = nullptr;
    if constexpr (OP == OP_DISTILL) {
        if (tail)
            map = reinterpret_cast<uint32_t *>(lds + a.list_k * 16 + a.slots * 4);
        if (lead && (tail || chunk == 0))
            ls = read_list<TYPE, FEAT>(a, r, row, List(a, lds), map, nullptr);
        if (tail)
            lds_barrier();
    } else {
        t = load_token<TYPE>(a, r, row);
    }
    if (row < a.streamed_rows)
        sum_groups<TYPE, FEAT, THREADS, 4, true>(a, r, map, 0, acc);
    else
        sum_groups<TYPE, FEAT, THREADS, 4, false>(a, r, map, 0, acc);
    acc_loose<TYPE, FEAT>(a, r, map, acc);
    Sums j = join_threads<FEAT, THREADS>(acc, sh);
    if (needs_care(j))
        j = careful_sums<TYPE, FEAT, THREADS>(a, r, map, sh.slot);
    if (OP == OP_PREFERENCE && chunk == 0 && threadIdx.x == 0 && a.row_grad)
        a.row_grad[row] = {0.0f, 0.0f, 0.0f, 0}; /* (of no pair yet) */
    if (threadIdx.x == 0)
        a.part[(long) row * a.chunks + chunk] = {
            j.s, j.t, j.ref(a.k), OP == OP_DISTILL ? ls.q_u : t.template w<FEAT>(a), ls.listed, ls.top, j.m, j.careful};
}

/* The gradient of a part of a row from the parts' sums; without one, a workgroup per row writes the
 * row's outputs. Parts of GRAD_VECS groups are read in one go: what short-lived workgroups that load first
 * move is the most this pattern of reads and writes reaches (a copy made so: 6.15 TB/s). */
constexpr int GRAD_U = 4;
template <int TYPE, int OP, int FEAT, int THREADS>
__global__ __launch_bounds__(THREADS) void k_loss_grad(LossArgs a, int chunks, int chunk_vecs) {
    __shared__ Shared sh;
    extern __shared__ __align__(16) char lds[];
    /* the last rows first: they are the likeliest to be in the cache still */
    const int row = a.rows - 1 - (int) (blockIdx.x / chunks), chunk = blockIdx.x % chunks;
    if constexpr (OP == OP_PREFERENCE) {
        if (row < a.seq_start[0] || row >= a.seq_start[2 * a.n_pairs])
            return;
    }
    const Row<TYPE> r(a, row, chunk, chunks, chunk_vecs);
    const bool      lead = threadIdx.x < 64;
    ListSums        ls   = {};
    Token<TYPE>     t    = {};
    if constexpr (OP != OP_DISTILL)
        t = load_token<TYPE>(a, r, row);
    /* the first groups are on their way while the scalars are formed */
    u32x4      raw[GRAD_U];
    const bool some = r.g && r.v1 > r.v0;
    if (some) {
#pragma unroll
        for (int i = 0; i < GRAD_U; ++i)
            raw[i] = r.load(min(r.v0 + i * THREADS + (int) threadIdx.x, r.v1 - 1));
    }
    Sums j = {};
    Coef c = {};
    if constexpr (OP == OP_PREFERENCE) {
        const LossRowGrad d = a.row_grad[row];
        c                   = {d.a, 0.0f, 0.0f, d.q, d.kind == 0};
        j.c = j.m = d.ref;
        j.careful = d.kind == 2;
    } else {
        if (lead) {
            const LossPart *p     = a.part + (long) row * a.chunks;
            const bool      first = chunk == 0 && threadIdx.x == 0;
            j                     = join_parts<FEAT>(p, a.chunks, a.k);
            const double at       = p[0].a;
            rebase(j);
            if constexpr (OP == OP_DISTILL) {
                ls = read_list<TYPE, FEAT>(a, r, row, List(a, lds), nullptr, &j.top);
                c  = distill_coef(a, row, ls, at, j, first);
            } else {
                c = policy_coef(a, row, t.id >= 0, at, j, FEAT & F_ENTROPY, first);
            }
            if (threadIdx.x == 0) {
                sh.sums = j;
                sh.coef = c;
            }
        }
    }
    if (!r.g)
        return;
    __syncthreads(); /* the part's values have been asked for before any is written */
    if constexpr (OP != OP_PREFERENCE) {
        j = sh.sums;
        c = sh.coef;
    }
    if (c.zero || j.careful) {
        write_rare<TYPE, FEAT, THREADS>(a, r, c, j);
    } else {
        if (some) {
#pragma unroll
            for (int i = 0; i < GRAD_U; ++i) {
                const int v = r.v0 + i * THREADS + (int) threadIdx.x;
                if (v < r.v1)
                    r.store(v, group_grad<TYPE, FEAT>(a, raw[i], keep_bits<TYPE, FEAT>(a, r, nullptr, v), c, j.c),
                            a.streamed);
            }
        }
        write_groups<TYPE, FEAT, THREADS, GRAD_U>(a, r, c, j, GRAD_U * THREADS);
        write_loose<TYPE, FEAT>(a, r, c, j);
    }
    if (c.zero)
        return;
    __syncthreads();
    if (lead) {
        if constexpr (OP == OP_DISTILL)
            write_listed<TYPE, FEAT>(a, r, List(a, lds), ls.n, c);
        else if (threadIdx.x == 0 && t.id >= 0 && r.mine(t.id))
            write_token<TYPE, FEAT>(a, r, t, c, j);
    }
}

constexpr int LDS_MOST = 158 * 1024; /* of 160 KB; the rest is what a kernel declares itself */
static_assert(sizeof(Shared) <= 2048, "beside the dynamic part");

/* groups per thread that go to LDS, of which a workgroup may use its share of the compute unit's */
template <int HELD> int stash_of(int threads, int vecs, size_t lds) {
    const int room = LDS_MOST * threads / 1024 - (int) ((lds + 15) / 16 * 16);
    return std::max(0, std::min(room / (threads * 16), (vecs + threads - 1) / threads - HELD));
}
template <int TYPE, int OP, int FEAT, int THREADS, int HELD>
void launch_held(LossArgs a, int vecs, size_t lds, hipStream_t stream) {
    a.stash          = stash_of<HELD>(THREADS, vecs, lds);
    a.stash_at       = (int) ((lds + 15) / 16 * 16);
    const size_t all = (size_t) a.stash_at + (size_t) a.stash * THREADS * 16;
    auto        *k   = k_loss_row<TYPE, OP, FEAT, THREADS, HELD>;
    /* (more than a launch gets unasked; where it is refused so is the launch, which the caller sees) */
    if (all > 64 * 1024)
        (void) hipFuncSetAttribute(reinterpret_cast<const void *>(k),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, LDS_MOST);
    k<<<dim3(a.rows), THREADS, all, stream>>>(a);
}

template <int TYPE, int OP, int FEAT>
void launch_one(LossStage stage, const LossArgs &a, size_t lds, int chunks, int chunk_vecs, hipStream_t stream) {
    if (stage == STAGE_ROW) {
        if constexpr (OP != OP_PREFERENCE) {
            const int vecs = a.n / Elem<TYPE>::N;
            if (!a.g && a.rows <= LOSS_WIDE_ROWS && vecs >= 4096) {
                k_loss_row<TYPE, OP, FEAT, 1024, 0><<<dim3(a.rows), 1024, lds, stream>>>(a);
            } else if (!a.g) {
                k_loss_row<TYPE, OP, FEAT, 256, 0><<<dim3(a.rows), 256, lds, stream>>>(a);
            } else {
                constexpr int H = Held<TYPE, OP, FEAT>::N;
                /* the smallest workgroup that holds the row, so that several share a compute unit and one
                 * loads while another computes; 512 threads also where they hold three quarters of it
                 * (4096 x 128256 bf16, of which they hold 80 %: 388 us, 1024 threads 401; 512 x 151936
                 * f32, 24 %: 159, 1024 threads 144). With no more rows than compute units none is shared:
                 * as many threads as there are. */
                auto held = [&](int threads) { return (H + stash_of<H>(threads, vecs, lds)) * threads; };
                const bool few = a.rows <= LOSS_WIDE_ROWS && vecs >= 4096;
                if (!few && held(128) >= vecs)
                    launch_held<TYPE, OP, FEAT, 128, H>(a, vecs, lds, stream);
                else if (!few && held(256) >= vecs)
                    launch_held<TYPE, OP, FEAT, 256, H>(a, vecs, lds, stream);
                else if (!few && held(512) >= vecs / 4 * 3)
                    launch_held<TYPE, OP, FEAT, 512, H>(a, vecs, lds, stream);
                else
                    launch_held<TYPE, OP, FEAT, 1024, H>(a, vecs, lds, stream);
            }
        }
    } else if (stage == STAGE_SUMS) {
        k_loss_sums<TYPE, OP, FEAT, 256><<<dim3((unsigned) a.rows * a.chunks), 256, lds, stream>>>(a);
    } else {
        k_loss_grad<TYPE, OP, FEAT, 256>
            <<<dim3((unsigned) a.rows * chunks), 256, lds, stream>>>(a, chunks, chunk_vecs);
    }
}

} // namespace

template <int TYPE>
void launch_loss(LossStage stage, int op, int feat, const LossArgs &a, size_t lds, int chunks,
                 int chunk_vecs, hipStream_t stream) {
#define GS_CASE(OP, FEAT)                                                                       \
    if (op == OP && feat == (FEAT))                                                             \
        return launch_one<TYPE, OP, (FEAT)>(stage, a, lds, chunks, chunk_vecs, stream);
    /* (soft-cap and mask together come with the entropy's sum, wanted or not) */
    GS_CASE(OP_TOKEN, 0)
    GS_CASE(OP_TOKEN, F_ENTROPY)
    GS_CASE(OP_TOKEN, F_CAP)
    GS_CASE(OP_TOKEN, F_CAP | F_ENTROPY)
    GS_CASE(OP_TOKEN, F_BITS)
    GS_CASE(OP_TOKEN, F_BITS | F_ENTROPY)
    GS_CASE(OP_TOKEN, F_CAP | F_BITS | F_ENTROPY)
    GS_CASE(OP_DISTILL, 0)
    GS_CASE(OP_DISTILL, F_CAP)
    GS_CASE(OP_DISTILL, F_BITS)
    GS_CASE(OP_DISTILL, F_CAP | F_BITS)
    GS_CASE(OP_PREFERENCE, 0)
    GS_CASE(OP_PREFERENCE, F_CAP)
    GS_CASE(OP_PREFERENCE, F_BITS)
    GS_CASE(OP_PREFERENCE, F_CAP | F_BITS)
    if constexpr (TYPE != GEIST_HIP_TYPE_F32) {
        GS_CASE(OP_TOKEN, F_CAP | F_WIDE | F_BITS | F_ENTROPY)
        GS_CASE(OP_DISTILL, F_CAP | F_WIDE | F_BITS)
        GS_CASE(OP_PREFERENCE, F_CAP | F_WIDE | F_BITS)
    }
#undef GS_CASE
}

} // namespace gs
#endif /* GEIST_LOSS_ROWS_KERNELS_H */
