"""The losses of include/geist_loss_hip.h written down in binary64 with numpy, row by row, and how far
a binary32 evaluation may be from them. Test infrastructure.

Tolerances. The device forms u_i = (y_i - m) k in binary32 (a rounded difference, a rounded k and a
rounded product: 3/2 units of 2^-24 |u_i| each way, at most 2 with the capped y's own rounding below),
2^u by an instruction good to one unit in the last place (2^-23), sums of positive terms per thread in
binary32 (fewer than 64 terms after one another here: 64 * 2^-24) and the rest in binary64, and rounds
a product or two more. So p_i is off by at most
    p_i * (ln2 * 2 |u_i| + 64 + 8) * 2^-24 =: p_i * rel_i
and a sum of log-probabilities by (72 + ln2 * 2 |u|) * 2^-24 per term. A soft-cap c forms
tanh from one 2^z and one reciprocal: y is off by at most c * 2^-21 (two ulps of 2^z near 1, one of the
reciprocal, two products), which moves u by c k 2^-21 and p by the same amount relative. A stored value is
rounded once more: half a step of its type, or half the smallest step there.
"""
import numpy as np

LN2 = np.log(2.0)
U24 = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SMALLEST = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}


class Row:
    """p, log p and slope of one row, and the tolerances of p and log p."""

    def __init__(self, x, temperature, cap, allowed):
        x = x.astype(np.float64)
        n = x.size
        self.ok = np.ones(n, bool) if allowed is None else allowed
        x = np.where(self.ok, x, 0.0)
        with np.errstate(over="ignore", invalid="ignore"):
            if cap:
                t = np.tanh(x / cap)
                y, slope = cap * t, 1.0 / np.cosh(np.clip(x / cap, -300, 300)) ** 2
            else:
                y, slope = x, np.ones(n)
            v = np.where(self.ok, y / temperature, -np.inf)
            m = v.max()
            self.empty = m == -np.inf
            if self.empty:
                self.lp = np.full(n, -np.inf)
                self.p = np.zeros(n)
            else:
                with np.errstate(divide="ignore"):
                    self.lp = (v - m) - np.log(np.exp(v - m).sum())
                self.p = np.exp(self.lp)
            u = np.where(self.p > 0, np.minimum(np.abs(v - m), 800.0), 0.0) / LN2
        self.slope = np.where(self.ok, slope / temperature, 0.0)
        self.rel = (LN2 * 2 * u + 72) * U24 + cap / temperature * 2.0 ** -21
        if cap:   # the slope 4 e / (1 + e)^2, e = 2^z: z is rounded, e and 1 / (1 + e) by an ulp
            self.rel = self.rel + (2 * np.minimum(np.abs(x) / cap, 200.0) * 2 + 8) * U24
        self.lp_tol = self.rel            # of log p_i, absolute
        self.lse_tol = 72 * U24 + cap / temperature * 2.0 ** -21


def stored(g, dtype):
    return np.abs(g) * HALF_STEP[dtype] * 1.001 + SMALLEST[dtype]


def distill(x, dtype, ids, values, tail, temperature=1.0, cap=0.0, allowed=None, weight=1.0):
    """(loss, gradient) and their tolerances for one row. ids, values: the entries that are given."""
    r = Row(x, temperature, cap, allowed)
    n = x.size
    seen, at, val = set(), [], []
    for i, v in zip(ids, values):
        if 0 <= i < n and v > -np.inf and r.ok[i] and i not in seen:
            seen.add(i)
            at.append(int(i))
            val.append(float(v))
    at, val = np.array(at, int), np.array(val, np.float64)
    zero = np.zeros(n)
    if weight == 0.0 or r.empty or (not tail and at.size == 0):
        return 0.0, zero, 0.0, zero
    mag = np.zeros(n)
    with np.errstate(divide="ignore", invalid="ignore"):
        if tail:
            q = np.exp(val)
            rest = max(0.0, 1.0 - q.sum())
            mass = max(1.0, q.sum())      # q.sum() + rest: what the row's log-sum is multiplied by
            out = np.ones(n, bool)
            out[at] = False
            out &= r.ok
            p_rest = r.p[out].sum()
            if p_rest == 0.0 and rest > 0.0:
                lp_rest = logsumexp(r.lp[out]) if out.any() else -np.inf
            else:
                lp_rest = np.log(p_rest)
            loss = (q * (val - r.lp[at])).sum() + (rest * (np.log(rest) - lp_rest) if rest > 0 else 0)
            share = np.exp(r.lp[out] - lp_rest) if np.isfinite(lp_rest) else 0.0
            g = np.zeros(n)
            g[out] = mass * r.p[out] - rest * share
            g[at] = mass * r.p[at] - q
            mag[out] = mass * r.p[out] + rest * share
            mag[at] = mass * r.p[at] + q
            tol = (q * (r.lp_tol[at] + (np.abs(val) + np.abs(r.lp[at])) * 4 * U24)).sum() \
                + rest * 2 * (r.lse_tol + 4 * U24)
            # rest share sits against a reference of its own: the same bound, u from there
        else:
            v = val / temperature
            lq = v - (v.max() + np.log(np.exp(v - v.max()).sum()))
            q = np.exp(lq)
            some = q > 0
            loss = (q[some] * (lq[some] - r.lp[at][some])).sum()
            g = r.p.copy()
            g[at] -= q
            mag = r.p.copy()
            mag[at] += q
            tol = (q * (r.lp_tol[at] + (np.abs(lq) + np.abs(r.lp[at])) * 4 * U24))[some].sum()
    scale = weight * r.slope
    g = g * scale
    g_tol = mag * np.abs(scale) * r.rel + stored(g, dtype)
    loss *= weight
    return loss, g, abs(weight) * tol + abs(loss) * 2.0 ** -23 + 1e-37, g_tol


def logsumexp(v):
    m = v.max()
    return -np.inf if m == -np.inf else m + np.log(np.exp(v - m).sum())


def policy(x, dtype, token, advantage, old, ref, weight=1.0, low=0.2, high=0.2, kl=0.0, ent=0.0,
           temperature=1.0, cap=0.0, allowed=None):
    """dict of loss, logprob, entropy, grad for one row and of their tolerances."""
    r = Row(x, temperature, cap, allowed)
    n = x.size
    some = r.p > 0
    H = -(r.p[some] * r.lp[some]).sum() if not r.empty else 0.0
    H_tol = (r.p[some] * (r.rel[some] * (1 + np.abs(r.lp[some])))).sum() + H * 8 * U24 + 1e-37
    used = 0 <= token < n
    lp = (r.lp[token] if r.ok[token] else -np.inf) if used else 0.0
    zero = np.zeros(n)
    res = {"loss": 0.0, "logprob": lp, "entropy": H, "grad": zero,
           "loss_tol": 0.0, "entropy_tol": H_tol, "grad_tol": zero,
           "logprob_tol": r.lp_tol[token] + abs(lp) * 4 * U24 if used and lp > -np.inf else 0.0}
    if not used or lp == -np.inf or weight == 0.0:
        return res
    e = res["logprob_tol"]
    d = loss = tol = d_tol = 0.0
    ratio = 1.0 if old is None else np.exp(lp - old)
    e_ratio = 0.0 if old is None else e
    if advantage != 0.0:
        free, held = ratio * advantage, min(max(ratio, 1 - low), 1 + high) * advantage
        loss = -min(free, held)
        d = -free if free <= held else 0.0
        tol = abs(free) * e_ratio
        d_tol = abs(d) * e_ratio
    if ref is not None:
        far = ref - lp
        loss += kl * (np.expm1(far) - far)
        d -= kl * np.expm1(far)
        tol += kl * abs(np.expm1(far)) * e
        d_tol += kl * np.exp(far) * e
    loss -= ent * H
    tol += abs(ent) * H_tol
    g = -d * r.p
    g[token] += d
    mag = abs(d) * r.p
    mag[token] += abs(d)
    lp_fin = np.where(some, r.lp, 0.0)
    g = g + ent * r.p * (lp_fin + H)
    mag = mag + abs(ent) * r.p * (1 + np.abs(lp_fin) + H) * 2
    scale = weight * r.slope
    delta = np.zeros(n)
    delta[token] = 1.0
    g_tol = (mag * r.rel + (r.p + delta) * d_tol + abs(ent) * r.p * H_tol) * np.abs(scale)
    res.update(loss=weight * loss, loss_tol=abs(weight) * tol + abs(weight * loss) * 2.0 ** -23 + 1e-37,
               grad=g * scale, grad_tol=g_tol + stored(g * scale, dtype))
    return res


def preference(x, dtype, tokens, ref, start, weight=None, kind="sigmoid", beta=0.1, margin=0.0,
               smoothing=0.0, normalised=False, temperature=1.0, cap=0.0, allowed=None):
    """dict of loss, ratios, logprob, grad over all rows (NaN where nothing is written) and tolerances."""
    rows, n = x.shape
    pairs = (len(start) - 1) // 2
    lp, lp_tol = np.full(rows, np.nan), np.zeros(rows)
    grad, grad_tol = np.full((rows, n), np.nan), np.zeros((rows, n))
    views = {}
    for r in range(start[0], start[-1]):
        views[r] = Row(x[r], temperature, cap, None if allowed is None else allowed[r])
        t = tokens[r]
        lp[r] = 0.0
        grad[r] = 0.0
        if 0 <= t < n:
            lp[r] = views[r].lp[t] if views[r].ok[t] else -np.inf
            if lp[r] > -np.inf:
                lp_tol[r] = views[r].lp_tol[t] + abs(lp[r]) * 4 * U24
    counts = [r in views and 0 <= tokens[r] < n and lp[r] > -np.inf for r in range(rows)]
    ratios, r_tol, share = np.zeros(2 * pairs), np.zeros(2 * pairs), np.ones(2 * pairs)
    for s in range(2 * pairs):
        mine = [r for r in range(start[s], start[s + 1]) if counts[r]]
        if normalised:
            share[s] = 1.0 / max(1, len(mine))
        ratios[s] = share[s] * sum(lp[r] - (0.0 if ref is None else float(ref[r])) for r in mine)
        r_tol[s] = share[s] * sum(lp_tol[r] for r in mine) + abs(ratios[s]) * 2.0 ** -23 + 1e-37
    loss, loss_tol = np.zeros(pairs), np.zeros(pairs)
    for i in range(pairs):
        w = 1.0 if weight is None else float(weight[i])
        gap, e = ratios[2 * i] - ratios[2 * i + 1], r_tol[2 * i] + r_tol[2 * i + 1]
        h = beta * gap - margin
        if kind == "squared":
            off = gap - 0.5 / beta
            loss[i], d, curve = off * off, 2 * off, 2.0
        elif kind == "hinge":
            loss[i], d, curve = max(0.0, 1 - h), (-beta if h < 1 else 0.0), 0.0
        else:
            loss[i] = (1 - smoothing) * np.logaddexp(0, -h) + smoothing * np.logaddexp(0, h)
            d, curve = beta * (smoothing - np.exp(-np.logaddexp(0, h))), beta * beta / 4
        if w == 0.0:
            loss[i] = d = curve = 0.0
        loss_tol[i] = abs(w) * (abs(d) * e + curve * e * e) + abs(w * loss[i]) * 2.0 ** -23 + 1e-37
        loss[i] *= w
        for side in (0, 1):
            s = 2 * i + side
            c = w * share[s] * (-d if side else d)
            c_tol = abs(w) * share[s] * curve * e + abs(c) * 2.0 ** -23
            for r in range(start[s], start[s + 1]):
                if not counts[r]:
                    continue
                v = views[r]
                g = -c * v.p
                g[tokens[r]] += c
                mag = v.p.copy()
                mag[tokens[r]] += 1.0
                scale = v.slope
                grad[r] = g * scale
                grad_tol[r] = (mag * v.rel * abs(c) + mag * c_tol) * np.abs(scale) + stored(
                    g * scale, dtype)
    return {"loss": loss, "ratios": ratios, "logprob": lp, "grad": grad, "loss_tol": loss_tol,
            "ratios_tol": r_tol, "logprob_tol": lp_tol, "grad_tol": grad_tol}
