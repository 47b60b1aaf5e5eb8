"""The losses over logit rows and their gradients (include/geist_loss_hip.h) through the C ABI, against
their binary64 statement (loss_reference.py) under the tolerances derived there."""
import numpy as np
import pytest

import loss_reference as ref
from gpu_util import pack_allowed

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAD = 7.0   # what gradients hold before a call


@pytest.fixture(scope="module")
def hs():
    from geistlib_amd import HipSampler
    s = HipSampler(1, 1)
    yield s
    s.close()


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


class Batch:
    """Rows in device memory with NaN around them, a gradient with PAD around it, and what the rows
    hold as float32 on the host."""

    def __init__(self, x, dtype, lead=0, pad=0, grad="apart", grad_lead=None, grad_pad=None, allowed=None,
                 temperature=1.0, cap=0.0):
        from geistlib_amd import HipSampler
        rows, n = x.shape
        self.rows, self.n, self.dtype = rows, n, dtype
        flat = torch.full((lead + rows * (n + pad) + 8,), float("nan"), dtype=TYPES[dtype], device="cuda")
        self.flat = flat
        self.logits = flat[lead: lead + rows * (n + pad)].view(rows, n + pad)[:, :n]
        self.logits.copy_(dev(x).to(TYPES[dtype]))
        self.x = self.logits.float().cpu().numpy()
        self.grad = self.gflat = None
        self.glead, self.gpad = lead if grad_lead is None else grad_lead, pad if grad_pad is None else grad_pad
        if grad == "apart":
            self.gflat = torch.full((self.glead + rows * (n + self.gpad) + 8,), PAD, dtype=TYPES[dtype],
                                    device="cuda")
            self.grad = self.gflat[self.glead: self.glead + rows * (n + self.gpad)].view(
                rows, n + self.gpad)[:, :n]
        elif grad == "in place":
            self.grad = self.logits
        self.d_allowed = None if allowed is None else dev(pack_allowed(allowed))
        self.ws = torch.full((max(16, HipSampler.loss_workspace_bytes(rows, n)),), 0xA5, dtype=torch.uint8,
                             device="cuda")
        self.view = HipSampler.loss_rows(self.logits, grad=self.grad, allowed=self.d_allowed,
                                         temperature=temperature, softcap=cap)

    def grads(self):
        """The gradient; nothing around it may have changed."""
        if self.gflat is not None:
            around = self.gflat.clone()
            around[self.glead: self.glead + self.rows * (self.n + self.gpad)].view(
                self.rows, self.n + self.gpad)[:, :self.n] = PAD
            assert bool((around == PAD).all())
        else:
            around = self.flat.clone()
            off = self.logits.storage_offset()
            around[off: off + self.rows * self.logits.stride(0)].view(self.rows, -1)[:, :self.n] = float("nan")
            assert bool(torch.isnan(around).all())
        return self.grad.double().cpu().numpy()


def out(n):
    return torch.full((n,), -77.0, device="cuda")


def near(got, want, tol, what):
    got, want, tol = (np.atleast_1d(np.asarray(v, np.float64)) for v in (got, want, tol))
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= tol))
    if bad.any():
        i = tuple(int(v[0]) for v in np.nonzero(bad))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off, first {i}: {got[i]!r} for "
                             f"{want[i]!r} +- {tol[i]:.3g}")


def logits(g, rows, n, scale=2.0):
    x = g.standard_normal((rows, n)) * scale
    for r in range(rows):
        x[r, g.integers(0, n, min(n, 6))] += g.uniform(2, 9)
    return x


# rows, vocabulary, type, elements in front of the first row, between rows
SHAPES = [(1, 1, "f32", 0, 0), (3, 2, "bf16", 1, 3), (5, 7, "f16", 3, 0), (2, 64, "f32", 1, 0),
          (4, 63, "bf16", 5, 1), (9, 1000, "f16", 0, 24), (3, 4097, "f32", 0, 0), (3, 20011, "bf16", 0, 0),
          (2, 20011, "f32", 3, 2), (4, 32768, "f16", 0, 0), (17, 9001, "bf16", 7, 0), (1, 40000, "f32", 0, 0),
          (700, 333, "bf16", 0, 0), (520, 1025, "f32", 2, 1), (600, 8200, "f16", 0, 0)]
# temperature, soft-cap, mask
OPTIONS = [(1.0, 0.0, False), (0.7, 0.0, True), (1.3, 20.0, False), (1.0, 30.0, True)]


def some_rows(rows):
    return range(rows) if rows <= 20 else sorted({0, 1, rows // 3, rows // 2, rows - 2, rows - 1})


def mask_of(g, rows, n, masked):
    if not masked:
        return None
    allowed = g.random((rows, n)) < 0.6
    allowed[:, g.integers(0, n)] = True
    if rows > 2:
        allowed[2] = False          # a row that may answer nothing
    return allowed


def distill_inputs(g, rows, n, k):
    ids = np.stack([g.permutation(max(n, k))[:k] for _ in range(rows)]).astype(np.int32)
    ids[ids >= n] = -1
    if k > 3:
        ids[:, 2] = ids[:, 0]       # listed before
        ids[0, 1] = n               # outside
    lead = g.standard_normal((rows, k)) * 1.5
    values = (lead - np.log(np.exp(lead).sum(1, keepdims=True)) - 0.2).astype(np.float32)
    if k > 4:
        values[-1, 4] = -np.inf
    return ids, values


def check_distill(hs, batch, ids, values, tail, count=None, weight=None, temperature=1.0, cap=0.0,
                  allowed=None, loss_too=True):
    from geistlib_amd import HipSampler
    rows, k = ids.shape
    d_ids, d_values = dev(ids), dev(values)
    d_count = None if count is None else dev(count.astype(np.int32))
    d_weight = None if weight is None else dev(weight.astype(np.float32))
    t = HipSampler.teacher(d_ids, d_values, d_count, d_weight, tail)
    loss = out(rows) if loss_too else None
    hs.distill(batch.view, t, loss, batch.ws)
    hs.sync()
    got = loss.cpu().numpy() if loss_too else None
    grads = batch.grads() if batch.grad is not None else None
    for r in some_rows(rows):
        m = k if count is None else min(k, max(0, int(count[r])))
        want, g, tol, g_tol = ref.distill(
            batch.x[r], batch.dtype, ids[r, :m], values[r, :m], tail, temperature, cap,
            None if allowed is None else allowed[r], 1.0 if weight is None else float(weight[r]))
        if loss_too:
            near(got[r], want, tol, f"loss of row {r}")
        if grads is not None:
            near(grads[r], g, g_tol, f"gradient of row {r}")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature,cap,masked", OPTIONS)
@pytest.mark.parametrize("rows,n,dtype,lead,pad", SHAPES)
def test_distill(hs, rows, n, dtype, lead, pad, temperature, cap, masked, tail):
    g = np.random.default_rng(rows * 7 + n + tail)
    allowed = mask_of(g, rows, n, masked)
    b = Batch(logits(g, rows, n), dtype, lead, pad, allowed=allowed, temperature=temperature, cap=cap)
    k = int(g.integers(1, 40))
    ids, values = distill_inputs(g, rows, n, k)
    check_distill(hs, b, ids, values, tail, count=g.integers(0, k + 2, rows), weight=g.uniform(0.1, 2, rows),
                  temperature=temperature, cap=cap, allowed=allowed)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,n", [(3, 50000), (520, 3000)])
def test_distill_with_the_longest_lists(hs, rows, n, tail):
    g = np.random.default_rng(n)
    b = Batch(logits(g, rows, n), "f32")
    ids, values = distill_inputs(g, rows, n, 1024)
    ids[:, 500:600] = ids[:, 100:200]
    ids[1] = ids[1, 0]              # one token a thousand times
    check_distill(hs, b, ids, values, tail)


def test_distill_lists_every_token(hs):
    """No token is left for the tail: with mass left over the loss is infinite, without it is not."""
    g = np.random.default_rng(1)
    n = 33
    b = Batch(logits(g, 2, n), "f32")
    ids = np.stack([g.permutation(n), g.permutation(n)]).astype(np.int32)
    values = np.log(np.full((2, n), 1 / n)).astype(np.float32)
    values[0] -= 0.5
    values[1] += 0.01
    check_distill(hs, b, ids, values, True)


def test_distill_mass_far_below_the_listed_tokens(hs):
    """The tail's and the list's sums have references of their own: neither vanishes."""
    g = np.random.default_rng(2)
    x = g.standard_normal((2, 300))
    x[0, 5:9] += 400.0
    x[1, 5:9] -= 400.0
    b = Batch(x, "f32")
    ids = np.tile(np.arange(5, 9, dtype=np.int32), (2, 1))
    values = np.log(np.full((2, 4), 0.2)).astype(np.float32)
    check_distill(hs, b, ids, values, True)


def policy_inputs(g, rows, n, batch, temperature, cap, allowed):
    tokens = g.integers(0, n, rows).astype(np.int32)
    for r in range(rows):
        if g.random() < 0.5:
            tokens[r] = int(np.argmax(batch.x[r] if allowed is None else np.where(allowed[r], batch.x[r], -1e30)))
    tokens[g.random(rows) < 0.15] = -1
    if rows > 4:
        tokens[4] = n
    lp = np.array([ref.policy(batch.x[r], "f32", int(tokens[r]), 1.0, None, None, temperature=temperature,
                              cap=cap, allowed=None if allowed is None else allowed[r])["logprob"]
                   if r in some_rows(rows) else -5.0 for r in range(rows)])
    lp = np.where(np.isfinite(lp), lp, -3.0)
    # (a ratio on the very border of the clip range would be decided by rounding)
    old = (lp + g.choice([-0.6, -0.1, 0.05, 0.1, 0.6], rows)).astype(np.float32)
    rf = (lp + 0.4 * g.standard_normal(rows)).astype(np.float32)
    advantage = g.standard_normal(rows).astype(np.float32)
    advantage[0] = 0.0
    return tokens, advantage, old, rf


@pytest.mark.parametrize("kl,ent,with_old", [(0.0, 0.0, True), (0.1, 0.02, True), (0.05, 0.0, False)])
@pytest.mark.parametrize("temperature,cap,masked", OPTIONS)
@pytest.mark.parametrize("rows,n,dtype,lead,pad", SHAPES)
def test_policy(hs, rows, n, dtype, lead, pad, temperature, cap, masked, kl, ent, with_old):
    from geistlib_amd import HipSampler
    g = np.random.default_rng(rows * 7 + n)
    allowed = mask_of(g, rows, n, masked)
    b = Batch(logits(g, rows, n), dtype, lead, pad, allowed=allowed, temperature=temperature, cap=cap)
    tokens, advantage, old, rf = policy_inputs(g, rows, n, b, temperature, cap, allowed)
    weight = g.uniform(0.1, 2, rows).astype(np.float32)
    weight[rows // 2] = 0.0
    d = [dev(v) for v in (tokens, advantage, old, rf, weight)]
    p = HipSampler.policy(d[0], d[1], old=d[2] if with_old else None, ref=d[3] if kl else None, weight=d[4],
                          clip_low=0.2, clip_high=0.28, kl_coef=kl, entropy_coef=ent)
    loss, lp, ent_out = out(rows), out(rows), out(rows)
    hs.policy_loss(b.view, p, loss, lp, ent_out, b.ws)
    hs.sync()
    grads = b.grads()
    for r in some_rows(rows):
        want = ref.policy(b.x[r], dtype, int(tokens[r]), float(advantage[r]),
                          float(old[r]) if with_old else None, float(rf[r]) if kl else None,
                          weight=float(weight[r]), low=float(np.float32(0.2)), high=float(np.float32(0.28)),
                          kl=float(np.float32(kl)), ent=float(np.float32(ent)), temperature=temperature, cap=cap,
                          allowed=None if allowed is None else allowed[r])
        for name, got in (("loss", loss), ("logprob", lp), ("entropy", ent_out)):
            near(got[r].item(), want[name], want[name + "_tol"] + abs(want[name]) * 2.0 ** -23
                 if np.isfinite(want[name]) else 0.0, f"{name} of row {r}")
        near(grads[r], want["grad"], want["grad_tol"], f"gradient of row {r}")
    # without the entropy asked for, and the gradient alone
    again = b.grad.clone()
    b.grad.fill_(3.0)
    hs.policy_loss(b.view, p, None, None, None, b.ws)
    hs.sync()
    for r in some_rows(rows):
        want = again[r].double().cpu().numpy()
        near(b.grad[r].double().cpu().numpy(), want, np.abs(want) * 2 * ref.HALF_STEP[dtype]
             + 2 * ref.SMALLEST[dtype] + np.abs(want).max() * 2.0 ** -20, f"row {r} alone")


PREFERENCES = [("sigmoid", 0.0, 0.0, False, True), ("sigmoid", 0.1, 0.5, True, False),
               ("hinge", 0.0, 0.25, False, True), ("squared", 0.0, 0.0, True, True)]


@pytest.mark.parametrize("kind,smoothing,margin,normalised,with_ref", PREFERENCES)
@pytest.mark.parametrize("temperature,cap,masked", OPTIONS[:3])
@pytest.mark.parametrize("rows,n,dtype,lead,pad", [s for s in SHAPES if s[0] < 100 and s[0] > 1]
                         + [(530, 70, "f16", 0, 0)])
def test_preference(hs, rows, n, dtype, lead, pad, temperature, cap, masked, kind, smoothing, margin,
                    normalised, with_ref):
    from geistlib_amd import HipSampler
    g = np.random.default_rng(rows + n)
    allowed = mask_of(g, rows, n, masked)
    b = Batch(logits(g, rows, n), dtype, lead, pad, allowed=allowed, temperature=temperature, cap=cap)
    pairs = 2 if rows < 9 else 3
    start = np.sort(g.integers(0, rows + 1, 2 * pairs + 1)).astype(np.int32)
    if rows >= 9:
        start[0], start[-1] = 1, rows - 2     # rows that belong to no sequence on either side
        start[2] = start[1]                   # an empty sequence
    tokens = np.argmax(b.x, 1).astype(np.int32)
    tokens[g.random(rows) < 0.3] = -1
    tokens[g.random(rows) < 0.3] = int(g.integers(0, n))
    rf = (-1.0 - g.random(rows)).astype(np.float32)
    weight = g.uniform(0.2, 2, pairs).astype(np.float32)
    d = [dev(v) for v in (tokens, start, rf, weight)]
    p = HipSampler.preference(d[0], d[1], ref=d[2] if with_ref else None, weight=d[3], kind=kind, beta=0.25,
                              margin=margin, label_smoothing=smoothing, length_normalised=normalised)
    loss, ratios, lp = out(pairs), out(2 * pairs), out(rows)
    hs.preference_loss(b.view, p, loss, ratios, lp, b.ws)
    hs.sync()
    want = ref.preference(b.x, dtype, tokens, rf if with_ref else None, start, weight, kind, 0.25, margin,
                          float(np.float32(smoothing)), normalised, temperature, cap, allowed)
    near(loss.cpu(), want["loss"], want["loss_tol"], "loss")
    near(ratios.cpu(), want["ratios"], want["ratios_tol"], "ratios")
    lps, grads = lp.cpu().numpy(), b.grads()
    inside = np.arange(rows)
    inside = (inside >= start[0]) & (inside < start[-1])
    assert (lps[~inside] == -77.0).all() and (grads[~inside] == PAD).all()
    near(lps[inside], want["logprob"][inside], want["logprob_tol"][inside] + 1e-30, "logprob")
    near(grads[inside], want["grad"][inside], want["grad_tol"][inside], "gradient")


@pytest.mark.parametrize("rows,n,dtype", [(4, 9001, "bf16"), (530, 1000, "f32"), (2, 30000, "f16")])
def test_gradient_in_the_place_of_the_logits(hs, rows, n, dtype):
    """d_grad == d_logits gives the same values as a gradient of its own, for all three losses."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n)
    x = logits(g, rows, n)
    ids, values = distill_inputs(g, rows, n, 12)
    tokens = g.integers(0, n, rows).astype(np.int32)
    half = rows // 2
    d_ids, d_val, d_tok = dev(ids), dev(values), dev(tokens)
    d_adv, d_start = dev(g.standard_normal(rows).astype(np.float32)), dev(np.array([0, half, rows], np.int32))
    for tail in (False, True):
        t = HipSampler.teacher(d_ids, d_val, tail=tail)
        p = HipSampler.policy(d_tok, d_adv, ref=d_adv, kl_coef=0.1, entropy_coef=0.01)
        q = HipSampler.preference(d_tok, d_start)
        for what in ("distill", "policy", "preference"):
            res = []
            for grad in ("apart", "in place"):
                b = Batch(x, dtype, 1, 3, grad=grad)
                loss = out(rows)
                if what == "distill":
                    hs.distill(b.view, t, loss, b.ws)
                elif what == "policy":
                    hs.policy_loss(b.view, p, loss, None, None, b.ws)
                else:
                    hs.preference_loss(b.view, q, loss, None, None, b.ws)
                hs.sync()
                res.append((loss.cpu().numpy(), b.grads()))
            assert (res[0][0] == res[1][0]).all() and (res[0][1] == res[1][1]).all(), what


def test_gradient_with_strides_of_its_own(hs):
    """Gradient rows that start elsewhere within 16 bytes than the logits' rows do."""
    g = np.random.default_rng(4)
    for dtype, lead, pad, gl, gp in [("bf16", 0, 0, 3, 1), ("f32", 1, 2, 0, 0), ("f16", 2, 6, 5, 6)]:
        for rows in (3, 515):
            n = 5003
            b = Batch(logits(g, rows, n), dtype, lead, pad, grad_lead=gl, grad_pad=gp)
            ids, values = distill_inputs(g, rows, n, 9)
            check_distill(hs, b, ids, values, True)


@pytest.mark.parametrize("rows", [4, 600])
@pytest.mark.parametrize("cap", [0.0, 10.0])
def test_special_values(hs, rows, cap):
    """Rows of the type's lowest value, infinities and NaN: in masked places, as logits, in one row only."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(6)
    n = 9000
    x = logits(g, rows, n)
    allowed = g.random((rows, n)) < 0.5
    allowed[:, :40] = True
    x[~allowed] = g.choice([np.nan, np.inf, -np.inf, 3e38], int((~allowed).sum()))
    x[0, 30:] = -np.finfo(np.float32).max       # a mask of the lowest value
    x[1] = -np.finfo(np.float32).max            # ... that leaves nothing else: uniform
    x[2, 5] = np.nan                            # one spoilt row
    x[3] = -np.inf                              # nothing left (a soft-cap makes it -cap everywhere: uniform)
    spoilt = (2,) if cap else (2, 3)
    tokens = np.full(rows, 3, np.int32)
    d_tok, d_adv = dev(tokens), dev(np.ones(rows, np.float32))
    ids = np.tile(np.array([3, 17, 8999], np.int32), (rows, 1))
    values = np.log(np.tile(np.array([0.5, 0.2, 0.1]), (rows, 1))).astype(np.float32)
    for tail in (False, True):
        b = Batch(x, "f32", allowed=allowed, cap=cap)
        loss = out(rows)
        d_ids, d_val = dev(ids), dev(values)
        hs.distill(b.view, HipSampler.teacher(d_ids, d_val, tail=tail), loss, b.ws)
        hs.sync()
        got, grads = loss.cpu().numpy(), b.grads()
        assert np.isnan(got[2]) and np.isnan(grads[2][allowed[2]]).all()
        assert cap or (got[3] == 0.0 and (grads[3] == 0).all())
        for r in [r for r in some_rows(rows) if r not in spoilt]:
            want, gr, tol, g_tol = ref.distill(b.x[r], "f32", ids[r], values[r], tail, 1.0, cap, allowed[r])
            near(got[r], want, tol, f"loss of row {r}")
            near(grads[r], gr, g_tol, f"gradient of row {r}")
    b = Batch(x, "f32", allowed=allowed, cap=cap)
    loss, lp, ent = out(rows), out(rows), out(rows)
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, entropy_coef=0.01), loss, lp, ent, b.ws)
    hs.sync()
    grads = b.grads()
    assert np.isnan(loss[2].item()) and np.isnan(ent[2].item())
    if not cap:
        assert loss[3].item() == 0.0 and lp[3].item() == -np.inf and ent[3].item() == 0.0
        assert (grads[3] == 0).all()
    for r in [r for r in some_rows(rows) if r not in spoilt]:
        want = ref.policy(b.x[r], "f32", 3, 1.0, None, None, ent=float(np.float32(0.01)), cap=cap,
                          allowed=allowed[r])
        near(loss[r].item(), want["loss"], want["loss_tol"], f"loss of row {r}")
        near(ent[r].item(), want["entropy"], want["entropy_tol"] + want["entropy"] * 2.0 ** -23, f"entropy {r}")
        near(grads[r], want["grad"], want["grad_tol"], f"gradient of row {r}")
    # the pair of a spoilt row is NaN, the other pair is not
    b = Batch(x[:4], "f32", allowed=allowed[:4], cap=cap)
    loss = out(2)
    d_start = dev(np.array([2, 3, 4, 4, 4], np.int32))
    hs.preference_loss(b.view, HipSampler.preference(d_tok[:4], d_start), loss, None, None, b.ws)
    hs.sync()
    assert np.isnan(loss[0].item()) and loss[1].item() == pytest.approx(np.log(2))


def test_a_weight_of_zero_leaves_a_row_out(hs):
    from geistlib_amd import HipSampler
    x = np.full((2, 500), np.nan)
    x[1] = 1.0
    d_w, d_tok = dev(np.array([0.0, 1.0], np.float32)), dev(np.array([3, 3], np.int32))
    d_adv = dev(np.ones(2, np.float32))
    b, loss = Batch(x, "f32"), out(2)
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, weight=d_w), loss, None, None, b.ws)
    hs.sync()
    assert loss[0].item() == 0.0 and (b.grads()[0] == 0).all() and loss[1].item() == -1.0
    b, loss = Batch(x, "f32"), out(2)
    d_ids, d_val = dev(np.zeros((2, 1), np.int32)), dev(np.zeros((2, 1), np.float32))
    hs.distill(b.view, HipSampler.teacher(d_ids, d_val, weight=d_w), loss, b.ws)
    hs.sync()
    assert loss[0].item() == 0.0 and (b.grads()[0] == 0).all()
    assert loss[1].item() == pytest.approx(np.log(500), rel=1e-6)


def test_rows_beyond_32_bit_offsets(hs):
    from geistlib_amd import HipSampler
    n, stride = 5000, 2 ** 32 + 64
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 20 GB of device memory")
    g = np.random.default_rng(9)
    base = torch.empty(stride + n, dtype=torch.bfloat16, device="cuda")
    gbase = torch.empty(stride + n, dtype=torch.bfloat16, device="cuda")
    x, gr = (t.as_strided((2, n), (stride, 1)) for t in (base, gbase))
    x.copy_(dev(logits(g, 2, n)))
    tokens, adv = dev(np.array([5, 6], np.int32)), dev(np.array([1.0, -1.0], np.float32))
    ws = torch.empty(HipSampler.loss_workspace_bytes(2, n), dtype=torch.uint8, device="cuda")
    loss = out(2)
    hs.policy_loss(HipSampler.loss_rows(x, grad=gr), HipSampler.policy(tokens, adv), loss, None, None, ws)
    hs.sync()
    for r in range(2):
        want = ref.policy(x[r].float().cpu().numpy(), "bf16", 5 + r, float(adv[r]), None, None)
        near(gr[r].double().cpu().numpy(), want["grad"], want["grad_tol"], f"gradient of row {r}")


@pytest.mark.parametrize("rows,n", [(3, 20000), (530, 2000)])
def test_recorded_calls_replay(rows, n):
    """Recorded into a graph, replayed on changing inputs with eager calls of the same sampler and
    other work in between; every replay gives what an eager call gives."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n)
    stream = torch.cuda.Stream()
    hs = HipSampler(1, 1, stream=stream.cuda_stream)
    b, e = (Batch(logits(g, rows, n), "bf16") for _ in range(2))
    ids, values = distill_inputs(g, rows, n, 10)
    d_ids, d_val = dev(ids), dev(values)
    d_tok, d_adv = dev(g.integers(0, n, rows).astype(np.int32)), dev(g.standard_normal(rows).astype(np.float32))
    d_start = dev(np.array([0, rows // 3, rows], np.int32))
    t = HipSampler.teacher(d_ids, d_val, tail=True)
    p = HipSampler.policy(d_tok, d_adv, entropy_coef=0.01)
    q = HipSampler.preference(d_tok, d_start)
    calls = [lambda v, l: hs.distill(v.view, t, l, v.ws),
             lambda v, l: hs.policy_loss(v.view, p, l, None, None, v.ws),
             lambda v, l: hs.preference_loss(v.view, q, l, None, None, v.ws)]
    for call in calls:
        l_graph, l_eager = out(rows), out(rows)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(b, l_graph)
        for k in range(4):
            x = dev(logits(g, rows, n)).to(torch.bfloat16)
            b.logits.copy_(x)
            e.logits.copy_(x)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            call(e, l_eager)
            stream.synchronize()
            assert torch.equal(l_graph, l_eager) and torch.equal(b.grad, e.grad), k
    hs.close()


def test_two_samplers_on_two_streams(hs):
    """Calls at the same time, each with its workspace, give what they give alone."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [HipSampler(1, 1, stream=s.cuda_stream) for s in streams]
    b = [Batch(logits(g, 5, 60000), "f32") for _ in range(2)]
    d_tok, d_adv = dev(np.arange(5, dtype=np.int32)), dev(np.ones(5, np.float32))
    p = HipSampler.policy(d_tok, d_adv)
    alone = []
    for v in b:
        loss, lp = out(5), out(5)
        hs.policy_loss(v.view, p, loss, lp, None, v.ws)
        hs.sync()
        alone.append((lp.clone(), v.grad.clone()))
    lps = [out(5) for _ in range(2)]
    losses = [out(5) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, v, lp, loss in zip(both, b, lps, losses):
            s.policy_loss(v.view, p, loss, lp, None, v.ws)
    for s in both:
        s.sync()
    for v, lp, want in zip(b, lps, alone):
        assert torch.equal(lp, want[0]) and torch.equal(v.grad, want[1])
    for s in both:
        s.close()


def test_same_inputs_same_bits(hs):
    """Nothing depends on the order of arrival: two calls give the same bits."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(12)
    for rows, n in [(2, 100000), (520, 4000)]:
        b = Batch(logits(g, rows, n), "f32")
        ids, values = distill_inputs(g, rows, n, 200)
        ids[:, 100:] = ids[:, :100]
        d_ids, d_val = dev(ids), dev(values)
        t = HipSampler.teacher(d_ids, d_val, tail=True)
        first = None
        for _ in range(3):
            loss = out(rows)
            hs.distill(b.view, t, loss, b.ws)
            hs.sync()
            now = (loss.clone(), b.grad.clone())
            assert first is None or (torch.equal(first[0], now[0]) and torch.equal(first[1], now[1]))
            first = now


def test_refusals(hs):
    from geistlib_amd import HipSampler
    from geistlib_amd.binding import GeistHipError
    b = Batch(np.zeros((4, 100)), "f32")
    d_tok, d_adv = dev(np.zeros(4, np.int32)), dev(np.zeros(4, np.float32))
    p = HipSampler.policy(d_tok, d_adv)
    loss = out(4)

    def refused(call, text):
        with pytest.raises(GeistHipError) as err:
            call()
        assert err.value.code == 2 and text in str(err.value), str(err.value)

    refused(lambda: hs.policy_loss(b.view, p, loss, None, None, b.ws[:8]), "workspace")
    refused(lambda: hs.policy_loss(b.view, p, loss, None, None, None), "workspace")
    view = HipSampler.loss_rows(b.logits, grad=b.grad, temperature=0.0)
    refused(lambda: hs.policy_loss(view, p, loss, None, None, b.ws), "temperature")
    view = HipSampler.loss_rows(b.logits)
    refused(lambda: hs.policy_loss(view, p, None, None, None, b.ws), "neither")
    q = HipSampler.policy(d_tok, d_adv, kl_coef=0.1)
    refused(lambda: hs.policy_loss(b.view, q, loss, None, None, b.ws), "KL term")
    assert (loss.cpu() == -77.0).all() and (b.grads() == PAD).all()


def test_sampled_scored_and_trained_on(hs, oracle):
    """The operators as they are used one after the other: tokens drawn by the sampler, their
    log-probabilities from the policy call agree with geist_hip_logprob_rows, a step down the policy
    gradient raises what was rewarded; a student moved along the distillation gradient comes nearer to
    its teacher, listed by its own top logits and their log-probabilities."""
    from geistlib_amd import HipSampler, SampleParams
    g = np.random.default_rng(21)
    rows, n, k = 24, 5000, 32
    teacher_x = (g.standard_normal((rows, n)) * 3).astype(np.float32)
    student = dev((teacher_x + g.standard_normal((rows, n))).astype(np.float32))
    teacher_d = dev(teacher_x)
    sampler = HipSampler(rows, n)
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    u = dev((g.integers(0, 1 << 24, rows) / np.float32(1 << 24)).astype(np.float32))
    sampler.sample(HipSampler.rows(student), SampleParams.make(temperature=1.0), u, tokens)
    scored = torch.empty((rows, 1), dtype=torch.float64, device="cuda")
    sampler.logprob(student, tokens.view(rows, 1), scored)
    grad = torch.empty_like(student)
    ws = torch.empty(HipSampler.loss_workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")
    loss, lp, lp2 = out(rows), out(rows), out(rows)
    adv = torch.ones(rows, device="cuda")
    sampler.policy_loss(HipSampler.loss_rows(student, grad=grad), HipSampler.policy(tokens, adv), loss, lp,
                        None, ws)
    sampler.sync()
    near(lp.cpu(), scored[:, 0].cpu(), (72 + 60) * ref.U24 + scored[:, 0].abs().cpu().numpy() * 4 * ref.U24,
         "logprob")
    # the gradient of -lp by the row, against a difference of the library's own double scores
    step = 1e-2
    moved = student - step * grad
    sampler.policy_loss(HipSampler.loss_rows(moved), HipSampler.policy(tokens, adv, old=lp), loss, lp2,
                        None, ws)
    sampler.sync()
    gain = step * (grad.double() ** 2).sum(1)
    rise = (lp2 - lp).double()
    # lp is concave in the row's logits along the step: second derivative at most 1 per squared length
    assert bool((rise <= gain + 2e-5).all()) and bool((rise >= gain - step * gain - 2e-5).all())
    # the teacher's leading tokens and their log-probabilities, from the library itself
    ids = torch.topk(teacher_d, k, 1).indices.to(torch.int32)
    values = torch.empty((rows, k), dtype=torch.float64, device="cuda")
    sampler.logprob(teacher_d, ids, values)
    vals = values.float()
    t = HipSampler.teacher(ids, vals, tail=True)
    l0, l1 = out(rows), out(rows)
    sampler.distill(HipSampler.loss_rows(student, grad=grad), t, l0, ws)
    moved = student - step * grad
    sampler.distill(HipSampler.loss_rows(moved), t, l1, ws)
    sampler.sync()
    gain = step * (grad.double() ** 2).sum(1)
    fall = (l0 - l1).double()
    # sum q log p with one merged event: its curvature along the step is at most 1 per squared length too
    assert bool((fall <= gain * (1 + step) + 2e-5).all()) and bool((fall >= gain * (1 - step) - 2e-5).all())
    # the teacher against itself: no loss, no gradient
    sampler.distill(HipSampler.loss_rows(teacher_d, grad=grad), t, l0, ws)
    sampler.sync()
    assert float(l0.abs().max()) < 2e-5 and float(grad.abs().max()) < 2e-5
    sampler.close()


# few long rows, cut into parts; and long rows of larger batches, of which a workgroup holds a part in
# registers, a part in LDS and reads the rest twice
LONG = [(2, 60001, "f32", 1, 3), (3, 130003, "bf16", 3, 0), (1, 300000, "f16", 0, 0), (40, 110001, "f32", 0, 0)]
HELD_ROWS = [(66, 60000, "f32", 0, 0), (70, 262144, "f32", 0, 0), (34, 131075, "bf16", 1, 2), (65, 262143, "f16", 0, 1),
        (40, 250001, "bf16", 0, 0)]


@pytest.mark.parametrize("temperature,cap,masked", OPTIONS)
@pytest.mark.parametrize("rows,n,dtype,lead,pad", LONG + HELD_ROWS)
def test_long_rows(hs, rows, n, dtype, lead, pad, temperature, cap, masked):
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n)
    base = logits(g, 3, n)
    x = base[np.arange(rows) % 3]
    allowed = None
    if masked:
        allowed = mask_of(g, 3, n, True)[np.arange(rows) % 3]
    look = sorted({0, min(1, rows - 1), min(2, rows - 1), rows - 1})
    b = Batch(x, dtype, lead, pad, allowed=allowed, temperature=temperature, cap=cap)
    weight = g.uniform(0.1, 2, rows).astype(np.float32)
    d_w = dev(weight)
    ids, values = distill_inputs(g, rows, n, 50)
    d_ids, d_val = dev(ids), dev(values)
    loss = out(rows)
    for tail in (False, True):
        hs.distill(b.view, HipSampler.teacher(d_ids, d_val, weight=d_w, tail=tail), loss, b.ws)
        hs.sync()
        grads = b.grads()
        for r in look:
            want, gr, tol, g_tol = ref.distill(b.x[r], dtype, ids[r], values[r], tail, temperature, cap,
                                               None if allowed is None else allowed[r], float(weight[r]))
            near(loss[r].item(), want, tol, f"tail {tail}: loss of row {r}")
            near(grads[r], gr, g_tol, f"tail {tail}: gradient of row {r}")
        alone = out(rows)
        view = HipSampler.loss_rows(b.logits, allowed=b.d_allowed, temperature=temperature, softcap=cap)
        hs.distill(view, HipSampler.teacher(d_ids, d_val, weight=d_w, tail=tail), alone, b.ws)
        hs.sync()
        near(alone.cpu(), loss.cpu(), loss.abs().cpu() * 3e-6 + 1e-7, "loss alone")
    tokens = np.argmax(b.x, 1).astype(np.int32)
    tokens[1::3] = n // 2
    advantage = g.standard_normal(rows).astype(np.float32)
    d_tok, d_adv = dev(tokens), dev(advantage)
    lp, ent = out(rows), out(rows)
    p = HipSampler.policy(d_tok, d_adv, weight=d_w, entropy_coef=0.01)
    hs.policy_loss(b.view, p, loss, lp, ent, b.ws)
    hs.sync()
    grads = b.grads()
    for r in look:
        want = ref.policy(b.x[r], dtype, int(tokens[r]), float(advantage[r]), None, None, float(weight[r]),
                          ent=float(np.float32(0.01)), temperature=temperature, cap=cap,
                          allowed=None if allowed is None else allowed[r])
        for name, got in (("loss", loss), ("logprob", lp), ("entropy", ent)):
            near(got[r].item(), want[name], want[name + "_tol"] + abs(want[name]) * 2.0 ** -23
                 if np.isfinite(want[name]) else 0.0, f"{name} of row {r}")
        near(grads[r], want["grad"], want["grad_tol"], f"gradient of row {r}")
    lp2, ent2 = out(rows), out(rows)
    view = HipSampler.loss_rows(b.logits, allowed=b.d_allowed, temperature=temperature, softcap=cap)
    hs.policy_loss(view, p, loss, lp2, ent2, b.ws)
    hs.sync()
    near(lp2.cpu(), lp.cpu(), lp.abs().cpu() * 3e-6 + 1e-6, "logprob alone")
    near(ent2.cpu(), ent.cpu(), ent.abs().cpu() * 3e-6 + 1e-6, "entropy alone")
    # in the place of the logits: the same bits
    want = b.grad.clone()
    c = Batch(x, dtype, lead, pad, grad="in place", allowed=allowed, temperature=temperature, cap=cap)
    hs.policy_loss(c.view, p, loss, lp, ent, c.ws)
    hs.sync()
    assert torch.equal(c.grad, want)


def test_long_rows_of_special_values(hs):
    """Parts of rows, and what LDS holds of a row, without anything that counts: all masked, of the lowest
    value, NaN behind the mask."""
    from geistlib_amd import HipSampler
    for rows in (3, 70):
        n = 150000
        x = np.zeros((rows, n))
        x[0, 100:] = -np.finfo(np.float32).max     # what counts lies in the first part
        x[1, :-5] = -np.inf                        # ... in the last one
        x[2, 70000:] = np.nan                      # behind the mask
        allowed = np.ones((rows, n), bool)
        allowed[2, 60000:] = False
        b = Batch(x, "f32", allowed=allowed)
        d_tok, d_adv = dev(np.full(rows, 3, np.int32)), dev(np.ones(rows, np.float32))
        loss, lp, ent = out(rows), out(rows), out(rows)
        hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, entropy_coef=0.1), loss, lp, ent, b.ws)
        hs.sync()
        grads = b.grads()
        for r in range(3):
            want = ref.policy(b.x[r], "f32", 3, 1.0, None, None, ent=float(np.float32(0.1)), allowed=allowed[r])
            near(ent[r].item(), want["entropy"], want["entropy_tol"] + want["entropy"] * 2.0 ** -23, f"entropy {r}")
            near(lp[r].item(), want["logprob"], want["logprob_tol"] + 1e-6, f"logprob {r}")
            near(grads[r], want["grad"], want["grad_tol"], f"gradient {r}")


def test_a_batch_beyond_the_cache(hs):
    """Non-temporal reads and writes, the preference loss's second pass from the last row back: what smaller
    batches of the same rows give."""
    from geistlib_amd import HipSampler
    rows, n = 1300, 131072
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn((rows, n), generator=gen, device="cuda") * 2).to(torch.bfloat16)
    g = np.random.default_rng(5)
    tokens = g.integers(0, n, rows).astype(np.int32)
    d_tok, d_adv = dev(tokens), dev(g.standard_normal(rows).astype(np.float32))
    d_start = dev(np.array([0, 300, 650, 1000, 1300], np.int32))
    ws = torch.empty(HipSampler.loss_workspace_bytes(rows, n), dtype=torch.uint8, device="cuda")
    grad = torch.empty_like(x)
    loss, lp = out(rows), out(rows)
    hs.policy_loss(HipSampler.loss_rows(x, grad=grad), HipSampler.policy(d_tok, d_adv), loss, lp, None, ws)
    part = torch.empty((100, n), dtype=torch.bfloat16, device="cuda")
    loss2, lp2 = out(100), out(100)
    for r in (0, 600, 1200):
        hs.policy_loss(HipSampler.loss_rows(x[r:r + 100], grad=part),
                       HipSampler.policy(d_tok[r:r + 100], d_adv[r:r + 100]), loss2, lp2, None, ws)
        hs.sync()
        # (another size is added up in another order: each side is within the bounds of loss_reference)
        near(lp2.cpu(), lp[r:r + 100].cpu(), 2 * (72 + 60) * ref.U24 + lp2.abs().cpu().numpy() * 8 * ref.U24,
             "logprob")
        a, b = part.float(), grad[r:r + 100].float()
        assert bool(((a - b).abs() <= b.abs() * (2 * ref.HALF_STEP["bf16"] + 300 * ref.U24)).all())
    p_loss, ratios = out(2), out(4)
    hs.preference_loss(HipSampler.loss_rows(x, grad=grad), HipSampler.preference(d_tok, d_start), p_loss,
                       ratios, lp, ws)
    hs.sync()
    for r in (0, 299, 300, 649, 1299):
        want = ref.policy(x[r].float().cpu().numpy(), "bf16", int(tokens[r]), 1.0, None, None)
        near(lp[r].item(), want["logprob"], want["logprob_tol"] + 1e-6, f"logprob {r}")
    half = torch.empty((650, n), dtype=torch.bfloat16, device="cuda")
    d_s2 = dev(np.array([0, 350, 650], np.int32))
    hs.preference_loss(HipSampler.loss_rows(x[650:], grad=half), HipSampler.preference(d_tok[650:], d_s2),
                       p_loss[:1].clone(), ratios[:2].clone(), None, ws)
    hs.sync()
    a, b = half.float(), grad[650:].float()
    assert bool(((a - b).abs() <= b.abs() * (2 * ref.HALF_STEP["bf16"] + 300 * ref.U24)).all())


def test_masks_that_leave_a_few_tokens(hs):
    """Most parts of a row, most wavefronts and most first groups have nothing that counts."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(31)
    for rows, n in [(4, 130001), (70, 70000), (300, 9001)]:
        x = logits(g, 3, n)[np.arange(rows) % 3]
        allowed = np.zeros((rows, n), bool)
        for r in range(rows):
            allowed[r, g.integers(0, n, 5)] = True
        tokens = np.array([np.flatnonzero(allowed[r])[0] for r in range(rows)], np.int32)
        adv = g.standard_normal(rows).astype(np.float32)
        d_tok, d_adv = dev(tokens), dev(adv)
        start = np.array([0, rows // 2, rows], np.int32)
        d_start = dev(start)
        b = Batch(x, "bf16", 1, 0, allowed=allowed)
        loss, lp, ent = out(rows), out(rows), out(rows)
        hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, entropy_coef=0.1), loss, lp, ent, b.ws)
        hs.sync()
        grads = b.grads()
        for r in some_rows(rows):
            want = ref.policy(b.x[r], "bf16", int(tokens[r]), float(adv[r]), None, None,
                              ent=float(np.float32(0.1)), allowed=allowed[r])
            near(ent[r].item(), want["entropy"], want["entropy_tol"] + want["entropy"] * 2.0 ** -23, f"entropy {r}")
            near(lp[r].item(), want["logprob"], want["logprob_tol"], f"logprob {r}")
            near(grads[r], want["grad"], want["grad_tol"], f"gradient {r}")
        b = Batch(x, "bf16", 1, 0, allowed=allowed)
        loss, lp = out(1), out(rows)
        hs.preference_loss(b.view, HipSampler.preference(d_tok, d_start, beta=0.25), loss, None, lp, b.ws)
        hs.sync()
        grads = b.grads()
        if rows < 100:
            want = ref.preference(b.x, "bf16", tokens, None, start, beta=0.25, allowed=allowed)
            near(loss.cpu(), want["loss"], want["loss_tol"], "loss")
            near(lp.cpu(), want["logprob"], want["logprob_tol"] + 1e-30, "logprob")
            for r in some_rows(rows):
                near(grads[r], want["grad"][r], want["grad_tol"][r], f"gradient {r}")


@pytest.mark.parametrize("offset", [-1e6, -726817.6, -726900.0, -3e5, 3e5, 4.6e7, 1e9, -3.3e38, 3.3e38])
def test_rows_far_from_zero(hs, offset):
    """Logits at an offset of any size: what the offset leaves of their differences is what counts."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(32)
    for rows, n in [(2, 60000), (3, 5000), (260, 2000)]:
        x = (logits(g, rows, n) + offset).astype(np.float32)
        tokens, adv = np.full(rows, 7, np.int32), np.ones(rows, np.float32)
        ids, values = distill_inputs(g, rows, n, 20)
        d_ids, d_val, d_tok, d_adv = dev(ids), dev(values), dev(tokens), dev(adv)
        d_start = dev(np.array([0, 1, 2], np.int32))
        b = Batch(x, "f32")
        loss, lp, ent = out(rows), out(rows), out(rows)
        hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, entropy_coef=0.1), loss, lp, ent, b.ws)
        hs.sync()
        grads = b.grads()
        for r in some_rows(rows):
            want = ref.policy(b.x[r], "f32", 7, 1.0, None, None, ent=float(np.float32(0.1)))
            near(lp[r].item(), want["logprob"], want["logprob_tol"] + 1e-6, f"logprob {r}")
            near(ent[r].item(), want["entropy"], want["entropy_tol"] + 1e-6, f"entropy {r}")
            near(grads[r], want["grad"], want["grad_tol"], f"gradient {r}")
        for tail in (False, True):
            hs.distill(b.view, HipSampler.teacher(d_ids, d_val, tail=tail), loss, b.ws)
            hs.sync()
            grads = b.grads()
            for r in some_rows(rows):
                want, gr, tol, g_tol = ref.distill(b.x[r], "f32", ids[r], values[r], tail)
                near(loss[r].item(), want, tol, f"tail {tail}: loss {r}")
                near(grads[r], gr, g_tol, f"tail {tail}: gradient {r}")
        p_loss = out(1)
        hs.preference_loss(b.view, HipSampler.preference(d_tok, d_start), p_loss, None, lp, b.ws)
        hs.sync()
        want = ref.preference(b.x[:2], "f32", tokens[:2], None, [0, 1, 2])
        near(p_loss.cpu(), want["loss"], want["loss_tol"], "preference loss")
        for r in range(2):
            near(b.grad[r].double().cpu().numpy(), want["grad"][r], want["grad_tol"][r], f"preference {r}")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [2.0, 64.0, 65.0, 3e4])
def test_soft_caps_small_and_large(hs, dtype, cap):
    """A cap far above the logits leaves them as they are, in 16 bits too; one below them flattens them."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(33)
    rows, n = 3, 5000
    x = logits(g, rows, n, 4.0)
    b = Batch(x, dtype, cap=cap)
    tokens = np.argmax(b.x, 1).astype(np.int32)
    d_tok, d_adv = dev(tokens), dev(np.ones(rows, np.float32))
    loss, lp = out(rows), out(rows)
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv), loss, lp, None, b.ws)
    hs.sync()
    grads = b.grads()
    for r in range(rows):
        want = ref.policy(b.x[r], dtype, int(tokens[r]), 1.0, None, None, cap=cap)
        # (above 64 every type's small arguments are formed to 2^-24 relative: y within 64 * 2^-23)
        slack = 64 * 2.0 ** -23 if cap > 64 else 0.0
        tol = want["logprob_tol"] if cap <= 64 else 100 * ref.U24 + abs(want["logprob"]) * 4 * ref.U24 + slack
        near(lp[r].item(), want["logprob"], tol, f"logprob {r}")
        near(grads[r], want["grad"], want["grad_tol"], f"gradient {r}")


def test_a_recorded_call_with_a_row_in_lds():
    """A workgroup that asks for more LDS than a launch gets unasked, in a graph."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(34)
    rows, n = 70, 200000
    stream = torch.cuda.Stream()
    hs = HipSampler(1, 1, stream=stream.cuda_stream)
    base = logits(g, 2, n)[np.arange(rows) % 2]
    b, e = Batch(base, "f32"), Batch(base, "f32")
    ids, values = distill_inputs(g, rows, n, 30)
    d_ids, d_val = dev(ids), dev(values)
    t = HipSampler.teacher(d_ids, d_val, tail=True)
    l_graph, l_eager = out(rows), out(rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        hs.distill(b.view, t, l_graph, b.ws)
    for k in range(3):
        b.logits.add_(0.01 * k)
        e.logits.copy_(b.logits)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        hs.distill(e.view, t, l_eager, e.ws)
        stream.synchronize()
        assert torch.equal(l_graph, l_eager) and torch.equal(b.grad, e.grad), k
    hs.close()
