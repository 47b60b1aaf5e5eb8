"""The losses over logit rows (include/geist_loss_hip.h) at their edges, against the binary64 statement
(loss_reference.py) under the tolerances derived there: logits of -inf and of the type's lowest value in the
elements outside a row's groups of 16 bytes, listed mass above 1, parts of a row without anything that counts."""
import numpy as np
import pytest

import loss_reference as ref
from test_gpu_loss_rows import TYPES, Batch, dev, distill_inputs, logits, near, out, some_rows

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# rows, vocabulary, type, elements in front of the first row: one launch in groups of several sizes, and rows
# of more than 200 000 bytes that are cut into parts; none of them a whole number of 16-byte groups
EDGES = [(3, 5003, "f32", 1), (3, 5003, "f16", 3), (3, 5003, "bf16", 5), (300, 1001, "f32", 3), (3, 60001, "f32", 1),
         (3, 110003, "f16", 1), (3, 110003, "bf16", 7)]


@pytest.fixture(scope="module")
def hs():
    from geistlib_amd import HipSampler
    s = HipSampler(1, 1)
    yield s
    s.close()


def lowest(dtype):
    return float(torch.finfo(TYPES[dtype]).min)


def check_policy(hs, b, tokens, advantage, weight=None, ent=0.0, cap=0.0, temperature=1.0, allowed=None,
                 want_entropy=True):
    """The policy loss of every row of b (old log-probabilities: the rows' own) against the statement."""
    from geistlib_amd import HipSampler
    rows = b.rows
    d = [dev(np.asarray(tokens, np.int32)), dev(np.asarray(advantage, np.float32))]
    d_w = None if weight is None else dev(np.asarray(weight, np.float32))
    loss, lp, H = out(rows), out(rows), out(rows) if want_entropy else None
    hs.policy_loss(b.view, HipSampler.policy(d[0], d[1], weight=d_w, entropy_coef=ent), loss, lp, H, b.ws)
    hs.sync()
    grads = b.grads() if b.grad is not None else None
    for r in some_rows(rows):
        want = ref.policy(b.x[r], b.dtype, int(tokens[r]), float(advantage[r]), None, None,
                          weight=1.0 if weight is None else float(np.float32(weight[r])), ent=float(np.float32(ent)),
                          temperature=temperature, cap=cap, allowed=None if allowed is None else allowed[r])
        near(loss[r].item(), want["loss"], want["loss_tol"], f"loss of row {r}")
        near(lp[r].item(), want["logprob"], want["logprob_tol"] + abs(want["logprob"]) * 2.0 ** -23
             if np.isfinite(want["logprob"]) else 0.0, f"logprob of row {r}")
        if want_entropy:
            near(H[r].item(), want["entropy"], want["entropy_tol"] + want["entropy"] * 2.0 ** -23, f"entropy of row {r}")
        if grads is not None:
            near(grads[r], want["grad"], want["grad_tol"], f"gradient of row {r}")


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,n,dtype,lead", EDGES)
def test_entropy_beside_logits_that_do_not_count(hs, rows, n, dtype, lead, masked):
    """-inf and the type's lowest value at the first and the last token, which lie outside the groups: no
    term of the entropy, and no NaN in the loss and the gradient that it is part of."""
    g = np.random.default_rng(n + lead)
    x = logits(g, rows, n)
    x[0, [0, -1]] = -np.inf
    x[1, [0, -1]] = lowest(dtype)
    x[2, [0, 1, n // 2, -2, -1]] = -np.inf
    allowed = None
    if masked:
        allowed = g.random((rows, n)) < 0.7
        allowed[:, [0, 1, 40, -2, -1]] = True
    for grad in ("apart", "in place", None):
        b = Batch(x, dtype, lead, 0, grad=grad, allowed=allowed)
        check_policy(hs, b, np.full(rows, 40), g.standard_normal(rows), ent=0.1, allowed=allowed)


@pytest.mark.parametrize("ent", [0.0, 0.1])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(3, 5003), (3, 110003)])
def test_a_token_of_the_lowest_value_with_entropy(hs, rows, n, dtype, ent):
    """The sampled token's logit is so low that its exponent is -inf in binary32: its probability is 0, the
    gradient at it is what the advantage makes of it, and not NaN."""
    g = np.random.default_rng(n)
    x = logits(g, rows, n)
    tokens = np.array([0, n // 2, n - 1])
    x[np.arange(3), tokens] = lowest(dtype)
    check_policy(hs, Batch(x, dtype, 1, 0), tokens, [1.0, -0.5, 2.0], ent=ent)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,n,dtype,lead", [e for e in EDGES if e[2] != "f16"])  # (it would overflow there)
def test_large_weights_of_the_entropy(hs, rows, n, dtype, lead, masked):
    """A weight (a loss scale) of 10^10: tokens that do not count get a gradient of 0, not 0 * inf."""
    g = np.random.default_rng(n + 2)
    x = logits(g, rows, n)
    x[:, [0, 3, n // 2, -1]] = -np.inf
    allowed = None
    if masked:
        allowed = g.random((rows, n)) < 0.7
        allowed[:, [0, 3, 40, n // 2, -1]] = True
        x[~allowed] = g.choice([np.nan, np.inf, -np.inf, 1.0], int((~allowed).sum()))
    b = Batch(x, dtype, lead, 0, allowed=allowed)
    check_policy(hs, b, np.full(rows, 40), g.standard_normal(rows), weight=np.full(rows, 1e10), ent=1.0,
                 allowed=allowed)
    # rows that are summed against a value outside the range of plain references
    low = np.where(np.isfinite(x), x - 1e6, x)
    b = Batch(low, "f32", lead, 0, allowed=allowed)
    check_policy(hs, b, np.full(rows, 40), g.standard_normal(rows), weight=np.full(rows, 1e10), ent=1.0,
                 allowed=allowed)


@pytest.mark.parametrize("rows,n,dtype,lead", EDGES)
def test_a_spoilt_row_of_any_policy_loss(hs, rows, n, dtype, lead):
    """NaN and +inf make a row's loss, log-probability and gradient NaN also where the loss does not look at
    the log-probability: without old ones, with an advantage of 0. Positions that are not trained on and
    weights of 0 stay 0, and the other rows what they are."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n + 1)
    x = logits(g, rows, n)
    x[0, n // 3], x[1, n - 1] = np.nan, np.inf
    d_tok, d_adv = dev(np.full(rows, 40, np.int32)), dev(np.concatenate([[1.0, 0.0], np.ones(rows - 2)]).astype(np.float32))
    b, loss, lp = Batch(x, dtype, lead, 0), out(rows), out(rows)
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv), loss, lp, None, b.ws)
    hs.sync()
    grads = b.grads()
    assert np.isnan(loss[:2].cpu().numpy()).all() and np.isnan(lp[:2].cpu().numpy()).all()
    assert np.isnan(grads[:2]).all() and (loss[2:].cpu() == -1.0).all() and np.isfinite(grads[2:]).all()
    d_w, d_tok = dev(np.where(np.arange(rows) == 0, 0.0, 1.0).astype(np.float32)), d_tok.clone()
    d_tok[1] = -1
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, weight=d_w), loss, lp, None, b.ws)
    hs.sync()
    assert (loss[:2].cpu() == 0.0).all() and (b.grads()[:2] == 0).all() and lp[1].item() == 0.0


@pytest.mark.parametrize("mass", [1.0, 1.01, 1.5, 8.0])
@pytest.mark.parametrize("cap,temperature,masked", [(0.0, 1.0, False), (20.0, 0.7, True)])
@pytest.mark.parametrize("rows,n,dtype,lead", EDGES)
def test_distill_listed_mass_above_one(hs, rows, n, dtype, lead, cap, temperature, masked, mass):
    """Nothing is left for the tail, and the listed mass multiplies the row's log-sum: the gradient is
    mass p_i - q_i, and 'mass p_i' for what is not listed."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n + int(8 * mass))
    x = logits(g, rows, n)
    allowed = None
    if masked:
        allowed = g.random((rows, n)) < 0.7
    k = 12
    ids = np.stack([g.permutation(n)[:k] for _ in range(rows)]).astype(np.int32)
    ids[:, 0] = np.argmax(x, 1)                   # the student's leading token among them
    if masked:
        for r in range(rows):
            allowed[r, ids[r]] = True
    q = g.random((rows, k)) + 0.05
    values = np.log(mass * q / q.sum(1, keepdims=True)).astype(np.float32)
    weight = g.uniform(0.2, 2, rows).astype(np.float32)
    d_ids, d_val, d_w = dev(ids), dev(values), dev(weight)
    t = HipSampler.teacher(d_ids, d_val, weight=d_w, tail=True)
    for grad in ("apart", "in place"):
        b = Batch(x, dtype, lead, 0, grad=grad, allowed=allowed, temperature=temperature, cap=cap)
        loss = out(rows)
        hs.distill(b.view, t, loss, b.ws)
        hs.sync()
        grads = b.grads()
        for r in some_rows(rows):
            want, gr, tol, g_tol = ref.distill(b.x[r], dtype, ids[r], values[r], True, temperature, cap,
                                               None if allowed is None else allowed[r], float(weight[r]))
            near(loss[r].item(), want, tol, f"loss of row {r}")
            near(grads[r], gr, g_tol, f"gradient of row {r}")
            if grad == "apart" and not cap and dtype == "f32":   # the probabilities' slopes cancel
                assert abs(grads[r].sum()) <= g_tol.sum()


@pytest.mark.parametrize("way", ["masked", "-inf"])
@pytest.mark.parametrize("offset,temperature,dtype", [(-1e6, 1.0, "f32"), (-3e38, 1.0, "f32"), (-100.0, 1e-4, "f32"),
                                                      (-100.0, 1e-4, "bf16"), (4.6e7, 1.0, "f32")])
@pytest.mark.parametrize("rows,n", [(4, 130001), (300, 2001)])
def test_parts_without_anything_that_counts(hs, rows, n, offset, temperature, dtype, way):
    """Rows far from zero of which whole parts are masked or -inf: the empty parts, whose values are none,
    do not stand above the others. (The larger batch has no parts and is the same rows.)"""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(41)
    # (differences that are a few units at the call's temperature)
    x = (logits(g, rows, n) * temperature + offset).astype(np.float32)
    kept = np.zeros((rows, n), bool)
    kept[0::4, :200] = True                       # the first part alone
    kept[1::4, -300:] = True                      # the last one
    kept[2::4, n // 2:n // 2 + 100] = True        # one between
    kept[3::4, [5, n - 7]] = True                 # both ends
    if way == "masked":
        allowed, x[~kept] = kept, np.nan
    else:
        allowed, x[~kept] = None, -np.inf
    tokens = np.array([np.flatnonzero(kept[r])[-1] for r in range(rows)], np.int32)
    advantage = g.standard_normal(rows).astype(np.float32)
    b = Batch(x, dtype, 1, 0, allowed=allowed, temperature=temperature)
    check_policy(hs, b, tokens, advantage, ent=0.1, temperature=temperature, allowed=allowed)
    bare = Batch(x, dtype, 1, 0, grad=None, allowed=allowed, temperature=temperature)
    check_policy(hs, bare, tokens, advantage, ent=0.1, temperature=temperature, allowed=allowed)
    ids = np.stack([np.flatnonzero(kept[r])[[0, -1]] for r in range(rows)]).astype(np.int32)
    values = np.log(np.tile(np.array([0.5, 0.2]), (rows, 1))).astype(np.float32)
    d_ids, d_val, loss = dev(ids), dev(values), out(rows)
    for tail in (False, True):
        hs.distill(b.view, HipSampler.teacher(d_ids, d_val, tail=tail), loss, b.ws)
        hs.sync()
        grads = b.grads()
        for r in some_rows(rows):
            want, gr, tol, g_tol = ref.distill(b.x[r], dtype, ids[r], values[r], tail, temperature, 0.0,
                                               None if allowed is None else allowed[r])
            near(loss[r].item(), want, tol, f"tail {tail}: loss {r}")
            near(grads[r], gr, g_tol, f"tail {tail}: gradient {r}")
    # (a pair's sums over 300 rows are not what is looked at here)
    b = Batch(x[:4], dtype, 1, 0, allowed=None if allowed is None else allowed[:4], temperature=temperature)
    d_tok, d_start = dev(tokens[:4]), dev(np.array([0, 1, 4], np.int32))
    loss, ratios, lp = out(1), out(2), out(4)
    hs.preference_loss(b.view, HipSampler.preference(d_tok, d_start), loss, ratios, lp, b.ws)
    hs.sync()
    want = ref.preference(b.x, dtype, tokens[:4], None, [0, 1, 4], temperature=temperature,
                          allowed=None if allowed is None else allowed[:4])
    grads = b.grads()
    near(loss.cpu(), want["loss"], want["loss_tol"], "preference loss")
    near(ratios.cpu(), want["ratios"], want["ratios_tol"], "ratios")
    near(lp.cpu(), want["logprob"], want["logprob_tol"] + 1e-30, "logprob")
    near(grads, want["grad"], want["grad_tol"], "preference gradient")


@pytest.mark.parametrize("way", ["masked", "-inf"])
def test_rows_cut_into_parts_that_are_all_empty(hs, way):
    """Nothing is left in any part: no distribution, everything 0 and the token's log-probability -inf."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(42)
    rows, n = 4, 130001
    x = logits(g, rows, n)
    x[1] = np.nan if way == "masked" else -np.inf
    allowed = None
    if way == "masked":
        allowed = np.ones((rows, n), bool)
        allowed[1] = False
    tokens = np.array([3, 4, 5, n - 1], np.int32)
    b = Batch(x, "f32", 1, 0, allowed=allowed)
    check_policy(hs, b, tokens, [1.0, 2.0, -1.0, 0.5], ent=0.1, allowed=allowed)
    d_ids, d_val, loss = dev(tokens[:, None].copy()), dev(np.full((rows, 1), -0.5, np.float32)), out(rows)
    for tail in (False, True):
        hs.distill(b.view, HipSampler.teacher(d_ids, d_val, tail=tail), loss, b.ws)
        hs.sync()
        assert loss[1].item() == 0.0 and (b.grads()[1] == 0).all()
    d_tok, d_start, lp = dev(tokens), dev(np.array([0, 2, 4], np.int32)), out(rows)
    hs.preference_loss(b.view, HipSampler.preference(d_tok, d_start), loss[:1], None, lp, b.ws)
    hs.sync()
    want = ref.preference(b.x, "f32", tokens, None, [0, 2, 4], allowed=allowed)
    near(lp.cpu(), want["logprob"], want["logprob_tol"] + 1e-30, "logprob")
    near(loss[:1].cpu(), want["loss"], want["loss_tol"], "loss")
    near(b.grads(), want["grad"], want["grad_tol"], "gradient")


def test_a_spoilt_part_beside_empty_ones(hs):
    """NaN or +inf in one part of a row whose other parts are empty: the row is NaN, the others are not."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(43)
    rows, n = 4, 130001
    x = np.full((rows, n), -np.inf)
    x[:, 60000:60100] = logits(g, rows, 100)
    x[1, 60050], x[2, 60050] = np.nan, np.inf
    tokens = np.full(rows, 60007, np.int32)
    b = Batch(x, "f32", 1, 0)
    d_tok, d_adv, loss, lp = dev(tokens), dev(np.ones(rows, np.float32)), out(rows), out(rows)
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv), loss, lp, None, b.ws)
    hs.sync()
    assert np.isnan(loss.cpu().numpy()).tolist() == [False, True, True, False]
    assert np.isnan(b.grads()[1:3]).all() and np.isfinite(b.grads()[[0, 3]]).all()
    d_start, two = dev(np.array([0, 1, 2, 3, 4], np.int32)), out(2)
    hs.preference_loss(b.view, HipSampler.preference(d_tok, d_start), two, None, lp, b.ws)
    hs.sync()
    assert np.isnan(two.cpu().numpy()).all() and np.isnan(lp.cpu().numpy()).tolist() == [False, True, True, False]


@pytest.mark.parametrize("rows,n", [(4, 5003), (4, 60001)])
def test_a_kl_term_that_is_switched_off(hs, rows, n):
    """kl_coef = 0 with reference log-probabilities of any value: what a call without them gives."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n)
    b = Batch(logits(g, rows, n), "f32")
    d_tok, d_adv = dev(np.full(rows, 9, np.int32)), dev(g.standard_normal(rows).astype(np.float32))
    d_ref = dev(np.array([-np.inf, 1e4, 3e38, np.nan], np.float32))
    res = []
    for r in (None, d_ref):
        loss = out(rows)
        hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, ref=r, kl_coef=0.0), loss, None, None, b.ws)
        hs.sync()
        res.append((loss, b.grad.clone()))
    assert bool(torch.isfinite(res[0][0]).all())
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


@pytest.mark.parametrize("cap", [0.0, 30.0, 100.0])
@pytest.mark.parametrize("rows,n,dtype,lead", EDGES)
def test_infinite_logits(hs, rows, n, dtype, lead, cap):
    """+inf makes its row NaN without a soft-cap; under one it is the cap itself, with no slope, as -inf is
    the cap's negative. At the row's ends and within it.
    With a cap of 100 other tokens' p_i reach 2^-126, below which 2^u is 0 (the instruction gives no subnormal
    results): p_i is off by up to 2^-126 more, the gradient by that times |A| + ent (|log p_i| + H) <=
    1 + 0.1 (2 * 100 + log n + log n) < 24 for n < 2^17, times a slope of at most 1."""
    flushed = 24 * 2.0 ** -126
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n + 5)
    x = logits(g, rows, n)
    x[0, 0] = x[1, n // 2] = x[2, -1] = np.inf
    if cap:
        x[0, 1] = x[1, 3] = x[2, -2] = -np.inf
    tokens = np.full(rows, 40, np.int32)
    tokens[:3] = 0, n // 2, 7
    ids = np.tile(np.array([0, n // 2, 7], np.int32), (rows, 1))
    values = np.log(np.tile(np.array([0.4, 0.3, 0.1]), (rows, 1))).astype(np.float32)
    spoilt = [] if cap else [0, 1, 2]
    d_tok, d_adv, d_ids, d_val = dev(tokens), dev(np.ones(rows, np.float32)), dev(ids), dev(values)
    b = Batch(x, dtype, lead, 0, cap=cap)
    loss, lp, H = out(rows), out(rows), out(rows)
    hs.policy_loss(b.view, HipSampler.policy(d_tok, d_adv, entropy_coef=0.1), loss, lp, H, b.ws)
    hs.sync()
    grads = b.grads()
    for r in some_rows(rows):
        if r in spoilt:
            assert all(np.isnan(v[r].item()) for v in (loss, lp, H)) and np.isnan(grads[r]).all()
            continue
        want = ref.policy(b.x[r], dtype, int(tokens[r]), 1.0, None, None, ent=float(np.float32(0.1)), cap=cap)
        near(loss[r].item(), want["loss"], want["loss_tol"], f"loss {r}")
        near(lp[r].item(), want["logprob"], want["logprob_tol"] + abs(want["logprob"]) * 2.0 ** -23, f"logprob {r}")
        near(H[r].item(), want["entropy"], want["entropy_tol"] + want["entropy"] * 2.0 ** -23, f"entropy {r}")
        near(grads[r], want["grad"], want["grad_tol"] + flushed, f"gradient {r}")
    for tail in (False, True):
        hs.distill(b.view, HipSampler.teacher(d_ids, d_val, tail=tail), loss, b.ws)
        hs.sync()
        grads = b.grads()
        for r in some_rows(rows):
            if r in spoilt:
                assert np.isnan(loss[r].item()) and np.isnan(grads[r]).all()
                continue
            want, gr, tol, g_tol = ref.distill(b.x[r], dtype, ids[r], values[r], tail, 1.0, cap)
            near(loss[r].item(), want, tol, f"tail {tail}: loss {r}")
            near(grads[r], gr, g_tol + flushed, f"tail {tail}: gradient {r}")
    b = Batch(x[:3], dtype, lead, 0, cap=cap)
    d_start, one, lp = dev(np.array([0, 1, 3], np.int32)), out(1), out(3)
    hs.preference_loss(b.view, HipSampler.preference(d_tok[:3], d_start), one, None, lp, b.ws)
    hs.sync()
    if spoilt:
        assert np.isnan(one.item()) and np.isnan(lp.cpu().numpy()).all() and np.isnan(b.grads()).all()
    else:
        want = ref.preference(b.x, dtype, tokens[:3], None, [0, 1, 3], cap=cap)
        near(one.item(), want["loss"], want["loss_tol"], "preference loss")
        near(lp.cpu(), want["logprob"], want["logprob_tol"] + np.abs(want["logprob"]) * 2.0 ** -23, "logprob")
        near(b.grads(), want["grad"], want["grad_tol"] + flushed, "preference gradient")


def test_outputs_without_room_are_refused(hs):
    """A vector that is too short or of another type is refused before anything is written; page-locked host
    memory is taken like device memory."""
    from geistlib_amd import HipSampler
    from geistlib_amd.binding import GeistHipError
    rows, n = 4, 1000
    b = Batch(logits(np.random.default_rng(50), rows, n), "f32")
    d_tok, d_adv = dev(np.full(rows, 9, np.int32)), dev(np.ones(rows, np.float32))
    d_ids, d_val = dev(np.full((rows, 1), 9, np.int32)), dev(np.zeros((rows, 1), np.float32))
    d_start = dev(np.array([0, 1, 2, 3, 4], np.int32))
    p, q = HipSampler.policy(d_tok, d_adv), HipSampler.preference(d_tok, d_start)
    t = HipSampler.teacher(d_ids, d_val)
    ok, short, other = out(rows), out(rows)[:rows - 1], torch.full((rows,), -77.0, dtype=torch.float16, device="cuda")
    other_rows, small = HipSampler.policy(d_tok[:3], d_adv[:3]), hs.host_buffer(4)
    for bad in (short, other, torch.zeros(rows), small):
        for call in (lambda: hs.distill(b.view, t, bad, b.ws),
                     lambda: hs.policy_loss(b.view, p, bad, None, None, b.ws),
                     lambda: hs.policy_loss(b.view, p, ok, bad, None, b.ws),
                     lambda: hs.policy_loss(b.view, p, ok, None, bad, b.ws),
                     lambda: hs.preference_loss(b.view, q, ok, bad, None, b.ws),
                     lambda: hs.preference_loss(b.view, q, ok, None, bad, b.ws),
                     lambda: hs.preference_loss(b.view, q, bad[:1] if torch.is_tensor(bad) else small, None, None, b.ws),
                     lambda: hs.policy_loss(b.view, other_rows, ok, None, None, b.ws)):
            with pytest.raises(GeistHipError) as err:
                call()
            assert err.value.code == 2
    hs.sync()
    assert (ok.cpu() == -77.0).all() and (short.cpu() == -77.0).all() and (other.cpu() == -77.0).all()
    assert (b.grads() == 7.0).all()
    hs.policy_loss(b.view, p, None, ok, None, b.ws)
    host, pinned = hs.host_buffer(4 * rows), torch.zeros(rows).pin_memory()
    hs.policy_loss(b.view, p, None, host, None, b.ws)
    hs.policy_loss(b.view, p, None, pinned, None, b.ws)
    hs.sync()
    assert (host.view(np.float32) == ok.cpu().numpy()).all() and torch.equal(pinned, ok.cpu())
    host.close()
    small.close()


@pytest.mark.parametrize("rows,n,dtype,lead", [(3, 5003, "f32", 1), (3, 110003, "bf16", 7), (300, 1001, "f16", 3)])
def test_scores_alone(hs, rows, n, dtype, lead):
    """Log-probabilities, entropies or ratios without a loss and without a gradient: the bits of a call that
    asks for the loss too."""
    from geistlib_amd import HipSampler
    g = np.random.default_rng(n + 9)
    b = Batch(logits(g, rows, n), dtype, lead, 0, grad=None)
    d_tok, d_adv = dev(g.integers(0, n, rows).astype(np.int32)), dev(np.ones(rows, np.float32))
    p = HipSampler.policy(d_tok, d_adv)
    loss, lp, H = out(rows), out(rows), out(rows)
    hs.policy_loss(b.view, p, loss, lp, H, b.ws)
    lp2, H2 = out(rows), out(rows)
    hs.policy_loss(b.view, p, None, lp2, H2, b.ws)
    hs.sync()
    assert torch.equal(lp, lp2) and torch.equal(H, H2)
    H3 = out(rows)
    hs.policy_loss(b.view, p, None, None, H3, b.ws)
    hs.sync()
    assert torch.equal(H, H3)
    d_start = dev(np.array([0, rows // 3, rows], np.int32))
    q = HipSampler.preference(d_tok, d_start)
    one, ratios, lp = out(1), out(2), out(rows)
    hs.preference_loss(b.view, q, one, ratios, lp, b.ws)
    ratios2, lp2 = out(2), out(rows)
    hs.preference_loss(b.view, q, None, ratios2, lp2, b.ws)
    hs.sync()
    assert torch.equal(ratios, ratios2) and torch.equal(lp, lp2)
