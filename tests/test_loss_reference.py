"""The binary64 statement of the losses (loss_reference.py): its gradients against central differences
of its losses, and closed forms. CPU only."""
import numpy as np
import pytest

import loss_reference as ref


def differences(f, x, at, h=1e-5):
    out = []
    for i in at:
        up, dn = x.copy(), x.copy()
        up[i] += h
        dn[i] -= h
        out.append((f(up) - f(dn)) / (2 * h))
    return np.array(out)


def row(seed, n):
    g = np.random.default_rng(seed)
    x = g.standard_normal(n) * 2
    x[g.integers(0, n, 3)] += 4
    allowed = g.random(n) < 0.7
    return g, x, allowed


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("cap,temperature,masked", [(0.0, 1.0, False), (5.0, 0.7, True), (0.0, 2.0, True)])
def test_distill_gradient_is_the_loss_differentiated(tail, cap, temperature, masked):
    g, x, allowed = row(3, 40)
    ids = np.array([4, 9, 9, 31, -1, 40, 17])
    values = np.log(np.array([0.2, 0.1, 0.4, 0.15, 0.1, 0.05, 0.05]))
    kw = dict(tail=tail, temperature=temperature, cap=cap, allowed=allowed if masked else None, weight=1.7)
    loss = lambda z: ref.distill(z, "f32", ids, values, **kw)[0]  # noqa: E731
    grad = ref.distill(x, "f32", ids, values, **kw)[1]
    np.testing.assert_allclose(grad, differences(loss, x, range(40)), atol=1e-8)


@pytest.mark.parametrize("advantage,shift", [(1.3, 0.0), (1.3, 0.5), (-0.7, -0.5), (-0.7, 0.5), (0.0, 0.2)])
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_policy_gradient_is_the_loss_differentiated(advantage, shift, cap):
    g, x, allowed = row(5, 30)
    allowed[7] = True
    kw = dict(weight=0.6, low=0.2, high=0.28, kl=0.3, ent=0.05, temperature=0.8, cap=cap, allowed=allowed)
    lp = ref.policy(x, "f32", 7, 1.0, None, None, temperature=0.8, cap=cap, allowed=allowed)["logprob"]
    old, rf = lp - shift, lp + 0.3
    loss = lambda z: ref.policy(z, "f32", 7, advantage, old, rf, **kw)["loss"]  # noqa: E731
    grad = ref.policy(x, "f32", 7, advantage, old, rf, **kw)["grad"]
    np.testing.assert_allclose(grad, differences(loss, x, range(30)), atol=1e-8)


@pytest.mark.parametrize("kind,smoothing,normalised", [("sigmoid", 0.0, False), ("sigmoid", 0.2, True),
                                                       ("hinge", 0.0, False), ("squared", 0.0, True)])
def test_preference_gradient_is_the_loss_differentiated(kind, smoothing, normalised):
    g = np.random.default_rng(8)
    x = g.standard_normal((9, 12))
    tokens = g.integers(0, 12, 9)
    tokens[3] = -1
    start, rf = [0, 2, 5, 5, 9], g.standard_normal(9)
    kw = dict(kind=kind, beta=0.4, margin=0.3 if kind != "squared" else 0.0, smoothing=smoothing,
              normalised=normalised, weight=[0.5, 1.5], cap=3.0)
    loss = lambda z: ref.preference(z.reshape(9, 12), "f32", tokens, rf, start, **kw)["loss"].sum()  # noqa: E731
    grad = ref.preference(x, "f32", tokens, rf, start, **kw)["grad"]
    np.testing.assert_allclose(grad.reshape(-1), differences(loss, x.reshape(-1), range(108)), atol=1e-8)


def test_closed_forms():
    n = 50
    flat = np.full(n, 3.25)
    # a one-hot teacher is the cross entropy; a row that agrees with its teacher has loss 0
    assert ref.distill(flat, "f32", [7], [0.0], False)[0] == pytest.approx(np.log(n))
    assert ref.distill(flat, "f32", [7, 9], [np.log(1 / n)] * 2, True)[0] == pytest.approx(0, abs=1e-15)
    assert np.abs(ref.distill(flat, "f32", [7], [np.log(1 / n)], True)[1]).max() < 1e-15
    res = ref.policy(flat, "f32", 3, 2.0, None, None)
    assert res["loss"] == -2.0 and res["entropy"] == pytest.approx(np.log(n))
    assert ref.preference(np.zeros((2, 4)), "f32", [0, 1], None, [0, 1, 2])["loss"][0] == pytest.approx(
        np.log(2))


@pytest.mark.parametrize("mass", [0.9, 1.01, 1.5, 4.0])
@pytest.mark.parametrize("cap,temperature,masked", [(0.0, 1.0, False), (5.0, 0.7, True)])
def test_tail_gradient_for_any_listed_mass(cap, temperature, masked, mass):
    """Above 1 nothing is left for the tail, and the loss holds the listed mass times the row's log-sum."""
    g, x, allowed = row(11, 40)
    allowed[[4, 9, 31]] = True
    q = np.array([0.5, 0.3, 0.2]) * mass
    kw = dict(tail=True, temperature=temperature, cap=cap, allowed=allowed if masked else None, weight=0.8)
    loss = lambda z: ref.distill(z, "f32", [4, 9, 31], np.log(q), **kw)[0]  # noqa: E731
    grad = ref.distill(x, "f32", [4, 9, 31], np.log(q), **kw)[1]
    np.testing.assert_allclose(grad, differences(loss, x, range(40)), atol=1e-8)
