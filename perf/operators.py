"""Losses over logit rows and their gradients, as measurable cases: distillation from a teacher's
top logits, the clipped policy loss with a KL term over sampled tokens, and the preference loss over
pairs of sequences.

A case is a dict of plain values. `listed()` gives the fixed ones, `draw(rng)` one more of the same
ranges; `prepare` makes what a training step holds before the call, `run` is one call of the operator
(its plain form where `own` is false), `exact` its value in 64 bits, `work` the bytes and operations
it cannot do without. Direction "loss" is the forward pass alone, "both" the loss and the gradient of
the logits in one step.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MOST_LOGITS = 4096 * 128256


def _distill(name, rows, vocab, dtype, k, tail, direction, temperature=1.0, softcap=0.0, ragged=False,
             mask=False, pad=0):
    case = {"kind": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "tail": tail,
            "direction": direction, "temperature": temperature, "softcap": softcap, "ragged": ragged,
            "mask": mask, "pad": pad}
    return {"name": name, **case} if name else case


def _policy(name, rows, vocab, dtype, direction, kl=0.0, entropy=0.0, temperature=1.0, softcap=0.0,
            mask=False, pad=0):
    case = {"kind": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "direction": direction,
            "kl": kl, "entropy": entropy, "temperature": temperature, "softcap": softcap,
            "mask": mask, "pad": pad}
    return {"name": name, **case} if name else case


def _preference(name, pairs, length, vocab, dtype, direction, loss="sigmoid", smoothing=0.0,
                normalised=False, reference=True, softcap=0.0, pad=0):
    case = {"kind": "preference", "pairs": pairs, "length": length, "vocab": vocab, "dtype": dtype,
            "direction": direction, "loss": loss, "smoothing": smoothing, "normalised": normalised,
            "reference": reference, "softcap": softcap, "pad": pad, "temperature": 1.0,
            "mask": False}
    return {"name": name, **case} if name else case


def listed():
    return [
        # a handful of positions against a teacher's 16 leading logits at temperature 2: the smallest
        # training call, where launches are the cost
        _distill("distill_8x32000_f32", 8, 32000, "f32", 16, False, "both", temperature=2.0),
        # a micro-batch of 1024 positions in bf16 with the teacher's top 64, as a drafter is trained
        # on what a server's top-k logged
        _distill("distill_1024x128256_bf16", 1024, 128256, "bf16", 64, False, "both"),
        # the teacher's top 128 log-probabilities with its remaining mass as one more event, in f32
        _distill("distill_tail_512x151936_f32", 512, 151936, "f32", 128, True, "both"),
        # an evaluation step: the loss alone, a vocabulary of odd size (rows that are not 16-byte
        # aligned) and teacher lists of different lengths
        _distill("distill_tail_2000x50257_f16_loss", 2000, 50257, "f16", 20, True, "loss",
                 ragged=True),
        # one sampled token scored under the current policy: the smallest call of all
        _policy("policy_1x128256_f32_loss", 1, 128256, "f32", "loss"),
        # a policy step over 4096 sampled tokens with KL and entropy terms: the largest batch
        _policy("policy_4096x128256_bf16", 4096, 128256, "bf16", "both", kl=0.05, entropy=0.001),
        # the widest vocabulary, with the soft-cap the rows were sampled under, at temperature 0.8
        _policy("policy_600x262144_f16_capped", 600, 262144, "f16", "both", kl=0.02, softcap=30.0,
                temperature=0.8),
        # tokens that were drawn under a grammar's mask, vocabulary of odd size
        _policy("policy_333x65537_bf16_mask", 333, 65537, "bf16", "both", mask=True),
        # two pairs of short answers
        _preference("preference_2x12x32000_f32", 2, 12, 32000, "f32", "both"),
        # four pairs of ordinary answers, labels smoothed
        _preference("preference_4x220x128256_bf16", 4, 220, 128256, "bf16", "both", smoothing=0.1),
        # eight pairs scored without a gradient, as a validation step does
        _preference("preference_8x150x151936_bf16_loss", 8, 150, 151936, "bf16", "loss"),
        # averaged log-probabilities without a reference model, a vocabulary of odd size
        _preference("preference_16x61x99991_f16_mean", 16, 61, 99991, "f16", "both",
                    normalised=True, reference=False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["distill", "policy", "preference"])
    vocab = _log_int(rng, 2000, 262144)
    if rng.random() < 0.5:
        vocab = vocab // 64 * 64
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    most = MOST_LOGITS // (2 if dtype == "f32" else 1)
    direction = rng.choice(["loss", "both", "both"])
    pad = 64 - vocab % 64 if rng.random() < 0.25 else 0
    softcap = 30.0 if rng.random() < 0.2 else 0.0
    temperature = round(rng.uniform(0.6, 2.0), 2) if rng.random() < 0.4 else 1.0
    if kind == "preference":
        rows = _log_int(rng, 16, 4096)
        pairs = max(1, min(_log_int(rng, 1, 32), rows // 4))
        length = max(1, min(rows, most // vocab) // (2 * pairs))
        return _preference(None, pairs, length, vocab, dtype, direction,
                           rng.choice(["sigmoid", "sigmoid", "hinge", "squared"]),
                           normalised=rng.random() < 0.3, reference=rng.random() < 0.7,
                           softcap=softcap, pad=pad)
    rows = max(1, min(_log_int(rng, 1, 8192), most // vocab))
    mask = rng.random() < 0.15
    if kind == "distill":
        return _distill(None, rows, vocab, dtype, _log_int(rng, 1, 512), rng.random() < 0.5,
                        direction, temperature, softcap, rng.random() < 0.3, mask, pad)
    return _policy(None, rows, vocab, dtype, direction, rng.choice([0.0, 0.02, 0.1]),
                   rng.choice([0.0, 0.0, 0.01]), temperature, softcap, mask, pad)


def _rows_of(case):
    return 2 * case["pairs"] * case["length"] if case["kind"] == "preference" else case["rows"]


def _view(rows, vocab, pad, dtype):
    """Rows of `vocab` values, `pad` more between them."""
    return torch.zeros((rows, vocab + pad), dtype=dtype, device="cuda")[:, :vocab]


def _allowed(words, vocab):
    """Mask words as truth values: bit e % 32 of word e // 32 stands for token e."""
    bits = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words[:, :, None] >> bits) & 1).bool().reshape(words.shape[0], -1)[:, :vocab]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def units(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    rows, vocab, dtype = _rows_of(case), case["vocab"], TYPES[case["dtype"]]
    st = {"case": case, "logits": _view(rows, vocab, case["pad"], dtype), "allowed": None,
          "grad": None, "ref": None}
    # a model's rows: a broad bulk and some two dozen tokens that share most of the mass
    x = normal(rows, vocab).mul_(2.0)
    part = vocab // 24
    lead = torch.randint(0, part, (rows, 24), generator=g, device="cuda")
    lead += torch.arange(24, device="cuda") * part
    boost = torch.linspace(math.log(vocab) + 4.0, math.log(vocab) - 5.0, 24, device="cuda")
    x.scatter_(1, lead, boost + normal(rows, 24))
    st["logits"].copy_(x)
    x.copy_(st["logits"])
    if case["softcap"]:
        x.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    x.div_(case["temperature"])
    if case["mask"]:
        words = (vocab + 31) // 32
        st["allowed"] = torch.randint(-2**31, 2**31, (rows, words), generator=g, device="cuda",
                                      dtype=torch.int64).to(torch.int32)
        st["allowed"][:, 0] |= 1
        x.masked_fill_(~_allowed(st["allowed"], vocab), -math.inf)
    if case["direction"] == "both":
        st["grad"] = _view(rows, vocab, case["pad"], dtype)
    st["loss"] = torch.zeros(case["pairs"] if case["kind"] == "preference" else rows, device="cuda")
    if case["kind"] == "distill":
        k = min(case["k"], vocab)
        t = x.add_(normal(rows, vocab))
        lse = torch.logsumexp(t, 1, keepdim=True)
        top = torch.topk(t, k, 1)
        st["ids"] = top.indices.to(torch.int32)
        # the teacher's own logits, or its log-probabilities where its tail counts
        st["values"] = (top.values - lse).clamp_min(-80.0) if case["tail"] \
            else top.values.clamp_min(-80.0) * case["temperature"]
        st["count"] = None
        if case["ragged"]:
            st["count"] = torch.randint(1, k + 1, (rows,), generator=g, device="cuda",
                                        dtype=torch.int32)
        st["weight"] = (0.5 + units(rows)) / rows
    else:
        lse = torch.logsumexp(x, 1)
        noise = units(rows, vocab).clamp_(1e-7, 1 - 1e-7).log_().neg_().log_()
        token = (x - noise).argmax(1)      # a draw from the row
        del noise
        logp = x.gather(1, token[:, None])[:, 0] - lse
        st["tokens"] = torch.where(units(rows) < 0.1, torch.full_like(token, -1), token).to(
            torch.int32)
        st["logprob"] = torch.zeros(rows, device="cuda")
        if case["kind"] == "policy":
            st["old"] = logp + 0.15 * normal(rows)
            st["ref"] = logp + 0.4 * normal(rows) if case["kl"] else None
            st["advantage"] = normal(rows)
            st["weight"] = (0.5 + units(rows)) / rows
            st["entropy"] = torch.zeros(rows, device="cuda")
        else:
            n = 2 * case["pairs"]
            cuts = torch.randint(0, rows + 1, (n - 1,), generator=g, device="cuda").sort().values
            even = torch.arange(1, n, device="cuda") * case["length"]
            ends = torch.tensor([rows], device="cuda")
            st["start"] = torch.cat([ends * 0, (cuts + 3 * even) // 4, ends]).to(torch.int32)
            st["ref"] = logp + 0.4 * normal(rows) if case["reference"] else None
            st["weight"] = (0.5 + units(case["pairs"])) / case["pairs"]
            st["ratios"] = torch.zeros(n, device="cuda")
    if own:
        _handles(st)
    return st


def _handles(st):
    """What a program that uses the library keeps: the sampler object of its stream, the workspace
    and the descriptions of its tensors."""
    from geistlib_amd import HipSampler
    case = st["case"]
    rows, vocab = st["logits"].shape
    hs = st["sampler"] = HipSampler(1, vocab, stream=torch.cuda.current_stream().cuda_stream)
    st["workspace"] = torch.zeros(hs.loss_workspace_bytes(rows, vocab), dtype=torch.uint8,
                                  device="cuda")
    st["rows"] = HipSampler.loss_rows(st["logits"], grad=st["grad"], allowed=st["allowed"],
                                      temperature=case["temperature"], softcap=case["softcap"])
    if case["kind"] == "distill":
        st["what"] = HipSampler.teacher(st["ids"], st["values"], count=st["count"],
                                        weight=st["weight"], tail=case["tail"])
    elif case["kind"] == "policy":
        st["what"] = HipSampler.policy(st["tokens"], st["advantage"], old=st["old"], ref=st["ref"],
                                       weight=st["weight"], clip_low=0.2, clip_high=0.28,
                                       kl_coef=case["kl"], entropy_coef=case["entropy"])
    else:
        st["what"] = HipSampler.preference(st["tokens"], st["start"], ref=st["ref"],
                                           weight=st["weight"], kind=case["loss"], beta=0.1,
                                           label_smoothing=case["smoothing"],
                                           length_normalised=case["normalised"])


def _own(st):
    hs, kind = st["sampler"], st["case"]["kind"]
    if kind == "distill":
        hs.distill(st["rows"], st["what"], st["loss"], st["workspace"])
        return {"loss": st["loss"], "grad": st["grad"]}
    if kind == "policy":
        hs.policy_loss(st["rows"], st["what"], st["loss"], st["logprob"], st["entropy"],
                       st["workspace"])
        return {"loss": st["loss"], "logprob": st["logprob"], "entropy": st["entropy"],
                "grad": st["grad"]}
    hs.preference_loss(st["rows"], st["what"], st["loss"], st["ratios"], st["logprob"],
                       st["workspace"])
    return {"loss": st["loss"], "ratios": st["ratios"], "logprob": st["logprob"],
            "grad": st["grad"]}


def run(st):
    if own:
        return _own(st)
    case = st["case"]
    x, slope = _scaled(st)
    m = x.amax(1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(1, keepdim=True, dtype=torch.float64)
    lse = m.double() + torch.log(total)
    p /= total.float()
    return {"distill": _plain_distill, "policy": _plain_policy,
            "preference": _plain_preference}[case["kind"]](st, slope, x, lse, p)


def _scaled(st):
    """The rows' values behind soft-cap, temperature and mask, and their slope by the logits."""
    case = st["case"]
    x, slope = st["logits"].float(), 1.0 / case["temperature"]
    if case["softcap"]:
        t = torch.tanh(x / case["softcap"])
        x = t * case["softcap"]
        if case["direction"] == "both":
            slope = (1.0 - t * t) / case["temperature"]
    x = x / case["temperature"]
    if st["allowed"] is not None:
        x = torch.where(_allowed(st["allowed"], x.shape[1]), x, -math.inf)
    return x, slope


def _plain_distill(st, slope, x, lse, p):
    case = st["case"]
    ids = st["ids"].long()
    listed_ = torch.ones_like(ids, dtype=torch.bool)
    if st["count"] is not None:
        listed_ = torch.arange(ids.shape[1], device="cuda") < st["count"][:, None]
    if st["allowed"] is not None:
        listed_ = listed_ & _allowed(st["allowed"], p.shape[1]).gather(1, ids)
    v = torch.where(listed_, st["values"], -math.inf)
    at = x.gather(1, ids).double() - lse
    if case["tail"]:
        q = torch.exp(v.double())
        q_rest = (1.0 - q.sum(1, keepdim=True)).clamp_min(0.0)
        inside = torch.zeros_like(p, dtype=torch.bool).scatter_(1, ids, listed_)
        p_rest = torch.where(inside, 0.0, p).sum(1, keepdim=True).double()
        terms = torch.where(listed_, q * (v.double() - at), 0.0).sum(1)
        loss = terms + torch.where(q_rest > 0, q_rest * (q_rest.log() - p_rest.log()), 0.0)[:, 0]
        share = torch.where(q_rest > 0, q_rest / p_rest, 0.0).float()
        if case["direction"] == "both":
            grad = torch.where(inside, p, p * (1.0 - share))
    else:
        v = v.double() / case["temperature"]
        some = listed_.any(1, keepdim=True)
        e = torch.where(listed_, torch.exp(v - torch.where(some, v.amax(1, keepdim=True), 0.0)), 0.0)
        total = torch.where(some, e.sum(1, keepdim=True), 1.0)
        q = e / total
        lq = torch.where(listed_, v - torch.where(some, v.amax(1, keepdim=True), 0.0), 0.0) \
            - total.log()
        loss = torch.where(q > 0, q * (lq - at), 0.0).sum(1)
        if case["direction"] == "both":
            grad = torch.where(some, p, 0.0)
    out = {"loss": (loss * st["weight"]).float(), "grad": None}
    if case["direction"] == "both":
        grad.scatter_add_(1, ids, -torch.where(listed_, q, 0.0).float())
        out["grad"] = (grad * st["weight"][:, None] * slope).to(st["logits"].dtype)
    return out


def _plain_policy(st, slope, x, lse, p):
    case = st["case"]
    used = st["tokens"] >= 0
    token = st["tokens"].long().clamp_min(0)
    lp = torch.where(used, (x.gather(1, token[:, None]).double() - lse)[:, 0], 0.0)
    logp = x - lse.float()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
    ratio = torch.exp(lp - st["old"])
    a = st["advantage"]
    free, held = ratio * a, ratio.clamp(0.8, 1.28) * a
    loss = -torch.minimum(free, held)
    d = torch.where(free <= held, -free, 0.0)
    if st["ref"] is not None:
        far = st["ref"] - lp
        loss = loss + case["kl"] * (torch.expm1(far) - far)
        d = d - case["kl"] * torch.expm1(far)
    loss = loss - case["entropy"] * entropy
    w = torch.where(used, st["weight"], 0.0)
    out = {"loss": (loss * w).float(), "logprob": lp.float(), "entropy": entropy, "grad": None}
    if case["direction"] == "both":
        d = d.float()
        grad = -d[:, None] * p
        grad.scatter_add_(1, token[:, None], d[:, None])
        if case["entropy"]:
            grad += case["entropy"] * torch.where(p > 0, p * (logp + entropy[:, None]), 0.0)
        out["grad"] = (grad * w[:, None] * slope).to(st["logits"].dtype)
    return out


def _plain_preference(st, slope, x, lse, p):
    case = st["case"]
    rows = p.shape[0]
    used = st["tokens"] >= 0
    token = st["tokens"].long().clamp_min(0)
    lp = torch.where(used, (x.gather(1, token[:, None]).double() - lse)[:, 0], 0.0)
    diff = lp if st["ref"] is None else lp - st["ref"].double()
    start = st["start"].long()
    seq = torch.searchsorted(start, torch.arange(rows, device="cuda"), right=True) - 1
    n = 2 * case["pairs"]
    sums = torch.zeros(n, dtype=torch.float64, device="cuda")
    sums = sums.index_add(0, seq, torch.where(used, diff, 0.0))
    share = torch.ones(n, dtype=torch.float64, device="cuda")
    if case["normalised"]:
        share = 1.0 / torch.zeros_like(sums).index_add(0, seq, used.double()).clamp_min(1.0)
    ratios = sums * share
    gap = ratios[0::2] - ratios[1::2]
    h = 0.1 * gap
    if case["loss"] == "sigmoid":
        s = case["smoothing"]
        loss = (1 - s) * torch.log1p(torch.exp(-h.abs())) + s * torch.log1p(torch.exp(-h.abs())) \
            + (1 - s) * (-h).clamp_min(0.0) + s * h.clamp_min(0.0)
        d = 0.1 * (s - 1.0 / (1.0 + torch.exp(h)))
    elif case["loss"] == "hinge":
        loss = (1.0 - h).clamp_min(0.0)
        d = torch.where(h < 1.0, -0.1, 0.0)
    else:
        loss = (gap - 5.0).square()
        d = 2.0 * (gap - 5.0)
    out = {"loss": (loss * st["weight"]).float(), "ratios": ratios.float(), "logprob": lp.float(),
           "grad": None}
    if case["direction"] == "both":
        d = torch.stack([d, -d], 1).reshape(-1) * st["weight"].double().repeat_interleave(2) * share
        d = torch.where(used, d[seq], 0.0).float()
        grad = -d[:, None] * p
        grad.scatter_add_(1, token[:, None], d[:, None])
        out["grad"] = (grad * slope).to(st["logits"].dtype)
    return out


def exact(case, seed):
    """The losses written down in double over blocks of rows; gradients by differentiating them."""
    st = prepare(case, seed)
    rows, vocab = st["logits"].shape
    block = max(1, min(rows, (1 << 26) // vocab))
    want = case["direction"] == "both"

    def log_rows(a, b):
        z = st["logits"][a:b].double().requires_grad_(want)
        y = z if not case["softcap"] else case["softcap"] * torch.tanh(z / case["softcap"])
        y = y / case["temperature"]
        if st["allowed"] is not None:
            y = y.masked_fill(~_allowed(st["allowed"][a:b], vocab), -math.inf)
        return z, y - torch.logsumexp(y, 1, keepdim=True)

    parts, grads = [], []
    if case["kind"] == "preference":
        return _exact_preference(st, case, log_rows, block, want)
    for a in range(0, rows, block):
        b = min(rows, a + block)
        z, lp = log_rows(a, b)
        one = _exact_distill if case["kind"] == "distill" else _exact_policy
        got = one(st, case, lp, a, b)
        if want:
            grads.append(torch.autograd.grad(got["loss"].sum(), z)[0])
        parts.append({k: v.detach() for k, v in got.items()})
    out = {k: torch.cat([x[k] for x in parts]) for k in parts[0]}
    return {**out, "grad": torch.cat(grads) if want else None}


def _exact_distill(st, case, lp, a, b):
    ids, w = st["ids"][a:b].long(), st["weight"][a:b].double()
    ok = torch.isfinite(lp.detach().gather(1, ids))
    if st["count"] is not None:
        ok &= torch.arange(ids.shape[1], device="cuda")[None] < st["count"][a:b, None]
    val = st["values"][a:b].double().masked_fill(~ok, -math.inf)
    at = lp.gather(1, ids).masked_fill(~ok, 0.0)
    if not case["tail"]:
        empty = ~ok.any(1, keepdim=True)
        lq = torch.log_softmax((val / case["temperature"]).masked_fill(empty, 0.0), 1)
        term = lq.exp() * (lq.masked_fill(~ok, 0.0) - at)
        return {"loss": w * term.masked_fill(~ok, 0.0).sum(1)}
    q = val.exp()
    left = (1.0 - q.sum(1)).clamp_min(0.0)
    hidden = torch.zeros(lp.shape, dtype=torch.bool, device="cuda").scatter_(1, ids, ok)
    rest = torch.logsumexp(lp.masked_fill(hidden, -math.inf), 1)
    loss = (q * (val - at).masked_fill(~ok, 0.0)).sum(1)
    return {"loss": w * (loss + torch.xlogy(left, left) - torch.where(left > 0, left * rest, 0.0))}


def _exact_policy(st, case, lp, a, b):
    token = st["tokens"][a:b].long()
    used = token >= 0
    at = lp.gather(1, token.clamp_min(0)[:, None])[:, 0].masked_fill(~used, 0.0)
    finite = lp.masked_fill(~torch.isfinite(lp.detach()), 0.0)
    entropy = -(lp.exp() * finite).sum(1)
    adv = st["advantage"][a:b].double()
    ratio = (at - st["old"][a:b].double()).exp()
    loss = -torch.min(ratio * adv, ratio.clamp(0.8, 1.28) * adv) - case["entropy"] * entropy
    if st["ref"] is not None:
        far = st["ref"][a:b].double() - at
        loss = loss + case["kl"] * (far.exp() - far - 1.0)
    w = st["weight"][a:b].double().masked_fill(~used, 0.0)
    return {"loss": w * loss, "logprob": at, "entropy": entropy}


def _exact_preference(st, case, log_rows, block, want):
    token = st["tokens"].long()
    rows, used = token.numel(), token >= 0
    with torch.no_grad():
        lp = torch.cat([log_rows(a, min(rows, a + block))[1].gather(
            1, token[a:a + block].clamp_min(0)[:, None])[:, 0] for a in range(0, rows, block)])
    lp = lp.masked_fill(~used, 0.0).requires_grad_(True)
    edges = st["start"].tolist()
    ratios = []
    for lo, hi in zip(edges[:-1], edges[1:]):
        one = lp[lo:hi] - (0.0 if st["ref"] is None else st["ref"][lo:hi].double())
        total = one.masked_fill(~used[lo:hi], 0.0).sum()
        ratios.append(total / max(1, int(used[lo:hi].sum())) if case["normalised"] else total)
    ratios = torch.stack(ratios)
    gap = ratios[0::2] - ratios[1::2]
    s = case["smoothing"]
    if case["loss"] == "sigmoid":
        loss = -(1 - s) * torch.nn.functional.logsigmoid(0.1 * gap) \
            - s * torch.nn.functional.logsigmoid(-0.1 * gap)
    elif case["loss"] == "hinge":
        loss = torch.relu(1.0 - 0.1 * gap)
    else:
        loss = (gap - 5.0) ** 2
    loss = loss * st["weight"].double()
    out = {"loss": loss.detach(), "ratios": ratios.detach(), "logprob": lp.detach(), "grad": None}
    if want:
        by_row = torch.autograd.grad(loss.sum(), lp)[0].masked_fill(~used, 0.0)
        grads = []
        for a in range(0, rows, block):
            z, y = log_rows(a, min(rows, a + block))
            at = y.gather(1, token[a:a + block].clamp_min(0)[:, None])[:, 0]
            grads.append(torch.autograd.grad((at * by_row[a:a + block]).sum(), z)[0])
        out["grad"] = torch.cat(grads)
    return out


def work(case):
    rows, vocab = _rows_of(case), case["vocab"]
    size = 4 if case["dtype"] == "f32" else 2
    passes = 2 if case["direction"] == "both" else 1
    read = rows * vocab * size * passes + rows * 32
    if case["kind"] == "distill":
        read += rows * case["k"] * 8
    if case["mask"]:
        read += rows * ((vocab + 31) // 32) * 4
    # a difference, an exponential and an addition for the sum, as much again for the gradient
    return {"bytes": read, "flops": 4 * rows * vocab * passes}
