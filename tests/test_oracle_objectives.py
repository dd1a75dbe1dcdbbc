"""The float64 objectives of the oracle against automatic differentiation of
torch's own functions and against differences of the losses (CPU only).

Tolerances: both sides are float64, so automatic differentiation has to agree to
some hundreds of ulps (1e-12); a central difference with step 1e-5 is off by its
third-order term, about 1e-10 times derivatives of order 1, and by rounding of
the loss, 1e-16 / 1e-5 = 1e-11."""

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import objectives as ob

ROWS, VOCAB = 7, 11
SEQS = [(0, 2), (2, 5), (5, 5), (5, 7)]


def inputs(seed=0):
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 2, (ROWS, VOCAB))
    tokens = rng.integers(0, VOCAB, ROWS)
    tokens[3] = -100
    return rng, x, tokens


def differences(fn, x, step=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += step
        b[i] -= step
        g[i] = (fn(a) - fn(b)) / (2 * step)
    return g


def auto(fn, x):
    t = torch.tensor(x, dtype=torch.float64, requires_grad=True)
    loss = fn(t)
    return loss.item(), torch.autograd.grad(loss, t)[0].numpy()


def chosen(t, tokens, temperature):
    lq = torch.log_softmax(t / temperature, -1)
    keep = torch.tensor(tokens != -100)
    return torch.where(keep, lq.gather(1, torch.tensor(np.maximum(tokens, 0))[:, None])[:, 0], 0.0), keep, lq


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_token_logprobs(temperature):
    rng, x, tokens = inputs()
    g, h = rng.normal(size=ROWS), rng.normal(size=ROWS)
    lp, ent, grad = ob.token_logprobs(x, tokens, temperature, dlogprobs=g, dentropy=h)

    def loss(t):
        c, keep, lq = chosen(t, tokens, temperature)
        e = torch.special.entr(lq.exp()).sum(-1) * keep
        return (c * torch.tensor(g)).sum() + (e * torch.tensor(h)).sum()

    value, expect = auto(loss, x)
    assert value == pytest.approx((lp * g + ent * h).sum(), rel=1e-12)
    np.testing.assert_allclose(grad, expect, rtol=1e-12, atol=1e-14)

    def plain(y):
        a, b, _ = ob.token_logprobs(y, tokens, temperature)
        return (a * g + b * h).sum()

    np.testing.assert_allclose(grad, differences(plain, x), atol=1e-8)


@pytest.mark.parametrize("by_sequence", [False, True])
@pytest.mark.parametrize("kl", [0.0, 0.3])
def test_policy_loss(by_sequence, kl):
    rng, x, tokens = inputs(1)
    lp, _, _ = ob.token_logprobs(x, tokens, 0.9)
    old, adv = lp + rng.normal(0, 0.3, ROWS), rng.normal(size=ROWS)
    ref = lp + rng.normal(0, 0.3, ROWS) if kl else None
    kw = dict(ref=ref, kl_coef=kl, clip=(0.2, 0.28), sequences=SEQS if by_sequence else None, temperature=0.9,
              scale=0.5)
    loss, _, _, clipped, grad = ob.policy_loss(x, tokens, old, adv, **kw)
    assert 0 < clipped < 1  # both branches are there

    def fn(t):
        c, keep, _ = chosen(t, tokens, 0.9)
        ratio = (c - torch.tensor(old)).exp()
        a = torch.tensor(adv)
        row = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.28) * a)
        if kl:
            d = torch.tensor(ref) - c
            row = row + kl * (d.exp() - d - 1)
        if not by_sequence:
            return 0.5 * row[keep].mean()
        means = [row[a:b][keep[a:b]].mean() for a, b in SEQS if keep[a:b].any()]
        return 0.5 * torch.stack(means).mean()

    value, expect = auto(fn, x)
    assert loss == pytest.approx(value, rel=1e-12)
    np.testing.assert_allclose(grad, expect, rtol=1e-11, atol=1e-14)
    np.testing.assert_allclose(grad, differences(lambda y: ob.policy_loss(y, tokens, old, adv, **kw)[0], x), atol=1e-8)


@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.1), ("ipo", 0.0), ("hinge", 0.0)])
@pytest.mark.parametrize("mean", [False, True])
def test_preference_loss(kind, smoothing, mean):
    rng, x, tokens = inputs(2)
    ref = rng.normal(-3, 2, len(SEQS))
    kw = dict(beta=0.3, kind=kind, label_smoothing=smoothing, length_average=mean)
    loss, _, _, grad = ob.preference_loss(x, tokens, ref, SEQS, **kw)

    def fn(t):
        c, keep, _ = chosen(t, tokens, 1.0)
        s = torch.stack([c[a:b].sum() / (max(1, int(keep[a:b].sum())) if mean else 1) for a, b in SEQS])
        r = 0.3 * (s - torch.tensor(ref))
        h = r[:2] - r[2:]
        if kind == "sigmoid":
            return (-(1 - smoothing) * F.logsigmoid(h) - smoothing * F.logsigmoid(-h)).mean()
        return ((h / 0.3 - 0.5 / 0.3) ** 2).mean() if kind == "ipo" else torch.relu(1 - h).mean()

    value, expect = auto(fn, x)
    assert loss == pytest.approx(value, rel=1e-12)
    np.testing.assert_allclose(grad, expect, rtol=1e-11, atol=1e-14)
    np.testing.assert_allclose(grad, differences(lambda y: ob.preference_loss(y, tokens, ref, SEQS, **kw)[0], x),
                               atol=1e-7 if kind == "ipo" else 1e-8)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_loss(tail):
    rng, x, _ = inputs(3)
    index = np.stack([rng.permutation(VOCAB)[:4] for _ in range(ROWS)])
    index[1, 2] = -1         # padding
    index[2, 3] = index[2, 0]  # an entry given twice
    t = rng.normal(2, 1, (ROWS, 4))
    t[4, 1] = -np.inf        # padding, too
    lse = np.logaddexp.reduce(t / 2.0, axis=1) + rng.uniform(0.05, 0.5, ROWS) if tail else None
    mask = np.array([1, 1, 1, 0, 1, 1, 1], bool)
    kw = dict(teacher_lse=lse, mask=mask, temperature=2.0, scale=0.5)
    loss, grad = ob.distill_loss(x, t, index, **kw)

    def fn(xt):
        lq = torch.log_softmax(xt / 2.0, -1)
        total = 0.0
        for r in np.flatnonzero(mask):
            keep = (index[r] >= 0) & np.isfinite(t[r])
            i, tt = torch.tensor(index[r][keep]), torch.tensor(t[r][keep]) / 2.0
            logp = tt - lse[r] if tail else torch.log_softmax(tt, 0)
            total = total + (logp.exp() * (logp - lq[r, i])).sum()
            if tail:
                out = torch.ones(VOCAB, dtype=torch.bool)
                out[i] = False
                rest = 1 - logp.exp().sum()
                total = total + rest * (rest.log() - torch.logsumexp(lq[r][out], 0))
        return 0.5 * 4.0 * total / int(mask.sum())

    value, expect = auto(fn, x)
    assert loss == pytest.approx(value, rel=1e-12)
    np.testing.assert_allclose(grad, expect, rtol=1e-10, atol=1e-13)
    np.testing.assert_allclose(grad, differences(lambda y: ob.distill_loss(y, t, index, **kw)[0], x), atol=1e-8)


def with_a_rest(x, t, index, lse):
    """(the loss by torch, its gradient): sum p (log p - log q) + P (log P - log Q), P at least 2^-20, T = 1."""
    def fn(xt):
        lq, total = torch.log_softmax(xt, -1), 0.0
        for r in range(len(x)):
            i, logp = torch.tensor(index[r]), torch.tensor(t[r] - lse[r])
            total = total + (logp.exp() * (logp - lq[r, i])).sum()
            out = torch.ones(x.shape[1], dtype=torch.bool)
            out[i] = False
            if out.any():
                rest = (1 - logp.exp().sum()).clamp(min=2.0**-20)
                total = total + rest * (rest.log() - torch.logsumexp(lq[r][out], 0))
        return total / len(x)

    return auto(fn, x)


@pytest.mark.parametrize("k", [4, VOCAB])
@pytest.mark.parametrize("extra", [0.5, 0.015, -0.4])
def test_distill_loss_of_probabilities_that_do_not_add_up(k, extra):
    """To 1 + extra, as a teacher's logits do that were rounded after their logsumexp was taken."""
    rng, x, _ = inputs(4)
    index = np.stack([rng.permutation(VOCAB)[:k] for _ in range(ROWS)])
    t = rng.normal(0, 1, (ROWS, k))
    lse = np.logaddexp.reduce(t, axis=1) - np.log1p(extra)
    loss, grad = ob.distill_loss(x, t, index, lse)
    value, expect = with_a_rest(x, t, index, lse)
    assert loss == pytest.approx(value, rel=1e-12)
    np.testing.assert_allclose(grad, expect, rtol=1e-10, atol=1e-13)
    np.testing.assert_allclose(grad, differences(lambda y: ob.distill_loss(y, t, index, lse)[0], x), atol=1e-8)


@pytest.mark.parametrize("gap", [30.0, 2000.0])
def test_distill_loss_of_a_rest_far_below(gap):
    """The student leaves next to nothing to the other entries: in 64 bits, too, it may underflow."""
    rng, x, _ = inputs(5)
    index = np.stack([rng.permutation(VOCAB)[:4] for _ in range(ROWS)])
    np.put_along_axis(x, index, np.take_along_axis(x, index, 1) + gap, 1)
    t = rng.normal(0, 1, (ROWS, 4))
    lse = np.logaddexp.reduce(t, axis=1) + 0.2
    loss, grad = ob.distill_loss(x, t, index, lse)
    value, expect = with_a_rest(x, t, index, lse)
    assert loss == pytest.approx(value, rel=1e-12)
    np.testing.assert_allclose(grad, expect, rtol=1e-10, atol=1e-13)
