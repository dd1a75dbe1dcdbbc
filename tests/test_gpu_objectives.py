"""The objectives' kernels against the float64 oracle, at the sizes, strides and
masks where they can go wrong.

Tolerances, with u = 2^-24 the rounding of one float32 operation.  y_j =
(x_j - M) log2(e)/T carries two roundings, so exp(y_j) is off by 3 u |y_j| + 4 u
of itself; summed with weights q_j that is at most 3 u (log V + 2) + 4 u, the sum
itself adds V/256 + 16 roundings at most, the logarithm 2 u log V, and a
log-probability l its own 3 u |l|:
    d = u (6 log V + V/256 + 32 + 3 |l|).
A gradient a ([j = t] - q_j) is off by 4 d of |a| max(q_j, [j = t]) and by what a
is off, plus half a place of the type it is rounded to (2^-9, 2^-12 or 2^-25 of
the value; float16 below 2^-14: 2^-25)."""

import math

import numpy as np
import pytest
import torch

from oracle import objectives as ob
from triton_muon_adamw import distill_loss, policy_loss, preference_loss, token_logprobs

pytestmark = pytest.mark.gpu

U = 2.0**-24
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_PLACE = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def lp_tol(vocab, lp):
    return U * (6 * math.log(max(vocab, 2)) + vocab / 256 + 32 + 3 * np.abs(lp))


def f64(x):
    return None if x is None else x.detach().double().cpu().numpy()


def check_grad(got, expect, tol):
    place = HALF_PLACE[got.dtype] * np.abs(expect) + (2.0**-25 if got.dtype == torch.float16 else 1e-38)
    got = f64(got)
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - expect) - (tol + place), initial=-1.0)
    assert worst <= 0, worst


def make(rows, vocab, dtype, seed=0, std=2.0, ignored=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty((rows, vocab), device="cuda").normal_(0, std, generator=gen)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=gen)
    x[torch.arange(rows), tokens] += math.log(vocab)
    tokens[torch.rand(rows, device="cuda", generator=gen) < ignored] = -100
    return x.to(DTYPES[dtype]), tokens, gen


def normal(shape, std, gen):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=gen)


def q_or_one(x64, tokens, temperature):
    """max(q_j, [j = token]) of each row."""
    q = np.stack([np.exp(ob.log_softmax(r / temperature)) for r in x64]) if len(x64) else x64
    for r, t in enumerate(tokens):
        if t >= 0:
            q[r, t] = 1.0
    return q


SIZES = [(1, 1), (3, 2), (5, 7), (4, 64), (6, 255), (7, 256), (5, 1003), (9, 2048), (4, 4099), (3, 8192), (3, 16390),
         (2, 32003), (3, 50257), (2, 65536), (2, 128256), (2, 131077)]


# ---- token_logprobs

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", SIZES + [(300, 517), (2500, 33)])
@pytest.mark.parametrize("entropy,temperature", [(False, 1.0), (True, 0.7)])
def test_token_logprobs(gpu, dtype, rows, vocab, entropy, temperature):
    x, tokens, gen = make(rows, vocab, dtype)
    g, h = normal(rows, 1.0, gen), normal(rows, 0.5, gen)
    x.requires_grad_()
    out = token_logprobs(x, tokens, temperature=temperature, entropy=entropy)
    lp, ent = out if entropy else (out, None)
    torch.autograd.backward([lp, ent] if entropy else [lp], [g, h] if entropy else [g])
    x64, t = f64(x), tokens.cpu().numpy()
    elp, eent, egrad = ob.token_logprobs(x64, t, temperature, dlogprobs=f64(g), dentropy=f64(h) if entropy else None)
    tol = lp_tol(vocab, elp)
    assert (np.abs(f64(lp) - elp) <= tol).all()
    a = np.abs(f64(g))
    if entropy:
        # sum q y: 4 d of sum q |log q|, which is the entropy
        tol_ent = 4 * lp_tol(vocab, eent) * (1 + eent)
        assert (np.abs(f64(ent) - eent) <= tol_ent).all()
        # q |log q| is at most 1/e, and log q has the absolute error d
        a = a + np.abs(f64(h)) * (2 + eent)
        ent_part = (np.abs(f64(h)) * tol_ent)[:, None]
    else:
        ent_part = 0.0
    # |log q| q <= sqrt(q): the relative error of small q grows with |log q|
    weight = np.sqrt(q_or_one(x64, t, temperature))
    check_grad(x.grad, egrad, (4 * a * tol / temperature)[:, None] * weight + ent_part * weight / temperature)
    assert not x.grad[tokens == -100].any()
    with torch.no_grad():
        again = token_logprobs(x, tokens, temperature=temperature, entropy=entropy)
    for p, q in zip(again if entropy else [again], [lp, ent] if entropy else [lp]):
        assert torch.equal(p, q)


# ---- policy_loss

def policy_case(rows, vocab, dtype, seed=0, temperature=1.0, **kw):
    x, tokens, gen = make(rows, vocab, dtype, seed, **kw)
    lp, _, _ = ob.token_logprobs(f64(x), tokens.cpu().numpy(), temperature)
    near = torch.tensor(lp, dtype=torch.float32, device="cuda")
    return x, tokens, near + normal(rows, 0.3, gen), normal(rows, 1.0, gen), near + normal(rows, 0.4, gen)


def check_policy(x, tokens, old, adv, ref, out, grad, factor=1.0, **kw):
    vocab, t = x.shape[-1], tokens.flatten().cpu().numpy()
    flat = lambda v: None if v is None else f64(v.expand(x.shape[:-1]).flatten())  # noqa: E731
    x64, o, a, rf = f64(x).reshape(-1, vocab), flat(old), flat(adv), flat(ref)
    loss, lp, kl, clipped, egrad = ob.policy_loss(x64, t, o, a, rf, **kw)
    temperature = kw.get("temperature", 1.0)
    weight = np.abs(kw.get("scale", 1.0)) * np.where(np.abs(egrad).max(-1) > 0, 1.0, (t != -100) * 1.0)
    n = max(1, int((t != -100).sum()))
    seqs = kw.get("sequences")
    if seqs is None:
        weight = weight / n
    else:
        lengths = [max(1, int((t[b:e] != -100).sum())) for b, e in seqs]
        some = max(1, sum(int((t[b:e] != -100).any()) for b, e in seqs))
        for (b, e), k in zip(seqs, lengths):
            weight[b:e] /= k * some
    d = lp_tol(vocab, lp)
    size = np.exp(lp - o) * np.abs(a) * (1 + np.abs(lp - o))
    if rf is not None:
        size = size + abs(kw.get("kl_coef", 0.0)) * (np.exp(rf - lp) + np.abs(rf - lp) + 1)
    active = t != -100
    assert (np.abs(f64(out.logprobs).flatten() - lp) <= d).all()
    assert abs(out.loss.item() - loss) <= 2 * (weight * size * d)[active].sum() + 1e-38
    if rf is not None:
        assert abs(out.kl.item() - kl) <= 4 * ((np.exp(rf - lp) + np.abs(rf - lp) + 1) * d)[active].max(initial=0)
    assert abs(out.clipped.item() - clipped) <= 64 * U
    if grad is not None:
        tol = (4 * factor * weight * size * d / temperature * active)[:, None]
        check_grad(grad.reshape(-1, vocab), factor * egrad, tol * np.sqrt(q_or_one(x64, t, temperature)))
        assert not grad.reshape(-1, vocab)[torch.tensor(t == -100, device="cuda")].any()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", SIZES + [(300, 517), (2500, 33)])
@pytest.mark.parametrize("kl,temperature", [(0.0, 1.0), (0.1, 0.8)])
def test_policy_loss(gpu, dtype, rows, vocab, kl, temperature):
    x, tokens, old, adv, ref = policy_case(rows, vocab, dtype, temperature=temperature)
    x.requires_grad_()
    ref = ref if kl else None
    out = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=kl, clip=(0.2, 0.28), temperature=temperature)
    out.loss.backward()
    check_policy(x, tokens, old, adv, ref, out, x.grad, kl_coef=kl, clip=(0.2, 0.28), temperature=temperature)
    with torch.no_grad():
        again = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=kl, clip=(0.2, 0.28),
                            temperature=temperature)
    assert all(torch.equal(p, q) for p, q in zip(again, out))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("average", ["token", "sequence"])
def test_policy_sequences(gpu, packed, average):
    """Sequences of lengths 0, 1 and more, one with no token that counts; int32 tokens and offsets; broadcast
    advantages."""
    x, tokens, old, adv, ref = policy_case(24, 301, "bf16", 3)
    if packed:
        seqs = [(0, 1), (1, 9), (9, 9), (9, 20), (20, 24)]
        tokens[20:] = -100
        offsets = torch.tensor([0, 1, 9, 9, 20, 24], dtype=torch.int32, device="cuda")
    else:
        x, tokens, old, ref = x.view(4, 6, -1), tokens.view(4, 6), old.view(4, 6), ref.view(4, 6)
        adv = adv[:4, None]
        seqs, offsets = [(0, 6), (6, 12), (12, 18), (18, 24)], None
        tokens[2] = -100
    tokens = tokens.int()
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=0.2, average=average, offsets=offsets, scale=0.25)
    out.loss.backward()
    check_policy(x, tokens, old, adv, ref, out, x.grad, kl_coef=0.2, scale=0.25,
                 sequences=seqs if average == "sequence" else None)


@pytest.mark.parametrize("packed", [False, True])
def test_policy_many_sequences(gpu, packed):
    """More sequences than are counted one by one; every third without a token that counts, packed ones also empty."""
    x, tokens, old, adv, ref = policy_case(3 * 131, 17, "fp32", 8)
    tokens.view(131, 3)[::3] = -100
    bounds = [min(2 * i, 393) for i in range(1 + 210)] if packed else list(range(0, 394, 3))
    kw = {}
    if packed:
        kw["offsets"] = torch.tensor(bounds, device="cuda")
    else:
        x, tokens, old, adv, ref = (t.view(131, 3, *t.shape[1:]) for t in (x, tokens, old, adv, ref))
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=0.2, average="sequence", **kw)
    out.loss.backward()
    check_policy(x, tokens, old, adv, ref, out, x.grad, kl_coef=0.2, sequences=list(zip(bounds, bounds[1:])))


def test_sequences_of_one_token(gpu):
    """Padded sequences of length 1: one value a sequence is one value a row, too."""
    x, tokens, old, adv, ref = policy_case(6, 130, "bf16", 2, ignored=0.0)
    x, tokens, old, adv, ref = x[:, None], tokens[:, None], old[:, None], adv[:, None], ref[:, None]
    tokens[3] = -100
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=0.2, average="sequence")
    out.loss.backward()
    check_policy(x, tokens, old, adv, ref, out, x.grad, kl_coef=0.2, sequences=[(i, i + 1) for i in range(6)])
    y, places = x.detach()[:, 0].requires_grad_(), torch.arange(7, device="cuda")
    x.grad = None
    padded = preference_loss(x, tokens, old[:, 0])
    packed = preference_loss(y, tokens[:, 0], old[:, 0], offsets=places)
    padded.loss.backward()
    packed.loss.backward()
    assert all(torch.equal(p, q) for p, q in zip(padded, packed)) and torch.equal(x.grad[:, 0], y.grad)


def test_policy_rows_outside_sequences(gpu):
    """Rows before the first offset and after the last do not count with average="sequence"."""
    x, tokens, old, adv, ref = policy_case(12, 65, "fp32", 5, ignored=0.0)
    offsets = torch.tensor([2, 5, 9], device="cuda")
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=0.2, average="sequence", offsets=offsets)
    out.loss.backward()
    inside = tokens.clone()
    inside[:2] = inside[9:] = -100
    check_policy(x, inside, old, adv, ref, out, x.grad, kl_coef=0.2, sequences=[(2, 5), (5, 9)])


@pytest.mark.parametrize("rows", [3, 5000])
def test_no_sequences(gpu, rows):
    """Offsets of one place: no sequence, so nothing counts."""
    x, tokens, old, adv, _ = policy_case(rows, 9, "fp32", 5, ignored=0.0)
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, average="sequence", offsets=torch.zeros(1, dtype=torch.int64, device="cuda"))
    out.loss.backward()
    assert out.loss == 0 and out.clipped == 0 and not x.grad.any()


def test_many_rows(gpu):
    """More rows than one workgroup adds up, and more than fit the first dimension of a launch's grid."""
    rows, vocab = 70001, 5
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = normal((rows, vocab), 2.0, gen)
    tokens = torch.randint(vocab, (rows,), device="cuda", generator=gen)
    old, adv = normal(rows, 0.3, gen) - 1.6, normal(rows, 1.0, gen) + 0.5
    y = x.clone().requires_grad_()
    out = policy_loss(y, tokens, old, adv)
    out.loss.backward()
    logq = torch.log_softmax(x.double(), -1)
    lp = logq.gather(1, tokens[:, None])[:, 0]
    ratio, a = (lp - old.double()).exp(), adv.double()
    bound = ratio.clamp(0.8, 1.2)
    size = (ratio.abs() * a.abs()).mean().item()
    assert abs(out.loss.item() + torch.minimum(ratio * a, bound * a).mean().item()) <= 64 * U * size
    slope = torch.where(bound * a < ratio * a, 0.0, -a * ratio) / rows
    g = (torch.nn.functional.one_hot(tokens, vocab) - logq.exp()) * slope[:, None]
    assert ((y.grad.double() - g).abs() <= 64 * U * (ratio * a.abs())[:, None] / rows).all()
    assert (token_logprobs(x, tokens).double() - lp).abs().max() <= 64 * U
    index = tokens[:, None]
    assert distill_loss(x, torch.zeros_like(index, dtype=torch.float32), index).item() == pytest.approx(
        -lp.mean().item(), rel=1e-6)
    half = preference_loss(x[:70000].view(1000, 70, 5), tokens[:70000].view(1000, 70), None)
    s = lp[:70000].view(2, 500, 70).sum(-1)
    assert half.loss.item() == pytest.approx(-torch.nn.functional.logsigmoid(0.1 * (s[0] - s[1])).mean().item(), rel=1e-5)


def test_offsets_that_hold_anything_stay_inside(gpu):
    """Offsets beyond the rows are cut to them; nothing is read outside."""
    x, tokens, old, adv, _ = policy_case(12, 65, "fp32", 5, ignored=0.0)
    for offsets in ([-5, 7, 4, 1 << 40], [0, 0, 0, 0], [12, 12, 40, 41]):
        o = torch.tensor(offsets, device="cuda")
        policy_loss(x.requires_grad_(), tokens, old, adv, average="sequence", offsets=o).loss.backward()
        preference_loss(x, tokens, None, offsets=o[:3]).loss.backward()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [37, 50257, 131077])
@pytest.mark.parametrize("factor", [0.125, 3.0, 65536.0])
def test_policy_scaled_backward(gpu, dtype, vocab, factor):
    """A gradient of the loss other than 1 (a scaler's, for one) is in the gradient before it is rounded."""
    x, tokens, old, adv, ref = policy_case(5, vocab, dtype, 7)
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=0.1)
    (out.loss * factor).backward()
    if dtype == "fp16" and factor > 1000:
        assert f64(x.grad).__abs__().max() < 65504
    check_policy(x, tokens, old, adv, ref, out, x.grad, factor=factor, kl_coef=0.1)


def test_retained_graph(gpu):
    """A second backward through the same graph gives the same gradient in memory of its own."""
    x, tokens, old, adv, _ = policy_case(6, 1003, "bf16", 9)
    x.requires_grad_()
    loss = policy_loss(x, tokens, old, adv).loss
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    keep = first.clone()
    second, = torch.autograd.grad(2 * loss, x, retain_graph=True)
    third, = torch.autograd.grad(loss, x)
    assert torch.equal(first, keep) and torch.equal(third, keep)
    assert first.data_ptr() != second.data_ptr()
    assert torch.equal(second, 2 * keep)  # a power of two rounds alike


def test_inputs_changed_in_place_are_noticed(gpu):
    x, tokens, old, adv, _ = policy_case(6, 103, "fp32", 9)
    x.requires_grad_()
    loss = policy_loss(x, tokens, old, adv).loss
    adv.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("which", ["logprobs", "policy", "preference", "distill"])
def test_graphs_used_twice(gpu, which):
    """Backward a second time without retain_graph is torch's error; a gradient with create_graph is the same, and
    differentiating it is an error."""
    x, tokens, old, adv, _ = policy_case(6, 103, "fp32", 9)
    x.requires_grad_()
    index = torch.arange(4, device="cuda").repeat(6, 1)
    make = {"logprobs": lambda: token_logprobs(x, tokens).sum(),
            "policy": lambda: policy_loss(x, tokens, old, adv).loss,
            "preference": lambda: preference_loss(x.view(2, 3, -1), tokens.view(2, 3), None).loss,
            "distill": lambda: distill_loss(x, torch.ones((6, 4), device="cuda"), index)}[which]
    loss = make()
    first, = torch.autograd.grad(loss, x)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, x)
    again, = torch.autograd.grad(make(), x, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError, match="differentiated a second time"):
        again.sum().backward()


def test_only_one_output_used(gpu):
    """Entropies alone in the loss, and a graph that reaches the logits through a view."""
    x, tokens, _ = make(6, 103, "fp32", 9)
    x.requires_grad_()
    a, = torch.autograd.grad(token_logprobs(x.view(2, 3, -1), tokens.view(2, 3), entropy=True)[1].sum(), x)
    _, _, egrad = ob.token_logprobs(f64(x), tokens.cpu().numpy(), dentropy=np.ones(6))
    check_grad(a, egrad, 1e-5)


# ---- preference_loss

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [1, 2, 517, 4099, 50257, 128256])
@pytest.mark.parametrize("kind,smoothing,mean", [("sigmoid", 0.0, False), ("sigmoid", 0.2, True), ("ipo", 0.0, True),
                                                 ("hinge", 0.0, False)])
@pytest.mark.parametrize("packed", [False, True])
def test_preference_loss(gpu, dtype, vocab, kind, smoothing, mean, packed):
    x, tokens, gen = make(24, vocab, dtype, 11)
    if packed:  # one sequence empty, one with no token that counts
        bounds = [0, 5, 5, 6, 13, 20, 24]
        tokens[20:] = -100
        offsets = torch.tensor(bounds, device="cuda")
    else:
        bounds = [0, 4, 8, 12, 16, 20, 24]
        x, tokens, offsets = x.view(6, 4, -1), tokens.view(6, 4), None
    seqs = list(zip(bounds[:-1], bounds[1:]))
    x64, t = f64(x).reshape(24, vocab), tokens.flatten().cpu().numpy()
    beta = 0.3
    elp = ob.preference_loss(x64, t, None, seqs, beta, length_average=mean)[1]
    ref = torch.tensor(elp, dtype=torch.float32, device="cuda") + normal(6, 2.0, gen)
    loss, elp, erew, egrad = ob.preference_loss(x64, t, f64(ref), seqs, beta, kind, smoothing, mean)
    x.requires_grad_()
    out = preference_loss(x, tokens, ref, beta=beta, kind=kind, label_smoothing=smoothing, length_average=mean,
                          offsets=offsets)
    out.loss.backward()
    row_lp = ob.token_logprobs(x64, t)[0]
    d = lp_tol(vocab, row_lp).max() * 13 + 16 * U * np.abs(elp).max()  # at most 13 rows a sequence
    assert (np.abs(f64(out.logprobs) - elp) <= d).all()
    dr = beta * (d + 4 * U * (np.abs(elp).max() + np.abs(f64(ref)).max()))
    assert (np.abs(f64(out.rewards) - erew) <= dr).all()
    h = erew[:3] - erew[3:]
    if kind == "ipo":
        slope, curve = 2 * np.abs(h / beta - 0.5 / beta).max() / beta, 2 / beta**2
    else:
        slope, curve = 1.0, (0.25 if kind == "sigmoid" else 0.0)
        assert kind != "hinge" or np.abs(h - 1).min() > 2 * dr  # no pair at the corner
    assert abs(out.loss.item() - loss) <= 2 * slope * dr + 16 * U * (abs(loss) + 1)
    a = beta / 3 * (slope * 4 * lp_tol(vocab, row_lp) + 2 * curve * dr + 8 * U * slope)
    check_grad(x.grad.reshape(24, vocab), egrad, a[:, None] * np.sqrt(q_or_one(x64, t, 1.0)))
    with torch.no_grad():
        again = preference_loss(x, tokens, ref, beta=beta, kind=kind, label_smoothing=smoothing, length_average=mean,
                                offsets=offsets)
    assert all(torch.equal(p, q) for p, q in zip(again, out))


def test_preference_scaled_backward_and_no_reference(gpu):
    x, tokens, _ = make(8, 999, "fp16", 13)
    x = x.view(2, 4, -1).requires_grad_()
    tokens = tokens.view(2, 4)
    loss = preference_loss(x, tokens, None).loss
    (loss * 1024).backward()
    _, _, _, egrad = ob.preference_loss(f64(x).reshape(8, -1), tokens.flatten().cpu().numpy(), None, [(0, 4), (4, 8)])
    check_grad(x.grad.reshape(8, -1), 1024 * egrad, 1024 * 0.1 * 1e-4)


def test_preference_extreme_margins(gpu):
    """|h| of some hundreds: the loss is |h| or 0, and nothing overflows."""
    x, tokens, _ = make(4, 77, "fp32", 15, ignored=0.0)
    x = x.view(2, 2, -1).requires_grad_()
    tokens = tokens.view(2, 2)
    for shift in (-5000.0, 5000.0):
        ref = torch.tensor([shift, 0.0], device="cuda")
        out = preference_loss(x, tokens, ref, beta=0.5)
        grad, = torch.autograd.grad(out.loss, x)
        loss, _, _, egrad = ob.preference_loss(f64(x).reshape(4, -1), tokens.flatten().cpu().numpy(), f64(ref),
                                               [(0, 2), (2, 4)], 0.5)
        assert out.loss.item() == pytest.approx(loss, rel=1e-5, abs=1e-30)
        check_grad(grad.reshape(4, -1), egrad, 1e-5)


# ---- distill_loss

def teacher(x, k, gen, dtype, temperature, tail):
    rows, vocab = x.shape
    index = torch.rand((rows, vocab), device="cuda", generator=gen).argsort(-1)[:, :k].contiguous()
    t = (normal((rows, k), 1.5, gen) + math.log(vocab)).to(DTYPES[dtype])
    rest = 0.02 + 0.4 * torch.rand(rows, device="cuda", generator=gen)
    lse = torch.logsumexp(t.double() / temperature, -1) - torch.log1p(-rest.double()) if tail else None
    return t, index, None if lse is None else lse.float()


def check_distill(x, t, index, lse, mask, temperature, loss, grad, factor=1.0, scale=1.0):
    vocab, k = x.shape[-1], t.shape[-1]
    x64, t64 = f64(x).reshape(-1, vocab), f64(t).reshape(-1, k)
    i = index.reshape(-1, k).cpu().numpy()
    m = np.ones(len(x64), bool) if mask is None else mask.flatten().cpu().numpy()
    l64 = None if lse is None else f64(lse).flatten()
    eloss, egrad = ob.distill_loss(x64, t64, i, l64, m, temperature, scale)
    logq = np.stack([ob.log_softmax(r / temperature) for r in x64])
    valid = (i >= 0) & (t64 != -np.inf)
    most = np.abs(np.where(valid, t64, 0.0)).max() / temperature
    ep = U * (k + 8 + 6 * most + (0 if lse is None else 3 * np.abs(l64).max()))  # of a teacher's probability, or their sum
    logqs = np.abs(np.where(valid, np.take_along_axis(logq, np.maximum(i, 0), 1), 0.0))
    d = lp_tol(vocab, logqs.max())
    per_row = d + ep * (logqs.max() + most + 1)
    if lse is not None:
        q = np.exp(logq)
        inside = np.zeros_like(q, dtype=bool)
        for r in range(len(q)):
            inside[r, i[r][valid[r]]] = True
        rest_q = np.maximum((q * ~inside).sum(-1), 1e-300)
        per_row += ep * (np.abs(np.log(rest_q)).max() + 21)
    assert abs(loss.item() - eloss) <= 2 * scale * temperature**2 * per_row
    if grad is not None:
        w = factor * scale * temperature / max(1, m.sum())
        size = np.sqrt(np.exp(logq))
        tol = w * 4 * d * size
        for r in range(len(size)):
            np.add.at(tol[r], i[r][valid[r]], 4 * w * ep)
        if lse is not None:
            tol += w * size * (ep / np.minimum(rest_q, 1.0) + 4 * d / rest_q)[:, None]
        check_grad(grad.reshape(-1, vocab), factor * egrad, tol * m[:, None])


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 1), (5, 7, 7), (6, 255, 8), (5, 1003, 64), (9, 2048, 1024),
                                          (3, 8192, 3), (3, 16390, 257), (3, 50257, 64), (2, 128256, 128),
                                          (2, 131077, 1000), (300, 517, 5)])
@pytest.mark.parametrize("tail,temperature", [(False, 2.0), (True, 1.0), (True, 3.0)])
def test_distill_loss(gpu, dtype, rows, vocab, k, tail, temperature):
    x, tokens, gen = make(rows, vocab, dtype, 21)
    t, index, lse = teacher(x, k, gen, dtype, temperature, tail)
    mask = tokens != -100
    x.requires_grad_()
    kw = dict(teacher_lse=lse, mask=mask, temperature=temperature, scale=0.5)
    loss = distill_loss(x, t, index, **kw)
    loss.backward()
    check_distill(x, t, index, lse, mask, temperature, loss, x.grad, scale=0.5)
    assert not x.grad[~mask].any()
    with torch.no_grad():
        assert torch.equal(distill_loss(x, t, index, **kw), loss)
    x.grad = None
    (distill_loss(x, t, index, **kw) * 48.0).backward()
    check_distill(x, t, index, lse, mask, temperature, loss, x.grad, factor=48.0, scale=0.5)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_padding_and_repeated_entries(gpu, tail):
    x, _, gen = make(8, 3001, "fp32", 23)
    t, index, lse = teacher(x, 12, gen, "fp32", 1.5, tail)
    index[0, 3:] = -1           # negative indices
    t[1, 5:] = -torch.inf       # logits of -inf,
    index[1, 5:] = 0            # whose indices repeat
    index[2] = -1               # nothing left
    index[3, 4] = index[3, 9] = index[3, 1]  # an entry given three times
    index[4, 0] = 0
    index[4, 1] = 3000
    if tail:
        lse = torch.logsumexp(torch.where(index < 0, -torch.inf, t / 1.5), -1).clamp(min=0.0) + 0.2
    x.requires_grad_()
    loss = distill_loss(x, t, index.int(), teacher_lse=lse, temperature=1.5)
    loss.backward()
    check_distill(x, t, index, lse, None, 1.5, loss, x.grad)
    assert torch.equal(loss, distill_loss(x, t, index.int(), teacher_lse=lse, temperature=1.5))


def test_distill_widest_tail(gpu):
    """The largest vocabulary with a rest: its table of bits takes 128 KiB of LDS."""
    x, _, gen = make(2, 1 << 20, "bf16", 25)
    index = torch.tensor([[0, 31, 32, 1048575], [5, 77777, 524288, 1000003]], device="cuda")
    t = normal((2, 4), 1.0, gen) + 14.0
    lse = torch.logsumexp(t, -1) + 0.3
    x.requires_grad_()
    loss = distill_loss(x, t, index, teacher_lse=lse)
    loss.backward()
    check_distill(x, t, index, lse, None, 1.0, loss, x.grad)
    wide = torch.zeros((1, (1 << 20) + 1), device="cuda")
    with pytest.raises(ValueError):
        distill_loss(wide, t[:1], index[:1], teacher_lse=lse[:1])


# ---- layouts

def everything(x, tokens, old, adv, ref, t, index, mask):
    """All four losses of one (batch, length, vocab) input with their gradients."""
    out = []
    for fn in (lambda y: (lambda o: (o[0].sum() + 0.1 * o[1].sum(), *o))(token_logprobs(y, tokens, entropy=True)),
               lambda y: policy_loss(y, tokens, old, adv, ref_logprobs=ref, kl_coef=0.1, average="sequence"),
               lambda y: preference_loss(y, tokens, ref.sum(-1)),
               lambda y: (distill_loss(y, t, index, mask=mask),)):
        y = x.detach().requires_grad_()
        res = fn(y)
        out += [*res, torch.autograd.grad(res[0], y)[0]]
    return [o.detach() for o in out]


def layout_inputs(vocab, dtype):
    x, tokens, gen = make(12, vocab, dtype, 31)
    shape = (4, 3)
    old, adv, ref = (normal(shape, 1.0, gen) - 3 for _ in range(3))
    t, index, _ = teacher(x, 5, gen, dtype, 1.0, False)
    return (x.view(4, 3, vocab), tokens.view(shape), old, adv, ref, t.view(4, 3, 5), index.view(4, 3, 5),
            (tokens != -100).view(shape))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [33, 1003, 9001, 50257, 70001])
def test_strides_and_alignment_change_nothing(gpu, dtype, vocab):
    """Padded and offset vocabularies, swapped dimensions, steps.  Which thread adds which logit goes by the row's
    place in memory, so results are equal to within their tolerance on either side: a log-probability's d, with
    values and gradients of order 1 here, and a place of the type."""
    dense = layout_inputs(vocab, dtype)
    expect = everything(*dense)
    x = dense[0]
    d = 16 * lp_tol(vocab, 40.0)

    def same(got, label):
        for i, (p, q) in enumerate(zip(got, expect)):
            off = np.abs(f64(p) - f64(q)) - (d * np.maximum(1.0, np.abs(f64(q))) + 2 * HALF_PLACE[q.dtype] * np.abs(f64(q)))
            assert off.max() <= 0, (label, i, off.max())

    def padded(v, left, right):
        wide = torch.full((*v.shape[:-1], v.shape[-1] + left + right), float("nan") if v.is_floating_point() else 1,
                          dtype=v.dtype, device="cuda")
        wide[..., left:left + v.shape[-1]] = v
        return wide[..., left:left + v.shape[-1]]

    def swapped(v):
        return v.transpose(0, 1).contiguous().transpose(0, 1)

    def stepped(v):
        wide = v.repeat_interleave(2, dim=1)
        return wide[:, ::2]

    for change in (lambda v: padded(v, 0, 7), lambda v: padded(v, 1, 2), lambda v: padded(v, 3, 64), swapped, stepped):
        same(everything(change(x), *[change(v) if v.dim() == 3 else swapped(v) for v in dense[1:]]), change)
    # logits that start off the 16-byte boundary
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    flat[1:] = x.flatten()
    same(everything(flat[1:].view(x.shape), *dense[1:]), "offset")


def test_broadcast_logits(gpu):
    x = torch.randn(1, 1003, device="cuda")
    tokens = torch.arange(6, device="cuda") * 100
    y = x.clone().requires_grad_()
    token_logprobs(y.expand(6, 1003), tokens).sum().backward()
    z = x.repeat(6, 1).requires_grad_()
    token_logprobs(z, tokens).sum().backward()
    assert torch.allclose(y.grad, z.grad.sum(0, keepdim=True), atol=1e-5)


@pytest.mark.parametrize("dtype", ["bf16"])
def test_offsets_beyond_32_bits(gpu, dtype):
    """Rows more than 2^31 elements and 2^32 bytes apart; off the 16-byte boundary where the near ones are on it, so
    to within the tolerance on either side (values of order 1)."""
    vocab, stride = 1003, (1 << 31) + 9
    flat = torch.empty(2 * stride + vocab, dtype=DTYPES[dtype], device="cuda")
    x, tokens, gen = make(3, vocab, dtype, 33, ignored=0.0)
    far = flat.as_strided((3, vocab), (stride, 1))
    far.copy_(x)
    old, adv = normal(3, 1.0, gen) - 4, normal(3, 1.0, gen)
    with torch.no_grad():
        pairs = [*zip(policy_loss(far, tokens, old, adv), policy_loss(x, tokens, old, adv)),
                 (token_logprobs(far, tokens), token_logprobs(x, tokens))]
    for a, b in pairs:
        assert (np.abs(f64(a) - f64(b)) <= 16 * lp_tol(vocab, f64(b)) * np.maximum(1.0, np.abs(f64(b)))).all()


def test_gradient_beyond_32_bits(gpu):
    """A gradient of more than 2^32 bytes and 2^31 elements: its last rows are as those of a small one."""
    vocab, rows = 128256, 16800
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device="cuda")
    tail, toks, gen = make(3, vocab, "bf16", 35, ignored=0.0)
    x[-3:] = tail
    tokens = torch.full((rows,), -100, device="cuda")
    tokens[-3:] = toks
    old, adv = normal(rows, 1.0, gen) - 4, normal(rows, 1.0, gen)
    small = tail.clone().requires_grad_()
    policy_loss(small, toks, old[-3:], adv[-3:]).loss.backward()
    x.requires_grad_()
    policy_loss(x, tokens, old, adv).loss.backward()
    assert torch.equal(x.grad[-3:], small.grad)
    assert not x.grad[:-3].any()
    grad, = torch.autograd.grad(token_logprobs(x, tokens).sum(), x)
    other, = torch.autograd.grad(token_logprobs(small, toks).sum(), small)
    assert torch.equal(grad[-3:], other)


# ---- values

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [9, 1003, 50257, 131077])
@pytest.mark.parametrize("masked", [-math.inf, "lowest"])
def test_masked_vocabulary(gpu, dtype, vocab, masked):
    """Entries at -inf or the type's lowest value have no probability and no gradient; nothing becomes NaN."""
    x, tokens, gen = make(6, vocab, dtype, 41, ignored=0.0)
    value = torch.finfo(x.dtype).min if masked == "lowest" else masked
    hidden = torch.rand((6, vocab), device="cuda", generator=gen) < 0.6
    hidden[0] = True  # all but the token
    hidden[torch.arange(6), tokens] = False
    x = x.masked_fill(hidden, value).requires_grad_()
    lp, ent = token_logprobs(x, tokens, entropy=True)
    (lp.sum() + ent.sum()).backward()
    elp, eent, egrad = ob.token_logprobs(f64(x), tokens.cpu().numpy(), dlogprobs=np.ones(6), dentropy=np.ones(6))
    assert (np.abs(f64(lp) - elp) <= lp_tol(vocab, elp)).all()
    assert (np.abs(f64(ent) - eent) <= 4 * lp_tol(vocab, eent) * (1 + eent)).all()
    check_grad(x.grad, egrad, 8 * lp_tol(vocab, elp).max() * (2 + eent.max()))
    assert not x.grad[hidden].any()
    y = x.detach().requires_grad_()
    old = torch.tensor(elp, device="cuda").float() + 0.1
    out = policy_loss(y, tokens, old, torch.ones(6, device="cuda"))
    out.loss.backward()
    check_policy(y, tokens, old, torch.ones(6, device="cuda"), None, out, y.grad)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [5, 1003, 50257, 131077])
def test_rows_of_the_lowest_value_are_uniform(gpu, dtype, vocab):
    low = torch.finfo(DTYPES[dtype]).min
    x = torch.full((2, vocab), low, dtype=DTYPES[dtype], device="cuda")
    x[1] = torch.finfo(DTYPES[dtype]).max
    x.requires_grad_()
    lp, ent = token_logprobs(x, torch.tensor([0, vocab - 1], device="cuda"), entropy=True, temperature=0.5)
    lp.sum().backward()
    assert torch.allclose(lp, torch.full_like(lp, -math.log(vocab)), atol=1e-4)
    assert torch.allclose(ent, torch.full_like(ent, math.log(vocab)), atol=1e-4)
    expect = np.full((2, vocab), -2.0 / vocab)
    expect[0, 0] += 2.0
    expect[1, -1] += 2.0
    check_grad(x.grad, expect, 1e-4 / vocab)


def test_rows_of_minus_infinity_or_nan_are_nan(gpu):
    x = torch.randn(4, 600, device="cuda")
    x[0] = -math.inf
    x[1, 7] = math.nan
    x[2, 599] = math.inf
    tokens = torch.tensor([3, 4, 5, 6], device="cuda")
    x.requires_grad_()
    lp = token_logprobs(x, tokens)
    assert lp[:3].isnan().all() and lp[3].isfinite()
    lp.sum().backward()
    assert x.grad[:2].isnan().all() and x.grad[3].isfinite().all()
    # and a token at -inf has probability 0
    y = torch.randn(1, 600, device="cuda")
    y[0, 9] = -math.inf
    assert token_logprobs(y, torch.tensor([9], device="cuda")).item() == -math.inf


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_that_do_not_count_are_not_read(gpu, dtype, bad):
    dense = list(layout_inputs(1003, dtype))
    tokens = dense[1]
    tokens[1] = -100
    tokens[0, 0] = 5
    dense[7] = tokens != -100
    out = ~dense[7]
    for i in (0, 2, 3, 5):  # logits, old, advantages, the teacher's logits
        dense[i] = dense[i].masked_fill(out if dense[i].dim() == 2 else out[..., None], 0.0)
    expect = everything(*dense)
    for i in (0, 2, 3, 5):
        dense[i] = dense[i].masked_fill(out if dense[i].dim() == 2 else out[..., None], bad)
    for p, q in zip(everything(*dense), expect):
        assert torch.equal(p, q)


def test_nothing_counts(gpu):
    x = torch.full((4, 3, 50), math.nan, device="cuda", requires_grad=True)
    tokens = torch.full((4, 3), 7, device="cuda")
    zeros = torch.zeros((4, 3), device="cuda")
    for average in ("token", "sequence"):
        out = policy_loss(x, tokens, zeros, zeros, ref_logprobs=zeros, kl_coef=0.1, average=average, ignore_index=7)
        grad, = torch.autograd.grad(out.loss, x)
        assert out.loss == 0 and out.kl == 0 and out.clipped == 0 and not grad.any() and not out.logprobs.any()
    out = preference_loss(x, tokens, None, ignore_index=7)
    grad, = torch.autograd.grad(out.loss, x)
    assert out.loss.item() == pytest.approx(math.log(2)) and not grad.any()
    loss = distill_loss(x, zeros[..., None], tokens[..., None], mask=zeros.bool())
    grad, = torch.autograd.grad(loss, x)
    assert loss == 0 and not grad.any()


def test_entropies_changed_in_place_raise(gpu):
    x, tokens, _ = make(4, 65, "fp32", 0)
    x.requires_grad_()
    lp, ent = token_logprobs(x, tokens, entropy=True)
    ent.mul_(0.5)
    with pytest.raises(RuntimeError, match="inplace"):
        ent.sum().backward()
    lp, ent = token_logprobs(x, tokens, entropy=True)
    (lp.sum() + (0.5 * ent).sum()).backward()
    assert x.grad.isfinite().all()


@pytest.mark.parametrize("which", ["logits", "shape", "tokens", "old"])
def test_inputs_given_other_memory_raise(gpu, which):
    """t.data = ... is seen by no version counter; backward reads by address."""
    x, tokens, old, adv, _ = policy_case(4, 65, "fp32", 0, ignored=0.0)
    leaf = x.clone().requires_grad_()
    for loss in (lambda y: policy_loss(y, tokens, old, adv).loss, lambda y: token_logprobs(y, tokens).sum()):
        if which == "old" and loss(leaf).grad_fn.name() != "PolicyLossBackward":
            continue
        y = leaf * 1.0
        out = loss(y)
        kept = tokens.data, old.data
        if which == "logits":
            y.data = torch.zeros_like(y)
        elif which == "shape":
            y.data = y.data[:2]
        elif which == "tokens":
            tokens.data = tokens.clone()
        else:
            old.data = old.clone()
        with pytest.raises(RuntimeError, match="after the forward pass"):
            out.backward()
        tokens.data, old.data = kept
        loss(leaf * 1.0).backward()


@pytest.mark.parametrize("shape", [(0, 9), (0, 3, 9), (2, 0, 9)])
def test_no_rows(gpu, shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True)
    tokens = torch.zeros(shape[:-1], dtype=torch.int64, device="cuda")
    f = torch.zeros(shape[:-1], device="cuda")
    lp, ent = token_logprobs(x, tokens, entropy=True)
    assert lp.shape == ent.shape == shape[:-1]
    (lp.sum() + ent.sum()).backward()
    assert x.grad.shape == shape
    out = policy_loss(x, tokens, f, f)
    out.loss.backward()
    assert out.loss == 0
    loss = distill_loss(x, torch.zeros((*shape[:-1], 2), device="cuda"),
                        torch.zeros((*shape[:-1], 2), dtype=torch.int64, device="cuda"))
    loss.backward()
    assert loss == 0
    if shape[0] == 2:
        out = preference_loss(x, tokens, torch.zeros(2, device="cuda"))
        out.loss.backward()
        assert out.loss.item() == pytest.approx(math.log(2))


def test_tokens_beyond_the_vocabulary_give_nan(gpu):
    x, tokens, gen = make(5, 1003, "fp32", 51, ignored=0.0)
    tokens[1], tokens[3] = 1003, -7
    x.requires_grad_()
    lp = token_logprobs(x, tokens)
    lp.sum().backward()
    assert lp.isnan().tolist() == [False, True, False, True, False]
    assert x.grad.isnan().any(-1).tolist() == [False, True, False, True, False]
    f = torch.zeros(5, device="cuda")
    assert policy_loss(x, tokens, f, f + 1).loss.isnan()
    assert preference_loss(x[:4], tokens[:4], None, offsets=torch.tensor([0, 2, 4], device="cuda")).loss.isnan()
    assert distill_loss(x, torch.zeros((5, 1), device="cuda"), tokens.clamp(min=0)[:, None]).isnan()


# ---- differences

def directional(loss_of, x, gen, step):
    """(difference of the loss along a random direction, the gradient along it)."""
    y = x.clone().requires_grad_()
    grad, = torch.autograd.grad(loss_of(y), y)
    d = normal(x.shape, 1.0, gen)
    with torch.no_grad():
        diff = (loss_of(x + step * d).double() - loss_of(x - step * d).double()) / (2 * step)
    return diff.item(), (grad.double() * d.double()).sum().item()


@pytest.mark.parametrize("which", ["logprobs", "entropy", "policy", "preference", "distill", "tail"])
def test_gradients_against_differences(gpu, which):
    """float32 losses of order 1 carry errors of about 1e-6, so a central difference with step 0.02 one of 5e-5; its
    third-order term is 0.02^2 / 6 times a third derivative along a direction in which each row's logits move by
    about one: some 1e-3 at most."""
    x, tokens, old, adv, ref = policy_case(16, 131, "fp32", 61)
    gen = torch.Generator(device="cuda").manual_seed(1)
    # no token near the corners of the clamp, where there is no derivative
    lp = token_logprobs(x, tokens)
    old = lp + torch.where(torch.arange(16, device="cuda") % 2 == 0, 0.02, 0.6)
    t, index, lse = teacher(x, 9, gen, "fp32", 1.0, True)
    fns = {
        "logprobs": lambda y: token_logprobs(y, tokens).mean(),
        "entropy": lambda y: token_logprobs(y, tokens, entropy=True)[1].mean(),
        "policy": lambda y: policy_loss(y, tokens, old, adv, ref_logprobs=ref, kl_coef=0.3).loss,
        "preference": lambda y: preference_loss(y.view(4, 4, -1), tokens.view(4, 4), None, beta=0.3).loss,
        "distill": lambda y: distill_loss(y, t, index),
        "tail": lambda y: distill_loss(y, t, index, teacher_lse=lse),
    }
    diff, grad = directional(fns[which], x, gen, 0.02)
    assert abs(diff - grad) <= 2e-3 * (1 + abs(grad)), (diff, grad)


# ---- streams and graphs

def test_another_stream(gpu):
    x, tokens, old, adv, ref = policy_case(64, 5003, "bf16", 71)
    expect = everything_flat(x, tokens, old, adv, ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything_flat(x, tokens, old, adv, ref)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, expect))


def everything_flat(x, tokens, old, adv, ref):
    y = x.detach().requires_grad_()
    out = policy_loss(y, tokens, old, adv, ref_logprobs=ref, kl_coef=0.1)
    (out.loss * 2).backward()
    return [o.detach() for o in out] + [y.grad]


def test_graph_capture(gpu):
    """One pass recorded and replayed with new logits: every replay as the eager call on the same values."""
    x, tokens, old, adv, ref = policy_case(32, 5003, "bf16", 73)
    index = torch.arange(8, device="cuda") * 500 + torch.arange(32, device="cuda")[:, None]
    t = normal((32, 8), 1.0, torch.Generator(device="cuda").manual_seed(3))

    def one_pass(y):
        p = policy_loss(y, tokens, old, adv, ref_logprobs=ref, kl_coef=0.1)
        q = distill_loss(y, t, index)
        r = preference_loss(y.view(4, 8, -1), tokens.view(4, 8), None)
        grads = [torch.autograd.grad(v, y)[0] for v in (p.loss, q, r.loss)]
        return [v.detach() for v in (*p, q, *r)] + grads

    static = x.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one_pass(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = one_pass(static)
    for seed in range(4):
        new = (x.float() + normal(x.shape, 0.3, torch.Generator(device="cuda").manual_seed(seed))).to(x.dtype)
        with torch.no_grad():
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(recorded, one_pass(new.requires_grad_())):
            assert torch.equal(p, q), seed


def test_same_bits_every_time(gpu):
    dense = layout_inputs(9001, "bf16")
    first = everything(*dense)
    for _ in range(3):
        for p, q in zip(everything(*dense), first):
            assert torch.equal(p, q)
