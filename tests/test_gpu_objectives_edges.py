"""The objectives' kernels where values leave the ordinary range: rows far from 0 with hidden entries, large and small
quotients of logits and temperature, shares that underflow, entries and rows that are left out; and backward passes
whose inputs were kept by someone else.

Tolerances are those of test_gpu_objectives (u = 2^-24, d the error of a log-probability); what is derived here stands
at its test."""

import math

import numpy as np
import pytest
import torch
from test_gpu_objectives import (
    DTYPES,
    U,
    check_distill,
    check_grad,
    check_policy,
    f64,
    lp_tol,
    make,
    normal,
    policy_case,
    q_or_one,
)

from oracle import objectives as ob
from triton_muon_adamw import distill_loss, policy_loss, preference_loss, token_logprobs

pytestmark = pytest.mark.gpu


# ---- rows whose largest logit is far below 0

def hidden_rows(vocab, dtype, level, temperature, seed):
    """Six rows of logits around `level` T, from half to all but one of their entries at -inf."""
    x, tokens, gen = make(6, vocab, "fp32", seed, ignored=0.0)
    share = torch.tensor([0.5, 0.75, 0.9, 0.97, 0.99, 1.0], device="cuda")[:, None]
    hidden = torch.rand((6, vocab), device="cuda", generator=gen) < share
    hidden[torch.arange(6), tokens] = False
    x = ((x + level) * temperature).to(DTYPES[dtype]).masked_fill(hidden, -math.inf)
    return x, tokens, hidden, gen


LEVELS = [(-100.0, 1.0), (-1000.0, 1.0), (-100.0, 0.125), (1000.0, 1.0)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [9, 1003, 2048, 4099, 8192, 16390, 32003, 50257, 65536, 131077])
@pytest.mark.parametrize("level,temperature", LEVELS)
def test_policy_of_hidden_entries_at_any_level(gpu, dtype, vocab, level, temperature):
    x, tokens, hidden, gen = hidden_rows(vocab, dtype, level, temperature, 81)
    lp = ob.token_logprobs(f64(x), tokens.cpu().numpy(), temperature)[0]
    old = torch.tensor(lp, device="cuda").float() + normal(6, 0.3, gen)
    adv = normal(6, 1.0, gen)
    adv[1] = 0.0
    x.requires_grad_()
    out = policy_loss(x, tokens, old, adv, temperature=temperature)
    out.loss.backward()
    assert x.grad.isfinite().all() and not x.grad[hidden].any() and not x.grad[1].any()
    check_policy(x, tokens, old, adv, None, out, x.grad, temperature=temperature)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [1003, 2048, 4099, 8192, 16390, 32003, 50257, 65536, 131077])
@pytest.mark.parametrize("level,temperature", LEVELS)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_of_hidden_entries_at_any_level(gpu, dtype, vocab, level, temperature, tail):
    x, _, hidden, gen = hidden_rows(vocab, dtype, level, temperature, 83)
    keep = (~hidden).sum(-1) > 5  # some are left beside the entries
    x, hidden = x[keep].contiguous(), hidden[keep]
    index = x.float().topk(5, -1).indices
    t = normal(index.shape, 1.0, gen) * temperature
    lse = torch.logsumexp(t / temperature, -1) + 0.3 if tail else None
    x.requires_grad_()
    loss = distill_loss(x, t, index, teacher_lse=lse, temperature=temperature)
    loss.backward()
    assert x.grad.isfinite().all() and not x.grad[hidden].any()
    check_distill(x, t, index, lse, None, temperature, loss, x.grad)


# ---- logits that are large beside the temperature

@pytest.mark.parametrize("vocab", [33, 1003, 50257])
@pytest.mark.parametrize("level,temperature", [(1e4, 1.0), (1e5, 1.0), (-1e6, 1.0), (1e7, 1.0), (-1e8, 1.0), (1e6, 0.5),
                                               (0.0, 2.0**-10), (0.0, 2.0**-14), (0.0, 2.0**-20)])
def test_logits_large_beside_the_temperature(gpu, vocab, level, temperature):
    """A logit's difference to the largest one is exact here, so the tolerances are those of any row."""
    x, tokens, gen = make(8, vocab, "fp32", 85)
    x = x + level
    g, h = normal(8, 1.0, gen), normal(8, 0.5, gen)
    x.requires_grad_()
    lp, ent = token_logprobs(x, tokens, temperature=temperature, entropy=True)
    torch.autograd.backward([lp, ent], [g, h])
    x64, t = f64(x), tokens.cpu().numpy()
    elp, eent, egrad = ob.token_logprobs(x64, t, temperature, dlogprobs=f64(g), dentropy=f64(h))
    tol = lp_tol(vocab, elp)
    assert (np.abs(f64(lp) - elp) <= tol).all()
    tol_ent = 4 * lp_tol(vocab, eent) * (1 + eent)
    assert (np.abs(f64(ent) - eent) <= tol_ent).all()
    a, b = np.abs(f64(g)), np.abs(f64(h))
    weight = np.sqrt(q_or_one(x64, t, temperature)) / temperature
    check_grad(x.grad, egrad, (4 * (a + b * (2 + eent)) * lp_tol(vocab, eent) + b * tol_ent)[:, None] * weight)
    with torch.no_grad():
        out = preference_loss(x.view(2, 4, -1), tokens.view(2, 4), None, temperature=temperature)
    sums = elp.reshape(2, 4).sum(-1)
    assert (np.abs(f64(out.logprobs) - sums) <= tol.reshape(2, 4).sum(-1) + 4 * U * np.abs(sums)).all()


# ---- distillation: what the teacher and the student leave to the other entries

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab,k", [(7, 7), (7, 3), (1003, 12), (16390, 12), (50257, 64), (131077, 5)])
@pytest.mark.parametrize("extra", [0.5, 0.015, -0.4])
def test_distill_with_probabilities_that_do_not_add_up(gpu, dtype, vocab, k, extra):
    """A teacher's logits that were rounded after its logsumexp was taken: their probabilities add up to 1 + extra, and
    the gradient is that of the loss as it is."""
    x, _, gen = make(5, vocab, dtype, 87)
    index = torch.rand((5, vocab), device="cuda", generator=gen).argsort(-1)[:, :k].contiguous()
    t = normal((5, k), 1.5, gen).to(DTYPES[dtype])
    lse = (torch.logsumexp(t.double() / 2.0, -1) - math.log1p(extra)).float()
    x.requires_grad_()
    loss = distill_loss(x, t, index, teacher_lse=lse, temperature=2.0)
    loss.backward()
    check_distill(x, t, index, lse, None, 2.0, loss, x.grad)
    if k == vocab:  # no others: as sharp a tolerance without what they add, (S q_j - p_j) off by 4 d sqrt(q_j) S + 4 ep
        _, egrad = ob.distill_loss(f64(x), f64(t), index.cpu().numpy(), f64(lse), None, 2.0)
        size = np.exp(np.stack([ob.log_softmax(row / 2.0) for row in f64(x)]) / 2)
        ep = U * (k + 8 + 6 * np.abs(f64(t)).max() / 2 + 3 * np.abs(f64(lse)).max())
        check_grad(x.grad, egrad, 2.0 / 5 * (4 * lp_tol(vocab, 0.0) * (1 + extra) * size + 4 * ep))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [300, 1003, 16390, 50257, 131077])
@pytest.mark.parametrize("gap,temperature", [(80.0, 1.0), (110.0, 1.0), (900.0, 1.0), (200.0, 0.125), (5000.0, 4.0)])
def test_distill_with_a_rest_far_below(gpu, dtype, vocab, gap, temperature):
    """All other logits lie `gap` T below the teacher's entries: Q underflows, log Q and the others' gradient do not.

    With r the softmax over the others alone, d' the error of log r and of log Q's two logarithms, ep that of a
    probability of the teacher's: P log(P / Q) is off by P (d' + 3 u |log Q|) + ep (|log P / Q| + 1), the gradient of
    the others, w (q_j (S + P) - P r_j), by w sqrt(r_j) (4 d' P + ep)."""
    x, _, gen = make(4, vocab, "fp32", 89)
    index = torch.rand((4, vocab), device="cuda", generator=gen).argsort(-1)[:, :6].contiguous()
    x.scatter_(1, index, gap + normal((4, 6), 1.0, gen))
    x = (x * temperature).to(DTYPES[dtype])
    t = normal((4, 6), 1.5, gen) * temperature
    lse = (torch.logsumexp(t.double() / temperature, -1) + 0.2).float()
    x.requires_grad_()
    loss = distill_loss(x, t, index, teacher_lse=lse, temperature=temperature)
    loss.backward()
    x64, t64, i = f64(x), f64(t) / temperature, index.cpu().numpy()
    eloss, egrad = ob.distill_loss(x64, f64(t), i, f64(lse), None, temperature)
    outside = np.ones(x64.shape, bool)
    np.put_along_axis(outside, i, False, 1)
    logq = np.stack([ob.log_softmax(row / temperature) for row in x64])
    log_rest = np.array([np.logaddexp.reduce(l[o]) for l, o in zip(logq, outside)])
    logr = np.where(outside, logq - log_rest[:, None], -np.inf)
    p = np.exp(t64 - f64(lse)[:, None])
    rest_p = 1.0 - p.sum(-1)
    ep = U * (6 + 8 + 6 * np.abs(t64).max() + 3 * np.abs(f64(lse)).max())
    d = lp_tol(vocab, np.maximum(np.abs(np.take_along_axis(logq, i, 1)).max(-1), 0.0))
    dr = 2 * lp_tol(vocab, 0.0)
    row = (d + ep * (np.abs(np.take_along_axis(logq, i, 1)).max() + np.abs(t64).max() + 1) +
           rest_p * (dr + 3 * U * np.abs(log_rest)) + ep * (np.abs(np.log(rest_p) - log_rest) + 1))
    assert abs(loss.item() - eloss) <= 2 * temperature**2 * row.max()
    w = temperature / 4
    tol = w * (4 * d[:, None] * np.exp(logq / 2) + np.exp(logr / 2) * (4 * dr * rest_p + ep)[:, None])
    np.put_along_axis(tol, i, np.take_along_axis(tol, i, 1) + 4 * w * ep, 1)
    check_grad(x.grad, egrad, tol)


@pytest.mark.parametrize("tail", [False, True])
def test_padding_may_point_anywhere(gpu, tail):
    """An entry with a logit of -inf is left out whatever its index."""
    x, _, gen = make(4, 1003, "fp32", 91)
    index = torch.rand((4, 1003), device="cuda", generator=gen).argsort(-1)[:, :9].contiguous()
    t = normal((4, 9), 1.5, gen)
    t[:, 6:] = -math.inf
    lse = torch.logsumexp(t, -1) + 0.3 if tail else None
    losses, grads = [], []
    for padding in (-1, 0, 1003, 1 << 40):
        index[:, 6:] = padding
        y = x.clone().requires_grad_()
        loss = distill_loss(y, t, index, teacher_lse=lse)
        loss.backward()
        check_distill(y, t, index.clamp(max=1002), lse, None, 1.0, loss, y.grad)
        losses.append(loss.detach())
        grads.append(y.grad)
    assert all(torch.equal(p, losses[0]) for p in losses) and all(torch.equal(g, grads[0]) for g in grads)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [257, 1003, 4099, 16390, 50257, 131077])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_of_entries_at_the_lowest_value(gpu, dtype, vocab, tail):
    """Twelve entries a row are visible, six of them the teacher's; all others are at the type's lowest value, so most
    threads see nothing else."""
    x, _, gen = make(12, vocab, dtype, 93)
    seen = torch.rand((12, vocab), device="cuda", generator=gen).argsort(-1)[:, :12].contiguous()
    hidden = torch.ones((12, vocab), dtype=torch.bool, device="cuda").scatter_(1, seen, False)
    x = x.masked_fill(hidden, torch.finfo(x.dtype).min).requires_grad_()
    index = seen[:, :6].contiguous()
    t = normal((12, 6), 1.5, gen)
    lse = torch.logsumexp(t, -1) + 0.3 if tail else None
    loss = distill_loss(x, t, index, teacher_lse=lse)
    loss.backward()
    check_distill(x, t, index, lse, None, 1.0, loss, x.grad)
    assert not x.grad[hidden].any()


# ---- preference

@pytest.mark.parametrize("smoothing", [0.0, 1.0])
def test_an_impossible_sequence_is_no_contradiction(gpu, smoothing):
    """A token of no probability in the sequence that ought to be unlikely: its reward is -inf, the loss 0."""
    x, tokens, _ = make(4, 77, "fp32", 95, ignored=0.0)
    unlikely = 2 if smoothing == 0.0 else 0
    x[unlikely, tokens[unlikely]] = -math.inf
    x = x.view(2, 2, -1).requires_grad_()
    out = preference_loss(x, tokens.view(2, 2), None, label_smoothing=smoothing)
    grad, = torch.autograd.grad(out.loss, x)
    assert out.loss == 0 and out.rewards[unlikely // 2] == -math.inf
    assert not grad.any()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_outside_the_pairs_do_not_count(gpu, dtype, bad):
    """Rows before the first offset and after the last, whatever they hold."""
    x, tokens, _ = make(12, 1003, dtype, 97, ignored=0.0)
    offsets = torch.tensor([2, 5, 9], device="cuda")
    y = x[2:9].clone().requires_grad_()
    expect = preference_loss(y, tokens[2:9].clone(), None, offsets=offsets - 2)
    expect.loss.backward()
    x[:2] = x[9:] = bad
    x.requires_grad_()
    out = preference_loss(x, tokens, None, offsets=offsets)
    out.loss.backward()
    d = 16 * lp_tol(1003, 40.0)
    for p, q in zip(out, expect):  # to within the place of the rows in memory
        assert (np.abs(f64(p) - f64(q)) <= d * np.maximum(1.0, np.abs(f64(q)))).all()
    assert not x.grad[:2].any() and not x.grad[9:].any()
    check_grad(x.grad[2:9], f64(y.grad), d + 2.0**-8 * np.abs(f64(y.grad)))


# ---- what backward keeps

ROWS, WIDTH, VOCAB = 24, 16, 5003


def losses():
    _, tokens, old, adv, ref = policy_case(ROWS, VOCAB, "bf16", 99)
    gen = torch.Generator(device="cuda").manual_seed(1)
    index = torch.rand((ROWS, VOCAB), device="cuda", generator=gen).argsort(-1)[:, :9].contiguous()
    t = normal((ROWS, 9), 1.0, gen)
    lse = torch.logsumexp(t, -1) + 0.3
    places = torch.tensor([0, 5, 11, 12, ROWS], dtype=torch.int32, device="cuda")
    return {
        "logprobs": lambda x: (lambda o: o[0].sum() + 0.1 * o[1].sum())(token_logprobs(x, tokens, entropy=True)),
        "policy": lambda x: policy_loss(x, tokens, old, adv, ref_logprobs=ref, kl_coef=0.1, average="sequence",
                                        offsets=places).loss,
        "policy rows": lambda x: policy_loss(x.view(4, 6, VOCAB), tokens.view(4, 6), old.view(4, 6), adv[:4, None]).loss,
        "preference": lambda x: preference_loss(x, tokens, None, offsets=places).loss,
        "distill": lambda x: distill_loss(x, t, index, mask=tokens != -100),
        "rest": lambda x: distill_loss(x, t, index, teacher_lse=lse),
    }


@pytest.mark.parametrize("which", ["logprobs", "policy", "policy rows", "preference", "distill", "rest"])
@pytest.mark.parametrize("factor", [1.0, 3.0])
@pytest.mark.parametrize("how", ["checkpoint", "cpu"])
def test_saved_tensors_kept_elsewhere(gpu, which, factor, how):
    """Recomputed by a checkpoint or brought back from host memory, the logits lie elsewhere in the backward pass."""
    from torch.utils.checkpoint import checkpoint

    loss_of = losses()[which]
    gen = torch.Generator(device="cuda").manual_seed(5)
    hidden = normal((ROWS, WIDTH), 1.0, gen)
    head = normal((WIDTH, VOCAB), 0.5, gen).bfloat16().requires_grad_()

    def step(h):
        return loss_of(h.bfloat16() @ head)

    def grads(run):
        h = hidden.clone().requires_grad_()
        loss = run(h)
        junk = [torch.full((1 << 18,), math.nan, device="cuda") for _ in range(8)]  # where freed logits were
        return [loss.detach(), *torch.autograd.grad(loss * factor, [h, head])], junk

    def on_cpu(h):
        with torch.autograd.graph.save_on_cpu():
            return step(h)

    expect, _ = grads(step)
    got, _ = grads((lambda h: checkpoint(step, h, use_reentrant=False)) if how == "checkpoint" else on_cpu)
    for p, q in zip(got, expect):
        assert torch.equal(p, q)


@pytest.mark.parametrize("which", ["logprobs", "policy", "preference", "distill"])
def test_saved_strided_tensors_come_back_dense(gpu, which):
    loss_of = losses()[which]
    gen = torch.Generator(device="cuda").manual_seed(5)
    wide = normal((ROWS, VOCAB + 13), 2.0, gen).bfloat16()
    grads = []
    for hooked in (False, True):
        x = wide.clone().requires_grad_()
        if hooked:
            with torch.autograd.graph.save_on_cpu():
                loss = loss_of(x[:, 3:VOCAB + 3])
        else:
            loss = loss_of(x[:, 3:VOCAB + 3])
        grads.append(torch.autograd.grad(3 * loss, x)[0])
    d = 16 * lp_tol(VOCAB, 40.0)
    assert f64(grads[0]).any()
    check_grad(grads[1], f64(grads[0]), d * np.sqrt(np.abs(f64(grads[0]))) + 2.0**-8 * np.abs(f64(grads[0])))


@pytest.mark.parametrize("which", ["logprobs", "policy", "preference", "distill"])
def test_saved_tensors_kept_elsewhere_are_let_go(gpu, which):
    """Neither the logits nor a gradient of their size stays on the device."""
    loss_of = losses()[which]
    x = normal((ROWS, VOCAB), 2.0, torch.Generator(device="cuda").manual_seed(5)).requires_grad_()
    loss_of(x * 1.0)  # what is allocated once
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        loss = loss_of(x * 1.0)
    assert torch.cuda.memory_allocated() - before < x.numel() * 4 // 2
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    second, = torch.autograd.grad(loss, x)
    assert torch.equal(first, second)


def test_inputs_of_inference_mode(gpu):
    """What an inference-mode pass computed goes with a loss that is trained on, as a constant."""
    x, tokens, old, adv, ref = policy_case(8, 1003, "bf16", 101)
    with torch.inference_mode():
        kept = [v.clone() for v in (tokens, old, adv, ref)]
        mask = kept[0] != -100
        index, top = torch.arange(8, device="cuda")[:, None].clone(), kept[1][:, None].clone()
    index_, top_ = torch.arange(8, device="cuda")[:, None], old[:, None]

    def run(tokens, old, adv, ref, mask, index, top):
        y = x.clone().requires_grad_()
        out = [policy_loss(y, tokens, old, adv, ref_logprobs=ref, kl_coef=0.1).loss, token_logprobs(y, tokens).sum(),
               distill_loss(y, top, index, mask=mask),
               preference_loss(y.view(2, 4, -1), tokens.view(2, 4), ref[:2]).loss]
        return [torch.autograd.grad(3 * v, y)[0] for v in out]

    expect = run(tokens, old, adv, ref, tokens != -100, index_, top_)
    for p, q in zip(run(*kept, mask, index, top), expect):
        assert torch.equal(p, q)
