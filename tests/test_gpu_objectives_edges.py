"""The objectives' kernels where values leave the ordinary range: rows far from 0 with hidden entries, large and small
quotients of logits and temperature, shares that underflow, entries and rows that are left out; and backward passes
whose inputs were kept by someone else.

Tolerances are those of test_gpu_objectives (u = 2^-24, d the error of a log-probability); what is derived here stands
at its test."""

import math

import pytest
import torch
from test_gpu_objectives import (
    DTYPES,
    check_distill,
    check_policy,
    f64,
    make,
    normal,
)

from oracle import objectives as ob
from triton_muon_adamw import distill_loss, policy_loss, token_logprobs

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
