"""The objectives of a training step, for timing and for comparing results.

A case is one pass through an operator that turns a language model's logits
into a loss and the gradient that the optimizer works from: log-probabilities
of tokens (``token_logprobs``), a clipped policy loss with a KL term
(``policy_loss``), a preference loss over pairs of sequences
(``preference_loss``) and distillation from a teacher's top logits
(``distill_loss``).

With ``own`` false, ``run`` computes the operator from elementary torch
operations in 32 bits; with ``own`` true it calls the framework's.  ``exact``
is the definition in 64 bits, its gradients by automatic differentiation.

Logits are N(0, 2) with a few raised entries in each row, as a trained model's
are: the token that follows in nine rows of ten, with most of the probability,
and in a distillation the entries the teacher ranks first.  Sequences have a prompt that is not trained
on and end before the padding does; which tokens count depends on the case
alone, so that a case's work does not depend on the seed.
"""

import math
import random
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT / "triton-muonadamw_amd") not in sys.path:
    sys.path.insert(0, str(ROOT / "triton-muonadamw_amd"))

own = False

IGNORE = -100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # The log-probability of one sampled token over the GPT-2 vocabulary (an odd size): latency alone.
        {"name": "logprobs_one_token", "op": "logprobs", "dtype": "bf16", "seqs": 1, "length": 1, "vocab": 50257,
         "packed": False, "entropy": False, "grad": False, "temperature": 1.0},
        # A batch scored by a frozen model (the old policy, the reference): forward only, entropies for the log.
        {"name": "logprobs_gpt2", "op": "logprobs", "dtype": "bf16", "seqs": 8, "length": 1024, "vocab": 50257,
         "packed": False, "entropy": True, "grad": False, "temperature": 1.0},
        # Log-probabilities and entropies in a loss of the user's own: both directions, half precision, odd sizes.
        {"name": "logprobs_grad_odd", "op": "logprobs", "dtype": "fp16", "seqs": 3, "length": 333, "vocab": 32003,
         "packed": False, "entropy": True, "grad": True, "temperature": 0.7},
        # A few tokens of a toy model, averaged by sequence: launches and the host's part.
        {"name": "policy_small", "op": "policy", "dtype": "fp32", "seqs": 4, "length": 16, "vocab": 1003,
         "packed": False, "kl": True, "by": "sequence", "advantages": "sequence", "temperature": 1.0},
        # A step of reinforcement learning on the GPT-2 set, whose parameters and logits are fp32.
        {"name": "policy_gpt2", "op": "policy", "dtype": "fp32", "seqs": 4, "length": 1024, "vocab": 50257,
         "packed": False, "kl": True, "by": "token", "advantages": "token", "temperature": 1.0},
        # The same for the Llama-8B set in bf16, as it is trained: the largest pass, one advantage a sequence.
        {"name": "policy_llama", "op": "policy", "dtype": "bf16", "seqs": 8, "length": 1024, "vocab": 128256,
         "packed": False, "kl": True, "by": "token", "advantages": "sequence", "temperature": 0.9},
        # Two pairs of short sequences packed end to end.
        {"name": "preference_small", "op": "preference", "dtype": "fp32", "seqs": 4, "length": 15, "vocab": 517,
         "packed": True, "kind": "sigmoid", "smoothing": 0.0, "mean": False},
        # Eight pairs of ragged sequences, packed: no padding is computed on.
        {"name": "preference_gpt2", "op": "preference", "dtype": "bf16", "seqs": 16, "length": 375, "vocab": 50257,
         "packed": True, "kind": "sigmoid", "smoothing": 0.1, "mean": False},
        # Four padded pairs over the largest vocabulary, log-probabilities averaged over each answer.
        {"name": "preference_llama", "op": "preference", "dtype": "bf16", "seqs": 8, "length": 512, "vocab": 128256,
         "packed": False, "kind": "ipo", "smoothing": 0.0, "mean": True},
        # A toy student and eight teacher logits a token, half precision.
        {"name": "distill_small", "op": "distill", "dtype": "fp16", "seqs": 1, "length": 16, "vocab": 1003,
         "packed": False, "k": 8, "tail": False, "temperature": 2.0},
        # A GPT-2 student in fp32 and the teacher's 64 first logits, taken as the whole of its distribution.
        {"name": "distill_gpt2", "op": "distill", "dtype": "fp32", "seqs": 2, "length": 1024, "vocab": 50257,
         "packed": False, "k": 64, "tail": False, "temperature": 2.0},
        # The Llama-8B vocabulary in bf16, 128 teacher logits with the mass of all others known.
        {"name": "distill_llama", "op": "distill", "dtype": "bf16", "seqs": 4, "length": 1024, "vocab": 128256,
         "packed": False, "k": 128, "tail": True, "temperature": 1.0},
    ]


def draw(rng):
    def size(lo, hi):
        """Log-uniform in [lo, hi]; a third of the draws rounded to a multiple of 64 where that fits."""
        x = min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
        return x // 64 * 64 if x // 64 * 64 >= lo and rng.random() < 0.34 else x

    op = rng.choice(["logprobs", "policy", "preference", "distill"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    vocab = size(300, 128256)
    tokens = min(size(4, 8192), int(6144 * 128256 * 2 / (vocab * (4 if dtype == "fp32" else 2))))
    seqs = max(1, min(tokens, size(1, 32)))
    case = {"op": op, "dtype": dtype, "vocab": vocab, "packed": rng.random() < 0.4}
    if op == "preference":
        seqs = max(2, seqs // 2 * 2)
        case.update(kind=rng.choice(["sigmoid", "sigmoid", "ipo", "hinge"]), smoothing=0.0, mean=rng.random() < 0.3)
        if case["kind"] == "sigmoid" and rng.random() < 0.5:
            case["smoothing"] = 0.1
    elif op == "policy":
        case.update(kl=rng.random() < 0.7, by=rng.choice(["token", "sequence"]),
                    advantages=rng.choice(["token", "sequence"]), temperature=rng.choice([1.0, 0.9, 1.3]))
    elif op == "distill":
        case.update(k=size(1, min(256, vocab // 4)), tail=rng.random() < 0.5, temperature=rng.choice([1.0, 2.0, 4.0]))
    else:
        case.update(entropy=rng.random() < 0.5, grad=rng.random() < 0.6, temperature=rng.choice([1.0, 0.7]))
    case.update(seqs=seqs, length=max(1, tokens // seqs))
    return case


# ---------------------------------------------------------------------------
# Which tokens there are, and which of them count.

def _spans(case):
    """[(start, first that counts, end of those that count, end)] of each sequence, as places in the rows of logits.
    Padded sequences all have `length` rows and stop before the last; packed ones have lengths of their own that fill
    all rows."""
    seqs, length = case["seqs"], case["length"]
    rng = random.Random(seqs * 1000003 + length * 101 + case["vocab"])
    if case["packed"]:
        cuts = sorted(rng.sample(range(1, seqs * length), seqs - 1))
        bounds = list(zip([0] + cuts, cuts + [seqs * length]))
    else:
        bounds = [(i * length, (i + 1) * length) for i in range(seqs)]
    spans = []
    for start, end in bounds:
        n = end - start
        first = start + rng.randint(0, n // 3)
        last = end if case["packed"] else rng.randint(max(first + 1, start + n // 2 + 1), end)
        spans.append((start, first, last, end))
    return spans


def _normal(shape, std, gen):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen)


def _logsumexp(x):
    m = x.amax(-1, keepdim=True)
    return (m + (x - m).exp().sum(-1, keepdim=True).log()).squeeze(-1)


def _by_sequence(x, sequence, seqs):
    """The sums of `x` over each sequence, in the same order every time."""
    return torch.where(sequence == torch.arange(seqs, device="cuda")[:, None], x, 0.0).sum(1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    seqs, length, vocab, op = case["seqs"], case["length"], case["vocab"], case["op"]
    rows = seqs * length
    spans = _spans(case)
    counts = torch.zeros(rows, dtype=torch.bool)
    sequence = torch.zeros(rows, dtype=torch.int64)
    for i, (start, first, last, end) in enumerate(spans):
        counts[first:last] = True
        sequence[start:end] = i
    counts, sequence = counts.cuda(), sequence.cuda()

    logits = _normal((rows, vocab), 2.0, gen)
    follows = torch.randint(vocab, (rows, 1), device="cuda", generator=gen)
    # against all the others together, which at a temperature t have log(vocab) + 2 / t^2: from -1 to 2 above
    t = case.get("temperature", 1.0)
    raised = t * (math.log(vocab) + 2.0 / t**2 - 1.0 + 3.0 * torch.rand((rows, 1), device="cuda", generator=gen))
    other = torch.randint(vocab, (rows, 1), device="cuda", generator=gen)
    tokens = torch.where(torch.rand((rows, 1), device="cuda", generator=gen) < 0.9, follows, other).squeeze(1)
    state = {"case": dict(case)}
    if op == "distill":
        # One entry from each of k equal parts of the vocabulary, the teacher's logits falling from the first on.
        k, part = case["k"], vocab // case["k"]
        index = torch.arange(k, device="cuda") * part + torch.randint(part, (rows, k), device="cuda", generator=gen)
        top = math.log(vocab) + 3.0 - 9.0 * torch.rand((rows, k), device="cuda", generator=gen).sort(-1).values
        logits.scatter_(1, index, top + _normal((rows, k), 1.0, gen))
        state["top"], state["index"] = top.to(DTYPES[case["dtype"]]), index
        if case["tail"]:  # all others hold between 1% and 30% of the teacher's mass
            rest = 0.01 + 0.29 * torch.rand(rows, device="cuda", generator=gen)
            state["lse"] = _logsumexp(state["top"].float() / case["temperature"]) - (1.0 - rest).log()
    else:
        logits.scatter_(1, follows, raised)
    logits = logits.to(DTYPES[case["dtype"]])

    def logprob(part):
        x = logits[part].float() / t
        return x.gather(1, tokens[part, None]).squeeze(1) - _logsumexp(x)

    near = torch.zeros(rows, device="cuda")  # the log-probabilities, for what an earlier model said of the same tokens
    if op in ("policy", "preference"):
        for part in torch.arange(rows, device="cuda").split(max(1, (1 << 28) // vocab)):
            near[part] = logprob(part)
    if op == "policy":
        state["old"] = near + _normal(rows, 0.15, gen)
        state["ref"] = near + _normal(rows, 0.3, gen) if case["kl"] else None
        if case["advantages"] == "sequence":
            state["advantage"] = (0.5 + _normal(seqs, 1.0, gen))[sequence]
            if not case["packed"]:
                state["advantage"] = state["advantage"].view(seqs, length)[:, :1]
        else:
            state["advantage"] = 0.5 + _normal(rows, 1.0, gen)
    if op == "preference":
        total = _by_sequence(near.double() * counts, sequence, seqs)
        if case["mean"]:
            total = total / _by_sequence(counts.double(), sequence, seqs).clamp(min=1)
        state["ref"] = total.float() + _normal(seqs, 0.05 if case["mean"] else 10.0, gen)
    if op == "logprobs" and case["grad"]:
        state["dlogprobs"] = _normal(rows, 1.0, gen)
        state["dentropy"] = _normal(rows, 0.1, gen)
    if op != "distill":
        state["tokens"] = torch.where(counts, tokens, IGNORE)
    state["counts"], state["sequence"] = counts, sequence
    state["offsets"] = torch.tensor([s[0] for s in spans] + [rows], device="cuda")
    if not case["packed"]:
        for name, x in list(state.items()):
            if isinstance(x, torch.Tensor) and x.shape[:1] == (rows,) and name not in ("sequence", "offsets"):
                state[name] = x.view(seqs, length, *x.shape[1:])
        logits = logits.view(seqs, length, vocab)
    state["logits"] = logits.requires_grad_(op != "logprobs" or case["grad"])
    return state


BETA = 0.1
KL = 0.05
CLIP = (0.2, 0.28)


# ---------------------------------------------------------------------------
# The framework's operators.

def _own(state):
    from triton_muon_adamw import distill_loss, policy_loss, preference_loss, token_logprobs

    case, logits = state["case"], state["logits"]
    logits.grad = None
    offsets = state["offsets"] if case["packed"] else None
    if case["op"] == "logprobs":
        out = token_logprobs(logits, state["tokens"], temperature=case["temperature"], entropy=case["entropy"])
        out = {"logprobs": out[0], "entropy": out[1]} if case["entropy"] else {"logprobs": out}
        if case["grad"]:
            torch.autograd.backward(list(out.values()),
                                    [state["dlogprobs"], state["dentropy"]][:len(out)])
    elif case["op"] == "policy":
        out = policy_loss(logits, state["tokens"], state["old"], state["advantage"], ref_logprobs=state["ref"],
                          kl_coef=KL if case["kl"] else 0.0, clip=CLIP, average=case["by"], offsets=offsets,
                          temperature=case["temperature"])
        out.loss.backward()
        out = {"loss": out.loss, "logprobs": out.logprobs, "kl": out.kl, "clipped": out.clipped}
    elif case["op"] == "preference":
        out = preference_loss(logits, state["tokens"], state["ref"], beta=BETA, kind=case["kind"],
                              label_smoothing=case["smoothing"], length_average=case["mean"], offsets=offsets)
        out.loss.backward()
        out = {"loss": out.loss, "logprobs": out.logprobs, "rewards": out.rewards}
    else:
        loss = distill_loss(logits, state["top"], state["index"], teacher_lse=state.get("lse"), mask=state["counts"],
                            temperature=case["temperature"])
        loss.backward()
        out = {"loss": loss}
    if logits.grad is not None:
        out["grad"] = logits.grad
    return out


# ---------------------------------------------------------------------------
# Their plain form: rows of logits in 32 bits, gradients by their formulas.

def _log_softmax(logits, temperature):
    x = logits.detach().float().flatten(0, -2) / temperature
    x = x - x.amax(-1, keepdim=True)
    return x - x.exp().sum(-1, keepdim=True).log()


def _grad(logits, probs, coef, index, at):
    """at * [entry is index] - coef * probs, a row each, rounded to the logits' type."""
    g = probs * -coef[:, None]
    g.scatter_add_(1, index, at)
    return g.to(logits.dtype).view(logits.shape)


def _plain(state):
    case, logits = state["case"], state["logits"]
    shape, counts = logits.shape[:-1], state["counts"].flatten()
    zero = torch.zeros((), device="cuda")
    temperature = case.get("temperature", 1.0)
    logq = _log_softmax(logits, temperature)
    if case["op"] == "distill":
        p = state["top"].float().flatten(0, -2) / temperature
        index = state["index"].flatten(0, -2)
        at = logq.gather(1, index)
        if case["tail"]:
            logp = p - state["lse"].flatten()[:, None]
        else:
            logp = p - p.amax(-1, keepdim=True)
            logp = logp - logp.exp().sum(-1, keepdim=True).log()
        p = logp.exp()
        q = logq.exp()
        row = (p * (logp - at)).sum(-1)
        weight = counts / counts.sum().clamp(min=1) * temperature
        share = torch.ones_like(row)
        if case["tail"]:
            rest_p = (1.0 - p.sum(-1)).clamp(min=2.0**-20)
            rest_q = q.scatter(1, index, 0.0).sum(-1)
            row = row + rest_p * (rest_p / rest_q).log()
            share = 1.0 - rest_p / rest_q
        g = q * (weight * share)[:, None]
        g.scatter_(1, index, (at.exp() - p) * weight[:, None])
        loss = (torch.where(counts, row, zero) * weight).sum() * temperature
        return {"loss": loss, "grad": g.to(logits.dtype).view(logits.shape)}

    tokens = state["tokens"].flatten().clamp(min=0)[:, None]
    logprob = torch.where(counts, logq.gather(1, tokens).squeeze(1), zero)
    if case["op"] == "logprobs":
        out = {"logprobs": logprob.view(shape)}
        if case["entropy"] or case["grad"]:
            q = logq.exp()
        if case["entropy"]:
            entropy = torch.where(counts, -(q * logq).sum(-1), zero)
            out["entropy"] = entropy.view(shape)
        if case["grad"]:
            at = torch.where(counts, state["dlogprobs"].flatten(), zero) / temperature
            if case["entropy"]:
                h = torch.where(counts, state["dentropy"].flatten(), zero) / temperature
                g = q * -(at[:, None] + h[:, None] * (logq + entropy[:, None]))
                g.scatter_add_(1, tokens, at[:, None])
                out["grad"] = g.to(logits.dtype).view(logits.shape)
            else:
                out["grad"] = _grad(logits, q, at, tokens, at[:, None])
        return out

    sequence, seqs = state["sequence"], case["seqs"]
    n = _by_sequence(counts.float(), sequence, seqs)
    if case["op"] == "policy":
        if case["by"] == "sequence":
            weight = counts / (n.clamp(min=1) * (n > 0).sum().clamp(min=1))[sequence]
        else:
            weight = counts / n.sum().clamp(min=1)
        advantage = state["advantage"].expand(shape).flatten()
        ratio = (logprob - state["old"].flatten()).exp()
        bound = ratio.clamp(1.0 - CLIP[0], 1.0 + CLIP[1])
        clipped = bound * advantage < ratio * advantage
        row = -torch.where(clipped, bound, ratio) * advantage
        slope = torch.where(clipped, zero, -advantage * ratio)
        kl = torch.zeros_like(row)
        if case["kl"]:
            d = state["ref"].flatten() - logprob
            kl = d.exp() - d - 1.0
            row = row + KL * kl
            slope = slope + KL * (1.0 - d.exp())
        coef = slope * weight / temperature
        return {"loss": (row * weight).sum(), "logprobs": logprob.view(shape), "kl": (kl * weight).sum(),
                "clipped": (clipped * weight).sum(), "grad": _grad(logits, logq.exp(), coef, tokens, coef[:, None])}

    total = _by_sequence(logprob, sequence, seqs)
    if case["mean"]:
        total = total / n.clamp(min=1)
    pairs = seqs // 2
    rewards = BETA * (total - state["ref"])
    h = rewards[:pairs] - rewards[pairs:]
    if case["kind"] == "sigmoid":
        s = case["smoothing"]
        softplus = torch.log1p((-h.abs()).exp())
        row = (1.0 - s) * (softplus + (-h).clamp(min=0.0)) + s * (softplus + h.clamp(min=0.0))
        slope = s - 1.0 / (1.0 + h.exp())
    elif case["kind"] == "ipo":
        row = (h / BETA - 0.5 / BETA).square()
        slope = 2.0 * (h / BETA - 0.5 / BETA) / BETA
    else:
        row = (1.0 - h).clamp(min=0.0)
        slope = -(h < 1.0).float()
    slope = torch.cat([slope, -slope]) * (BETA / pairs)
    if case["mean"]:
        slope = slope / n.clamp(min=1)
    coef = slope[sequence] * counts
    return {"loss": row.mean(), "logprobs": total, "rewards": rewards,
            "grad": _grad(logits, logq.exp(), coef, tokens, coef[:, None])}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------------

def work(case):
    rows = case["seqs"] * case["length"]
    active = sum(last - first for _, first, last, _ in _spans(case))
    size = 4 if case["dtype"] == "fp32" else 2
    grad = case["op"] != "logprobs" or case["grad"]
    # Rows that do not count need no reading; the gradient is written whole.
    nbytes = active * case["vocab"] * size + (rows * case["vocab"] * size if grad else 0) + rows * 8
    # Scale, subtract, exponential and sum of each entry; another exponential, product and sum for its gradient.
    flops = active * case["vocab"] * (9.0 if grad else 5.0)
    if case["op"] == "policy":
        nbytes += rows * (12 + (4 if case["advantages"] == "token" else 0) + (4 if case["kl"] else 0))
    elif case["op"] == "distill":
        nbytes += rows * (case["k"] * (8 + size) + (4 if case["tail"] else 0) - 7)
        flops += active * case["k"] * 10.0
    elif case["op"] == "logprobs":
        nbytes += rows * 4 * (1 + case["entropy"]) * (1 + case["grad"])
        flops += active * case["vocab"] * (2.0 + 3.0 * case["grad"]) * case["entropy"]
    else:
        nbytes += case["seqs"] * 12
    return {"bytes": float(nbytes), "flops": float(flops)}


# ---------------------------------------------------------------------------
# 64 bits, from the definitions; gradients by automatic differentiation.

def exact(case, seed):
    state = prepare(case, seed)
    x = state["logits"].detach().double().requires_grad_()
    z = x / case.get("temperature", 1.0)
    logq = torch.log_softmax(z, -1)
    counts = state["counts"]
    if case["op"] == "distill":
        t = state["top"].double() / case["temperature"]
        logp = t - state["lse"].double()[..., None] if case["tail"] else torch.log_softmax(t, -1)
        divergence = torch.nn.functional.kl_div(logq.gather(-1, state["index"]), logp, reduction="none",
                                                log_target=True).sum(-1)
        if case["tail"]:
            rest = (-torch.expm1(torch.logsumexp(logp, -1))).clamp(min=2.0**-20)
            outside = torch.logsumexp(z.scatter(-1, state["index"], -math.inf), -1) - torch.logsumexp(z, -1)
            divergence = divergence + rest * (rest.log() - outside)
        loss = case["temperature"] ** 2 * divergence[counts].mean()
        return {"loss": loss, "grad": torch.autograd.grad(loss, x)[0]}

    logprobs = torch.zeros(counts.shape, dtype=torch.float64, device="cuda")
    chosen = -torch.nn.functional.nll_loss(logq[counts], state["tokens"][counts], reduction="none")
    logprobs = logprobs.masked_scatter(counts, chosen)
    if case["op"] == "logprobs":
        out, ups = {"logprobs": logprobs}, [state["dlogprobs"].double()] if case["grad"] else []
        if case["entropy"]:
            out["entropy"] = torch.special.entr(logq.exp()).sum(-1) * counts
            ups += [state["dentropy"].double()] if case["grad"] else []
        if case["grad"]:
            g = torch.autograd.grad(list(out.values()), x, ups)[0]
            out["grad"] = g
        return out

    seq = state["sequence"].view(counts.shape)
    member = torch.nn.functional.one_hot(seq[counts], case["seqs"]).double()  # tokens x sequences
    lengths = member.sum(0)
    if case["op"] == "policy":
        advantage = state["advantage"].double().expand(counts.shape)[counts]
        log_ratio = chosen - state["old"].double()[counts]
        surrogate = torch.minimum(log_ratio.exp() * advantage,
                                  log_ratio.exp().clamp(1.0 - CLIP[0], 1.0 + CLIP[1]) * advantage)
        over = torch.where(advantage > 0, log_ratio > math.log1p(CLIP[1]),
                           (advantage < 0) & (log_ratio < math.log1p(-CLIP[0])))
        kl = torch.zeros_like(chosen)
        if case["kl"]:
            gap = state["ref"].double()[counts] - chosen
            kl = torch.expm1(gap) - gap

        def mean(v):
            if case["by"] == "token":
                return v.mean()
            return ((v[:, None] * member).sum(0) / lengths)[lengths > 0].mean()

        loss = mean(KL * kl - surrogate)
        return {"loss": loss, "logprobs": logprobs, "kl": mean(kl), "clipped": mean(over.double()),
                "grad": torch.autograd.grad(loss, x)[0]}

    total = (chosen[:, None] * member).sum(0)
    if case["mean"]:
        total = total / lengths.clamp(min=1)
    rewards = BETA * (total - state["ref"].double())
    good, bad = rewards.chunk(2)
    if case["kind"] == "sigmoid":
        loss = torch.nn.functional.binary_cross_entropy_with_logits(
            good - bad, torch.full_like(good, 1.0 - case["smoothing"]))
    elif case["kind"] == "ipo":
        loss = ((good - bad) / BETA - 1.0 / (2.0 * BETA)).pow(2).mean()
    else:
        loss = torch.relu(1.0 - (good - bad)).mean()
    return {"loss": loss, "logprobs": total, "rewards": rewards, "grad": torch.autograd.grad(loss, x)[0]}
