"""The objectives of a training step in float64: losses over rows of logits and
their gradients by the formulas, plainly and row by row.

No counterpart in the reference, which starts at gradients.  Pinned by
``tests/test_oracle_objectives.py`` against automatic differentiation and
against differences of the losses.  Logits are ``(rows, vocab)`` arrays;
``sequences`` is a list of ``(start, end)`` rows.
"""

from __future__ import annotations

import numpy as np

SMALLEST_TAIL = 2.0**-20


def log_softmax(z):
    z = z - z.max()
    return z - np.log(np.exp(z).sum())


def token_logprobs(logits, tokens, temperature=1.0, ignore_index=-100, dlogprobs=None, dentropy=None):
    """(logprobs, entropies, gradient of sum(dlogprobs * logprobs + dentropy * entropies))."""
    n, _ = logits.shape
    lp, ent, grad = np.zeros(n), np.zeros(n), np.zeros(logits.shape)
    for r in range(n):
        if tokens[r] == ignore_index:
            continue
        logq = log_softmax(logits[r].astype(np.float64) / temperature)
        q = np.exp(logq)
        lp[r] = logq[tokens[r]]
        safe = np.where(q > 0, logq, 0.0)
        ent[r] = -(q * safe).sum()
        a = 0.0 if dlogprobs is None else dlogprobs[r]
        h = 0.0 if dentropy is None else dentropy[r]
        grad[r] = -q * (a + h * (safe + ent[r]))
        grad[r, tokens[r]] += a
        grad[r] /= temperature
    return lp, ent, grad


def policy_loss(logits, tokens, old, advantages, ref=None, kl_coef=0.0, clip=(0.2, 0.2), sequences=None,
                temperature=1.0, ignore_index=-100, scale=1.0):
    """(loss, logprobs, kl, clipped, gradient); the mean over ``sequences`` where they are given."""
    n = logits.shape[0]
    active = np.array([t != ignore_index for t in tokens])
    weight = np.zeros(n)
    if sequences is None:
        weight[active] = 1.0 / max(1, active.sum())
    else:
        lengths = [int(active[a:b].sum()) for a, b in sequences]
        some = max(1, sum(k > 0 for k in lengths))
        for (a, b), k in zip(sequences, lengths):
            weight[a:b] = active[a:b] / (max(1, k) * some)
    active &= weight > 0
    lp = np.zeros(n)
    loss = kl = clipped = 0.0
    grad = np.zeros(logits.shape)
    for r in np.flatnonzero(active):
        logq = log_softmax(logits[r].astype(np.float64) / temperature)
        lp[r] = logq[tokens[r]]
        ratio, adv = np.exp(lp[r] - old[r]), advantages[r]
        bound = min(max(ratio, 1.0 - clip[0]), 1.0 + clip[1])
        is_clipped = bound * adv < ratio * adv
        row = -min(ratio * adv, bound * adv)
        slope = 0.0 if is_clipped else -adv * ratio
        if ref is not None:
            d = ref[r] - lp[r]
            k = np.expm1(d) - d
            row += kl_coef * k
            slope -= kl_coef * np.expm1(d)
            kl += weight[r] * k
        loss += scale * weight[r] * row
        clipped += weight[r] * is_clipped
        grad[r] = -np.exp(logq)
        grad[r, tokens[r]] += 1.0
        grad[r] *= scale * weight[r] * slope / temperature
    return loss, lp, kl, clipped, grad


def preference_loss(logits, tokens, ref, sequences, beta=0.1, kind="sigmoid", label_smoothing=0.0,
                    length_average=False, temperature=1.0, ignore_index=-100):
    """(loss, logprobs of the sequences, rewards, gradient)."""
    row_lp, _, _ = token_logprobs(logits, tokens, temperature, ignore_index)
    active = np.array([t != ignore_index for t in tokens])
    count = [max(1, int(active[a:b].sum())) if length_average else 1 for a, b in sequences]
    lp = np.array([row_lp[a:b].sum() / c for (a, b), c in zip(sequences, count)])
    rewards = beta * (lp - (0.0 if ref is None else ref))
    pairs = len(sequences) // 2
    loss, coef = 0.0, np.zeros(len(tokens))
    for i in range(pairs):
        h = rewards[i] - rewards[i + pairs]
        if kind == "sigmoid":
            e = label_smoothing
            loss += (1 - e) * np.logaddexp(0.0, -h) + e * np.logaddexp(0.0, h)
            slope = e - np.exp(-np.logaddexp(0.0, h))
        elif kind == "ipo":
            loss += (h / beta - 0.5 / beta) ** 2
            slope = 2.0 * (h / beta - 0.5 / beta) / beta
        else:
            loss += max(0.0, 1.0 - h)
            slope = -1.0 if h < 1.0 else 0.0
        for s, sign in ((i, 1.0), (i + pairs, -1.0)):
            a, b = sequences[s]
            coef[a:b] = sign * slope * beta / (pairs * count[s])
    _, _, grad = token_logprobs(logits, tokens, temperature, ignore_index, dlogprobs=coef)
    return loss / pairs, lp, rewards, grad


def distill_loss(logits, teacher_logits, teacher_indices, teacher_lse=None, mask=None, temperature=1.0, scale=1.0):
    """(loss, gradient)."""
    n, vocab = logits.shape
    active = np.ones(n, bool) if mask is None else np.asarray(mask, bool)
    loss, grad = 0.0, np.zeros(logits.shape)
    weight = scale * temperature**2 / max(1, active.sum())
    for r in np.flatnonzero(active):
        logq = log_softmax(logits[r].astype(np.float64) / temperature)
        q = np.exp(logq)
        keep = (teacher_indices[r] >= 0) & (teacher_logits[r] != -np.inf)
        index, t = teacher_indices[r][keep], teacher_logits[r][keep].astype(np.float64) / temperature
        if teacher_lse is not None:
            logp = t - np.float64(teacher_lse[r])
        else:
            logp = log_softmax(t) if len(t) else t
        p = np.exp(logp)
        loss += weight * (p * (logp - logq[index])).sum()
        target = np.zeros(vocab)
        np.add.at(target, index, p)
        inside = np.zeros(vocab, bool)
        inside[index] = True
        if teacher_lse is None:
            g = q * (1.0 if len(t) else 0.0) - target
        else:
            # of sum p (log p - log q): (sum p) q - p; of P (log P - log Q): P (q - the others' own softmax)
            total = p.sum()
            g = -target
            if not inside.all():
                rest_p, log_rest = max(1.0 - total, SMALLEST_TAIL), np.logaddexp.reduce(logq[~inside])
                loss += weight * rest_p * (np.log(rest_p) - log_rest)
                g[~inside] -= rest_p * np.exp(logq[~inside] - log_rest)
                total += rest_p
            g += total * q
        grad[r] = weight * g / temperature
    return loss, grad
