"""Losses over rows of logits: the part of a training step before the optimizer.

The reference starts at gradients; these have no counterpart there.  Logits
are ``(rows, vocab)`` or ``(batch, length, vocab)`` in float32, bfloat16 or
float16, with any strides but a contiguous vocabulary; what goes with them has
one value for each row and may be broadcast.  Between the logits and the
gradient, which has the logits' type, everything is float32.  Work is queued on
the current stream without a host synchronisation, results do not depend on
the order in which anything runs, and a HIP graph can record a pass.

Rows whose token is ``ignore_index`` (or whose mask is false) are not read:
infinities and NaN in them change nothing, and where no row is left the loss is
0.  Values on the device are not looked at by the host, so a token beyond the
vocabulary cannot raise: it reads nothing and gives NaN.
"""

from __future__ import annotations

import ctypes
from typing import Literal, NamedTuple

import torch

from .. import _lib

_FLOATS = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_INTS = {torch.int32: _lib.I32, torch.int64: _lib.I64}
_BOOLS = {torch.bool: _lib.BOOL}
_F32 = {torch.float32: _lib.F32}
_KINDS = {"sigmoid": 0, "ipo": 1, "hinge": 2}


class PolicyLoss(NamedTuple):
    """``loss`` carries the gradient; the rest are values for the log."""

    loss: torch.Tensor
    logprobs: torch.Tensor  # of the tokens, 0 where they do not count
    kl: torch.Tensor        # mean of exp(ref - logprob) - (ref - logprob) - 1, 0 without ref_logprobs
    clipped: torch.Tensor   # share of the tokens that the clamp keeps from contributing


class PreferenceLoss(NamedTuple):
    """``loss`` carries the gradient; the rest are values for the log, one a sequence."""

    loss: torch.Tensor
    logprobs: torch.Tensor  # sums (or means) over each sequence's tokens
    rewards: torch.Tensor   # beta * (logprobs - ref_logprobs)


def _rows(logits: torch.Tensor) -> _lib.Rows:
    _lib.require_gpu_tensor(logits, "logits")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits must be float32, bfloat16 or float16 (got {logits.dtype})")
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits must be (rows, vocab) or (batch, length, vocab) (got {tuple(logits.shape)})")
    vocab = logits.shape[-1]
    if vocab == 0:
        raise ValueError("logits have an empty vocabulary")
    if vocab > 1 and logits.stride(-1) != 1 and logits.numel() > 0:
        raise ValueError("logits must be contiguous along the vocabulary")
    outer, so = (1, 0) if logits.dim() == 2 else (logits.shape[0], logits.stride(0))
    return _lib.Rows(logits.data_ptr(), outer, logits.shape[-2], vocab, so, logits.stride(-2), _FLOATS[logits.dtype], 0)


def _per_row(x: torch.Tensor | None, name: str, logits: torch.Tensor, types: dict, k: int = 0) -> _lib.PerRow:
    """One value (``k`` > 0: ``k`` values) for each row of ``logits``, broadcast to them."""
    if x is None:
        return _lib.PerRow(None, 0, 0, 0, 0)
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor (got {type(x).__name__})")
    if x.dtype not in types:
        raise TypeError(f"{name} must be {' or '.join(str(t).split('.')[1] for t in types)} (got {x.dtype})")
    if x.device != logits.device:
        raise ValueError(f"{name} is on {x.device}, logits on {logits.device}")
    shape = logits.shape[:-1] + ((k,) if k else ())
    if x.shape != shape:
        if k and x.shape[-1:] != (k,):
            raise ValueError(f"{name} must have {k} values for each row (got {tuple(x.shape)})")
        try:
            x = x.expand(shape)
        except RuntimeError:
            raise ValueError(f"{name} of shape {tuple(x.shape)} does not go with rows of shape "
                             f"{tuple(logits.shape[:-1])}") from None
    so = x.stride(0) if logits.dim() == 3 else 0
    return _lib.PerRow(x.data_ptr(), so, x.stride(logits.dim() - 2), types[x.dtype], 0)


def _sequences(offsets: torch.Tensor | None, logits: torch.Tensor, needed: bool) -> tuple[torch.Tensor | None, int]:
    """(offsets for the device, how many sequences there are)."""
    if offsets is None:
        if logits.dim() == 2:
            if needed:
                raise ValueError("logits of shape (rows, vocab) need offsets: where each sequence starts, and the end "
                                 "of the last")
            return None, 1
        return None, logits.shape[0]
    if logits.dim() != 2:
        raise ValueError("offsets go with logits of shape (rows, vocab)")
    if not isinstance(offsets, torch.Tensor) or offsets.dtype not in _INTS:
        raise TypeError("offsets must be an int32 or int64 tensor")
    if offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError(f"offsets must hold a place for each sequence and the end (got shape {tuple(offsets.shape)})")
    if offsets.device != logits.device:
        raise ValueError(f"offsets are on {offsets.device}, logits on {logits.device}")
    return offsets.to(torch.int64).contiguous(), offsets.numel() - 1


def _ptr(x: torch.Tensor | None) -> int | None:
    return None if x is None else x.data_ptr()


def _workspace(fn, logits: torch.Tensor, *args) -> torch.Tensor:
    nbytes = ctypes.c_size_t()
    _lib.check(fn(*args, ctypes.byref(nbytes)), fn.__name__)
    return torch.empty(max(nbytes.value, 256), dtype=torch.uint8, device=logits.device)


def _wants_grad(logits: torch.Tensor) -> bool:
    return logits.requires_grad and torch.is_grad_enabled()


def _grad_like(logits: torch.Tensor) -> torch.Tensor:
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def _scale_of(grad_output: torch.Tensor) -> torch.Tensor:
    return grad_output.to(torch.float32)


# ---------------------------------------------------------------------------

def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100,
                   entropy: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Log-probability of ``tokens`` under ``softmax(logits / temperature)``,
    float32, 0 where the token is ``ignore_index``; with ``entropy`` also the
    distribution's entropy.  Both are differentiable."""
    rows = _rows(logits)
    toks = _per_row(tokens, "tokens", logits, _INTS)
    args = (logits, tokens, rows, toks, float(temperature), int(ignore_index), bool(entropy))
    if _wants_grad(logits):
        out = _TokenLogprobs.apply(*args)
    else:
        out = _token_logprobs(*args)[:2]
    return out if entropy else out[0]


def _token_logprobs(logits, tokens, rows, toks, temperature, ignore_index, entropy, stats=False):
    shape, dev = logits.shape[:-1], logits.device
    logprobs = torch.empty(shape, dtype=torch.float32, device=dev)
    ent = torch.empty(shape, dtype=torch.float32, device=dev) if entropy else None
    st = torch.empty((*shape, 2), dtype=torch.float32, device=dev) if stats else None
    with _lib.device_guard(dev):
        _lib.check(_lib.load().mamw_token_logprobs(
            ctypes.byref(rows), ctypes.byref(toks), ignore_index, temperature, logprobs.data_ptr(), _ptr(ent),
            _ptr(st), _lib.raw_stream(dev)), "token_logprobs")
    return logprobs, ent, st


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, rows, toks, temperature, ignore_index, entropy):
        logprobs, ent, stats = _token_logprobs(logits, tokens, rows, toks, temperature, ignore_index, entropy, True)
        ctx.save_for_backward(logits, tokens, stats, ent)
        ctx.hyper = temperature, ignore_index
        return logprobs, ent

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogprobs, dentropy):
        logits, tokens, stats, ent = ctx.saved_tensors
        temperature, ignore_index = ctx.hyper
        coef = _per_row(dlogprobs, "gradient", logits, _F32)
        with_entropy = ent is not None and dentropy is not None
        grad = _grad_like(logits)
        dev = logits.device
        with _lib.device_guard(dev):
            _lib.check(_lib.load().mamw_logits_grad(
                ctypes.byref(_rows(logits)), ctypes.byref(_per_row(tokens, "tokens", logits, _INTS)), ignore_index,
                temperature, stats.data_ptr(), ctypes.byref(coef),
                ctypes.byref(_per_row(dentropy, "gradient", logits, _F32)) if with_entropy else None,
                _ptr(ent), None, grad.data_ptr(), _lib.raw_stream(dev)), "token_logprobs backward")
        return grad, None, None, None, None, None, None


# ---------------------------------------------------------------------------

class _OnePass(torch.autograd.Function):
    """A loss whose forward kernel writes the gradient as well: a row's gradient
    needs nothing beyond that row.  ``backward`` hands it out; a gradient of the
    loss other than 1 has it computed again from the logits with that factor (the
    device decides, so nothing waits), which rounds once and keeps float16
    gradients of a scaled loss from vanishing first."""

    @staticmethod
    def forward(ctx, logits, call):
        grad = _grad_like(logits)
        out = call.loss(grad)
        ctx.save_for_backward(logits, *call.tensors)
        ctx.call, ctx.grad = call, grad
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output, *_):
        logits = ctx.saved_tensors[0]  # raises where an input was changed in place since
        grad, ctx.grad = ctx.grad, None
        fresh = grad is None  # the graph was retained and the first one is someone else's now
        if fresh:
            grad = _grad_like(logits)
        ctx.call.again(_scale_of(grad_output), not fresh, grad)
        return grad, None


class _PolicyCall:
    def __init__(self, logits, rows, desc, tensors):
        self.rows, self.desc, self.tensors, self.device = rows, desc, tensors, logits.device
        self.shape = logits.shape[:-1]
        lib = _lib.load()
        self.ws = _workspace(lib.mamw_policy_workspace_bytes, logits, ctypes.byref(rows), ctypes.byref(desc))

    def loss(self, grad):
        result = torch.empty(3, dtype=torch.float32, device=self.device)
        logprobs = torch.empty(self.shape, dtype=torch.float32, device=self.device)
        with _lib.device_guard(self.device):
            _lib.check(_lib.load().mamw_policy_loss(
                ctypes.byref(self.rows), ctypes.byref(self.desc), result.data_ptr(), logprobs.data_ptr(), _ptr(grad),
                self.ws.data_ptr(), self.ws.numel(), _lib.raw_stream(self.device)), "policy_loss")
        return result[0], logprobs, result[1], result[2]

    def again(self, scale, unless_one, grad):
        with _lib.device_guard(self.device):
            _lib.check(_lib.load().mamw_policy_grad(
                ctypes.byref(self.rows), ctypes.byref(self.desc), scale.data_ptr(), int(unless_one), grad.data_ptr(),
                self.ws.data_ptr(), self.ws.numel(), _lib.raw_stream(self.device)), "policy_loss backward")


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: torch.Tensor | None = None, kl_coef: float = 0.0,
                clip: tuple[float, float] = (0.2, 0.2), average: Literal["token", "sequence"] = "token",
                offsets: torch.Tensor | None = None, temperature: float = 1.0, ignore_index: int = -100,
                scale: float = 1.0) -> PolicyLoss:
    """Clipped policy loss: with ``ratio = exp(logprob - old_logprobs)``, the mean of
    ``-min(ratio * A, clamp(ratio, 1 - clip[0], 1 + clip[1]) * A)`` plus, with
    ``ref_logprobs``, ``kl_coef * (exp(d) - d - 1)`` for ``d = ref_logprobs - logprob``.

    The mean is over all tokens that count, or with ``average="sequence"`` over
    the sequences' own means (those with a token that counts): one for each
    element of the batch, or for ``(rows, vocab)`` logits from ``offsets[i]`` to
    ``offsets[i + 1]``.  ``scale`` multiplies the loss; a factor that is known
    beforehand (of gradient accumulation, for one) is given here rather than
    multiplied afterwards, which has the gradient computed a second time."""
    if average not in ("token", "sequence"):
        raise ValueError(f"average must be 'token' or 'sequence' (got {average!r})")
    rows = _rows(logits)
    offs, n = _sequences(offsets, logits, average == "sequence")
    desc = _lib.Policy(
        _per_row(tokens, "tokens", logits, _INTS), _per_row(old_logprobs, "old_logprobs", logits, _F32),
        _per_row(advantages, "advantages", logits, _F32), _per_row(ref_logprobs, "ref_logprobs", logits, _F32),
        _ptr(offs), n, int(ignore_index), float(clip[0]), float(clip[1]), float(kl_coef), float(temperature),
        float(scale), int(average == "sequence"))
    tensors = [t for t in (tokens, old_logprobs, advantages, ref_logprobs, offs) if t is not None]
    call = _PolicyCall(logits, rows, desc, [t.detach() for t in tensors])
    if _wants_grad(logits):
        return PolicyLoss(*_OnePass.apply(logits, call))
    return PolicyLoss(*call.loss(None))


# ---------------------------------------------------------------------------

class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, rows, desc, temperature, ignore_index):
        loss, logprobs, rewards, stats, coef = _preference(logits, rows, desc, True)
        ctx.save_for_backward(logits, tokens, stats, coef)
        ctx.hyper = temperature, ignore_index
        ctx.mark_non_differentiable(logprobs, rewards)
        return loss, logprobs, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output, *_):
        logits, tokens, stats, coef = ctx.saved_tensors
        temperature, ignore_index = ctx.hyper
        grad = _grad_like(logits)
        dev = logits.device
        scale = _scale_of(grad_output)
        with _lib.device_guard(dev):
            _lib.check(_lib.load().mamw_logits_grad(
                ctypes.byref(_rows(logits)), ctypes.byref(_per_row(tokens, "tokens", logits, _INTS)), ignore_index,
                temperature, stats.data_ptr(), ctypes.byref(_per_row(coef, "coefficients", logits, _F32)), None, None,
                scale.data_ptr(), grad.data_ptr(), _lib.raw_stream(dev)), "preference_loss backward")
        return grad, None, None, None, None, None


def _preference(logits, rows, desc, with_grad):
    lib, dev, shape = _lib.load(), logits.device, logits.shape[:-1]
    ws = _workspace(lib.mamw_preference_workspace_bytes, logits, ctypes.byref(rows), ctypes.byref(desc))
    loss = torch.empty((), dtype=torch.float32, device=dev)
    per_sequence = torch.empty((2, desc.sequences), dtype=torch.float32, device=dev)
    stats = torch.empty((*shape, 2), dtype=torch.float32, device=dev) if with_grad else None
    coef = torch.empty(shape, dtype=torch.float32, device=dev) if with_grad else None
    with _lib.device_guard(dev):
        _lib.check(lib.mamw_preference_loss(
            ctypes.byref(rows), ctypes.byref(desc), loss.data_ptr(), per_sequence[0].data_ptr(),
            per_sequence[1].data_ptr(), _ptr(stats), _ptr(coef), ws.data_ptr(), ws.numel(), _lib.raw_stream(dev)),
            "preference_loss")
    return loss, per_sequence[0], per_sequence[1], stats, coef


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, ref_logprobs: torch.Tensor | None, *,
                    beta: float = 0.1, kind: Literal["sigmoid", "ipo", "hinge"] = "sigmoid",
                    label_smoothing: float = 0.0, length_average: bool = False, offsets: torch.Tensor | None = None,
                    temperature: float = 1.0, ignore_index: int = -100) -> PreferenceLoss:
    """Preference loss over pairs: of ``2 P`` sequences the first ``P`` are the
    preferred ones, sequence ``i`` against ``i + P``.  A sequence's reward is
    ``beta * (logprob - ref_logprobs)`` with the sum (``length_average``: the
    mean) of its tokens' log-probabilities; ``h`` is the difference of a pair's.

    ``kind``: ``"sigmoid"`` ``-log sigmoid(h)`` (with ``label_smoothing`` e,
    ``1 - e`` of it and ``e`` of ``-log sigmoid(-h)``), ``"ipo"``
    ``(h / beta - 1 / (2 beta))**2``, ``"hinge"`` ``max(0, 1 - h)``; the loss is
    the mean over the pairs.  Sequences as in :func:`policy_loss`;
    ``ref_logprobs`` holds one value for each, ``None`` for 0."""
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {sorted(_KINDS)} (got {kind!r})")
    rows = _rows(logits)
    offs, n = _sequences(offsets, logits, True)
    if n < 2 or n % 2:
        raise ValueError(f"pairs need an even number of sequences, at least 2 (got {n})")
    if ref_logprobs is not None:
        if ref_logprobs.dtype != torch.float32:
            raise TypeError(f"ref_logprobs must be float32 (got {ref_logprobs.dtype})")
        if ref_logprobs.shape != (n,) or ref_logprobs.device != logits.device:
            raise ValueError(f"ref_logprobs must hold one value for each of {n} sequences on {logits.device} "
                             f"(got {tuple(ref_logprobs.shape)} on {ref_logprobs.device})")
        ref_logprobs = ref_logprobs.contiguous()
    desc = _lib.Preference(_per_row(tokens, "tokens", logits, _INTS), _ptr(ref_logprobs), _ptr(offs), n,
                           int(ignore_index), float(beta), float(label_smoothing), float(temperature), _KINDS[kind],
                           int(bool(length_average)), 0)
    if _wants_grad(logits):
        return PreferenceLoss(*_Preference.apply(logits, tokens, rows, desc, float(temperature), int(ignore_index)))
    return PreferenceLoss(*_preference(logits, rows, desc, False)[:3])


# ---------------------------------------------------------------------------

class _DistillCall:
    def __init__(self, logits, rows, desc, tensors):
        self.rows, self.desc, self.tensors, self.device = rows, desc, tensors, logits.device
        lib = _lib.load()
        self.ws = _workspace(lib.mamw_distill_workspace_bytes, logits, ctypes.byref(rows), ctypes.byref(desc))

    def loss(self, grad):
        result = torch.empty(3, dtype=torch.float32, device=self.device)
        with _lib.device_guard(self.device):
            _lib.check(_lib.load().mamw_distill_loss(
                ctypes.byref(self.rows), ctypes.byref(self.desc), result.data_ptr(), _ptr(grad), self.ws.data_ptr(),
                self.ws.numel(), _lib.raw_stream(self.device)), "distill_loss")
        return (result[0],)

    def again(self, scale, unless_one, grad):
        with _lib.device_guard(self.device):
            _lib.check(_lib.load().mamw_distill_grad(
                ctypes.byref(self.rows), ctypes.byref(self.desc), scale.data_ptr(), int(unless_one), grad.data_ptr(),
                self.ws.data_ptr(), self.ws.numel(), _lib.raw_stream(self.device)), "distill_loss backward")


def distill_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_indices: torch.Tensor, *,
                 teacher_lse: torch.Tensor | None = None, mask: torch.Tensor | None = None, temperature: float = 1.0,
                 scale: float = 1.0) -> torch.Tensor:
    """``temperature**2`` times the mean divergence KL(teacher || student) at
    ``temperature``, from the teacher's ``k`` first logits of each row and their
    places in the vocabulary (``k`` up to 1024, in any order).

    Without ``teacher_lse`` the ``k`` entries are the teacher's whole distribution.
    With ``teacher_lse``, the ``logsumexp(teacher / temperature)`` over its whole
    vocabulary, they have their true probabilities, and all other entries
    together count as one more, of which at least ``2**-20`` is taken to be left.
    Entries with a negative index or a logit of ``-inf`` are padding.  Rows with a
    false ``mask`` do not count.  ``scale`` as in :func:`policy_loss`."""
    rows = _rows(logits)
    if not isinstance(teacher_logits, torch.Tensor) or teacher_logits.dim() < 1:
        raise ValueError("teacher_logits must have k values for each row")
    k = teacher_logits.shape[-1]
    if not 1 <= k <= _lib.MAX_TEACHER:
        raise ValueError(f"teacher_logits must have between 1 and {_lib.MAX_TEACHER} values for each row (got {k})")
    if k > 1 and teacher_logits.stride(-1) != 1:
        teacher_logits = teacher_logits.contiguous()
    if k > 1 and isinstance(teacher_indices, torch.Tensor) and teacher_indices.dim() and teacher_indices.stride(-1) != 1:
        teacher_indices = teacher_indices.contiguous()
    desc = _lib.Distill(
        _per_row(teacher_logits, "teacher_logits", logits, _FLOATS, k),
        _per_row(teacher_indices, "teacher_indices", logits, _INTS, k),
        _per_row(teacher_lse, "teacher_lse", logits, _F32), _per_row(mask, "mask", logits, _BOOLS), k,
        float(temperature), float(scale))
    tensors = [t for t in (teacher_logits, teacher_indices, teacher_lse, mask) if t is not None]
    call = _DistillCall(logits, rows, desc, [t.detach() for t in tensors])
    if _wants_grad(logits):
        return _OnePass.apply(logits, call)[0]
    return call.loss(None)[0]
