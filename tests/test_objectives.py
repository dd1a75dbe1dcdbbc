"""What the objectives refuse, on the host and before anything is queued: through
Python (arguments are checked before the device, so CPU tensors do) and at the C
ABI, where device pointers are fake addresses that validation never reads."""

import ctypes

import pytest
import torch

from triton_muon_adamw import _lib, distill_loss, policy_loss, preference_loss, token_logprobs

NULL, COUNT, NUMEL, SHAPE, ALIGN, WS, HYPER, ALIAS = -1, -2, -3, -4, -5, -6, -7, -9

X = torch.zeros(6, 9)
T = torch.zeros(6, dtype=torch.int64)
F = torch.zeros(6)
OFF = torch.tensor([0, 3, 6])


def logprobs(logits=X, tokens=T, **kw):
    return token_logprobs(logits, tokens, **kw)


def policy(logits=X, tokens=T, old=F, adv=F, **kw):
    return policy_loss(logits, tokens, old, adv, **kw)


def preference(logits=X, tokens=T, ref=None, offsets=OFF, **kw):
    return preference_loss(logits, tokens, ref, offsets=offsets, **kw)


def distill(logits=X, teacher=torch.zeros(6, 2), index=torch.zeros(6, 2, dtype=torch.int64), **kw):
    return distill_loss(logits, teacher, index, **kw)


ALL = [logprobs, policy, preference, distill]


@pytest.mark.parametrize("fn", ALL)
def test_cpu_tensors_are_refused(fn):
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        fn()


@pytest.mark.parametrize("fn", ALL)
@pytest.mark.parametrize("logits,error,text", [
    (X.double(), TypeError, "float32, bfloat16 or float16"),
    (X.long(), TypeError, "float32, bfloat16 or float16"),
    (torch.zeros(9), ValueError, "rows, vocab"),
    (torch.zeros(1, 2, 3, 9), ValueError, "rows, vocab"),
    (torch.zeros(6, 0), ValueError, "empty vocabulary"),
    (torch.zeros(9, 6).t(), ValueError, "contiguous along the vocabulary"),
    (torch.zeros(6, 18)[:, ::2], ValueError, "contiguous along the vocabulary"),
    ([[0.0]], TypeError, "logits must be a tensor"),
])
def test_logits_refused(fn, logits, error, text):
    with pytest.raises(error, match=text):
        fn(logits)


@pytest.mark.parametrize("call,error,text", [
    (lambda: logprobs(tokens=T.float()), TypeError, "tokens must be int32 or int64"),
    (lambda: logprobs(tokens=T[:5]), ValueError, "does not go with"),
    (lambda: logprobs(tokens=T.view(2, 3)), ValueError, "does not go with"),
    (lambda: logprobs(tokens=None), TypeError, "tokens must be a tensor"),
    (lambda: logprobs(temperature="warm"), TypeError, "real number|float"),
    (lambda: policy(old=F.double()), TypeError, "old_logprobs must be float32"),
    (lambda: policy(adv=F.bfloat16()), TypeError, "advantages must be float32"),
    (lambda: policy(adv=torch.zeros(4)), ValueError, "advantages of shape"),
    (lambda: policy(ref_logprobs=T), TypeError, "ref_logprobs must be float32"),
    (lambda: policy(average="batch"), ValueError, "average must be"),
    (lambda: policy(average="sequence"), ValueError, "need offsets"),
    (lambda: policy(clip=(-0.1, 0.2)), ValueError, "hyper-parameter"),
    (lambda: policy(clip=(0.1, float("nan"))), ValueError, "hyper-parameter"),
    (lambda: policy(kl_coef=float("inf")), ValueError, "hyper-parameter"),
    (lambda: policy(scale=float("nan")), ValueError, "hyper-parameter"),
    (lambda: policy(temperature=0.0), ValueError, "hyper-parameter"),
    (lambda: policy(temperature=-1.0), ValueError, "hyper-parameter"),
    (lambda: policy(temperature=float("inf")), ValueError, "hyper-parameter"),
    (lambda: policy(temperature=1e-40), ValueError, "hyper-parameter"),
    (lambda: policy(offsets=OFF.float()), TypeError, "offsets must be int32 or int64"),
    (lambda: policy(offsets=OFF[None]), ValueError, "offsets must hold"),
    (lambda: policy(offsets=OFF[:0]), ValueError, "offsets must hold"),
    (lambda: policy(X.view(2, 3, 9), T.view(2, 3), F.view(2, 3), F.view(2, 3), offsets=OFF), ValueError,
     "offsets go with"),
    (lambda: preference(offsets=None), ValueError, "need offsets"),
    (lambda: preference(offsets=torch.tensor([0, 2, 4, 6])), ValueError, "even number"),
    (lambda: preference(offsets=OFF[:1]), ValueError, "even number"),
    (lambda: preference(ref=torch.zeros(3)), ValueError, "one value for each of 2"),
    (lambda: preference(ref=torch.zeros(2, dtype=torch.float64)), TypeError, "ref_logprobs must be float32"),
    (lambda: preference(kind="log"), ValueError, "kind must be"),
    (lambda: preference(beta=0.0), ValueError, "hyper-parameter"),
    (lambda: preference(label_smoothing=1.5), ValueError, "hyper-parameter"),
    (lambda: preference(kind="ipo", label_smoothing=0.1), ValueError, "hyper-parameter"),
    (lambda: distill(teacher=torch.zeros(6, 0)), ValueError, "between 1 and 1024"),
    (lambda: distill(teacher=torch.zeros(6, 1025)), ValueError, "between 1 and 1024"),
    (lambda: distill(teacher=torch.zeros(())), ValueError, "between 1 and 1024"),
    (lambda: distill(teacher=torch.zeros(6, 2).double()), TypeError, "teacher_logits must be"),
    (lambda: distill(index=torch.zeros(6, 3, dtype=torch.int64)), ValueError, "2 values for each row"),
    (lambda: distill(index=torch.zeros(6, 2)), TypeError, "teacher_indices must be int32 or int64"),
    (lambda: distill(teacher_lse=torch.zeros(6, 1)), ValueError, "teacher_lse of shape"),
    (lambda: distill(mask=F), TypeError, "mask must be bool"),
    (lambda: distill(mask=torch.ones(5, dtype=torch.bool)), ValueError, "mask of shape"),
])
def test_refused(call, error, text):
    with pytest.raises(error, match=text):
        call()


@pytest.mark.parametrize("fn", ALL)
def test_forward_mode_is_refused(fn):
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        fn(fwd.make_dual(X, torch.ones_like(X)))


# ---- the C ABI

BASE = 1 << 40


def rows(**kw):
    r = _lib.Rows(BASE, 2, 3, 9, 27, 9, _lib.F32, 0)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def per_row(kind, at=BASE + (1 << 30), **kw):
    p = _lib.PerRow(at, 3, 1, kind, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def a_policy(**kw):
    p = _lib.Policy(per_row(_lib.I64), per_row(_lib.F32), per_row(_lib.F32), _lib.PerRow(None, 0, 0, 0, 0), None, 2,
                    -100, 0.2, 0.2, 0.0, 1.0, 1.0, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def a_preference(**kw):
    p = _lib.Preference(per_row(_lib.I64), None, None, 2, -100, 0.1, 0.0, 1.0, 0, 0, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def a_distill(**kw):
    none = _lib.PerRow(None, 0, 0, 0, 0)
    p = _lib.Distill(per_row(_lib.BF16), per_row(_lib.I32), none, none, 4, 1.0, 1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def ws_bytes(kind, r, p):
    n = ctypes.c_size_t()
    st = getattr(_lib.load(), f"mamw_{kind}_workspace_bytes")(ctypes.byref(r), ctypes.byref(p), ctypes.byref(n))
    return st, n.value


@pytest.mark.parametrize("change,status", [
    ({"type": _lib.I32}, HYPER), ({"reserved": 1}, HYPER), ({"outer": -1}, SHAPE), ({"inner": -1}, SHAPE),
    ({"vocab": 0}, SHAPE), ({"vocab": (1 << 30) + 1}, SHAPE), ({"outer_stride": -1}, SHAPE),
    ({"inner_stride": -1}, SHAPE), ({"outer": 1 << 31}, COUNT), ({"outer": 1 << 16, "inner": 1 << 16}, COUNT),
    ({"outer": 2, "outer_stride": 1 << 62}, NUMEL), ({"data": None}, NULL), ({"data": BASE + 2}, ALIGN),
])
def test_abi_rows(change, status):
    r = rows(**change)
    for kind, p in (("policy", a_policy()), ("distill", a_distill())):
        assert ws_bytes(kind, r, p)[0] == status
    lib = _lib.load()
    st = lib.mamw_token_logprobs(ctypes.byref(r), ctypes.byref(per_row(_lib.I64)), -100, 1.0, BASE, None, None, None)
    assert st == status


@pytest.mark.parametrize("kind,make,change,status", [
    ("policy", a_policy, {"tokens": per_row(_lib.F32)}, HYPER),
    ("policy", a_policy, {"tokens": _lib.PerRow(None, 0, 0, _lib.I64, 0)}, NULL),
    ("policy", a_policy, {"old_logprobs": per_row(_lib.F32, at=BASE + 1)}, ALIGN),
    ("policy", a_policy, {"advantages": per_row(_lib.F32, inner_stride=-1)}, SHAPE),
    ("policy", a_policy, {"advantages": per_row(_lib.F32, reserved=3)}, HYPER),
    ("policy", a_policy, {"sequences": 3}, COUNT),
    ("policy", a_policy, {"sequences": -1}, COUNT),
    ("policy", a_policy, {"offsets": BASE + 4, "sequences": 5}, ALIGN),
    ("policy", a_policy, {"clip_low": -1.0}, HYPER),
    ("policy", a_policy, {"temperature": float("nan")}, HYPER),
    ("preference", a_preference, {"sequences": 1}, COUNT),
    ("preference", a_preference, {"sequences": 3, "offsets": BASE}, COUNT),
    ("preference", a_preference, {"beta": float("inf")}, HYPER),
    ("preference", a_preference, {"smoothing": -0.1}, HYPER),
    ("preference", a_preference, {"kind": 3}, HYPER),
    ("preference", a_preference, {"reserved": 1}, HYPER),
    ("preference", a_preference, {"ref_logprobs": BASE + 2}, ALIGN),
    ("distill", a_distill, {"k": 0}, SHAPE),
    ("distill", a_distill, {"k": 1025}, SHAPE),
    ("distill", a_distill, {"teacher_logits": per_row(_lib.I32)}, HYPER),
    ("distill", a_distill, {"teacher_indices": per_row(_lib.BOOL)}, HYPER),
    ("distill", a_distill, {"mask": per_row(_lib.I32)}, HYPER),
    ("distill", a_distill, {"scale": float("inf")}, HYPER),
])
def test_abi_descriptions(kind, make, change, status):
    assert ws_bytes(kind, rows(), make())[0] == 0
    assert ws_bytes(kind, rows(), make(**change))[0] == status


def test_abi_wide_tail():
    lse = per_row(_lib.F32)
    assert ws_bytes("distill", rows(vocab=1 << 20), a_distill(teacher_lse=lse))[0] == 0
    assert ws_bytes("distill", rows(vocab=(1 << 20) + 1), a_distill(teacher_lse=lse))[0] == SHAPE
    assert ws_bytes("distill", rows(vocab=(1 << 20) + 1), a_distill())[0] == 0


def test_abi_workspaces_outputs_and_overlap():
    lib = _lib.load()
    r, p, f, d = rows(), a_policy(), a_preference(), a_distill()
    far = BASE + (1 << 34)
    for kind, desc, loss in (("policy", p, lambda ws, n, g=far, out=far: lib.mamw_policy_loss(
                                 ctypes.byref(r), ctypes.byref(p), out, far, g, ws, n, None)),
                             ("distill", d, lambda ws, n, g=far, out=far: lib.mamw_distill_loss(
                                 ctypes.byref(r), ctypes.byref(d), out, g, ws, n, None)),
                             ("preference", f, lambda ws, n, g=far, out=far: lib.mamw_preference_loss(
                                 ctypes.byref(r), ctypes.byref(f), out, far, far, far, far, ws, n, None))):
        st, n = ws_bytes(kind, r, desc)
        assert st == 0 and n > 0
        assert loss(None, n) == WS and loss(far + 8, n) == WS and loss(far, n - 1) == WS
        assert loss(far, n, out=None) == NULL
        if kind != "preference":
            assert loss(far, n, g=BASE + 27 * 4) == ALIAS  # inside the logits
            assert loss(far, n, g=far + 2) == ALIGN
    for grad, desc in ((lib.mamw_policy_grad, p), (lib.mamw_distill_grad, d)):
        assert grad(ctypes.byref(r), ctypes.byref(desc), None, 0, far, far, 1 << 20, None) == NULL
        assert grad(ctypes.byref(r), ctypes.byref(desc), far, 0, None, far, 1 << 20, None) == NULL
    toks, coef = per_row(_lib.I64), per_row(_lib.F32)
    assert lib.mamw_logits_grad(ctypes.byref(r), ctypes.byref(toks), -100, 1.0, None, ctypes.byref(coef), None, None,
                                None, far, None) == NULL
    assert lib.mamw_logits_grad(ctypes.byref(r), ctypes.byref(toks), -100, 1.0, far, ctypes.byref(coef), None, None,
                                None, BASE, None) == ALIAS
    assert lib.mamw_logits_grad(ctypes.byref(r), ctypes.byref(toks), -100, 1.0, far, ctypes.byref(coef),
                                ctypes.byref(coef), None, None, far, None) == NULL
    assert lib.mamw_token_logprobs(ctypes.byref(r), None, -100, 1.0, far, None, None, None) == NULL
    assert lib.mamw_token_logprobs(ctypes.byref(r), ctypes.byref(toks), -100, 0.0, far, None, None, None) == HYPER
    assert lib.mamw_token_logprobs(ctypes.byref(r), ctypes.byref(toks), -100, 1.0, None, None, None, None) == NULL
    for kind in ("policy", "preference", "distill"):
        assert getattr(lib, f"mamw_{kind}_workspace_bytes")(ctypes.byref(r), None, ctypes.byref(ctypes.c_size_t())) \
            == NULL


def test_no_rows_need_no_pointers():
    r = rows(outer=0, data=None)
    p = a_policy(tokens=_lib.PerRow(None, 0, 0, 0, 0), old_logprobs=_lib.PerRow(None, 0, 0, 0, 0),
                 advantages=_lib.PerRow(None, 0, 0, 0, 0), sequences=0)
    assert ws_bytes("policy", r, p)[0] == 0
    lib = _lib.load()
    assert lib.mamw_token_logprobs(ctypes.byref(r), ctypes.byref(p.tokens), -100, 1.0, None, None, None, None) == 0


def test_a_missing_native_module_is_an_error(monkeypatch):
    import sys

    import triton_muon_adamw

    monkeypatch.setattr(_lib, "_objectives", None)
    monkeypatch.delattr(triton_muon_adamw, "_objectives", raising=False)
    monkeypatch.setitem(sys.modules, "triton_muon_adamw._objectives", None)
    with pytest.raises(RuntimeError, match="_objectives cannot be used"):
        logprobs()


def test_abi_types_that_are_none():
    """In a process of its own: what ends it is not an error status."""
    import subprocess
    import sys
    from pathlib import Path

    code = f"""
import sys
sys.path[:0] = {[str(Path(__file__).parent), *sys.path]!r}
from test_objectives import *
for kind, make, name in [("policy", a_policy, "old_logprobs"), ("policy", a_policy, "advantages"),
                         ("policy", a_policy, "ref_logprobs"), ("distill", a_distill, "teacher_lse"),
                         ("distill", a_distill, "mask")]:
    for number in (-1, 6, 1 << 30):
        assert ws_bytes(kind, rows(), make(**{{name: per_row(number)}}))[0] == HYPER, (name, number)
print("refused")
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert (res.returncode, res.stdout.strip()) == (0, "refused"), res.stderr[-500:]
