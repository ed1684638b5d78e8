"""What the serving operators refuse before anything is launched.  Without a GPU the tensors say they are on one and have no memory."""
from contextlib import nullcontext

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

ON = pytest.mark.parametrize("tensors", [pytest.param(FakeTensorMode, id="no GPU"), pytest.param(nullcontext, id="GPU", marks=pytest.mark.gpu)])
F32, F64, BF16, I32, I64 = torch.float32, torch.float64, torch.bfloat16, torch.int32, torch.int64


@pytest.fixture(scope="module")
def ops():
    from rwkvstic_amd import ops as _ops
    return _ops


def _e(*s, dtype=F32, device="cuda"):
    return torch.empty(*s, dtype=dtype, device=device)


def _arguments(op):
    if op == "lora_rows":
        return dict(x=_e(6, 32), a=_e(3, 4, 32, dtype=BF16), b=_e(3, 20, 4, dtype=BF16), adapter=_e(6, dtype=I32), scale=_e(3), base=_e(6, 20), out=_e(6, 20))
    if op == "delta_rule":
        return dict(q=_e(6, 2, 16), k=_e(6, 2, 16), v=_e(6, 4, 8), g=_e(6, 4), beta=_e(6, 4), state=_e(2, 4, 16, 8), starts=_e(3, dtype=I32), out=_e(6, 4, 8))
    return dict(logits=_e(2, 4, 50, dtype=F64), drafts=_e(2, 3, dtype=I64), u=_e(2, 4), draft_logits=_e(2, 3, 50, dtype=F64), lengths=_e(2, dtype=I32))


WRONG = {
    "short": lambda t: t[:-1],
    "narrow": lambda t: t[..., :-1].contiguous(),
    "other type": lambda t: t.new_empty(t.shape, dtype=torch.int16),
    "strided": lambda t: torch.stack((t, t), -1)[..., 0],
    "on the host": lambda t: _e(*t.shape, dtype=t.dtype, device="cpu"),
    "no tensor": lambda t: 3.0,
}


@ON
@pytest.mark.parametrize("op,which", [(op, which) for op in ("lora_rows", "delta_rule", "verify_drafts") for which in {
    "lora_rows": ("x", "a", "b", "adapter", "scale", "base", "out"), "delta_rule": ("q", "k", "v", "g", "beta", "state", "starts", "out"),
    "verify_drafts": ("logits", "drafts", "u", "draft_logits", "lengths")}[op]])
@pytest.mark.parametrize("how", WRONG)
def test_an_argument_that_does_not_fit_is_refused(ops, tensors, op, which, how):
    with tensors():
        args = _arguments(op)
        args[which] = WRONG[how](args[which])
        with pytest.raises((ValueError, TypeError)):
            getattr(ops, op)(**args)


@ON
def test_results_and_arguments_that_cannot_be(ops, tensors):
    with tensors():
        a = _arguments("lora_rows")
        with pytest.raises(ValueError):               # rows of the result in the same memory
            ops.lora_rows(**{**a, "out": _e(1, 20).expand(6, 20)})
        with pytest.raises(TypeError):                # base of another type than x
            ops.lora_rows(**{**a, "base": _e(6, 20, dtype=F64)})
        a = _arguments("delta_rule")
        with pytest.raises(ValueError):               # 6 rows, 4 sequences
            ops.delta_rule(**{**a, "state": _e(4, 4, 16, 8), "starts": None})
        with pytest.raises(ValueError):
            ops.delta_rule(**{**a, "state": _e(2, 4, 16, 8).transpose(0, 1)})
        a = _arguments("verify_drafts")
        with pytest.raises(ValueError):
            ops.verify_drafts(**{**a, "u": None})
        for temp in (0.0, -1.0, float("nan")):
            with pytest.raises(ValueError):
                ops.verify_drafts(**a, temp=temp)


def test_the_library_looks_for_itself():
    """Sizes, types, strides and workspaces, at the C entry points; nothing is launched."""
    from rwkvstic_amd import _native
    L = _native.lib()
    ARG, ALIGN, SIZE, WORKSPACE = -1, -2, -3, -4
    ws = 1 << 40

    def lora(T=2, n_in=8, n_out=8, N=1, R=4, real=0, x=16, xs=8, low=2, a=16, b=16, adapter=16, base=16, bs=8, out=16, os=8, work=16, n=ws):
        return L.rwkv_lora_rows(None, T, n_in, n_out, N, R, real, x, xs, low, a, b, adapter, None, base, bs, out, os, work, n)
    for kw in ({"x": None}, {"adapter": None}, {"out": None}, {"T": 0}, {"R": 0}, {"N": -1}, {"real": 2}, {"low": 1}, {"low": 9}, {"os": 7}, {"xs": -1}):
        assert lora(**kw) == ARG, kw
    assert lora(R=257) == SIZE and lora(n=0) == WORKSPACE and lora(work=None) == WORKSPACE and lora(work=8) == ALIGN
    assert L.rwkv_lora_rows_workspace_bytes(0, 8, 8, 1, 4, 0) == 0

    def delta(T=4, B=2, Hk=1, Hv=2, dk=16, dv=16, type=0, q=16, st=16, starts=16, state=16, work=16, n=ws):
        return L.rwkv_delta_rule(None, T, B, Hk, Hv, dk, dv, type, q, st, 16, st, 16, st, 16, 16, 1.0, starts, state, 16, work, n)
    for kw in ({"q": None}, {"state": None}, {"T": 0}, {"B": 0}, {"Hk": 3}, {"dk": 0}, {"type": 1}, {"st": -1}, {"starts": None, "T": 5}):
        assert delta(**kw) == ARG, kw
    assert delta(dk=257) == SIZE
    assert L.rwkv_delta_rule_workspace_bytes(0, 1, 1, 1, 16, 16) == 0

    def verify(B=2, K=3, V=50, real=1, logits=16, s=200, drafts=16, u=16, temp=1.0, greedy=0, tokens=16, work=16, n=ws):
        return L.rwkv_verify_drafts(None, B, K, V, real, logits, s, 50, None, 0, 0, drafts, None, u, temp, greedy, tokens, 16, work, n)
    for kw in ({"logits": None}, {"drafts": None}, {"u": None}, {"tokens": None}, {"B": 0}, {"K": -1}, {"V": 0}, {"real": 2}, {"temp": 0.0}, {"s": -1}):
        assert verify(**kw) == ARG, kw
    assert verify(K=65) == SIZE and verify(n=0) == WORKSPACE and verify(work=8) == ALIGN
    assert L.rwkv_verify_drafts_workspace_bytes(0, 3, 50) == 0


def test_results_in_the_memory_of_what_is_read():
    """Rows of base and of the result may lie between each other, and be the same; nothing is launched."""
    from rwkvstic_amd import _native
    L = _native.lib()
    ARG, WORKSPACE, base = -1, -4, 1 << 20

    def lora(T, at, bs, os, n_out=8):
        return L.rwkv_lora_rows(None, T, 8, n_out, 1, 4, 0, 16, 8, 2, 16, 16, 16, None, base, bs, base + 4 * at, os, 16, 0)
    for at, bs, os, shared in [(0, 8, 8, False), (0, 8, 9, True), (8, 8, 8, True), (24, 8, 8, False), (-24, 8, 8, False), (-23, 8, 8, True), (8, 16, 16, False),
                               (-8, 16, 16, False), (7, 16, 16, True), (9, 16, 16, True), (9, 17, 17, False), (24, 8, 100, False), (5, 0, 8, True), (8, 0, 8, False)]:
        assert lora(3, at, bs, os) == (ARG if shared else WORKSPACE), (at, bs, os)
    assert lora(1, 8, 8, 8) == WORKSPACE and lora(1, 7, 8, 8) == ARG

    far = [(i + 1) << 24 for i in range(7)]

    def delta(**at):
        q, k, v, g, beta, state, o = [at.get(n, f) for n, f in zip(("q", "k", "v", "g", "beta", "state", "o"), far)]
        return L.rwkv_delta_rule(None, 100, 1, 1, 2, 16, 16, 0, q, 16, k, 16, v, 32, g, beta, 1.0, None, state, o, 16, 0)
    assert delta() == WORKSPACE and delta(k=far[0]) == WORKSPACE
    for kw in ({"o": far[2]}, {"o": far[0] + 4}, {"o": far[5]}, {"state": far[4]}, {"o": far[3] + 800 - 4}, {"o": far[1] - 4 * 3200 + 4}):
        assert delta(**kw) == ARG, kw
    assert delta(o=far[3] + 800) == WORKSPACE and delta(o=far[1] - 4 * 3200) == WORKSPACE
