"""Results in the memory of what is read: refused by the library before anything is launched, and served where they only lie beside it."""
import pytest
import torch

import serving_plain as P

ARG = -1
WS, FAR = 1 << 50, [(i + 1) << 24 for i in range(12)]


@pytest.fixture(scope="module")
def ops():
    from rwkvstic_amd import ops as _ops
    return _ops


@pytest.mark.parametrize("T,stride", [(1, 8), (5, 8), (5, 40), (300, 8)])
@pytest.mark.parametrize("at,size", [("a", 3 * 4 * 16 * 2), ("b", 3 * 8 * 4 * 2), ("adapter", None), ("scale", 3 * 4)])
def test_adapters_into_what_they_read(T, stride, at, size):
    from rwkvstic_amd import _native
    x, a, b, adapter, scale, work = FAR[:6]
    start = dict(a=a, b=b, adapter=adapter, scale=scale)[at]
    size = T * 4 if size is None else size
    rows = ((T - 1) * stride + 8) * 4

    def into(out):
        return _native.lib().rwkv_lora_rows(None, T, 16, 8, 3, 4, 0, x, 16, 2, a, b, adapter, scale, None, 0, out, stride, work, WS)
    for out in (start, start + size - 4, start - rows + 4):
        assert into(out) == ARG, out - start


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 200])
def test_adapters_beside_what_they_read_and_into_their_rows(ops, T):
    g = torch.Generator().manual_seed(T)
    f = lambda *s: torch.randn(*s, generator=g)
    x, a, b, scale = f(T, 16), f(3, 4, 16), f(3, 16, 4), f(3)
    adapter = torch.arange(T, dtype=torch.int32) % 4
    want, bound = P.lora_rows(x, a, b, adapter, scale)
    near = lambda got: bool(((got.cpu().double() - want).abs() <= 2.0 ** -24 * (bound + want.abs())).all())
    sizes = [3 * 4 * 16, T * 16, 3 * 16 * 4, T, T * 16, 3]             # a, out, b, adapter, out, scale: one after the other
    whole = torch.zeros(sum(sizes)).cuda()
    A, first, B, I, second, S = whole.split(sizes)
    A.copy_(a.flatten()), B.copy_(b.flatten()), I.view(torch.int32).copy_(adapter), S.copy_(scale)
    for out in (first, second):
        assert near(ops.lora_rows(x.cuda(), A.view(3, 4, 16), B.view(3, 16, 4), I.view(torch.int32), S, out=out.view(T, 16)))
    own = x.cuda()                                    # rows that have been read are free for the result
    assert near(ops.lora_rows(own, A.view(3, 4, 16), B.view(3, 16, 4), I.view(torch.int32), S, out=own))
    wide = torch.zeros(T, 48).cuda()
    wide[:, :16] = x.cuda()
    assert near(ops.lora_rows(wide[:, :16], A.view(3, 4, 16), B.view(3, 16, 4), I.view(torch.int32), S, out=wide[:, 8:24]))


@pytest.mark.parametrize("greedy", [0, 1])
@pytest.mark.parametrize("which", ["tokens", "accepted"])
@pytest.mark.parametrize("at", ["logits", "draft", "drafts", "lengths", "u", "other"])
def test_verdicts_into_what_they_are_made_of(greedy, which, at):
    """Sequences of logits 1000 apart, their rows 100 apart: to the last logit of the last row."""
    from rwkvstic_amd import _native
    B, K, V = 5, 3, 50
    memory = dict(zip(("logits", "draft", "drafts", "lengths", "u", "tokens", "accepted"), FAR))
    work = FAR[7]
    size = {"logits": (4 * 1000 + 3 * 100 + 50) * 8, "draft": (4 * 1000 + 2 * 100 + 50) * 8, "drafts": B * K * 8, "lengths": B * 4, "u": B * (K + 1) * 4,
            "tokens": B * (K + 1) * 8, "accepted": B * 8}
    if greedy and at in ("draft", "u"):
        pytest.skip("not read")
    other = {"tokens": "accepted", "accepted": "tokens"}[which] if at == "other" else at
    for to in (memory[other], memory[other] + size[other] - 4, memory[other] - size[which] + 4):
        m = {**memory, which: to}
        got = _native.lib().rwkv_verify_drafts(None, B, K, V, 1, m["logits"], 1000, 100, m["draft"], 1000, 100, m["drafts"], m["lengths"], m["u"], 1.0, greedy,
                                               m["tokens"], m["accepted"], work, WS)
        assert got == ARG, to - memory[other]


@pytest.mark.parametrize("T", [6, 500])
@pytest.mark.parametrize("which,size", [("o", 2 * 16 * 4), ("state", 3 * 2 * 16 * 16 * 4)])
def test_outputs_and_states_into_the_starts(T, which, size):
    from rwkvstic_amd import _native
    q, k, v, g, beta, starts, state, o, work = FAR[:9]
    size *= T if which == "o" else 1
    for to in (starts, starts + 4 * 4 - 4, starts - size + 4):
        m = {"state": state, "o": o, which: to}
        assert _native.lib().rwkv_delta_rule(None, T, 3, 1, 2, 16, 16, 0, q, 16, k, 16, v, 32, g, beta, 1.0, starts, m["state"], m["o"], work, WS) == ARG, to - starts


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 500])
def test_the_delta_rule_beside_what_it_reads(ops, T):
    """Everything that is read and written in one buffer, one after the other."""
    c = P.delta_inputs(T, 3, 1, 2, 16, 16, torch.float32, T)
    starts = [0, T // 3, T // 2, T]
    want, after = P.delta_rule(*c, starts, 0.25)
    s = torch.tensor(starts, dtype=torch.int32)
    parts = [c[5], s.view(torch.float32), torch.zeros(T, 2, 16), c[0], c[1], c[2], c[3], c[4]]
    whole = torch.cat([t.flatten() for t in parts]).cuda()
    at, views = 0, []
    for t in parts:
        views.append(whole[at:at + t.numel()].view(t.shape))
        at += t.numel()
    state, st, out, q, k, v, g, beta = views
    ops.delta_rule(q, k, v, g, beta, state, starts=st.view(torch.int32), scale=0.25, out=out)
    off = 4 * ((T + 64) * (16 + 64)) ** 0.5 * 2.0 ** -24           # rounded sums at random, as elsewhere
    assert float((out.cpu() - want).abs().max()) <= off * float(want.abs().max()) and float((state.cpu() - after).abs().max()) <= off * float(after.abs().max())
    assert torch.equal(st.cpu().view(torch.int32), s)


def test_more_than_a_launch_can_take():
    """Refused for their size before the workspace is looked at; nothing is launched."""
    from rwkvstic_amd import _native
    L = _native.lib()
    SIZE, WORKSPACE = -3, -4
    far = [(i + 1) << 50 for i in range(10)]

    def lora(T, N, real=0):
        return L.rwkv_lora_rows(None, T, 16, 8, N, 4, real, far[0], 16, 2, far[1], far[2], far[3], None, None, 0, far[4], 8, far[5], 0)
    assert lora(1 << 24, 1) == WORKSPACE and lora(1 << 22, 500) == WORKSPACE and lora(1 << 22, 1024) == SIZE and lora(1 << 21, 1024, 1) == SIZE

    def delta(B, T=None, Hv=64):
        T = B if T is None else T
        return L.rwkv_delta_rule(None, T, B, 1, Hv, 4, 4, 0, far[0], 4, far[1], 4, far[2], 4 * Hv, far[3], far[4], 1.0, far[5], far[6], far[7], far[8], 0)
    assert delta(1 << 20) == SIZE and delta(1 << 20, 50 << 20, 1) == WORKSPACE and delta(1 << 24, 50 << 24, 1) == SIZE

    def verify(B, K):
        return L.rwkv_verify_drafts(None, B, K, 4, 0, far[0], 4 * (K + 1), 4, far[1], 4 * K, 4, far[2], None, far[3], 1.0, 0, far[4], far[5], far[6], 0)
    assert verify(1 << 21, 0) == WORKSPACE and verify(1 << 22, 0) == SIZE and verify(1 << 17, 63) == WORKSPACE and verify(1 << 18, 63) == SIZE
