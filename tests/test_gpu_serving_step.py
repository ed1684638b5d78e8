"""GPU: the serving operators as a program uses them: recorded into graphs, on several streams, from several threads, without their
native host side, and one after the other as a serving step of many requests."""
import threading

import pytest
import torch

import serving_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rwkvstic_amd import ops as _ops
    return _ops


def _calls(ops, seed, many):
    """One call of each operator (name, call, the tensors it reads that a caller would change), of few rows or of many."""
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g)
    T = 300 if many else 7
    x, a, b, base = f(T, 160).cuda(), f(5, 24, 160).bfloat16().cuda(), f(5, 96, 24).bfloat16().cuda(), f(T, 96).cuda()
    adapter = torch.randint(-1, 5, (T,), generator=g, dtype=torch.int32).cuda()
    yield "lora_rows", lambda: [ops.lora_rows(x, a, b, adapter, base=base)], (x, base)
    c = [t.cuda() for t in P.delta_inputs(T, 2, 2, 4, 64, 64, torch.bfloat16, seed)]
    starts = torch.tensor([0, T // 3, T], dtype=torch.int32).cuda()
    state = c[5].clone()
    def delta():
        s = c[5] * 1.0                                # (a new tensor: the state goes on from the same place at every call)
        return [ops.delta_rule(*c[:5], s, starts=starts), s]
    yield "delta_rule", delta, (c[2], c[5])
    logits, drafts, u, draft = (t.cuda() for t in P.verify_inputs(40 if many else 2, 3, 5000, torch.float64, seed))
    yield "verify_drafts", lambda: list(ops.verify_drafts(logits, drafts, u, draft_logits=draft, temp=0.7)), (u,)


def _change(tensors, step):
    for t in tensors:
        t.copy_(torch.rand_like(t) if t.dim() == 2 and t.dtype == torch.float32 and t.shape[1] <= 4 else t * (1.0 if step % 2 else -1.0))


@pytest.mark.parametrize("many", [False, True])
def test_recorded_calls(ops, many):
    """Each operator in a graph of its own: replayed with other inputs, with eager calls and synchronizations between."""
    for name, call, inputs in _calls(ops, 3, many):
        print(f"recorded {name} {many}", flush=True)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            recorded = call()
        for step in range(4):
            _change(inputs, step)
            want = [t.clone() for t in call()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(w, r) for w, r in zip(want, recorded)), (name, step)
            call()


def test_two_graphs_do_not_share_scratch(ops):
    """Graphs of the same operators replayed on two streams at once."""
    made = []
    for seed in (5, 6):
        calls = list(_calls(ops, seed, True))
        want = [[t.clone() for t in call()] for _, call, _ in calls]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [call() for _, call, _ in calls]
        made.append((graph, got, want, torch.cuda.Stream(), calls))
    for _ in range(20):
        for graph, _, _, stream, _ in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _, _ in made:
        assert all(torch.equal(w, r) for ws, rs in zip(want, got) for w, r in zip(ws, rs))


def test_calls_of_several_threads_and_streams(ops):
    """Every call gives what it gives alone, bit for bit, whatever runs beside it."""
    jobs = [(call, [t.clone() for t in call()]) for seed in (1, 2, 3, 4) for _, call, _ in _calls(ops, seed, seed % 2 == 0)]
    torch.cuda.synchronize()
    wrong = []

    def work(mine):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                for call, want in mine:
                    got = call()
                    stream.synchronize()
                    if not all(torch.equal(w, t) for w, t in zip(want, got)):
                        wrong.append(1)
    threads = [threading.Thread(target=work, args=(jobs[i::3],)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


@pytest.mark.parametrize("many", [False, True])
def test_results_are_the_same_without_the_native_host_side(ops, monkeypatch, many):
    from rwkvstic_amd import _native as N
    want = [call() for _, call, _ in _calls(ops, 9, many)]
    monkeypatch.setattr(N, "_host", (N.lib(), None))
    for w, (name, call, _) in zip(want, _calls(ops, 9, many)):
        assert all(torch.equal(a, b) for a, b in zip(w, call())), name


@pytest.mark.parametrize("requests,drafts", [(3, 4), (2, 63)])
def test_a_serving_step_of_many_requests(ops, requests, drafts):
    """A layer of a recurrent model over the drafted tokens of several requests, each with its adapter: quantised projections and
    adapters, the delta rule over the packed rows, the head, the verification."""
    C, Hk, Hv, d, V, R = 256, 2, 4, 64, 700, 8
    rows, T = drafts + 1, requests * (drafts + 1)
    g = torch.Generator().manual_seed(drafts)
    f = lambda *s: torch.randn(*s, generator=g)
    widths = {"q": Hk * d, "k": Hk * d, "v": Hv * d, "gate": 2 * Hv, "head": V}
    weight = {n: f(w, C if n != "head" else Hv * d) * C ** -0.5 for n, w in widths.items()}
    a = {n: f(3, R, weight[n].shape[1]) * C ** -0.5 for n in widths}
    b = {n: (f(3, w, R) * 0.3).bfloat16() for n, w in widths.items()}
    a = {n: t.bfloat16() for n, t in a.items()}
    scale = torch.tensor([1.0, 0.5, 2.0])
    adapter = torch.tensor([i % 4 - 1 for i in range(requests)], dtype=torch.int32).repeat_interleave(rows)
    x, state = f(T, C).double(), f(requests, Hv, d, d) * 0.1
    tokens, u = torch.randint(0, V, (requests, drafts), generator=g), torch.rand(requests, rows, generator=g)
    starts = torch.arange(0, T + 1, rows, dtype=torch.int32)

    def step(project, recur, unit):
        q, k, v, gate = (project(n, None) for n in ("q", "k", "v", "gate"))
        o = recur(unit(q.view(T, Hk, d)), unit(k.view(T, Hk, d)), v.view(T, Hv, d), -torch.nn.functional.softplus(gate[:, :Hv]), torch.sigmoid(gate[:, Hv:]))
        return project("head", o.reshape(T, Hv * d).double()).view(requests, rows, V)

    # on the device
    packed = {n: ops.quantize_packed(w.cuda())[1:] for n, w in weight.items()}
    dx, dstate = x.cuda(), state.cuda()

    def project(n, given):
        inp = dx if given is None else given
        y = ops.gemm8(inp, *packed[n], inp.shape[1], widths[n])
        return ops.lora_rows(inp, a[n].cuda(), b[n].cuda(), adapter.cuda(), scale.cuda(), base=y, out=y)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)
    logits = step(project, lambda q, k, v, gg, be: ops.delta_rule(q.float(), k.float(), v.float().contiguous(), gg.float().contiguous(), be.float().contiguous(), dstate, starts=starts.cuda()), unit)
    got = ops.verify_drafts(logits, tokens.cuda(), u.cuda(), temp=0.9)

    # from the definitions
    after = {}

    def plain(n, given):
        inp = x if given is None else given
        codes, rng, off = (t.cpu() for t in ops.quantize(weight[n].cuda()))
        return P.lora_rows(inp, a[n], b[n], adapter, scale, inp @ (codes.double() * rng.double()[:, None] + off[:, None]))[0]

    def recur(q, k, v, gg, be):
        o, after["state"] = P.delta_rule(q, k, v, gg, be, state, starts.tolist(), d ** -0.5)
        return o
    want = step(plain, recur, unit)
    # four stages of sums of some 256 terms, rounded at random to 2^-24 of the largest: sixteen each, and as much again for what follows
    off = 128 * 2.0 ** -24
    assert float((logits.cpu() - want).abs().max()) <= off * float(want.abs().max())
    assert float((dstate.cpu().double() - after["state"]).abs().max()) <= off * float(after["state"].abs().max())
    checked = P.verify_drafts(logits.cpu(), tokens, u, temp=0.9)
    assert torch.equal(got[0].cpu(), checked[0]) and torch.equal(got[1].cpu(), checked[1])
