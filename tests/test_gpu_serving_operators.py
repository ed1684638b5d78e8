"""GPU: adapters of many requests, the gated delta rule and the verification of drafts, against their definitions in float64."""
import math

import pytest
import torch

import serving_plain as P

pytestmark = pytest.mark.gpu

HALF = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # half a step


@pytest.fixture(scope="module")
def ops():
    from rwkvstic_amd import ops as _ops
    return _ops


def _cuda(t):
    return t.cuda() if isinstance(t, torch.Tensor) else t


# ------------------------------------------------------------------ adapters
def _adapters(T, n_in, n_out, N, R, real, low, seed, order="shuffled"):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g)
    adapter = torch.randint(-1, N, (T,), generator=g, dtype=torch.int32)
    if order == "segments":
        adapter = adapter.sort(stable=True).values.flip(0).contiguous()
    return dict(x=f(T, n_in).to(real), a=(f(N, R, n_in) * n_in ** -0.5).to(low), b=(f(N, n_out, R) * R ** -0.5).to(low), adapter=adapter,
                scale=0.5 + torch.rand(N, generator=g), base=f(T, n_out).to(real))


def _near(got, want, bound, half):
    got = got.cpu().double()
    assert torch.equal(got.isfinite(), want.isfinite())
    assert bool(((got - want).abs() <= half * (bound + want.abs()) + 1e-300)[want.isfinite()].all()), float(((got - want).abs() / (bound + want.abs())).max() / half)


@pytest.mark.parametrize("real", [torch.float32, torch.float64])
@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,n_in,n_out,N,R,order", [
    (1, 64, 64, 1, 1, "shuffled"), (1, 2560, 768, 4, 16, "shuffled"), (5, 33, 17, 3, 5, "shuffled"), (16, 256, 320, 1, 64, "segments"),
    (31, 1000, 999, 40, 8, "shuffled"), (64, 512, 512, 7, 33, "shuffled"), (65, 130, 260, 2, 17, "shuffled"), (200, 192, 1024, 3, 128, "segments"),
    (333, 768, 500, 16, 32, "shuffled"), (77, 96, 129, 64, 256, "shuffled"), (1030, 128, 64, 5, 4, "segments"), (129, 3, 2, 2, 2, "shuffled"),
    (40, 5000, 72, 2, 24, "segments"), (600, 80, 48, 300, 9, "shuffled"), (256, 64, 40, 9, 12, "shuffled"), (257, 64, 40, 9, 12, "shuffled"),
    (1024, 32, 36, 1500, 4, "shuffled"), (1025, 40, 24, 1, 40, "segments"), (2100, 24, 16, 1200, 3, "segments"), (6, 2048, 2048, 1, 64, "segments")])
def test_adapters_of_many_requests(ops, real, low, T, n_in, n_out, N, R, order):
    c = _adapters(T, n_in, n_out, N, R, real, low, T + n_in + R, order)
    print(f"adapters {T} {n_in} {n_out} {N} {R} {order} {real} {low}", flush=True)
    want, bound = P.lora_rows(**c)
    d = {k: v.cuda() for k, v in c.items()}
    got = ops.lora_rows(**d)
    _near(got, want, bound, HALF[real])
    # into base's own memory, the same values
    assert ops.lora_rows(**{**d, "out": d["base"]}) is d["base"] and torch.equal(d["base"], got)
    # without base and scale
    want, bound = P.lora_rows(c["x"], c["a"], c["b"], c["adapter"])
    _near(ops.lora_rows(d["x"], d["a"], d["b"], d["adapter"]), want, bound, HALF[real])


@pytest.mark.parametrize("real", [torch.float32, torch.float64])
@pytest.mark.parametrize("T", [3, 100])
def test_adapters_of_rows_that_lie_apart(ops, real, T):
    """Rows of wider tensors, at addresses that rule out wide loads; neighbours of what is written stay."""
    c = _adapters(T, 70, 45, 3, 12, real, torch.bfloat16, 9)
    want, bound = P.lora_rows(**c)
    wide = {k: torch.full((T, c[k].shape[1] + 9), 7.0, dtype=real).cuda() for k in ("x", "base")}
    d = {k: v.cuda() for k, v in c.items()}
    for k in wide:
        wide[k][:, 3:3 + c[k].shape[1]] = d[k]
        d[k] = wide[k][:, 3:3 + c[k].shape[1]]
    low = torch.zeros(3 * 12 * 70 + 1, dtype=torch.bfloat16).cuda()
    low[1:] = d["a"].flatten()
    d["a"] = low[1:].view(3, 12, 70)
    out = torch.full((T, 60), 5.0, dtype=real).cuda()
    got = ops.lora_rows(**d, out=out[:, 7:52])
    _near(got, want, bound, HALF[real])
    assert bool((out[:, :7] == 5).all()) and bool((out[:, 52:] == 5).all())
    one = c["x"][0].cuda().expand(T, 70)               # one row for all, in one row's memory
    want, bound = P.lora_rows(one.cpu(), c["a"], c["b"], c["adapter"])
    _near(ops.lora_rows(one, d["a"], d["b"], d["adapter"]), want, bound, HALF[real])


@pytest.mark.parametrize("T", [4, 40, 150, 400])
def test_rows_without_an_adapter_and_rows_that_are_not_numbers(ops, T):
    c = _adapters(T, 256, 192, 3, 16, torch.float32, torch.bfloat16, 2)
    c["adapter"][0], c["adapter"][1], c["adapter"][2], c["adapter"][3] = 3, -7, 1, 2 ** 31 - 1
    clean = ops.lora_rows(**{k: v.cuda() for k, v in c.items()})
    c["x"][2, 5], c["x"][0, 3], c["x"][1], c["base"][3, 4] = math.inf, math.nan, math.inf, math.nan
    got = ops.lora_rows(**{k: v.cuda() for k, v in c.items()})
    assert torch.equal(got[:2], c["base"][:2].cuda()) and torch.equal(got[4:], clean[4:])
    assert not bool(got[2].isfinite().any()) and bool(got[3, 4].isnan()) and torch.equal(got[3, 5:], c["base"][3, 5:].cuda())
    nobody = torch.full((T,), -1, dtype=torch.int32).cuda()
    base = torch.randn(T, 192).cuda()
    assert torch.equal(ops.lora_rows(c["x"].cuda(), c["a"].cuda(), c["b"].cuda(), nobody, base=base), base)
    assert not ops.lora_rows(c["x"].cuda(), c["a"].cuda(), c["b"].cuda(), nobody).any()


def test_no_rows_and_no_adapters(ops):
    e = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt).cuda()
    assert ops.lora_rows(e(0, 8), e(2, 4, 8), e(2, 3, 4), e(0, dt=torch.int32)).shape == (0, 3)


def test_adapters_of_rows_past_32_bits(ops):
    """out has more than 2^31 values; the last rows are what a call of them alone gives, to the rounding of its sums."""
    T, n_out = 70000, 32768
    x, a, b = torch.randn(T, 16).cuda(), torch.randn(2, 4, 16).cuda(), torch.randn(2, n_out, 4).cuda()
    adapter = (torch.arange(T, dtype=torch.int32) % 3 - 1).cuda()
    out = ops.lora_rows(x, a, b, adapter)
    for rows in (slice(0, 5), slice(65534, 65540), slice(T - 5, T)):
        want, bound = P.lora_rows(x[rows].cpu(), a.cpu(), b.cpu(), adapter[rows].cpu())
        _near(out[rows], want, bound, HALF[torch.float32])


# ------------------------------------------------------------------ the gated delta rule
def _delta_near(got, want, T, dk, half):
    """Half a step of the value, and what the sums before it may be off: a row's step makes some dk roundings of 2^-24 of the
    largest value, at random, and states do not grow (unit keys, 0 <= beta <= 1), so that after T steps sqrt(T dk) of them have
    added up; four times that."""
    got, there = got.cpu().double(), ~want.isnan()
    off = 4 * math.sqrt((T + 64) * (dk + 64)) * 2.0 ** -24 * float(want[there].abs().max() if there.any() else 0.0)
    assert bool(((got - want).abs()[there] <= half * want.abs()[there] + off).all()), (float((got - want).abs()[there].max()), off)


def _delta(ops, c, starts, scale=None, half=None, **kw):
    q, k, v, g, beta, state = c
    T, dk, dtype = q.shape[0], q.shape[2], q.dtype
    want, after = P.delta_rule(*c, starts, dk ** -0.5 if scale is None else scale)
    d = [t.cuda() for t in c]
    out = torch.full(v.shape, 3.0, dtype=dtype).cuda()
    got = ops.delta_rule(*d, starts=torch.tensor(starts, dtype=torch.int32).cuda(), scale=scale, out=out, **kw)
    assert got is out
    longest = max(b - a for a, b in zip(starts, starts[1:]))
    _delta_near(got, want, longest, dk, HALF[dtype])
    _delta_near(d[5], after, longest, dk, HALF[torch.float32])
    assert bool((got.cpu()[want.isnan()] == 3).all())
    return got, d[5]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,Hv,dk,dv,starts", [
    (1, 1, 16, 16, [0, 1]), (2, 4, 64, 64, [0, 1, 2, 3, 4]), (3, 3, 33, 17, [0, 2, 2, 9]), (2, 2, 128, 128, [0, 64, 65, 200]),
    (1, 4, 256, 100, [0, 130, 131]), (5, 5, 64, 64, [0, 300]), (2, 6, 96, 32, [3, 70, 70, 75, 333]), (1, 1, 1, 1, [0, 70]),
    (1, 2, 200, 256, [0, 63, 127, 192]), (40, 40, 64, 64, [0, 5, 10, 15, 16]), (1, 1, 128, 65, [0, 1000]), (2, 2, 20, 24, [0, 17, 97])])
def test_delta_rule(ops, dtype, Hk, Hv, dk, dv, starts):
    print(f"delta rule {Hk} {Hv} {dk} {dv} {starts} {dtype}", flush=True)
    _delta(ops, P.delta_inputs(starts[-1] + 5, len(starts) - 1, Hk, Hv, dk, dv, dtype, sum(starts) + dk), starts)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hk,Hv,dk,dv,starts", [(1, 2, 64, 64, [0, 2500]), (1, 1, 33, 70, [0, 60, 2600]), (2, 4, 128, 128, [0, 1300]), (1, 1, 256, 24, [0, 1100]),
                                                (1, 1, 20, 8, [5, 5, 70, 71, 5000]), (1, 3, 96, 200, [0, 1030, 2060])])
def test_delta_rule_of_long_sequences(ops, dtype, Hk, Hv, dk, dv, starts):
    """Few heads and long sequences: cut into segments, one sequence of a single segment among them."""
    print(f"delta rule {Hk} {Hv} {dk} {dv} {starts} {dtype}", flush=True)
    _delta(ops, P.delta_inputs(starts[-1] + 3, len(starts) - 1, Hk, Hv, dk, dv, dtype, sum(starts) + dk, rate=-6.0), starts)


@pytest.mark.parametrize("T,B", [(4, 4), (6, 2), (200, 2), (129, 1), (1600, 2)])
def test_delta_rule_without_starts(ops, T, B):
    c = P.delta_inputs(T, B, 2, 2, 64, 48, torch.float32, T)
    want, after = P.delta_rule(*c, [T // B * i for i in range(B + 1)], 0.25)
    d = [t.cuda() for t in c]
    got = ops.delta_rule(*d, scale=0.25)
    _delta_near(got, want, T // B, 64, HALF[torch.float32])
    _delta_near(d[5], after, T // B, 64, HALF[torch.float32])


@pytest.mark.parametrize("n", [5, 150])
def test_delta_rule_on_parts_of_one_projection(ops, n):
    """q, k, v as columns of one matrix, at addresses that rule out wide loads."""
    Hk, Hv, dk, dv = 2, 4, 64, 32
    q, k, v, g, beta, state = P.delta_inputs(n, 1, Hk, Hv, dk, dv, torch.bfloat16, n)
    wide = torch.zeros(n, 1 + 2 * Hk * dk + Hv * dv + 2, dtype=torch.bfloat16).cuda()
    at, views = 1, []
    for t in (q, k, v):
        w = t[0].numel()
        wide[:, at:at + w] = t.flatten(1).cuda()
        views.append(wide[:, at:at + w].view(n, *t.shape[1:]))
        at += w
    want, after = P.delta_rule(q, k, v, g, beta, state, [0, n], dk ** -0.5)
    s = state.cuda()
    _delta_near(ops.delta_rule(*views, g.cuda(), beta.cuda(), s), want, n, dk, HALF[torch.bfloat16])
    _delta_near(s, after, n, dk, HALF[torch.float32])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", ["no decay", "decays of all sizes", "all forgotten", "nothing learnt", "one key", "one key, learnt whole", "no keys", "keys by turns"])
def test_delta_rule_at_the_edges(ops, dtype, case):
    """Decays of 0 and e^-infinity, beta of 0 and 1, keys that are all the same or nothing."""
    starts = [0, 7, 200, 333]
    q, k, v, g, beta, state = P.delta_inputs(333, 3, 2, 2, 64, 64, dtype, 5)
    if case == "no decay":
        g.zero_()
    elif case == "decays of all sizes":
        g = -torch.exp(torch.rand(g.shape, generator=torch.Generator().manual_seed(1)) * 20 - 13)
    elif case == "all forgotten":
        g[::5] = -math.inf
        g[3::50] = -3e38
    elif case == "nothing learnt":
        beta.zero_()
    elif case == "one key":
        k[:] = k[:1]
        g.zero_()
    elif case == "one key, learnt whole":
        k[:] = k[:1]
        g.zero_()
        beta.fill_(1.0)
    elif case == "no keys":
        k.zero_()
    else:
        k[1::2] = -k[:-1:2]
        beta.fill_(1.0)
    _delta(ops, (q, k, v, g, beta, state), starts)


@pytest.mark.parametrize("long", [False, True])
def test_starts_that_name_rows_there_are_not(ops, long):
    """Cut to the rows there are: before the first, behind the last."""
    c = P.delta_inputs(150 if long else 12, 4, 1, 1, 32, 32, torch.float32, 3)
    _delta(ops, c, [-50, 100, 100, 140, 99999] if long else [-5, 3, 3, 9, 99999])


def test_delta_rule_in_parts_is_the_whole(ops):
    """A prompt in three calls with the state handed on; single steps after it."""
    c = [t.cuda() for t in P.delta_inputs(420, 1, 2, 4, 64, 80, torch.float32, 8)]
    state = c[5].clone()
    whole = ops.delta_rule(*c[:5], state)
    part = c[5].clone()
    got = torch.cat([ops.delta_rule(*(t[a:b].contiguous() for t in c[:5]), part) for a, b in [(0, 100), (100, 101), (101, 400)] + [(i, i + 1) for i in range(400, 420)]])
    _delta_near(got, whole.double().cpu(), 420, 64, HALF[torch.float32])
    _delta_near(part, state.double().cpu(), 420, 64, HALF[torch.float32])


def test_delta_rule_of_rows_past_32_bits(ops):
    """v and o have more than 2^31 values: the sequences at the end are what a call of them alone gives."""
    Hk, Hv, dk, dv = 1, 32, 16, 128
    n = [524288, 300, 1, 40]
    starts = [0]
    for i in n:
        starts.append(starts[-1] + i)
    T = starts[-1]
    g = torch.Generator(device="cuda").manual_seed(1)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")
    q, k, v = unit(f(T, Hk, dk)).bfloat16(), unit(f(T, Hk, dk)).bfloat16(), torch.empty(T, Hv, dv, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    decay, beta, state = -f(T, Hv).abs() * 0.1, torch.sigmoid(f(T, Hv)), f(len(n), Hv, dk, dv)
    own, at = state[1:].clone(), starts[1]
    o = ops.delta_rule(q, k, v, decay, beta, state, starts=torch.tensor(starts, dtype=torch.int32).cuda())
    want, after = P.delta_rule(*(t[at:].cpu() for t in (q, k, v, decay, beta)), own.cpu(), [s - at for s in starts[1:]], dk ** -0.5)
    _delta_near(o[at:], want, 300, dk, HALF[torch.bfloat16])
    _delta_near(state[1:], after, 300, dk, HALF[torch.float32])


# ------------------------------------------------------------------ verification of drafts
def _verify(ops, logits, drafts, u, **kw):
    want = P.verify_drafts(logits, drafts, u, **kw)
    got = ops.verify_drafts(logits.cuda(), drafts.cuda(), u.cuda(), **{k: _cuda(v) for k, v in kw.items()})
    assert torch.equal(got[0].cpu(), want[0]), (got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu(), want[1])
    return want


@pytest.mark.parametrize("real", [torch.float64, torch.float32])
@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (1, 4, 50277), (3, 2, 5), (9, 5, 1000), (2, 64, 777), (40, 3, 4097), (5, 8, 65536), (130, 1, 63), (1, 1, 200001), (150, 13, 9000), (2, 2, 300000)])
def test_drafts_by_sampling(ops, real, B, K, V):
    print(f"verify {B} {K} {V} {real}", flush=True)
    g = torch.Generator().manual_seed(V)
    logits, drafts, u, draft = P.verify_inputs(B, K, V, real, B + K + V)
    lengths = torch.randint(-1, K + 3, (B,), generator=g, dtype=torch.int32)
    for temp in (1.0, 0.3, 5.0):
        _verify(ops, logits, drafts, u, draft_logits=draft, temp=temp)
    _verify(ops, logits, drafts, u, draft_logits=draft, lengths=lengths, temp=0.8)
    _verify(ops, logits, drafts, u, lengths=lengths)
    likely = torch.where(torch.rand(drafts.shape, generator=g) < 0.8, logits[:, :K].argmax(-1), drafts)
    _verify(ops, logits, likely, u, greedy=True)
    _verify(ops, logits, likely, u, lengths=lengths, greedy=True)


@pytest.mark.parametrize("real", [torch.float64, torch.float32])
def test_drafts_at_the_edges(ops, real):
    """Rows with no weight at all, +infinity, NaN, ties; drafts that are no tokens; random numbers of 0, next to 1, and outside."""
    B, K, V = 14, 3, 700
    logits, drafts, u, draft = P.verify_inputs(B, K, V, real, 4)
    logits[0] = -math.inf
    logits[1, 1] = -math.inf
    logits[2, 0, 5] = logits[2, 0, 9] = math.inf
    drafts[2, 0] = 9
    logits[3, :, ::2] = math.nan
    logits[4] = math.nan
    draft[5, 0] = -math.inf
    draft[6, :, 7] = math.inf
    drafts[6] = 7
    drafts[7, 0], drafts[8, 1], drafts[9, 2] = -1, V, 2 ** 40
    logits[10] = 0.0
    drafts[10] = 0
    u[11], u[12] = 0.0, 1.0 - 2.0 ** -24
    draft[13] = logits[13, :K]                        # the same distribution: accepted whatever u is
    accepted = _verify(ops, logits, drafts, u, draft_logits=draft)[1]
    assert int(accepted[13]) == K and int(accepted[7]) == 0 and int(accepted[0]) == 0
    _verify(ops, logits, drafts, u)
    _verify(ops, logits, drafts, u, greedy=True)
    u[11], u[12] = -1.0, 2.0
    _verify(ops, logits, drafts, u, draft_logits=draft)


@pytest.mark.parametrize("V", [9, 5000, 270000])
def test_nothing_left_of_the_distribution(ops, V):
    """Target and drafter agree to the last bit and the random number refuses all the same (it is 1): the token is drawn from p."""
    logits, drafts, u, draft = P.verify_inputs(5, 2, V, torch.float64, V)
    draft = logits[:, :2].clone()
    u[:, :2] = 1.0
    tokens = _verify(ops, logits, drafts, u, draft_logits=draft)[0]
    assert bool((tokens[:, 0] >= 0).all()) and bool((tokens[:, 1:] == -1).all())


@pytest.mark.parametrize("greedy", [False, True])
def test_logits_of_one_step_after_the_other(ops, greedy):
    """Logits as a model gives them, [V] more than the vocabulary wide and step by step: a view whose sequences lie closer than its rows."""
    B, K, V = 6, 3, 301
    logits, drafts, u, draft = P.verify_inputs(B, K, V, torch.float64, 11)
    want = P.verify_drafts(logits, drafts, u, draft_logits=draft, greedy=greedy)
    steps, d = torch.full((K + 1, B, V + 3), math.inf, dtype=torch.float64).cuda(), torch.full((K, B, V + 3), math.inf, dtype=torch.float64).cuda()
    steps[..., 1:V + 1], d[..., 1:V + 1] = logits.transpose(0, 1), draft.transpose(0, 1)
    got = ops.verify_drafts(steps[..., 1:V + 1].transpose(0, 1), drafts.cuda(), u.cuda(), draft_logits=d[..., 1:V + 1].transpose(0, 1), greedy=greedy)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_logits_past_32_bits(ops):
    """More than 2^31 logits; the last sequences are what a call of them alone gives."""
    B, K, V = 700, 1, 1600000
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.empty(B, K + 1, V, device="cuda").normal_(generator=g)
    drafts, u = torch.randint(0, V, (B, K), generator=g, device="cuda"), torch.rand(B, K + 1, generator=g, device="cuda")
    tokens, accepted = ops.verify_drafts(logits, drafts, u, temp=0.2)
    for rows in (slice(0, 2), slice(B - 2, B)):
        want = P.verify_drafts(logits[rows].cpu(), drafts[rows].cpu(), u[rows].cpu(), temp=0.2)
        assert torch.equal(tokens[rows].cpu(), want[0]) and torch.equal(accepted[rows].cpu(), want[1])


def test_tokens_follow_the_target_distribution(ops):
    """Whatever the drafter, the first token of a sequence is distributed as the target's: 200000 sequences over 8 tokens; a count of
    n p is off by more than 6 sqrt(n p (1 - p)) once in 10^9."""
    n, V = 200000, 8
    g = torch.Generator(device="cuda").manual_seed(6)
    p, q = torch.randn(V, generator=g, device="cuda").double(), torch.randn(V, generator=g, device="cuda").double()
    drafts = torch.multinomial(torch.softmax(q, 0), n, replacement=True, generator=g).view(n, 1)
    u = torch.rand(n, 2, generator=g, device="cuda")
    tokens, _ = ops.verify_drafts(p.expand(n, 2, V), drafts, u, draft_logits=q.expand(n, 1, V))
    want = torch.softmax(p, 0)
    count = torch.bincount(tokens[:, 0], minlength=V).double()
    assert bool(((count - n * want).abs() <= 6 * (n * want * (1 - want)).sqrt()).all())


@pytest.mark.parametrize("temp", [1e-310, 5e-324])
def test_hardly_any_temperature_is_none(ops, temp):
    """All weight on the first maximum: a temperature whose reciprocal overflows gives the greedy choice."""
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(4, 3, 700, generator=g, dtype=torch.float64)
    drafts = logits[:, :2].argmax(-1)
    drafts[1, 0] = (drafts[1, 0] + 1) % 700
    u = torch.rand(4, 3, generator=g)
    want = ops.verify_drafts(logits.cuda(), drafts.cuda(), greedy=True)
    got = ops.verify_drafts(logits.cuda(), drafts.cuda(), u.cuda(), temp=temp)
    assert all(torch.equal(a, b) for a, b in zip(got, want)), (got, want)


@pytest.mark.parametrize("T", [63, 64, 65, 127, 128, 129])
def test_adapters_where_tiles_are_found_another_way(ops, T):
    c = _adapters(T, 70, 50, 3, 5, torch.float32, torch.float16, T)
    c["adapter"][::7] = -1
    want, bound = P.lora_rows(**c)
    _near(ops.lora_rows(**{k: v.cuda() for k, v in c.items()}), want, bound, HALF[torch.float32])


@pytest.mark.parametrize("B", [64, 65])
def test_delta_rule_of_many_ragged_sequences_in_chunks(ops, B):
    """The longest begun first, up to a wavefront's number of sequences: equal ones, empty ones, the longest last."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 60, (B,), generator=g)
    lens[:5], lens[9], lens[-1] = 0, 0, 60 * B
    starts = [0] + lens.cumsum(0).tolist()
    assert starts[-1] >= 64 * B
    _delta(ops, P.delta_inputs(starts[-1], B, 1, 2, 16, 24, torch.float32, B, rate=-3.0), starts)
