"""Serving operators beside the quantised products, the recurrence and the sampler, as cases that can be timed and compared.

Kinds of case (the key ``"kind"``):

``adapters``  ``ops.lora_rows``: the low-rank adapters of many requests added to the result of a projection that they share.
``delta``     ``ops.delta_rule``: the gated delta rule over packed sequences, its state updated in place.
``verify``    ``ops.verify_drafts``: drafted tokens held against the target's logits.

With ``own`` false ``run`` computes the same in elementary torch operations; with ``own`` true it calls the framework.
"""
from __future__ import annotations

import math
import random

import torch

own = False

VOCAB = 50277
WIDTHS = (512, 768, 1024, 1536, 2048, 2560, 4096, 5120)
TYPES = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64


def listed():
    return [
        # One request on the smallest model of the family: one row, a small adapter; launches and latency decide.
        dict(name="adapters-one", kind="adapters", rows=1, n_in=768, n_out=768, rank=16, adapters=4, type="bf16", real="f32", order="segments"),
        # One token for each of 32 requests beside the 3B shape's ffn key, float64 as the batched product returns it.
        dict(name="adapters-batch", kind="adapters", rows=32, n_in=2560, n_out=10240, rank=64, adapters=24, type="bf16", real="f64", order="shuffled"),
        # The prompts of a few requests, packed, beside a square matrix of the 3B shape.
        dict(name="adapters-prompts", kind="adapters", rows=1024, n_in=2560, n_out=2560, rank=32, adapters=5, type="f16", real="f64", order="segments"),
        # The largest shape's ffn key for a full pass of short requests in any order.
        dict(name="adapters-wide", kind="adapters", rows=2048, n_in=5120, n_out=20480, rank=128, adapters=8, type="bf16", real="f32", order="shuffled"),
        # One token for each of 32 requests: the state is read and written once, nothing else weighs.
        dict(name="delta-tokens", kind="delta", seqs=32, rows=32, key_heads=40, value_heads=40, dk=64, dv=64, type="f32", lengths="even"),
        # A handful of drafted tokens for each of 16 requests, heads of keys shared by two heads of values.
        dict(name="delta-drafts", kind="delta", seqs=16, rows=80, key_heads=16, value_heads=32, dk=128, dv=128, type="bf16", lengths="ragged"),
        # A whole prompt of one request in the framework's own type.
        dict(name="delta-prompt", kind="delta", seqs=1, rows=1024, key_heads=40, value_heads=40, dk=64, dv=64, type="f32", lengths="even"),
        # Prompts of different lengths packed into one pass.
        dict(name="delta-packed", kind="delta", seqs=7, rows=8192, key_heads=8, value_heads=32, dk=128, dv=128, type="bf16", lengths="ragged"),
        # Four drafted tokens of one request: a few rows of logits, latency decides.
        dict(name="verify-one", kind="verify", seqs=1, drafts=4, vocab=VOCAB, real="f64", source="model", pick="sample"),
        # The same for 16 requests, some with fewer drafts.
        dict(name="verify-batch", kind="verify", seqs=16, drafts=4, vocab=VOCAB, real="f64", source="model", pick="sample"),
        # Drafts looked up in the text (no distribution of their own), longer, the most likely token wanted.
        dict(name="verify-lookup", kind="verify", seqs=32, drafts=7, vocab=VOCAB, real="f32", source="lookup", pick="greedy"),
        # Many requests with long drafts over a larger vocabulary.
        dict(name="verify-many", kind="verify", seqs=64, drafts=8, vocab=65536, real="f32", source="model", pick="sample"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("adapters", "delta", "verify"))
    case = dict(kind=kind)
    if kind == "adapters":
        n_in = rng.choice(WIDTHS) if rng.random() < 0.7 else _log(rng, 64, 5120)
        n_out = rng.choice((1, 1, 4)) * rng.choice(WIDTHS) if rng.random() < 0.7 else _log(rng, 64, 20480)
        case.update(rows=_log(rng, 1, 2048), n_in=n_in, n_out=n_out, rank=rng.choice((4, 8, 16, 32, 64, 128, _log(rng, 1, 128))),
                    adapters=_log(rng, 1, 32), type=rng.choice(("bf16", "f16", "f32")), real=rng.choice(("f32", "f64")),
                    order=rng.choice(("segments", "shuffled")))
    elif kind == "delta":
        case["lengths"] = rng.choice(("even", "ragged"))
        case["seqs"] = _log(rng, 1, 32)
        case["rows"] = case["seqs"] * _log(rng, 1, 8) if rng.random() < 0.4 else max(case["seqs"], _log(rng, 16, 8192))
        case["key_heads"] = rng.randint(1, 16)
        case["value_heads"] = case["key_heads"] * rng.choice((1, 1, 2, 4))
        case["dk"] = rng.choice((32, 64, 64, 96, 128, 128, 200, 256, rng.randint(16, 128)))
        case["dv"] = rng.choice((32, 64, 64, 96, 128, 128, 256, rng.randint(16, 128)))
        case["type"] = rng.choice(("f32", "bf16", "f16"))
        # (no more than the largest listed one's work, and 128 MB of state)
        head = case["value_heads"] * case["dk"] * case["dv"]
        case["seqs"] = max(1, min(case["seqs"], (1 << 25) // head))
        case["rows"] = max(case["seqs"], min(case["rows"], 8192 * 32 * 128 * 128 // head))
    else:
        case.update(seqs=_log(rng, 1, 64), drafts=rng.randint(0, 8), vocab=VOCAB if rng.random() < 0.6 else _log(rng, 300, 65536),
                    real=rng.choice(("f32", "f64")), source=rng.choice(("model", "model", "lookup")), pick=rng.choice(("sample", "sample", "greedy")))
    return case


# ---------------------------------------------------------------- inputs
class _State:
    pass


def _lengths(total, seqs, ragged, rng):
    """``seqs`` lengths that add up to ``total``; ragged ones spread over a wide range, some empty."""
    if not ragged:
        return [total // seqs + (i < total % seqs) for i in range(seqs)]
    cuts = sorted(rng.randint(0, total) for _ in range(seqs - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def prepare(case, seed):
    s = _State()
    s.case, kind = case, case["kind"]
    host = random.Random(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 17)
    randn = lambda *shape, scale=1.0, dtype=torch.float32: (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)
    rand = lambda *shape, dtype=torch.float32: torch.rand(*shape, generator=g, device="cuda", dtype=dtype)
    if kind == "adapters":
        T, N, R, n_in, n_out = case["rows"], case["adapters"], case["rank"], case["n_in"], case["n_out"]
        real, low = TYPES[case["real"]], TYPES[case["type"]]
        s.x, s.base = randn(T, n_in, dtype=real), randn(T, n_out, dtype=real)
        s.a, s.b = randn(N, R, n_in, scale=n_in ** -0.5, dtype=low), randn(N, n_out, R, scale=R ** -0.5, dtype=low)
        s.scale = 0.5 + rand(N)
        # one row in eight or so is of a request without an adapter
        if case["order"] == "segments":
            lens = _lengths(T, min(T, N + 1 + T // 256), True, host)
            of = [host.randrange(-1 if host.random() < 0.5 else 0, N) for _ in lens]
            rows = [i for i, n in zip(of, lens) for _ in range(n)]
        else:
            rows = [-1 if T > 1 and host.random() < 0.125 else host.randrange(N) for _ in range(T)]
        if all(i < 0 for i in rows):
            rows[-1] = host.randrange(N)
        s.adapter = torch.tensor(rows, dtype=torch.int32).cuda()
    elif kind == "delta":
        T, B, Hk, Hv, dk, dv = (case[k] for k in ("rows", "seqs", "key_heads", "value_heads", "dk", "dv"))
        low = TYPES[case["type"]]
        unit = lambda t: t / t.norm(dim=-1, keepdim=True)
        s.q, s.k, s.v = unit(randn(T, Hk, dk)).to(low), unit(randn(T, Hk, dk)).to(low), randn(T, Hv, dv, dtype=low)
        # decays of a step from almost none to a factor of a few, as exp(log rate) * softplus(input) gives them
        s.g = -torch.exp(randn(Hv) - 2.0) * torch.nn.functional.softplus(randn(T, Hv))
        s.beta = torch.sigmoid(randn(T, Hv))
        s.state = randn(B, Hv, dk, dv, scale=0.3)
        s.lens = _lengths(T, B, case["lengths"] == "ragged", host)
        starts = [0]
        for n in s.lens:
            starts.append(starts[-1] + n)
        s.starts = torch.tensor(starts, dtype=torch.int32).cuda()
        s.scale = dk ** -0.5
    else:
        B, K, V = case["seqs"], case["drafts"], case["vocab"]
        real = TYPES[case["real"]]
        # a few likely tokens over a long tail; one token in fifty is banned (-inf)
        logits = randn(B, K + 1, V, scale=2.0) + 6.0 * (rand(B, K + 1, V) < 20.0 / V)
        logits.masked_fill_(rand(1, 1, V) < 0.02, -math.inf)
        s.logits = logits.to(real)
        s.temp = 0.8
        s.drafts = torch.zeros(B, K, dtype=torch.int64, device="cuda")
        s.draft_logits = None
        if K and case["source"] == "model":
            s.draft_logits = (logits[:, :K] + randn(B, K, V, scale=0.7)).to(real)
            s.drafts = torch.multinomial(torch.softmax(s.draft_logits.float() / s.temp, -1).view(B * K, V), 1, generator=g).view(B, K)
        elif K:
            s.drafts = torch.where(rand(B, K) < 0.7, logits[:, :K].argmax(-1), torch.randint(0, V, (B, K), generator=g, device="cuda"))
        s.lengths = torch.tensor([K if host.random() < 0.7 else host.randint(0, K) for _ in range(B)], dtype=torch.int32).cuda()
        s.u = rand(B, K + 1)
        s.greedy = case["pick"] == "greedy"
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    kind = s.case["kind"]
    if own:
        from rwkvstic_amd import ops

        if kind == "adapters":
            return ops.lora_rows(s.x, s.a, s.b, s.adapter, s.scale, base=s.base)
        if kind == "delta":
            return [ops.delta_rule(s.q, s.k, s.v, s.g, s.beta, s.state, starts=s.starts, scale=s.scale), s.state]
        return list(ops.verify_drafts(s.logits, s.drafts, s.u, draft_logits=s.draft_logits, lengths=s.lengths, temp=s.temp, greedy=s.greedy))
    if kind == "adapters":
        return _adapters(s)
    if kind == "delta":
        return _delta(s)
    return _verify(s)


def _adapters(s):
    """Few rows: the adapters gathered row by row; many: all adapters for all rows, each row's own kept."""
    real, (N, R, n_in), T = s.x.dtype, s.a.shape, s.x.shape[0]
    i = s.adapter.long().clamp(0, N - 1)
    scale = torch.where(s.adapter >= 0, s.scale[i], 0.0).to(real)
    if T <= 64:
        h = torch.bmm(s.a[i].to(real), s.x.unsqueeze(2)) * scale.view(T, 1, 1)
        return s.base + torch.bmm(s.b[i].to(real), h).squeeze(2)
    every = (s.x @ s.a.to(real).view(N * R, n_in).t()).view(T, N, R)
    kept = torch.zeros_like(every)
    rows = torch.arange(T, device=s.x.device)
    kept[rows, i] = every[rows, i] * scale.unsqueeze(1)
    return s.base + kept.view(T, N * R) @ s.b.to(real).transpose(1, 2).reshape(N * R, -1)


def _delta(s):
    """Chunks of 64 rows: what is within a chunk for all chunks at once, the state from chunk to chunk."""
    (T, Hv, dv), dk, B = s.v.shape, s.q.shape[2], len(s.lens)
    C = min(CHUNK, max(s.lens))
    n = -(-max(s.lens) // C)
    at = torch.arange(n * C, device=s.v.device)
    starts = s.starts.long()
    there = at < (starts[1:] - starts[:-1]).unsqueeze(1)                                    # [B, n * C]
    row = torch.where(there, starts[:-1].unsqueeze(1) + at, 0)
    mask = there.view(B, n * C, 1)
    pad = lambda t: torch.where(mask.unsqueeze(-1), t[row].float(), 0.0).view(B, n, C, t.shape[1], -1).transpose(2, 3)    # [B, n, H, C, d]
    share = lambda t: t.repeat_interleave(Hv // t.shape[2], dim=2)
    q, k, v = share(pad(s.q)) * s.scale, share(pad(s.k)), pad(s.v)
    g = torch.where(mask, s.g[row], 0.0).double().view(B, n, C, Hv).transpose(2, 3).cumsum(-1)  # [B, n, H, C]
    beta = torch.where(mask, s.beta[row], 0.0).view(B, n, C, Hv).transpose(2, 3).unsqueeze(-1)
    decay = torch.exp(torch.clamp(g.unsqueeze(-1) - g.unsqueeze(-2), max=0.0).float()).tril()
    m = -(beta * decay * (k @ k.transpose(-1, -2))).tril(-1)
    inverse = torch.eye(C, device=v.device) + m
    width = 2
    while width < C:                                                                        # (1 + m)(1 + m^2)(1 + m^4)...
        m = m @ m
        inverse = inverse + inverse @ m
        width *= 2
    within = decay * (q @ k.transpose(-1, -2))
    e = torch.exp(g.float()).unsqueeze(-1)
    u, w = inverse @ (beta * v), inverse @ (beta * e * k)
    qe, last = q * e, torch.exp(g[..., -1].float()).unsqueeze(-1).unsqueeze(-1)
    kt = (k * torch.exp((g[..., -1:] - g).float()).unsqueeze(-1)).transpose(-1, -2).contiguous()
    state, out = s.state, torch.empty_like(v)
    for c in range(n):
        new = u[:, c] - w[:, c] @ state
        out[:, c] = qe[:, c] @ state + within[:, c] @ new
        state = last[:, c] * state + kt[:, c] @ new
    s.state.copy_(state)
    return [out.transpose(2, 3).reshape(B, n * C, Hv, dv)[there].to(s.v.dtype), s.state]


def _verify(s):
    (B, K1, V), K = s.logits.shape, s.drafts.shape[1]
    at = torch.arange(K, device=s.u.device)
    counted = at < s.lengths.unsqueeze(1)
    rows = torch.arange(B, device=s.u.device)
    if s.greedy:
        best = s.logits.argmax(-1)
        accepted = ((best[:, :K] == s.drafts) & counted).long().cumprod(1).sum(1)
        drawn = best[rows, accepted]
    else:
        p = torch.softmax(s.logits.double() / s.temp, -1)
        q = torch.zeros_like(p)
        if s.draft_logits is not None:
            q[:, :K] = torch.softmax(s.draft_logits.double() / s.temp, -1)
        else:
            q[:, :K].scatter_(2, s.drafts.unsqueeze(2), 1.0)
        of = lambda t: t[:, :K].gather(2, s.drafts.unsqueeze(2)).squeeze(2)
        accepted = ((s.u[:, :K].double() * of(q) < of(p)) & counted).long().cumprod(1).sum(1)
        p = p[rows, accepted]
        left = torch.where((accepted < s.lengths).unsqueeze(1), (p - q[rows, accepted]).clamp(min=0.0), p)
        left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
        running = left.cumsum(1)
        drawn = torch.searchsorted(running, s.u[:, K:].double() * running[:, -1:], right=True).squeeze(1).clamp(max=V - 1)
    at = torch.arange(K1, device=s.u.device)
    tokens = torch.where(at < accepted.unsqueeze(1), torch.nn.functional.pad(s.drafts, (0, 1)), -1)
    return [torch.where(at == accepted.unsqueeze(1), drawn.unsqueeze(1), tokens), accepted]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}
    if case["kind"] == "adapters":
        T, N, R, n_in, n_out = case["rows"], case["adapters"], case["rank"], case["n_in"], case["n_out"]
        used = min(N, T)
        return {"bytes": T * (n_in + 2 * n_out) * size[case["real"]] + used * R * (n_in + n_out) * size[case["type"]] + 4 * T,
                "flops": 2 * T * R * (n_in + n_out)}
    if case["kind"] == "delta":
        T, B, Hk, Hv, dk, dv = (case[k] for k in ("rows", "seqs", "key_heads", "value_heads", "dk", "dv"))
        return {"bytes": T * (2 * Hk * dk + 2 * Hv * dv) * size[case["type"]] + 8 * T * Hv + 8 * B * Hv * dk * dv, "flops": 7 * T * Hv * dk * dv}
    B, K, V = case["seqs"], case["drafts"], case["vocab"]
    with_drafts = K if case["source"] == "model" and case["pick"] == "sample" else 0
    return {"bytes": B * (K + 1 + with_drafts) * V * size[case["real"]] + 24 * B * (K + 1), "flops": 4 * B * (K + 1 + with_drafts) * V}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adapters":
        out = s.base.double().clone()
        for i in set(s.adapter.tolist()) - {-1}:
            rows = s.adapter == i
            out[rows] += s.scale[i].double() * (s.x[rows].double() @ s.a[i].double().t() @ s.b[i].double().t())
        return out
    if case["kind"] == "delta":
        (T, Hv, dv), Hk = s.v.shape, s.q.shape[1]
        out, state = torch.zeros(T, Hv, dv, dtype=torch.float64, device="cuda"), s.state.double().clone()
        head = torch.arange(Hv, device="cuda") // (Hv // Hk)
        lens = torch.tensor(s.lens, device="cuda")
        for t in range(max(s.lens)):
            live = (lens > t).nonzero().squeeze(1)
            row = s.starts.long()[live] + t
            q, k, v = s.q[row][:, head].double(), s.k[row][:, head].double(), s.v[row].double()
            S = state[live] * s.g[row].double().exp()[..., None, None]
            u = s.beta[row].double()[..., None] * (v - (S * k[..., None]).sum(2))
            S = S + k[..., None] * u[..., None, :]
            state[live] = S
            out[row] = s.scale * (S * q[..., None]).sum(2)
        return [out, state]
    B, K = s.drafts.shape
    tokens, counts = torch.full((B, K + 1), -1, dtype=torch.int64), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        drafts, u, count = s.drafts[b].tolist(), s.u[b].double().tolist(), int(s.lengths[b])
        n, left = 0, None
        while True:
            x = s.logits[b, n].double()
            p = torch.exp(x / s.temp - torch.logsumexp(x / s.temp, 0))
            if n == count:
                left = p
                break
            if s.greedy:
                taken = int(torch.nonzero(x == x.max())[0]) == drafts[n]
            else:
                q = torch.zeros_like(p)
                if s.draft_logits is None:
                    q[drafts[n]] = 1.0
                else:
                    y = s.draft_logits[b, n].double() / s.temp
                    q = torch.exp(y - torch.logsumexp(y, 0))
                taken = u[n] * float(q[drafts[n]]) < float(p[drafts[n]])
                left = torch.relu(p - q)
            if not taken:
                break
            n += 1
        if s.greedy:
            last = int(torch.nonzero(x == x.max())[0])
        else:
            running = torch.cumsum(left, 0)
            last = int(torch.nonzero(running > u[K] * float(running[-1]))[0])
        tokens[b, :n], tokens[b, n], counts[b] = torch.tensor(drafts[:n], dtype=torch.int64), last, n
    return [tokens, counts]
