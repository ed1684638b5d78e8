"""The serving operators from their definitions, in float64 on the CPU, and the inputs their tests share."""
import math

import torch


def lora_rows(x, a, b, adapter, scale=None, base=None):
    """The result, and a bound on the error of sums in any order, in units of half a step of the sums' type: each of the n_in + R terms
    behind a value goes through at most n_in + R roundings, the scale and the addition to base are three more."""
    x, a, b = x.double(), a.double(), b.double()
    (T, n_in), (N, R, _), n_out = x.shape, a.shape, b.shape[1]
    out = base.double().clone() if base is not None else torch.zeros(T, n_out, dtype=torch.float64)
    off = out.abs()
    for t, i in enumerate(adapter.tolist()):
        if 0 <= i < N:
            s = float(scale[i]) if scale is not None else 1.0
            out[t] += s * (b[i] @ (a[i] @ x[t]))
            off[t] += (n_in + R + 3) * abs(s) * (b[i].abs() @ (a[i].abs() @ x[t].abs()))
    return out, off


def delta_rule(q, k, v, g, beta, state, starts, scale):
    """Outputs (NaN in rows of no sequence) and the states after the last rows."""
    (T, Hv, dv), Hk = v.shape, q.shape[1]
    of = torch.arange(Hv) // (Hv // Hk)
    q, k, v, g, beta, state = q.double()[:, of], k.double()[:, of], v.double(), g.double(), beta.double(), state.double().clone()
    out = torch.full((T, Hv, dv), math.nan, dtype=torch.float64)
    for n in range(len(starts) - 1):
        S = state[n]
        for t in range(max(0, min(starts[n], T)), max(0, min(starts[n + 1], T))):
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
            S = S + k[t][:, :, None] * u[:, None, :]
            out[t] = scale * (S * q[t][:, :, None]).sum(1)
        state[n] = S
    return out, state


def delta_inputs(T, B, Hk, Hv, dk, dv, dtype, seed, rate=-2.0):
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True).clamp(min=1e-20)
    return (unit(f(T, Hk, dk)).to(dtype), unit(f(T, Hk, dk)).to(dtype), f(T, Hv, dv).to(dtype),
            -torch.exp(f(Hv) + rate) * torch.nn.functional.softplus(f(T, Hv)), torch.sigmoid(f(T, Hv)), f(B, Hv, dk, dv) * 0.3)


def softmax(x, temp):
    """Weights of float64 logits: none for -infinity and NaN, all of it for +infinity; None where there are none."""
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.max()
    if top == -math.inf:
        return None
    w = torch.where(x == top, 1.0, torch.exp((x - top) / temp).nan_to_num(0.0))
    return w / w.sum()


def verify_drafts(logits, drafts, u, draft_logits=None, lengths=None, temp=1.0, greedy=False):
    (B, K1, V), K = logits.shape, drafts.shape[1]
    tokens, accepted = torch.full((B, K1), -1), torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        count, n, drawn = K if lengths is None else max(0, min(K, int(lengths[b]))), 0, -1
        while True:
            x, d = logits[b, n].double(), int(drafts[b, n]) if n < count else -1
            known = 0 <= d < V
            if greedy:
                x = torch.where(x.isnan(), -math.inf, x)
                drawn = int((x == x.max()).nonzero()[0]) if x.max() > -math.inf else -1
                taken = known and d == drawn
            else:
                p = softmax(x, temp)
                q = torch.zeros(V, dtype=torch.float64)
                if n < count and draft_logits is not None:
                    q = softmax(draft_logits[b, n].double(), temp)
                    q = torch.zeros(V, dtype=torch.float64) if q is None else q
                elif known:
                    q[d] = 1.0
                taken = known and p is not None and float(u[b, n]) * float(q[d]) < float(p[d])
            if n >= count or not taken:
                break
            n += 1
        if not greedy and p is not None:
            left = (p - q).clamp(min=0.0) if n < count else p
            left = left if left.sum() > 0 else p
            run = left.cumsum(0)
            over = ((run > float(u[b, K]) * float(run[-1])) & (left > 0)).nonzero()
            drawn = int(over[0]) if len(over) else int(left.nonzero()[-1])
        elif not greedy:
            drawn = -1
        tokens[b, :n], tokens[b, n], accepted[b] = drafts[b, :n], drawn, n
    return tokens, accepted


def verify_inputs(B, K, V, real, seed, banned=0.02):
    """Logits with a few likely tokens over a tail, some banned, and a drafter that is near them."""
    g = torch.Generator().manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g)
    logits = 2.0 * f(B, K + 1, V) + 6.0 * (torch.rand(B, K + 1, V, generator=g) < 20.0 / V)
    gone = torch.rand(V, generator=g) < banned
    gone[0] = False
    logits[:, :, gone] = -math.inf
    draft = logits[:, :K] + 0.7 * f(B, K, V)
    drafts = torch.multinomial(torch.softmax(draft.reshape(B * K, V), -1), 1, generator=g).view(B, K) if K else torch.zeros(B, 0, dtype=torch.int64)
    return logits.to(real), drafts, torch.rand(B, K + 1, generator=g), draft.to(real)
