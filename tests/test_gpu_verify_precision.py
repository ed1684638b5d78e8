"""GPU: `verify_drafts` decides by probabilities of float64, to the last bits of them."""
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from rwkvstic_amd import ops as _ops
    return _ops


def _next_to(x0, count):
    """Random numbers u (float32) near e^x0 / (1 + e^x0), each with logits x on both sides of where a token of logit x beside one of
    logit 0 has that probability, 2^-50 of it away and as little further as float64 allows; and whether it is above u."""
    getcontext().prec = 50
    u, found = np.float32(1.0 / (1.0 + np.exp(-x0))), []
    for _ in range(count):
        u = np.nextafter(u, np.float32(1.0))
        for sign in (1, -1):
            p = Decimal(float(u)) * (1 + sign * Decimal(2) ** -50)
            exact = (p / (1 - p)).ln()
            x = float(exact)
            if sign * (Decimal(x) - exact) < 0:
                x = float(np.nextafter(x, sign * np.inf))
            found.append((float(u), x, sign > 0))
    return found


@pytest.mark.parametrize("lo,hi", [(-45.5, -18.0), (-900.0, -46.0)])
def test_random_numbers_next_to_the_probability(ops, lo, hi):
    """Two tokens, a draft without a distribution: accepted while u < p, p = w / (1 + w), w = e^x.  In units of 2^-53: w is off by 3 (a
    value of the table by 1/2, the series and its product with the table by 1 each, the rest of the series by 1/32), and by |x| / 8 for
    32 log2 e, which is known to 2^-56, at most 2.5 here; p is off by (1 - p) times that, and the sum and the quotient add 1 each.  Both
    sides of u are 8 units, 2^-50, away.  Arguments by eighths of 32nds of a power of two."""
    cases = [c for t in np.arange(lo, hi, (hi - lo) / 230) for c in _next_to(np.round(t * 8) / 8 * np.log(2.0) / 32, 2)]
    us, xs, above = zip(*cases)
    n = len(us)
    logits, u = torch.zeros(n, 2, 2, dtype=torch.float64), torch.zeros(n, 2)
    logits[:, 0, 1], u[:, 0] = torch.tensor(xs, dtype=torch.float64), torch.tensor(us, dtype=torch.float64).float()
    accepted = ops.verify_drafts(logits.cuda(), torch.ones(n, 1, dtype=torch.int64).cuda(), u.cuda())[1].cpu()
    wrong = accepted != torch.tensor(above).long()
    assert not bool(wrong.any()), f"{int(wrong.sum())} of {n}"
