"""GPU: what the definition makes of infinities in rows, adapters and scales is what `lora_rows` gives, whatever the types."""
import math

import pytest
import torch

import serving_plain as P

pytestmark = pytest.mark.gpu

HALF = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24}       # half a step
TYPES = pytest.mark.parametrize("real,low", [(r, l) for r in (torch.float32, torch.float64) for l in (torch.bfloat16, torch.float16, torch.float32)])


@pytest.fixture(scope="module")
def ops():
    from rwkvstic_amd import ops as _ops
    return _ops


def _same(ops, c, half):
    """Infinities and what is no number where the definition has them; the rest within the bound of sums in any order."""
    want, bound = P.lora_rows(**c)
    got = ops.lora_rows(**{k: v.cuda() for k, v in c.items()}).cpu().double()
    assert torch.equal(got.isnan(), want.isnan()), (int(got.isnan().sum()), int(want.isnan().sum()))
    there = want.isfinite()
    assert torch.equal(got[want.isinf()], want[want.isinf()]) and torch.equal(got.isfinite(), there)
    assert bool(((got - want).abs()[there] <= half * (bound + want.abs())[there]).all())
    return want


def _case(T, n_in, n_out, R, real, low, seed):
    """Three adapters and rows without one; every weight at least 2^-4, so that no product with an infinity is of a zero."""
    g = torch.Generator().manual_seed(seed)
    away = lambda *s: (lambda t: t + t.sign() * 2.0 ** -4 + (t == 0) * 1.0)(torch.randn(*s, generator=g))
    return dict(x=away(T, n_in).to(real), a=away(3, R, n_in).to(low), b=away(3, n_out, R).to(low), adapter=torch.arange(T, dtype=torch.int32) % 4,
                scale=0.5 + torch.rand(3, generator=g), base=away(T, n_out).to(real))


SIZES = pytest.mark.parametrize("T,n_in,n_out,R", [(9, 64, 40, 1), (9, 64, 40, 8), (50, 300, 72, 40), (200, 64, 40, 1), (200, 136, 48, 24), (300, 70, 33, 100), (1100, 33, 20, 130)])


@TYPES
@SIZES
def test_rows_that_are_infinite(ops, real, low, T, n_in, n_out, R):
    c = _case(T, n_in, n_out, R, real, low, T + R)
    for t, k, v in ((0, 0, math.inf), (5, n_in - 1, -math.inf), (6, 3, math.inf), (3, 1, math.inf)):              # (row 3 has no adapter)
        c["x"][t, k] = v
    c["x"][4], c["x"][8] = math.inf, -math.inf
    c["a"][2] = c["a"][2].abs()                       # (row 6: all of h is +infinity, and with these b all of its outputs)
    c["b"][2] = c["b"][2].abs()
    want = _same(ops, c, HALF[real])
    assert bool((want[6] == math.inf).all()) and bool(want[3].isfinite().all()) and (R > 1 or bool(want[:1].isinf().all()))


@TYPES
@SIZES
def test_adapters_that_are_infinite(ops, real, low, T, n_in, n_out, R):
    """Rows of few bits too: 1 is 1 + 0 + 0 where it is cut in parts, and no part of it may meet the infinity as a zero."""
    c = _case(T, n_in, n_out, R, real, low, T + R)
    c["x"][::5] = 1.0
    c["x"][1::5] = 1.0 + 2.0 ** -12
    c["a"][0, 0, 2], c["a"][1, R - 1, n_in - 1] = math.inf, -math.inf
    c["b"][2, 7, R - 1], c["b"][2, 8, 0] = -math.inf, math.inf
    assert bool(_same(ops, c, HALF[real]).isinf().any())


@TYPES
@pytest.mark.parametrize("T", [2, 140])
def test_an_infinite_weight_of_a_product_that_is_one(ops, real, low, T):
    one = dict(x=torch.ones(T, 1, dtype=real), a=torch.ones(2, 1, 1, dtype=low), b=torch.ones(2, 16, 1, dtype=low), adapter=torch.zeros(T, dtype=torch.int32))
    one["b"][0, 3], one["b"][0, 5] = math.inf, -math.inf
    want = _same(ops, one, HALF[real])
    assert bool((want[:, 3] == math.inf).all()) and bool((want[:, 5] == -math.inf).all()) and int(want.isfinite().sum()) == 14 * T


@TYPES
@SIZES
def test_scales_that_are_infinite(ops, real, low, T, n_in, n_out, R):
    c = _case(T, n_in, n_out, R, real, low, T + R)
    for k in ("x", "a", "b"):
        c[k] = c[k].abs()
    c["scale"][1] = math.inf
    assert bool((_same(ops, c, HALF[real])[1] == math.inf).all())
