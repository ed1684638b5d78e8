"""GPU: rows next to nothing.  Where float32 rows are cut in bfloat16 parts, a part under 2^-126 counts as 0; nothing else is lost."""
import pytest
import torch

import serving_plain as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,n_in,n_out,R", [(5, 64, 40, 8), (200, 64, 40, 8), (300, 70, 33, 100)])
@pytest.mark.parametrize("power", [90, 104, 112, 120, 128, 140])
def test_small_rows_of_large_adapters(low, T, n_in, n_out, R, power):
    """Of each value of x, and of h, less than two times 2^-126 is lost (its parts do not overlap); what a float32 product itself rounds
    to a step of 2^-149 is below that too."""
    from rwkvstic_amd import ops
    g = torch.Generator().manual_seed(power + R)
    f = lambda *s: torch.randn(*s, generator=g)
    x, b = (f(T, n_in).double() * 2.0 ** -power).float(), f(3, n_out, R).to(low)
    a = (f(3, R, n_in) * 2.0 ** (10 if low == torch.float16 else 60)).to(low)
    adapter = torch.arange(T, dtype=torch.int32) % 4
    want, bound = P.lora_rows(x, a, b, adapter)
    got = ops.lora_rows(x.cuda(), a.cuda(), b.cuda(), adapter.cuda()).cpu().double()
    A, B = a.double().abs().sum(2), b.double().abs()
    lost = torch.stack([B[i] @ (A[i] + 1.0) for i in range(3)] + [torch.zeros(n_out, dtype=torch.float64)])[adapter.long()] * 2.0 ** -125
    assert bool(((got - want).abs() <= 2.0 ** -24 * (bound + want.abs()) + lost).all()), float(((got - want).abs() / (bound * 2.0 ** -24 + lost + 1e-300)).max())
