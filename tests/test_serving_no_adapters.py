"""`lora_rows` of a pool that is empty: every row gets base."""
import pytest
import torch


def test_the_library_takes_no_adapters():
    """Up to the look at the workspace; nothing is launched."""
    from rwkvstic_amd import _native
    L = _native.lib()
    ARG, WORKSPACE = -1, -4

    def lora(N, R, a):
        return L.rwkv_lora_rows(None, 2, 8, 8, N, R, 0, 1 << 24, 8, 2, a, a, 1 << 25, None, None, 0, 1 << 26, 8, 16, 0)
    assert lora(0, 4, None) == WORKSPACE and lora(0, 0, None) == WORKSPACE and lora(0, 4, 1 << 27) == WORKSPACE
    assert lora(1, 4, None) == ARG and lora(1, 0, 1 << 27) == ARG and lora(-1, 4, 1 << 27) == ARG and lora(0, 257, None) == -3
    assert L.rwkv_lora_rows_workspace_bytes(2, 8, 8, 0, 0, 0) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("real", [torch.float32, torch.float64])
@pytest.mark.parametrize("T,n_out,R", [(1, 8, 4), (7, 33, 0), (128, 64, 300), (129, 64, 16), (2000, 260, 0)])
def test_rows_get_base(real, T, n_out, R):
    from rwkvstic_amd import ops
    g = torch.Generator().manual_seed(T)
    x, base = torch.randn(T, 24, generator=g, dtype=real).cuda(), torch.randn(T, n_out, generator=g, dtype=real).cuda()
    a, b, adapter = torch.empty(0, R, 24).cuda(), torch.empty(0, n_out, R).cuda(), (torch.arange(T, dtype=torch.int32) % 3 - 1).cuda()
    if R > 256:
        with pytest.raises(RuntimeError):
            ops.lora_rows(x, a, b, adapter, base=base)
        return
    want, x[0, 0] = base.clone(), float("nan")
    assert torch.equal(ops.lora_rows(x, a, b, adapter, torch.empty(0).cuda(), base=base), want)
    assert torch.equal(ops.lora_rows(x, a, b, adapter, base=base, out=base), want)
    assert not ops.lora_rows(x, a, b, adapter).any()
