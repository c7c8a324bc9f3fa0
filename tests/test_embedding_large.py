"""The token embedding at the limits of its sizes."""
import pytest
import torch

from zorse_amd import _abi


def test_sizes_beyond_the_launches_are_refused():
    """Tokens times columns from 2^40 on (CPU; more than the GPU's memory)."""
    ws = _abi.lib().zk_embedding_bwd_workspace
    assert ws(1 << 28, 8, 1 << 12) < 0 and ws(1 << 18, 8, 1 << 22) < 0
    assert ws(1 << 28, 8, (1 << 12) - 1) > 0 and ws(300, (1 << 28) - 1, (1 << 23) - 1) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [100, 200])
def test_gradient_of_a_table_with_many_rows(dev, tokens):
    """2^24 rows of 4112 bytes, 69 GB: a workgroup for each of them would be 2^32
    threads and more.  All rows are written, those without a token with zeros."""
    from zorse_amd import kernels
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of the GPU's memory")
    V, h = 1 << 24, 2056
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randperm(1 << 12, generator=g)[:tokens] * 4096 + 7
    ids[:2] = torch.tensor([0, V - 1])
    dy = torch.randn(tokens, h, generator=g).to(dev, torch.bfloat16)
    ids = ids.to(dev)
    dw = torch.full((V, h), float("nan"), device=dev, dtype=torch.bfloat16)
    kernels.embedding_bwd(ids, dy, V, dw=dw)
    assert torch.equal(dw[ids], dy)
    dw[ids] = 0
    for part in dw.split(1 << 20):
        assert not bool(part.any())  # NaN counts
    del dw, part
    torch.cuda.empty_cache()
