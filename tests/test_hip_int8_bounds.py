"""What the int8 operators do at the borders of their domain: more rows than a launch has threads for, arguments that would lose a gradient, tall and narrow
products, memory that is shared or copied."""
import pytest
import torch

from saunet_amd import functional as HF, lib as L


def rows(m, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(1, k, generator=g))).to(dtype)


@pytest.mark.gpu
def test_quantize_rows_in_more_than_one_launch():
    """2^23 rows are one launch; each row is a function of itself alone: the same as in a short call"""
    m, k = (1 << 23) + 37, 6
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(m, k, generator=gen, device="cuda", dtype=torch.bfloat16)
    r = HF.quantize_rows(x)
    # (float64 of the exact maximum, rounded once)
    assert torch.equal(r.scale, (x.abs().amax(1).double() / 127).float())
    for lo, hi in ((0, 1000), ((1 << 23) - 500, (1 << 23) + 37), (m - 3, m)):
        part = HF.quantize_rows(x[lo:hi].clone())
        assert torch.equal(r.data[lo:hi], part.data) and torch.equal(r.scale[lo:hi], part.scale)
    q = torch.round(x.double() / r.scale.double()[:, None])
    assert torch.equal(r.data[:, :k].double(), q) and not r.data[:, k:].any()
