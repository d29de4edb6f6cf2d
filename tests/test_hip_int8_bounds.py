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


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(200100, 520, 8), (200100, 520, 64), (70001, 580, 65), (50003, 1000, 192), (33000, 700, 193), (8, 520, 200100), (64, 577, 70001), (65, 600, 60003),
                                   (40000, 4096, 20)])
def test_tall_and_narrow_products(m, k, n):
    """more than three thousand 64 x 64 tiles with one short side, on either side of the tile rule.  The integer sum is exact (float64 holds it), its conversion,
    the two scalings and the bias addition are half a step of float32 each, the result half a step of bfloat16."""
    gen = torch.Generator(device="cuda").manual_seed(m + n)
    q, w = (torch.randint(-127, 128, (r, k), generator=gen, device="cuda", dtype=torch.int8) for r in (m, n))
    sq, sw = (torch.rand(r, generator=gen, device="cuda") * 1e-3 + 1e-4 for r in (m, n))
    bias = torch.randn(n, generator=gen, device="cuda")
    y = HF.matmul_int8(HF.Int8Rows(q, sq), HF.Int8Rows(w, sw), bias=bias, relu=True)
    p = (q.double() @ w.double().t()) * sq.double()[:, None] * sw.double()
    ref, size = (p + bias.double()).clamp(min=0), p.abs() + bias.double().abs()
    tol = 4 * 2.0 ** -24 * size + 2.0 ** -8 * (ref + 4 * 2.0 ** -24 * size)
    assert ((y.double() - ref).abs() <= tol).all()
