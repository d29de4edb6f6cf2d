"""What the int8 operators do at the borders of their domain: more rows than a launch has threads for, arguments that would lose a gradient, tall and narrow
products, memory that is shared or copied."""
import ctypes as C
import threading

import pytest
import torch

from saunet_amd import functional as HF, lib as L


def rows(m, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(1, k, generator=g))).to(dtype)


def test_more_channels_than_an_index_holds_are_refused():
    d = L.Int8Desc(4096, 4096, 64, 1, 4096, 4096, 64, (1 << 30) + 1, 64, None, 4096, (1 << 30) + 1, L.F32, 0)
    assert L.load().saunet_matmul_int8(C.byref(d), None) == -1 and L.load().saunet_linear_int8(C.byref(d), L.F32, 4096, 64, 4096, 1 << 20, None) == -1
    with pytest.raises(RuntimeError, match="channels"):
        HF._int8_out((1,), 1, (1 << 30) + 1, torch.float32, torch.device("cuda:0"), None)


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


@pytest.mark.gpu
def test_a_bias_or_affine_that_asks_for_a_gradient_is_refused():
    x, w = rows(5, 96, 1).cuda(), HF.quantize_rows(rows(7, 96, 2).cuda())
    bias, sc, sh = (torch.randn(n).cuda().requires_grad_() for n in (7, 96, 96))
    a = HF.quantize_rows(x)
    for f in (lambda: HF.matmul_int8(a, w, bias=bias), lambda: HF.linear_int8(x, w, bias=bias), lambda: HF.quantize_rows(x, affine=(sc, sh)),
              lambda: HF.quantize_rows(x, affine=(sc.detach(), sh)), lambda: HF.pointwise_int8(x.view(5, 96, 1, 1), w, bias)):
        with pytest.raises(RuntimeError, match="inference"):
            f()
    with torch.no_grad():
        y, r = HF.linear_int8(x, w, bias=bias), HF.quantize_rows(x, affine=(sc, sh))
    assert torch.equal(y, HF.linear_int8(x, w, bias=bias.detach())) and torch.equal(r.data, HF.quantize_rows(x, affine=(sc.detach(), sh.detach())).data)


@pytest.mark.gpu
def test_int8_rows_share_or_copy():
    q, s = torch.randint(-127, 128, (6, 128), dtype=torch.int8).cuda(), torch.rand(6).cuda()
    shared, copied = HF.Int8Rows(q, s), HF.Int8Rows(q[:, :100], s)
    assert shared.data.data_ptr() == q.data_ptr() and copied.data.data_ptr() != q.data_ptr()
    w = HF.quantize_rows(rows(9, 128, 3).cuda())
    before = HF.matmul_int8(shared, w, dtype=torch.float32)
    q.zero_()
    assert before.any() and not HF.matmul_int8(shared, w, dtype=torch.float32).any() and copied.q.any()


@pytest.mark.gpu
def test_pointwise_int8_of_an_empty_batch_and_one_pixel():
    w = HF.quantize_rows(rows(20, 64, 4).cuda())
    assert HF.pointwise_int8(torch.zeros(0, 64, 8, 8).cuda(), w).shape == (0, 20, 8, 8)
    x = rows(1, 64, 5).cuda()
    y = HF.pointwise_int8(x.view(1, 64, 1, 1), w)
    assert torch.equal(y.view(1, 20), HF.linear_int8(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(1, 4096), (3, 1024), (8, 512), (40, 300)])
def test_linear_int8_into_its_own_input(m, k):
    x, w = rows(m, k, 7).cuda(), HF.quantize_rows((rows(k, k, 8) / k).cuda())
    ref = HF.linear_int8(x, w)
    wide = torch.zeros(m, k + 8, device="cuda")
    wide[:, 8:] = x
    for buf, out in ((x.clone(), None), (wide[:, 8:], wide[:, :k])):        # the same memory, and rows shifted against each other
        out = buf if out is None else out
        assert HF.linear_int8(buf, w, out=out) is out and torch.equal(out, ref)


@pytest.mark.gpu
def test_two_threads_at_once():
    """each on a stream of its own, the first calls of several kernels among them"""
    x, w = rows(700, 900, 1).cuda(), HF.quantize_rows(rows(5000, 900, 2).cuda())
    g = [1e-2 * rows(m, n, m).cuda() for m, n in ((20, 70), (150, 400), (500, 600))]
    torch.cuda.synchronize()
    outs, errors = {}, []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    outs[k] = (HF.linear_int8(x, w), HF.linear_int8(x[:1], w), *HF.newton_schulz(g, steps=5 + k))
                torch.cuda.current_stream().synchronize()
        except Exception as e:              # noqa: BLE001 -- reported by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for k in range(2):
        want = (HF.linear_int8(x, w), HF.linear_int8(x[:1], w), *HF.newton_schulz(g, steps=5 + k))
        assert all(torch.equal(a, b) for a, b in zip(outs[k], want))
