"""int8 matrix products and the quantisation in front of them, against their definitions in float64.

Tolerances.  The integer sum is exact, its conversion to float32 is off by half a step of float32 (2^-24), each of the two scalings and the bias addition by
another: 4 * 2^-24 of |product| + |bias|, then half a step of the output type.  Quantised values and scales are equal."""
import ctypes as C

import pytest
import torch

from saunet_amd import functional as HF, lib as L

TINY = torch.finfo(torch.float32).tiny
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def quant64(x, affine=None, relu=False):
    """x on the CPU -> (q, scale)"""
    v = x.float()
    if affine is not None:      # one float32 fused multiply-add: exact in float64, rounded once
        v = (v.double() * affine[0].double() + affine[1].double()).float()
    if relu:
        v = torch.where(v < 0, torch.zeros_like(v), v)
    top = v.abs().amax(1)
    bad = ~torch.isfinite(v).all(1)
    s = (top.double() / 127).float()
    s = torch.where(s < TINY, torch.zeros_like(s), s)
    q = torch.where((s > 0)[:, None], (v.double() / s.double()[:, None]).round(), torch.zeros(1, dtype=torch.float64))
    q[bad] = 0
    s[bad] = float("nan")
    return q.to(torch.int8), s


def product64(q, s, wq, ws, bias, relu):
    p = (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()
    y = p if bias is None else p + bias.double()
    return (y.clamp(min=0) if relu else y), p.abs() + (0 if bias is None else bias.double().abs())


def check_product(y, ref, size, dtype):
    d = (y.cpu().double() - ref).abs()
    half = torch.finfo(dtype).eps / 2
    # float16 has a smallest step of 2^-24 below 2^-14
    tol = 4 * 2.0 ** -24 * size + half * (ref.abs() + 4 * 2.0 ** -24 * size) + (2.0 ** -25 if dtype == torch.float16 else 0)
    over = d > tol
    assert not over.any(), (int(over.sum()), float((d / tol).max()))


def rows(m, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(1, k, generator=g))).to(dtype)


def random_rows(m, k, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8), torch.rand(m, generator=g) + 0.01


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
def test_refuses_cpu_tensors():
    for f in (lambda: HF.quantize_rows(torch.zeros(2, 4)), lambda: HF.Int8Rows(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2)),
              lambda: HF.linear_int8(torch.zeros(2, 4), None)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
    with pytest.raises(RuntimeError, match="Int8Rows"):
        HF.matmul_int8(torch.zeros(2, 4), torch.zeros(2, 4))


def test_c_entries_refuse_before_any_launch():
    h = L.load()

    def quant(dtype=L.F32, x=4096, ldx=64, rows=2, k=64, scale=None, shift=None, q=4096, ldq=64, s=4096):
        return h.saunet_quantize_rows(dtype, x, ldx, rows, k, scale, shift, 0, q, ldq, s, None)

    assert quant(rows=-1) == -1 and quant(k=0) == -1 and quant(k=131072, ldx=131072, ldq=131072) == -1 and quant(ldx=63) == -1
    assert quant(ldq=80) == -1 and quant(ldq=0) == -1 and quant(x=None) == -1 and quant(scale=4096) == -1
    assert quant(dtype=5) == -2 and quant(q=4100) == -4 and quant(rows=0) == 0

    def mm(**kw):
        d = L.Int8Desc()
        v = dict(a=4096, a_scale=4096, lda=64, m=3, b=4096, b_scale=4096, ldb=64, n=5, k=33, bias=None, y=4096, ldy=5, dtype=L.F32, relu=0)
        v.update(kw)
        for name, val in v.items():
            setattr(d, name, val)
        return h.saunet_matmul_int8(C.byref(d), None)

    assert mm(m=-1) == -1 and mm(n=0) == -1 and mm(k=0) == -1 and mm(k=65) == -1 and mm(lda=72) == -1 and mm(ldb=48) == -1 and mm(ldy=4) == -1
    assert mm(k=131072, lda=131072, ldb=131072) == -1 and mm(a=None) == -1 and mm(y=None) == -1
    assert mm(dtype=9) == -2 and mm(a=4104) == -4 and mm(m=0) == 0

    def lin(x_dtype=L.F32, x=4096, ldx=64, ws=4096, wsb=1 << 20, **kw):
        d = L.Int8Desc()
        v = dict(m=30, b=4096, b_scale=4096, ldb=64, n=5, k=33, bias=None, y=4096, ldy=5, dtype=L.F32, relu=0)
        v.update(kw)
        for name, val in v.items():
            setattr(d, name, val)
        return h.saunet_linear_int8(C.byref(d), x_dtype, x, ldx, ws, wsb, None)

    assert lin(x_dtype=4) == -2 and lin(ldx=32) == -1 and lin(x=None) == -1 and lin(ws=None) == -1 and lin(wsb=30 * 68 - 1) == -1 and lin(ws=4104) == -1
    assert lin(b=4100) == -4 and lin(y=None) == -1 and lin(m=0) == 0


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 2), (5, 16), (7, 63), (4, 64), (9, 65), (33, 100), (2, 128), (17, 129), (300, 256), (5, 257), (6, 511), (3, 513), (4, 1024),
                                 (3, 2047), (2, 2049), (3, 4096), (2, 4100), (1, 9000), (1, 131071)])
def test_quantize_rows(m, k, dtype):
    x = rows(m, k, m * 131 + k, dtype)
    r = HF.quantize_rows(x.cuda())
    q, s = quant64(x)
    assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu(), q)
    assert r.shape == (m, k) and not r.data[:, k:].any() and r.data.shape[1] % 64 == 0
    assert torch.equal(r.dequantize().cpu(), q.float() * s[:, None])


@pytest.mark.gpu
def test_quantize_rows_ties_and_borders():
    # scale 1 exactly: halves round to even; a scale with a long mantissa: quotients one unit on either side of a half
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 125.5, 126.5, -126.5, 0.49999997, 0.50000006, 3.4999998]])
    cases = [x]
    for top in (0.1, 3.3333333, 1e-30, 7e30, 1.1754944e-36):
        s = torch.tensor(top) / 127
        h = (torch.arange(-127, 127).double() + 0.5) * s.double()
        f = h.float()
        near = torch.cat([f, torch.nextafter(f, torch.tensor(float("inf"))), torch.nextafter(f, torch.tensor(-float("inf")))])
        near = near[near.abs() <= top]
        cases.append(torch.cat([torch.tensor([top]), near]).view(1, -1))
    for x in cases:
        r = HF.quantize_rows(x.cuda())
        q, s = quant64(x)
        assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu(), q)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [40, 5000])
def test_quantize_rows_zero_tiny_and_nonfinite(k):
    x = rows(8, k, 3)
    x[0] = 0
    x[1] = 1e-40                      # the scale would be subnormal
    x[2, 5] = float("nan")
    x[3, 0] = float("-inf")
    x[4] = 0; x[4, 7] = TINY * 128
    x[6] = 3e38
    r = HF.quantize_rows(x.cuda())
    q, s = quant64(x)
    assert torch.equal(r.scale.cpu().nan_to_num(-1), s.nan_to_num(-1)) and torch.equal(r.q.cpu(), q)
    w = HF.quantize_rows(rows(6, k, 4).cuda())
    y = HF.matmul_int8(r, w, relu=True, dtype=torch.float32)
    assert y[2:4].isnan().all() and not y[:2].any() and not y[4:].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_affine_relu_and_strides(dtype):
    g = torch.Generator().manual_seed(0)
    for k in (48, 100, 700):
        x = rows(50, k, 8, dtype)
        sc, sh = torch.rand(k, generator=g) + 0.5, torch.randn(k, generator=g)
        for relu in (False, True):
            r = HF.quantize_rows(x.cuda(), affine=(sc.cuda(), sh.cuda()), relu=relu)
            q, s = quant64(x, (sc, sh), relu)
            assert torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu(), q)
    wide = rows(40, 300, 9, dtype).cuda()
    for v in (wide[:, 8:72], wide[:, 3:200], wide[::3, :64], wide.t(), wide[:1].expand(5, 300), wide.view(4, 10, 300)[:, 2:5, 16:48], wide[:, :1]):
        r = HF.quantize_rows(v)
        q, s = quant64(v.cpu().reshape(-1, v.shape[-1]))
        assert r.shape == tuple(v.shape) and torch.equal(r.scale.cpu(), s) and torch.equal(r.q.cpu().reshape(q.shape), q)
    assert HF.quantize_rows(wide[:0]).shape == (0, 300)


# ------------------------------------------------------------------------------------------------ the product
SHAPES = [(1, 1, 1), (1, 64, 16), (2, 65, 17), (3, 1000, 130), (16, 4096, 64), (17, 200, 515), (31, 64, 128), (33, 63, 129), (64, 512, 512), (127, 130, 255), (129, 257, 257),
          (200, 128, 1000), (513, 320, 96), (1000, 1001, 33), (2049, 256, 128), (70, 8192, 40), (64, 8075, 1), (500, 64, 17), (33, 1000, 8200), (16, 70, 16400), (900, 130, 600)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_int8(m, k, n, dtype):
    (q, s), (wq, ws) = random_rows(m, k, 1), random_rows(n, k, 2)
    s = s / k ** 0.5 / 127
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5))
    a, w = HF.Int8Rows(q.cuda(), s.cuda()), HF.Int8Rows(wq.cuda(), ws.cuda())
    for b, relu in ((None, False), (bias, True)):
        y = HF.matmul_int8(a, w, bias=None if b is None else b.cuda(), relu=relu, dtype=dtype)
        assert y.dtype == dtype and y.shape == (m, n)
        ref, size = product64(q, s, wq, ws, b, relu)
        check_product(y, ref, size, dtype)


@pytest.mark.gpu
def test_matmul_int8_largest_sum_is_exact():
    k = HF.INT8_K_MAX
    q = torch.full((2, k), -128, dtype=torch.int8)
    y = HF.matmul_int8(HF.Int8Rows(q.cuda(), torch.ones(2).cuda()), HF.Int8Rows(q[:1].cuda(), torch.ones(1).cuda()), dtype=torch.float32)
    assert torch.equal(y.cpu(), torch.full((2, 1), float(k * 128 * 128)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_matmul_int8_into_slices_leaves_the_rest_alone(dtype):
    for m, k, n, lo in ((100, 96, 40, 8), (5, 130, 33, 3), (300, 64, 128, 16), (1, 512, 256, 5)):
        (q, s), (wq, ws) = random_rows(m, k, 3), random_rows(n, k, 4)
        s = s / 1000
        wide = torch.full((m + 2, n + lo + 9), 7.0, dtype=dtype).cuda()
        out = wide[1:m + 1, lo:lo + n]
        y = HF.matmul_int8(HF.Int8Rows(q.cuda(), s.cuda()), HF.Int8Rows(wq.cuda(), ws.cuda()), dtype=dtype, out=out)
        assert y is out
        ref, size = product64(q, s, wq, ws, None, False)
        check_product(y, ref, size, dtype)
        keep = torch.ones_like(wide, dtype=torch.bool)
        keep[1:m + 1, lo:lo + n] = False
        assert (wide[keep] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 40, 300])
def test_linear_int8(m, dtype):
    for k, n in ((1, 1), (3, 33), (4096, 20), (8191, 18), (20000, 17), (64, 48), (200, 130), (1024, 512), (2049, 77), (6000, 20)):
        x, w = rows(m, k, k + m, dtype), rows(n, k, 7)
        wr = HF.quantize_rows(w.cuda())
        bias = torch.randn(n, generator=torch.Generator().manual_seed(1))
        q, s = quant64(x)
        for b, relu, od in ((None, False, None), (bias, True, torch.float32)):
            if od is None and dtype == torch.float16:
                od = torch.float32          # the products of these rows pass float16's largest value
            y = HF.linear_int8(x.cuda(), wr, bias=None if b is None else b.cuda(), relu=relu, dtype=od)
            ref, size = product64(q, s, wr.q.cpu(), wr.scale.cpu(), b, relu)
            check_product(y, ref, size, od or dtype)
            two = HF.matmul_int8(HF.quantize_rows(x.cuda()), wr, bias=None if b is None else b.cuda(), relu=relu, dtype=od or dtype)
            assert torch.equal(y, two)
    x = rows(m, 72, 3, dtype)
    x[0, 5] = float("nan")
    x[m // 2, 7] = float("inf")
    x[m - 1] = 0
    y = HF.linear_int8(x.cuda(), HF.quantize_rows(rows(20, 72, 4).cuda()), dtype=torch.float32).cpu()
    bad = ~torch.isfinite(x.float()).all(1)
    assert y[bad].isnan().all() and not y[~bad].isnan().any() and (bad[m - 1] or not y[m - 1].any())
    wide = rows(m, 300, 11, dtype).cuda()
    wr = HF.quantize_rows(rows(24, 96, 6).cuda())
    assert torch.equal(HF.linear_int8(wide[:, 101:197], wr, dtype=torch.float32), HF.linear_int8(wide[:, 101:197].contiguous(), wr, dtype=torch.float32))
    lead = rows(6 * m, 96, 5, dtype).view(2, 3, m, 96).cuda()
    wr = HF.quantize_rows(rows(24, 96, 6).cuda())
    assert torch.equal(HF.linear_int8(lead, wr, dtype=torch.float32), HF.linear_int8(lead.view(-1, 96), wr, dtype=torch.float32).view(2, 3, m, 24))
    assert HF.linear_int8(lead[:0], wr).shape == (0, 3, m, 24)
    one = HF.linear_int8(lead[0, 0, 0], wr, dtype=torch.float32)                      # a single vector
    assert one.shape == (24,) and torch.equal(one, HF.linear_int8(lead[0, 0, :1], wr, dtype=torch.float32)[0])
    assert HF.matmul_int8(HF.quantize_rows(lead[0, 0, 0]), wr, out=torch.empty(24, dtype=torch.bfloat16, device="cuda")).shape == (24,)


@pytest.mark.gpu
def test_int8_refusals_on_the_device():
    a, w = HF.quantize_rows(rows(4, 96, 1).cuda()), HF.quantize_rows(rows(8, 96, 2).cuda())
    for f, what in ((lambda: HF.matmul_int8(a, HF.quantize_rows(rows(8, 95, 2).cuda())), "does not meet"),
                    (lambda: HF.matmul_int8(a, w, dtype=torch.float64), "float32, bfloat16 or float16"),
                    (lambda: HF.matmul_int8(a, w, bias=torch.zeros(7).cuda()), "bias"),
                    (lambda: HF.matmul_int8(a, w, out=torch.zeros(4, 9).cuda()), "out has to be"),
                    (lambda: HF.matmul_int8(a, w, dtype=torch.float32, out=torch.zeros(8, 4).cuda().t()), "unit stride"),
                    (lambda: HF.quantize_rows(torch.zeros(2, 4).cuda().double()), "float32, bfloat16 or float16"),
                    (lambda: HF.quantize_rows(torch.zeros(2, 4).cuda(), affine=(torch.zeros(3).cuda(), torch.zeros(4).cuda())), "affine"),
                    (lambda: HF.linear_int8(torch.zeros(2, 96).cuda().requires_grad_(), w), "inference"),
                    (lambda: HF.Int8Rows(torch.zeros(2, 4, dtype=torch.int8).cuda(), torch.ones(3).cuda()), "one scale a row")):
        with pytest.raises(RuntimeError, match=what):
            f()


@pytest.mark.gpu
def test_int8_on_a_side_stream_and_replayed():
    x = rows(200, 700, 1).cuda()
    wr = HF.quantize_rows(rows(130, 700, 2).cuda())
    one = x[:1].clone()
    ref, ref1 = HF.linear_int8(x, wr), HF.linear_int8(one, wr)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side, side1 = HF.linear_int8(x, wr), HF.linear_int8(one, wr)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, ref) and torch.equal(side1, ref1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, y1 = HF.linear_int8(x, wr), HF.linear_int8(one, wr)
    for it in range(3):
        x.copy_(rows(200, 700, 10 + it)); one.copy_(x[3:4])
        g.replay()
        assert torch.equal(y, HF.linear_int8(x, wr)) and torch.equal(y1, HF.linear_int8(one, wr))
        torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ the 1x1 convolution and the network
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pointwise_int8(dtype):
    g = torch.Generator().manual_seed(2)
    for n, c, h, wd, co in ((2, 64, 9, 7, 128), (1, 33, 1, 1, 17), (3, 1, 2, 5, 4), (1, 96, 16, 16, 40)):
        buf = torch.randn(n, h, wd, c + 24, generator=g).to(dtype).cuda().permute(0, 3, 1, 2)
        sc, sh, bias = torch.rand(c, generator=g) + 0.5, torch.randn(c, generator=g), torch.randn(co, generator=g)
        w = HF.quantize_rows(rows(co, c, 3).cuda())
        for x in (buf[:, 8:8 + c], buf[:, :c].contiguous(memory_format=torch.channels_last), buf[:, :c].contiguous()):
            q, s = quant64(x.permute(0, 2, 3, 1).reshape(-1, c).cpu(), (sc, sh), True)
            ref, size = product64(q, s, w.q.cpu(), w.scale.cpu(), bias, True)
            y = HF.pointwise_int8(x, w, bias.cuda(), relu=True, affine=(sc.cuda(), sh.cuda()), affine_relu=True)
            assert y.shape == (n, co, h, wd) and y.dtype == dtype
            check_product(y.permute(0, 2, 3, 1).reshape(-1, co), ref, size, dtype)
            wide = torch.full((n, h, wd, co + 16), 3.0, dtype=dtype).cuda().permute(0, 3, 1, 2)
            z = HF.pointwise_int8(x, w, bias.cuda(), relu=True, affine=(sc.cuda(), sh.cuda()), affine_relu=True, out=wide[:, 8:8 + co])
            assert torch.equal(z, y) and (wide[:, :8] == 3).all() and (wide[:, 8 + co:] == 3).all()
    with pytest.raises(RuntimeError, match="Int8Rows"):
        HF.pointwise_int8(buf[:, :5], w)
    with pytest.raises(RuntimeError, match="inference"):
        HF.pointwise_int8(buf[:, :96].clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="out has to be"):
        HF.pointwise_int8(buf[:, :96], w, out=torch.zeros(1, 41, 16, 16, dtype=dtype).cuda())


@pytest.mark.gpu
def test_dense_block_int8_follows_its_definition(monkeypatch):
    """two dense layers with int8 conv1 against the same computation from the parts, everything but the int8 product in float32 of the existing kernels"""
    import saunet_amd
    from saunet_amd.modules import _DenseBlock
    monkeypatch.setattr(HF, "INT8_CHANNELS_MIN", 0)
    torch.manual_seed(0)
    saunet_amd.set_compute_dtype(torch.float32)
    blk = _DenseBlock(2, 64).cuda().eval()
    for m in blk.modules():
        if isinstance(m, torch.nn.BatchNorm2d):
            m.running_mean.normal_(); m.running_var.uniform_(0.5, 2.0); m.weight.data.uniform_(0.5, 1.5); m.bias.data.normal_()
    x = torch.randn(2, 64, 16, 16).cuda().contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        plain = blk(x).clone()
        blk.int8 = True
        y = blk(x).clone()
        blk.int8 = False
        assert torch.equal(blk(x), plain)
        buf = x
        for m in blk.values():
            s1 = m.norm1.weight / torch.sqrt(m.norm1.running_var + m.norm1.eps)
            s2 = m.norm2.weight / torch.sqrt(m.norm2.running_var + m.norm2.eps)
            a = torch.relu(buf * s1.view(1, -1, 1, 1) + (m.norm1.bias - m.norm1.running_mean * s1).view(1, -1, 1, 1))
            w = HF.quantize_rows(m.conv1.weight.flatten(1) * s2.view(-1, 1))
            b = m.norm2.bias - m.norm2.running_mean * s2
            q = HF.quantize_rows(a.permute(0, 2, 3, 1).reshape(-1, a.shape[1]))
            z = torch.relu(q.dequantize().double() @ w.dequantize().double().t() + b.double()).float().view(2, 16, 16, -1).permute(0, 3, 1, 2)
            buf = torch.cat([buf, HF.conv2d(z, m.conv2.weight, None, 1, 1)], 1)
    # Coefficients of the two BatchNorms are rounded differently (float64 there, float32 here), so a quantised value beside a half may come out one step away
    # (1/127 of the pixel's largest activation): of the sum over 64 channels that is one term in a few thousand.  A missing ReLU, scale or bias is of order one.
    assert not torch.equal(y, plain)
    for c0 in (64, 96):
        d, ref = (y - buf)[:, c0:c0 + 32].double(), buf[:, c0:c0 + 32].double()
        assert float(d.norm()) <= 1.0 / 127 * float(ref.norm()), (float(d.norm()), float(ref.norm()))


@pytest.mark.gpu
def test_saunet_int8_inference_switch(monkeypatch):
    import saunet_amd
    from saunet_amd import data
    saunet_amd.set_compute_dtype(torch.bfloat16)
    torch.manual_seed(0)
    net = saunet_amd.SAUNet(num_classes=4).cuda().eval()
    saunet_amd.set_compute_dtype(torch.float32)
    img = data.synthetic_batch(1, 64, 64, seed=1)[0].cuda()
    assert sum(m.int8 for m in net.modules() if hasattr(m, "int8")) == 0 and sum(m.int8 for m in net.int8_inference().modules() if hasattr(m, "int8")) == 4
    net.int8_inference(False)
    # compared at the encoder's last dense block: behind it the attention blocks add with float atomics, and two runs of one network differ in the last bits
    seen = []
    net.conv5[0].register_forward_hook(lambda m, i, o: seen.append(o[0] if isinstance(o, tuple) else o))

    def run():
        seen.clear()
        out = net(img)[0]
        return seen[0], out

    calls, inner = [], HF.pointwise_int8
    monkeypatch.setattr(HF, "pointwise_int8", lambda *a, **k: calls.append(1) or inner(*a, **k))
    with torch.no_grad():
        plain = run()[0].clone()
        assert not calls
        net.int8_inference()
        y, out = run()
        y = y.clone()
        assert len(calls) == 2 + 18 + 16                # layers of the second (128 + 32 i), third (256 + 32 i) and fourth (512 + 32 i) block with 448 channels or more
        assert torch.isfinite(out).all() and not torch.equal(y, plain)
        assert torch.equal(run()[0], y)
        net.int8_inference(False)
        assert torch.equal(run()[0], plain)
        net.int8_inference()
        g = torch.cuda.CUDAGraph()
        run()
        with torch.cuda.graph(g):
            z = run()[0]
        for it in range(3):
            img.copy_(data.synthetic_batch(1, 64, 64, seed=2 + it)[0].cuda())
            g.replay()
            got = z.clone()
            assert torch.equal(got, run()[0])
            torch.cuda.synchronize()
    net.train()
    out = net(img)[0]                                         # training is unaffected by the switch
    out.float().sum().backward()
    assert net.conv4["denselayer1"].conv1.weight.grad is not None
