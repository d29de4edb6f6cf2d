"""Newton-Schulz orthogonalisation and the Muon step against their formulas in float64.

Tolerance of the iteration.  The kernels multiply float16 pairs: an operand is off by 2^-24 of itself (float32's own half step) and the dropped lo lo
term by another 2^-24, so a product's error is at most three times that of the same product over float32 operands; a chain of products carries it on as the
float32 chain does.  The float32 chain's own distance from float64, measured on the same input, is therefore the yardstick: 4 times it, plus the rounding of the result to its type (half
a step of the value), plus a floor for inputs on which the float32 chain is exact by luck (a 1 x 1 matrix).  The floor is the worst case of the last step
alone at a singular value s near 1, in half steps d = 2^-24 of float32: S = s^2 carries 4 d (two operand roundings, the sum, its own storage), so
b S + c S^2 carries |b| 4 d + c (2 * 4 + 4) d = 43 d; with the storage of P (|P| < 2.8), the three roundings of the product P x and the two of a x that makes
43 + 2.8 + 8.4 + 6.9 = 61 d on a result of 0.7 ... 1.2: 64 d of the result's norm is not reached by correct arithmetic, and a lost low part is 2^-12."""
import copy
import ctypes as C
import math

import pytest
import torch

import saunet_amd
from saunet_amd import functional as HF, lib as L, optim

COEFF = (3.4445, -4.7750, 2.0315)


def chain(g, dtype, steps=5, coeff=COEFF, eps=1e-7):
    a, b, c = coeff
    x = g.to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / x.double().norm().clamp(min=eps).to(dtype)
    for _ in range(steps):
        s = x @ x.t()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t().contiguous() if tall else x


def check(out, g, noise=0.0, **kw):
    assert out.dtype == g.dtype and out.shape == g.shape
    ref = chain(g.cpu(), torch.float64, **kw)
    d32 = chain(g.cpu(), torch.float32, **kw).double() - ref
    d = out.cpu().double() - ref
    half = torch.finfo(g.dtype).eps / 2
    assert float(d.norm()) <= 4 * float(d32.norm()) + (64 * 2.0 ** -24 + noise + half) * float(ref.norm()), (float(d.norm()), float(d32.norm()), float(ref.norm()))
    top = float(ref.abs().max())
    assert float(d.abs().max()) <= 8 * float(d32.abs().max()) + (64 * 2.0 ** -24 + noise + half) * top, (float(d.abs().max()), float(d32.abs().max()), top)


def matrix(m, n, seed, dtype=torch.float32, kind="gauss"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=gen)
    if kind == "lowrank":
        r = max(1, min(m, n) // 8)
        x = torch.randn(m, r, generator=gen) @ torch.randn(r, n, generator=gen) + 0.02 * x
    return (1e-2 * x).to(dtype)


# ------------------------------------------------------------------------------------------------ refusals (no GPU needed)
def test_refuses_cpu_tensors_and_bad_arguments():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        HF.newton_schulz(torch.zeros(4, 4))
    for kw in (dict(steps=0), dict(steps=33), dict(steps=2.5), dict(eps=0.0), dict(eps=float("nan")), dict(coefficients=(1.0, 2.0)),
               dict(coefficients=(1.0, float("inf"), 0.0))):
        with pytest.raises(ValueError):
            HF.newton_schulz(torch.zeros(4, 4), **kw)
    assert HF.newton_schulz([]) == []


def test_muon_refuses_vectors_and_bad_hyperparameters():
    w, v = torch.nn.Parameter(torch.zeros(4, 4)), torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="another optimiser"):
        optim.FusedMuon([v])
    opt = optim.FusedMuon([w])
    with pytest.raises(ValueError, match="another optimiser"):
        opt.add_param_group({"params": [v]})
    assert len(opt.param_groups) == 1
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(ns_steps=0), dict(adjust_lr_fn="none")):
        with pytest.raises(ValueError):
            optim.FusedMuon([w], **kw)
    w.grad = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        opt.step(upload=False)


def test_c_entry_refuses_before_any_launch():
    h = L.load()
    ws = 1 << 20                                     # an address that is never used: every call below is refused on the host

    def desc(rows=8, cols=8, dtype=L.F32, steps=5, coeff=COEFF, eps=1e-7, ld=None, src=4096):
        return HF.ns_desc([src, 4096, 4096, ld or cols, ld or cols, rows, cols], dtype, steps, coeff, eps)

    def rc(d, bytes_=1 << 40, p=ws):
        return h.saunet_newton_schulz(C.byref(d[0]), p, bytes_, None)

    assert rc(desc(rows=0)) == -1 and rc(desc(rows=40000, cols=40000)) == -1 and rc(desc(cols=(1 << 20) + 1)) == -1
    assert rc(desc(ld=7)) == -1 and rc(desc(steps=0)) == -1 and rc(desc(eps=0.0)) == -1 and rc(desc(src=0)) == -1
    assert rc(desc(dtype=7)) == -2
    need = h.saunet_newton_schulz_workspace(C.byref(desc()[0]))
    assert need > 0 and rc(desc(), need - 1) == -1 and rc(desc(), need, None) == -1 and rc(desc(), need, ws + 128) == -1
    assert rc(desc(coeff=(50.0, 50.0, 50.0))) == -5                    # singular values leave the range
    assert b"out of range" in h.saunet_last_error()
    d = desc(dtype=L.BF16)
    assert h.saunet_muon_step(C.byref(d[0]), ws, ws, 1 << 40, None) == -2
    assert h.saunet_muon_step(C.byref(desc()[0]), None, ws, 1 << 40, None) == -1


def test_create_optimizers_muon_splits_matrices_and_vectors():
    net = saunet_amd.SAUNet(num_classes=4)
    muon, adam = optim.create_optimizers(net, "muon", lr=1e-3)
    assert isinstance(muon, optim.FusedMuon) and isinstance(adam, optim.FusedAdam)
    a, b = ([p for g in o.param_groups for p in g["params"]] for o in (muon, adam))
    assert all(p.shape[0] > 1 and p.numel() > p.shape[0] for p in a)
    assert not {id(p) for p in a} & {id(p) for p in b}
    both = {id(p) for g in optim.group_weight(net) for p in g["params"]}
    assert {id(p) for p in a} | {id(p) for p in b} == both


# ------------------------------------------------------------------------------------------------ the iteration
SIZES = [(1, 1), (1, 7), (5, 1), (3, 2), (17, 17), (32, 32), (33, 40), (31, 1152), (32, 1152), (127, 129), (128, 128), (129, 300), (200, 64), (1000, 130),
         (257, 1025), (64, 5000), (300, 900), (2, 100003), (70001, 33), (1100, 1200)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_newton_schulz_sizes(m, n, dtype):
    for kind in ("gauss", "lowrank"):
        g = matrix(m, n, m * 10007 + n, dtype, kind).cuda()
        before = g.clone()
        check(HF.newton_schulz(g), g)
        assert torch.equal(g, before)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(832, 840), (833, 900), (900, 833), (500, 1535), (1537, 500), (129, 2700), (128, 4096), (4100, 128), (65, 8321), (35, 36)])
def test_newton_schulz_on_either_side_of_the_tile_rules(m, n):
    """13 and 14 blocks of 64 rows, Gram sums of up to and above 1536 columns, up to and above 128 blocks of 64 x 64 of X"""
    g = matrix(m, n, m + n, torch.float32, "lowrank").cuda()
    check(HF.newton_schulz(g), g)


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(520, 530)] + [(130, 131)] * 100, [(200, 210)] * 60, [(516, 140)] + [(300, 290)] * 30], ids=["short behind", "uniform", "two rounds"])
def test_lists_of_more_than_one_round_of_tiles(shapes):
    """more 64 x 64 tiles than run at once, with short and with equal reductions behind the first round"""
    gs = [matrix(*s, 11 + i).cuda() for i, s in enumerate(shapes)]
    for out, g in zip(HF.newton_schulz(gs), gs):
        check(out, g)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [96, 97, 130])
def test_lists_on_either_side_of_the_tile_rules(count):
    """one 64-row block each: 32 x 32 tiles up to 96 of them, 64 x 64 behind; the parameters of a Muon step get what the same matrices get alone"""
    gs = [matrix(33 + i % 32, 34 + (i * 7) % 60, i).cuda() for i in range(count)]
    for i, out in enumerate(HF.newton_schulz(gs)):
        check(out, gs[i])
    ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in gs]
    opt = optim.FusedMuon(ps, lr=0.5, momentum=0.0, weight_decay=0.0, nesterov=False)
    for p, g in zip(ps, gs):
        p.grad = g.clone()
    opt.step()
    for p, g in zip(ps, gs):
        rate = 0.5 * math.sqrt(max(1.0, g.shape[0] / g.shape[1]))
        check(-p.detach() / rate, g, noise=4 * 2.0 ** -24)              # the rate, its product, this division and the subtraction: half a step each


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 8, 9, 12])
def test_newton_schulz_steps(steps):
    for m, n in ((40, 200), (200, 70), (20, 50), (50, 7)):
        g = matrix(m, n, steps).cuda()
        check(HF.newton_schulz(g, steps=steps), g, steps=steps)


@pytest.mark.gpu
@pytest.mark.parametrize("coeff", [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (4.0848, -6.8946, 2.9270)])
def test_newton_schulz_coefficients(coeff):
    g = matrix(90, 160, 5).cuda()
    check(HF.newton_schulz(g, coefficients=coeff), g, coeff=coeff)


@pytest.mark.gpu
def test_newton_schulz_batches_lists_and_strides():
    gs = [matrix(*s, 70 + i) for i, s in enumerate([(8, 16), (130, 257), (32, 1152), (300, 20), (1, 5)])]
    for out, g in zip(HF.newton_schulz([g.cuda() for g in gs]), gs):
        check(out, g)
    batch = torch.stack([matrix(33, 50, i) for i in range(6)]).view(2, 3, 33, 50)
    out = HF.newton_schulz(batch.cuda())
    for i in range(6):
        check(out.view(6, 33, 50)[i], batch.view(6, 33, 50)[i])
    wide = matrix(60, 300, 3).cuda()
    for view in (wide[:, 7:201], wide[::2, 1:130], wide.t(), wide.t()[5:200, ::3], wide[:, ::2]):
        check(HF.newton_schulz(view), view)
    one = wide[:1].expand(4, 300)                                   # rows that share memory
    check(HF.newton_schulz(one), one)
    assert HF.newton_schulz(torch.zeros(0, 5).cuda()).shape == (0, 5) and HF.newton_schulz(torch.zeros(2, 0, 5).cuda()).shape == (2, 0, 5)


@pytest.mark.gpu
def test_newton_schulz_many_matrices():
    gs = [matrix(4 + i % 37, 3 + i % 41, i) for i in range(205)]
    for i, (out, g) in enumerate(zip(HF.newton_schulz([g.cuda() for g in gs]), gs)):
        if i % 5 == 0 or i > 195:
            check(out, g)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_newton_schulz_scale(scale):
    g = (matrix(40, 90, 1).double() * 100 * scale).float().cuda()      # the sum of squares leaves float32's range on both sides
    check(HF.newton_schulz(g, eps=1e-30), g, eps=1e-30)


@pytest.mark.gpu
def test_newton_schulz_of_matrices_without_full_rank():
    """what an eigenvalue of rounding noise does over many steps: zero rows, repeated rows, rank one.

    A direction of singular value zero holds what rounding puts there -- a half step of |X| or so in each of the first steps -- and every later step multiplies
    it by a: 2 a^steps 2^-24 of the result in all.  Any float32 chain has that (a random rank-24 matrix of this size, eight steps: 2.2e-4 both here and in the plain
    chain); the plain chain escapes it only where rows are equal bit for bit and stay so."""
    g = matrix(48, 120, 9)
    zero, twice, one = g.clone(), g.clone(), g[:, :1] @ g[:1]
    zero[10:40] = 0
    twice[24:] = twice[:24]
    small = twice[:, :100][8:36].clone()
    for steps in (5, 8):
        for x in (zero, twice, one, small, one[:20].clone()):
            check(HF.newton_schulz(x.cuda(), steps=steps), x, noise=2 * COEFF[0] ** steps * 2.0 ** -24, steps=steps)


@pytest.mark.gpu
def test_newton_schulz_zero_and_nonfinite_matrices_stay_apart():
    gs = [matrix(50, 80, i).cuda() for i in range(5)]
    gs[1].zero_()
    gs[2][3, 4] = float("nan")
    gs[3][7, 0] = float("inf")
    out = HF.newton_schulz(gs)
    assert not out[1].any()
    assert out[2].isnan().all() and out[3].isnan().all()
    check(out[0], gs[0]); check(out[4], gs[4])


@pytest.mark.gpu
def test_newton_schulz_on_a_side_stream_and_replayed():
    g = matrix(150, 400, 2).cuda()
    ref = HF.newton_schulz(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = HF.newton_schulz(g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, ref)
    graphs = []
    for k in range(2):
        x = g.clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = HF.newton_schulz(x)
        graphs.append((gr, x, y))
    for it in range(3):
        for k, (gr, x, y) in enumerate(graphs):
            x.copy_(matrix(150, 400, 10 * it + k).cuda())
            gr.replay()
        for k, (gr, x, y) in enumerate(graphs):
            assert torch.equal(y, HF.newton_schulz(x))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_newton_schulz_needs_no_gradient():
    g = matrix(8, 8, 0).cuda().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        HF.newton_schulz(g)
    with torch.no_grad():
        check(HF.newton_schulz(g), g.detach())


# ------------------------------------------------------------------------------------------------ the step
def muon64(p, g, buf, lr, mom, wd, nesterov, adjust, gs=1.0):
    """-> (parameter, buffer, the scaled update) in float64; p, g, buf as [rows, cols]"""
    g = g.double() * gs
    buf = mom * buf.double() + (1 - mom) * g
    u = (1 - mom) * g + mom * buf if nesterov else buf
    m, n = u.shape
    rate = lr * (0.2 * math.sqrt(max(m, n)) if adjust else math.sqrt(max(1, m / n)))
    o = chain(u, torch.float64)
    d32 = chain(u.float(), torch.float32).double() - o
    # u itself is formed in float32: three roundings of 2^-24 of it, carried through the iteration like any other operand's
    tol = rate * (4 * float(d32.abs().max()) * 2 + 64 * 2.0 ** -24 * float(o.abs().max()))
    return p.double() * (1 - lr * wd) - rate * o, buf, tol


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,adjust,wd", [(True, None, 0.1), (False, "original", 0.0), (True, "match_rms_adamw", 0.01)])
def test_muon_step(nesterov, adjust, wd):
    shapes = [(32, 128, 3, 3), (128, 96, 1, 1), (64, 3, 7, 7), (17, 17, 1, 1), (200, 30), (16, 8, 4, 4), (9, 2)]
    gen = torch.Generator().manual_seed(3)
    ps = [torch.nn.Parameter(torch.randn(*s, generator=gen).cuda()) for s in shapes]
    opt = optim.FusedMuon(ps, lr=0.03, momentum=0.9, weight_decay=wd, nesterov=nesterov, adjust_lr_fn=adjust)
    opt.grad_scale = 0.5
    bufs = [torch.zeros(s[0], math.prod(s[1:])) for s in shapes]
    for it in range(3):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).cuda()
        if it == 2:
            opt.param_groups[0]["lr"] = 0.01
            ps[3].grad = None
        old = [p.detach().cpu().view(p.shape[0], -1).clone() for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            got = p.detach().cpu().view(p.shape[0], -1).double()
            if p.grad is None:
                assert torch.equal(got, old[i].double())
                continue
            ref, buf, tol = muon64(old[i], p.grad.cpu().view(p.shape[0], -1), bufs[i], opt.param_groups[0]["lr"], 0.9, wd, nesterov, adjust == "match_rms_adamw", 0.5)
            hb = opt.state[p]["momentum_buffer"].cpu().view(p.shape[0], -1)
            assert float((hb.double() - buf).abs().max()) <= 4 * 2.0 ** -24 * float(buf.abs().max() + bufs[i].abs().max() + p.grad.abs().max())
            bufs[i] = hb
            # parameter: rounding of keep, of the product and of the sum
            assert float((got - ref).abs().max()) <= tol + 3 * 2.0 ** -24 * float(old[i].abs().max() + ref.abs().max())


@pytest.mark.gpu
def test_muon_state_dict_round_trip():
    def build():
        torch.manual_seed(1)
        return torch.nn.Conv2d(8, 24, 3, bias=False).cuda()
    a, b = build(), build()
    oa, ob = optim.FusedMuon(a.parameters(), lr=0.02), optim.FusedMuon(b.parameters(), lr=0.5)
    gs = [torch.randn(24, 8, 3, 3).cuda() for _ in range(3)]
    a.weight.grad = gs[0]; oa.step()
    b.load_state_dict(a.state_dict()); ob.load_state_dict(copy.deepcopy(oa.state_dict()))      # (without the copy both optimisers would hold one buffer)
    for g in gs[1:]:
        a.weight.grad, b.weight.grad = g.clone(), g.clone()
        oa.step(); ob.step()
    assert torch.equal(a.weight, b.weight)


@pytest.mark.gpu
def test_muon_step_captured_and_replayed_with_a_new_learning_rate():
    def build():
        torch.manual_seed(2)
        return [torch.nn.Parameter(torch.randn(40, 90).cuda()), torch.nn.Parameter(torch.randn(130, 20).cuda())]
    pa, pb = build(), build()
    oa, ob = optim.FusedMuon(pa, lr=0.02), optim.FusedMuon(pb, lr=0.02)
    grads = [torch.randn_like(p) for p in pa]
    for p, q, g in zip(pa, pb, grads):
        p.grad, q.grad = g.clone(), g.clone()
    step = saunet_amd.graph.GraphedStep(lambda: oa.step(upload=False), warmup=1, optimizers=[oa])
    ob.step()                                                            # the warm-up step
    for it in range(4):
        lr = 0.02 / (it + 1)
        oa.param_groups[0]["lr"] = ob.param_groups[0]["lr"] = lr
        for p, q in zip(pa, pb):
            g = torch.randn_like(p)
            p.grad.copy_(g); q.grad.copy_(g)
        step.replay()
        ob.step()
        for p, q in zip(pa, pb):
            assert torch.equal(p, q)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_muon_step_then_int8_inference_uses_the_new_weights():
    """the operators one behind the other, as a training program uses them: gradient, Muon step, validation with int8 convolutions"""
    saunet_amd.set_compute_dtype(torch.float32)
    torch.manual_seed(0)
    net = saunet_amd.SAUNet(num_classes=4).cuda()
    muon, adam = optim.create_optimizers(net, "muon", lr=1e-2)
    sm = saunet_amd.SegmentationModule(saunet_amd.DualLoss(mode="train"), net, 4)
    img, seg, edge = saunet_amd.data.synthetic_batch(2, 64, 64, seed=3)
    feed = {"image": img.cuda(), "mask": (seg.cuda(), edge.cuda())}
    layer = net.conv5[0]["denselayer3"]

    def block_input():
        seen = []
        hook = net.conv5[0].register_forward_hook(lambda m, i, o: seen.append((i[0].clone(), (o[0] if isinstance(o, tuple) else o).clone())))
        with torch.no_grad():
            net.eval()(feed["image"][:1])
        hook.remove()
        return seen[0]

    net.int8_inference()
    before = HF.folded_conv_bn_int8(layer.conv1.weight, layer.norm2)[0].dequantize()
    for _ in range(2):
        net.train()
        net.zero_grad(set_to_none=True)
        loss, _ = sm(feed, 1)
        loss.backward()
        old = layer.conv1.weight.detach().clone()
        g, b = layer.conv1.weight.grad.clone(), muon.state[layer.conv1.weight].get("momentum_buffer", torch.zeros_like(layer.conv1.weight)).clone()
        muon.step(); adam.step()
        ref, _, tol = muon64(old.cpu().flatten(1), g.cpu().flatten(1), b.cpu().flatten(1), 1e-2, 0.9, 1e-4, True, True)
        assert float((layer.conv1.weight.detach().cpu().flatten(1).double() - ref).abs().max()) <= tol + 3 * 2.0 ** -24 * float(old.abs().max() + ref.abs().max())
    x, y = block_input()
    assert torch.isfinite(y).all()
    with torch.no_grad():
        w, bias = HF.folded_conv_bn_int8(layer.conv1.weight, layer.norm2)
        scale = layer.norm2.weight / torch.sqrt(layer.norm2.running_var + layer.norm2.eps)
        want = layer.conv1.weight.flatten(1) * scale.view(-1, 1)
    assert not torch.equal(w.dequantize(), before)
    # one quantisation step of each row, half of it to either side, and the two roundings of the folded weight
    assert ((w.dequantize() - want).abs() <= w.scale[:, None] * 0.5 + 4 * 2.0 ** -24 * want.abs() + 2.0 ** -22 * w.scale[:, None] * 127).all()


@pytest.mark.gpu
def test_train_command_runs_with_muon(tmp_path):
    from saunet_amd import train
    hist = train.main(["--num_epoch", "1", "--synthetic", "4", "--size", "64", "--val_slices", "1", "--batch_size_per_gpu", "2", "--workers", "0",
                       "--optimizer", "muon", "--val_int8", "--lr_encoder", "1e-4", "--ckpt", str(tmp_path)])
    assert math.isfinite(hist["train"]["loss"][0])
