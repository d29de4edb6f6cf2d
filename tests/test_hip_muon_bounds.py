"""What the Newton-Schulz kernels and the Muon step do at the borders of their domain: coefficients beside the range that the float16 pairs hold, matrices
below eps, lists that outgrow one workspace, lists of long and short matrices, arguments that have to be refused."""
import ctypes as C
import math
import random

import numpy as np
import pytest
import torch

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


# ------------------------------------------------------------------------------------------------ the number format (no GPU needed)
def test_what_a_pair_of_float16_holds():
    """the figures that the tolerances below count with: x = hi + lo to 2^-23 of x, and |lo| <= 2^-11 |x|"""
    x = np.float32(1) + np.random.default_rng(0).integers(0, 1 << 23, 1 << 20).astype(np.float32) * np.float32(2.0 ** -23)
    hi = x.astype(np.float16)
    rest = x - hi.astype(np.float32)                                     # exact
    lo = rest.astype(np.float16)
    off = np.abs(x.astype(np.float64) - hi.astype(np.float64) - lo.astype(np.float64)) / x
    assert off.max() <= 2.0 ** -23 and (np.abs(lo.astype(np.float64)) <= 2.0 ** -11 * x).all()
    assert 0.2 < (off > 2.0 ** -24).mean() < 0.3


# ------------------------------------------------------------------------------------------------ coefficients (no GPU needed)
def workspace(rows, cols, steps, coeff):
    """bytes, or the status of a call that cannot be made: nothing is launched"""
    d, hold = HF.ns_desc([0, 0, 0, cols, cols, rows, cols], L.F32, steps, coeff, 1e-7)
    return L.load().saunet_newton_schulz_workspace(C.byref(d))


def largest(steps, coeff, first, later, x):
    """the largest |eigenvalue| of anything that the chain keeps, over the starting singular values x: X, S = X^2, R = (a + P) S and, of the composed
    product of the factors a + P, what is kept of it"""
    a, b, c = (float(np.float32(v)) for v in coeff)
    top, done = 0.0, 0
    with np.errstate(all="ignore"):
        while done < steps:
            nb = min(steps - done, later if done else first)
            base = 1.0 if done else a
            t = np.ones_like(x)
            for j in range(nb):
                s = x * x
                f = a + (c * s + b) * s
                t = t * f
                kept = [s, f - base, t - base ** (j + 1)] + ([f * s] if j < nb - 1 else [])
                top = max([top] + [float(np.abs(v).max()) for v in kept])
                x = f * x
            done += nb
            if done < steps:
                top = max(top, float(np.abs(x).max()))
    return top


def test_a_peak_between_two_samples_is_refused():
    # a polynomial of degree 5^5 whose largest value, 2e8, is taken on an interval far narrower than a hundredth of its domain
    for steps in (5, 6, 8):
        assert workspace(300, 400, steps, (1.5012, -3.8716, 1.2536)) == -5
    assert b"out of range" in L.load().saunet_last_error()
    assert workspace(300, 400, 5, COEFF) > 0


def test_accepted_coefficients_stay_in_range():
    """everything kept stays below 4096, the limit of the scales, on a fine grid; and the usual
    coefficients are accepted"""
    x = np.linspace(0, 1, 200001) ** 4
    rng = random.Random(5)
    accepted = 0
    for i in range(600):
        coeff, steps = (rng.uniform(0.5, 4.0), rng.uniform(-8, 1), rng.uniform(-1, 4)), (3, 5, 8)[i % 3]
        rows, first, later = ((64, 1, 1), (200, 2, 2), (300, 3, 2))[i // 3 % 3]
        if workspace(rows, 400, steps, coeff) < 0:
            continue
        accepted += 1
        # (float32's rounding of the coefficients aside, the host's interval is exact)
        assert largest(steps, coeff, first, later, x) <= 4096 * (1 + 1e-6), (coeff, steps, rows)
    assert accepted > 60
    for coeff in (COEFF, (1.5, -0.5, 0.0), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (4.0848, -6.8946, 2.9270)):
        for rows in (20, 64, 200, 300):
            for steps in (1, 5, 12, 32):
                assert workspace(rows, 400, steps, coeff) > 0


@pytest.mark.gpu
def test_a_narrow_finite_peak_comes_out_finite():
    """one singular value where (a + P) S reaches 1346 and X 451, twenty times what the neighbourhood suggests.

    Tolerance: after three steps X = 1.55 carries the rounding of a product kept to 30 with 2^-21 of it, 1.4e-5; the two steps behind multiply that by their
    slopes, 30 and 860: 0.4 of 451, and as much again from the second block's own matrices (289 kept with 2^-21): below one per cent."""
    coeff, peak = (3.04314876, -6.77973318, 2.62109327), 0.9766965
    gen = torch.Generator().manual_seed(4)
    m, n = 260, 300
    u, v = torch.linalg.qr(torch.randn(m, m, generator=gen, dtype=torch.float64))[0], torch.linalg.qr(torch.randn(n, m, generator=gen, dtype=torch.float64))[0]
    s = torch.full((m,), math.sqrt((1 - peak * peak) / (m - 1)), dtype=torch.float64)
    s[0] = peak
    g = ((u * s) @ v.t()).float()
    out = HF.newton_schulz(g.cuda(), coefficients=coeff).cpu()
    ref = chain(g, torch.float64, coeff=coeff)
    assert 400 < float(ref.norm()) < 500 and torch.isfinite(out).all()
    assert float((out.double() - ref).norm()) <= 0.01 * float(ref.norm())


# ------------------------------------------------------------------------------------------------ lists that outgrow one workspace
def test_the_workspace_of_a_long_list_is_bounded():
    def need(shapes):
        d, hold = HF.ns_desc([v for m, n in shapes for v in (0, 0, 0, n, n, m, n)], L.F32, 5, COEFF, 1e-7)
        return L.load().saunet_newton_schulz_workspace(C.byref(d))

    one = need([(4096, 4096)])
    assert 32 * 4096 ** 2 <= one <= 32 * 4096 ** 2 + (1 << 27)
    cap = (4 << 30) + (1 << 28)
    for shapes in ([(4096, 4096)] * 32, [(4096, 11008)] * 100, [(300, 700)] * 4000, [(24, 1152), (2000, 2100), (100, 9000)] * 1300):
        assert one < need(shapes) <= cap
    assert need([(16384, 16384)] * 3) <= need([(16384, 16384)]) + (1 << 28)            # a matrix of 8 GiB is a part of its own
    assert need([(30, 30)] * 4096) < 1 << 28


@pytest.mark.gpu
def test_a_list_of_more_matrices_than_a_call_takes():
    gs = [1e-2 * torch.randn(3 + i % 5, 4 + i % 3, generator=torch.Generator().manual_seed(i)) for i in range(L.NS_ITEMS_MAX + 5)]
    outs = HF.newton_schulz([g.cuda() for g in gs])
    ps = [torch.nn.Parameter(torch.zeros(g.shape).cuda()) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = g.cuda()
    optim.FusedMuon(ps, lr=0.5, momentum=0.0, weight_decay=0.0, nesterov=False).step()
    for i in list(range(0, 40)) + list(range(L.NS_ITEMS_MAX - 3, L.NS_ITEMS_MAX + 5)):
        ref = chain(gs[i], torch.float64)
        tol = 4 * float((chain(gs[i], torch.float32).double() - ref).norm()) + 128 * 2.0 ** -24 * float(ref.norm())
        assert float((outs[i].cpu().double() - ref).norm()) <= tol
        rate = 0.5 * math.sqrt(max(1.0, ref.shape[0] / ref.shape[1]))
        assert float((-ps[i].detach().cpu().double() / rate - ref).norm()) <= tol + 4 * 2.0 ** -24 * float(ref.norm())


@pytest.mark.gpu
def test_a_list_that_goes_in_parts():
    """1400 matrices, 7 GiB of intermediate matrices: each as exact as alone, the first, the last and those around the border between the parts among them.
    The Muon step of the same list too.  Tolerance: see the matrices below eps; s is not small here, so 128 d bounds the chain's own roundings of the last step"""
    shapes = [(600, 700), (310, 40), (20, 300), (450, 460)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    gs = [1e-2 * torch.randn(*shapes[i % 4], generator=gen, device="cuda") for i in range(1400)]
    d, hold = HF.ns_desc([v for g in gs for v in (0, 0, 0, g.shape[1], g.shape[1], *g.shape)], L.F32, 5, COEFF, 1e-7)
    assert sum(12 * m * n + 20 * min(m, n) ** 2 for m, n in (g.shape for g in gs)) > L.load().saunet_newton_schulz_workspace(C.byref(d)) > 1 << 31
    outs = HF.newton_schulz(gs)
    flat = [torch.nn.Parameter(torch.zeros_like(g)) for g in gs]
    for p, g in zip(flat, gs):
        p.grad = g
    optim.FusedMuon(flat, lr=0.5, momentum=0.0, weight_decay=0.0, nesterov=False).step()
    for i, (g, out, p) in enumerate(zip(gs, outs, flat)):
        size = 0.5 * math.sqrt(max(1.0, g.shape[0] / g.shape[1]))
        near = (-p.detach() / size - out).norm() <= 2e-5 * out.norm()        # all of them are there (a matrix left out or mixed up is off by its size)
        assert near and out.norm() > 0, i
        if i % 97 and i not in (1, 1398, 1399):
            continue
        ref = chain(g.cpu(), torch.float64)
        tol = 4 * float((chain(g.cpu(), torch.float32).double() - ref).norm()) + 128 * 2.0 ** -24 * float(ref.norm())
        assert float((out.cpu().double() - ref).norm()) <= tol
        assert float((-p.detach().cpu().double() / size - ref).norm()) <= tol + 4 * 2.0 ** -24 * float(ref.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("shapes,dtype", [([(1000, 1024)] * 6, torch.bfloat16), ([(300, 900)], torch.float32), ([(520, 530)] + [(130, 131)] * 100, torch.float32),
                                          ([(200, 210)] * 60, torch.float16), ([(64, 5000), (30, 40)], torch.float32)],
                         ids=["stack", "one", "short behind", "uniform", "wide"])
def test_a_call_repeats_itself_bit_for_bit(shapes, dtype):
    """whatever the workspace held before"""
    gen = torch.Generator(device="cuda").manual_seed(2)
    gs = [(1e-2 * torch.randn(*s, generator=gen, device="cuda")).to(dtype) for s in shapes]
    ref = [x.clone() for x in HF.newton_schulz(gs)]
    for i in range(4):
        junk = torch.full((1 << 27,), (float("nan"), 1e30, float("-inf"), 0.0)[i], device="cuda")
        del junk
        assert all(torch.equal(a, b) for a, b in zip(HF.newton_schulz(gs), ref))


# ------------------------------------------------------------------------------------------------ matrices below eps
@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(40, 90), (300, 500), (700, 140), (1100, 1200), (20, 60), (200, 4000)])
def test_matrices_whose_norm_is_below_eps_keep_their_digits(m, n):
    """X = G / eps there, far below one: the result is small and as exact as any other.  Matrices of both kinds in one call.

    Tolerance, in half steps d = 2^-24 of float32, for singular values so small that every factor is a I + (next to nothing): a composed factor keeps
    q + Q with |Q| below q's size, 2 d + 4 d (its two operands) + 4 d (the dropped low parts) a product, at most six products and three applications of it, the
    stored X, 2 d each time, and the result's own rounding: below 100 d.  Where s is not small the float32 chain is the yardstick as everywhere."""
    gen = torch.Generator().manual_seed(m)
    gs, ratio = [], [1e3, 0.7, 1e-2, 1e-4, 1e-6, 1e-9, 1e-14, 1e-30]
    for r in ratio:
        g = torch.randn(m, n, generator=gen)
        gs.append((g.double() / g.double().norm() * 1e-7 * r).float() if r > 1e-20 else torch.zeros(m, n).index_put_((torch.tensor(m - 1), torch.tensor(1)), torch.tensor(1e-37)))
    for out, g, r in zip(HF.newton_schulz([g.cuda() for g in gs]), gs, ratio):
        ref = chain(g, torch.float64)
        d32 = (chain(g, torch.float32).double() - ref).norm()
        tol = 4 * float(d32) + 100 * 2.0 ** -24 * float(ref.norm()) + 2.0 ** -149 * (m * n) ** 0.5
        assert float((out.cpu().double() - ref).norm()) <= tol, (r, float((out.cpu().double() - ref).norm()), float(ref.norm()))
    for dtype in (torch.bfloat16, torch.float16):
        g = gs[2].to(dtype) if dtype == torch.bfloat16 else (gs[2] * 1e4).half()
        eps = 1e-7 if dtype == torch.bfloat16 else 1e-2
        out = HF.newton_schulz(g.cuda(), eps=eps).cpu()
        ref = chain(g, torch.float64, eps=eps)
        tol = 4 * float((chain(g, torch.float32, eps=eps).double() - ref).norm()) + (100 * 2.0 ** -24 + torch.finfo(dtype).eps / 2) * float(ref.norm())
        assert float((out.double() - ref).norm()) <= tol + (2.0 ** -25 * (m * n) ** 0.5 if dtype == torch.float16 else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(40, 90), (150, 120), (300, 500)])
@pytest.mark.parametrize("steps", [8, 11, 14, 20])
def test_matrices_below_eps_grow_into_range(m, n, steps):
    """X grows by 3.4445 a step until it arrives near one, in the middle of a block or between two: the scale t ends at 1 wherever that is"""
    gen = torch.Generator().manual_seed(m + steps)
    gs = []
    for r in (0.3, 1e-2, 1e-4, 1e-5, 1e-6, 1e-8):
        g = torch.randn(m, n, generator=gen)
        gs.append((g.double() / g.double().norm() * 1e-7 * r).float())
    for out, g in zip(HF.newton_schulz([g.cuda() for g in gs], steps=steps), gs):
        ref = chain(g, torch.float64, steps=steps)
        # as above, one more product and application for every further step (100 / 5 a step)
        tol = 4 * float((chain(g, torch.float32, steps=steps).double() - ref).norm()) + 20 * steps * 2.0 ** -24 * float(ref.norm())
        assert float((out.cpu().double() - ref).norm()) <= tol, (float(g.double().norm()), float((out.cpu().double() - ref).norm()), tol)


@pytest.mark.gpu
def test_muon_update_of_a_gradient_below_eps():
    gen = torch.Generator().manual_seed(8)
    ps, gs = [], []
    for m, n, r in ((60, 100, 1e-5), (300, 400, 1e-5), (24, 50, 1e-5), (90, 80, 1e3)):
        g = torch.randn(m, n, generator=gen)
        gs.append((g.double() / g.double().norm() * 1e-7 * r).float())
        ps.append(torch.nn.Parameter(torch.zeros(m, n).cuda()))
        ps[-1].grad = gs[-1].cuda()
    optim.FusedMuon(ps, lr=0.5, momentum=0.0, weight_decay=0.0, nesterov=False).step()
    for p, g in zip(ps, gs):
        ref = -0.5 * math.sqrt(max(1.0, g.shape[0] / g.shape[1])) * chain(g, torch.float64)
        d32 = -0.5 * math.sqrt(max(1.0, g.shape[0] / g.shape[1])) * chain(g, torch.float32).double() - ref
        # as above; the rate and the product with it two roundings more
        assert float((p.detach().cpu().double() - ref).norm()) <= 4 * float(d32.norm()) + 102 * 2.0 ** -24 * float(ref.norm())


# ------------------------------------------------------------------------------------------------ lists of long and short matrices
def composed(g, dtype, first=3, later=2, coeff=COEFF, eps=1e-7):
    """five steps of the chain with `first` and then `later` of them composed on the m x m matrices before X is touched: S' = (a + P)^2 S and Q, the product
    of the factors a + P less the product of the a, with P = b S + c S^2 in the first block and (a - 1) more, a = 1, behind it"""
    a0, b, c = coeff
    x = g.to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    x = x / x.double().norm().clamp(min=eps).to(dtype)
    done = 0
    while done < 5:
        nb = min(5 - done, later if done else first)
        a = 1.0 if done else a0
        s = x @ x.t()
        eye = torch.eye(s.shape[0], dtype=dtype)
        for j in range(nb):
            p = b * s + c * (s @ s) + (a0 - a) * eye
            big, q = (p, a) if j == 0 else (a * big + q * p + p @ big, q * a)
            if j < nb - 1:
                r = a * s + p @ s
                s = a * r + r @ p
        x = q * x + big @ x
        done += nb
    return x.t().contiguous() if tall else x


LISTS = {"40 to 300 rows": [(40, 90), (300, 500), (700, 200), (20, 60), (33, 40), (171, 70), (128, 736), (64, 576), (257, 33)],
         "wide and tall": [(520, 4000), (33, 50), (4000, 520), (100, 3000)],
         "few": [(130, 140), (40, 50)]}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("kind", ["gauss", "lowrank"])
def test_muon_update_in_a_list_of_long_and_short_matrices(name, kind):
    """One matrix of more than 128 rows takes the whole list of a Muon step into the composed chain; the bare update (parameters zero) of each.

    Tolerance: an operand of a product is off by 2^-23 of itself and the dropped low parts are another 2^-22 of the product, four times float32's two half
    steps; so four times the distance of the same composed recurrences in float32, and 128 half steps of the result for inputs on which those are exact by
    luck.  The rate, its product, this division and the subtraction are half a step each.  Both rules of the rate, and a parameter that is not zero."""
    gen = torch.Generator().manual_seed(12)
    shapes = LISTS[name]
    gs = []
    for m, n in shapes:
        g = torch.randn(m, n, generator=gen)
        if kind == "lowrank":
            r = max(1, min(m, n) // 16)
            g = torch.randn(m, r, generator=gen) @ torch.randn(r, n, generator=gen) / r ** 0.5 + 0.5 * g
        gs.append(1e-3 * g)
    refs, tols = [], []
    for g in gs:
        ref = chain(g, torch.float64)
        assert float((composed(g, torch.float64) - ref).norm()) <= 1e-9 * float(ref.norm())
        own = chain if min(g.shape) <= 32 else composed
        refs.append(ref)
        tols.append(4 * float((own(g, torch.float32).double() - ref).norm()) + 128 * 2.0 ** -24 * float(ref.norm()))
    for adjust, wd, p0 in ((None, 0.0, 0.0), ("match_rms_adamw", 0.1, 0.5)):
        starts = [p0 * torch.randn(g.shape, generator=gen) for g in gs]
        ps = [torch.nn.Parameter(p.cuda()) for p in starts]
        for p, g in zip(ps, gs):
            p.grad = g.cuda()
        optim.FusedMuon(ps, lr=0.25, momentum=0.0, weight_decay=wd, nesterov=False, adjust_lr_fn=adjust).step()
        for p, start, ref, tol in zip(ps, starts, refs, tols):
            m, n = ref.shape
            rate = 0.25 * (0.2 * math.sqrt(max(m, n)) if adjust else math.sqrt(max(1, m / n)))
            want = start.double() * (1 - 0.25 * wd) - rate * ref
            d = float((p.detach().cpu().double() - want).norm())
            assert d <= rate * (tol + 4 * 2.0 ** -24 * float(ref.norm())) + 3 * 2.0 ** -24 * float(start.norm() + want.norm()), (m, n, d / rate, tol)


# ------------------------------------------------------------------------------------------------ the step's arguments
def test_whole_steps_of_any_number_type():
    for steps in (5, 5.0, np.int64(5), np.float32(5)):
        HF.ns_check_hyper(steps, COEFF, 1e-7)
        assert HF.ns_desc([0] * 7, L.F32, steps, COEFF, 1e-7)[0].steps == 5


@pytest.mark.gpu
@pytest.mark.parametrize("make", [lambda ps: optim.FusedMuon(ps), lambda ps: optim.FusedSGD(ps, lr=0.1), lambda ps: optim.FusedAdam(ps), lambda ps: optim.FusedRAdam(ps)],
                         ids=["muon", "sgd", "adam", "radam"])
def test_a_group_that_begins_on_the_cpu_is_refused(make):
    """the hyper-parameters lie beside the group's first parameter: on the CPU no kernel may read them"""
    host, dev = torch.nn.Parameter(torch.ones(4, 4)), torch.nn.Parameter(torch.ones(4, 4).cuda())
    dev.grad = torch.ones_like(dev)
    with pytest.raises(RuntimeError, match="GPU only"):
        make([host, dev]).step()
    assert (dev == 1).all()


@pytest.mark.gpu
def test_muon_step_evaluates_its_closure():
    torch.manual_seed(0)
    w = torch.nn.Parameter(torch.randn(8, 12).cuda())
    x = torch.randn(12, 5).cuda()
    ref = torch.nn.Parameter(w.detach().clone())
    a, b = optim.FusedMuon([w], lr=0.1), optim.FusedMuon([ref], lr=0.1)

    def closure():
        a.zero_grad()
        loss = (w @ x).square().sum()
        loss.backward()
        return loss

    for _ in range(2):
        want = (ref @ x).square().sum()
        b.zero_grad()
        want.backward()
        loss = a.step(closure)
        b.step()
        assert torch.equal(loss, want) and torch.equal(w, ref)
    assert b.step() is None
