"""Cases that measure the matrix-update and 8-bit matrix-product operators of saunet_amd.

  newton_schulz   ``functional.newton_schulz``: the orthogonal factor of a matrix (or a batch of matrices) by an odd quintic iteration
  muon            ``optim.FusedMuon.step``: momentum, orthogonalised update, decoupled weight decay over a whole list of parameters
  matmul_int8     ``functional.matmul_int8``: int8 x int8 with one float32 scale a row (token, pixel) and one a channel
  linear_int8     ``functional.linear_int8``: the same product from floating-point rows, quantised on the way

``run`` computes them in their plain form (elementary torch operations) or, with ``own`` set, through the package.
"""
import math

import torch

own = False

COEFF = (3.4445, -4.7750, 2.0315)
NS_STEPS, NS_EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = torch.finfo(torch.float32).tiny

# every matrix-shaped convolution weight of SAUNet (4 classes, 32 filters) seen as [out, in * kh * kw], with its multiplicity
SAUNET = (
    [(32, 1152)] * 58 + [(128, 64 + 32 * i) for i in range(6)] + [(128, 128 + 32 * i) for i in range(12)] +
    [(128, 256 + 32 * i) for i in range(24)] + [(128, 512 + 32 * i) for i in range(16)] +
    [(64, 147), (128, 256), (256, 512), (512, 1024), (16, 144), (16, 144), (32, 288), (32, 288), (64, 576), (64, 576), (48, 576), (32, 576),
     (64, 2304), (128, 4608), (256, 9216), (512, 9216), (512, 13824), (512, 8192), (512, 8192), (256, 4096), (128, 2048), (48, 512),
     (32, 64), (64, 128), (128, 8), (8, 128), (256, 16), (16, 256), (512, 32), (32, 512), (17, 17), (33, 33), (9, 9), (16, 32), (8, 16)])
DENSE_LAYER = [(128, 256), (32, 1152)]
SETS = {"saunet": SAUNET, "layer": DENSE_LAYER}


def listed():
    return [
        # the second convolution of one DenseNet layer: the smallest call, a chain of dependent products where latency is all
        {"name": "ns_layer_f32", "op": "newton_schulz", "batch": 1, "rows": 32, "cols": 1152, "dtype": "f32"},
        # the widest decoder convolution (1536 -> 512 channels, 3 x 3): a short, very wide matrix
        {"name": "ns_decoder_f32", "op": "newton_schulz", "batch": 1, "rows": 512, "cols": 13824, "dtype": "f32"},
        # a stack of classifier-shaped updates in bfloat16: ragged sizes, several matrices in one call
        {"name": "ns_stack_bf16", "op": "newton_schulz", "batch": 6, "rows": 1000, "cols": 1024, "dtype": "bf16"},
        # a large square projection, float32
        {"name": "ns_square_f32", "op": "newton_schulz", "batch": 1, "rows": 4096, "cols": 4096, "dtype": "f32"},
        # one DenseNet layer's two weights: the smallest optimiser step
        {"name": "muon_layer", "op": "muon", "set": "layer", "scale": 1.0},
        # the optimiser step of the whole network: a hundred and fifty matrices between 8 x 16 and 512 x 13824
        {"name": "muon_saunet", "op": "muon", "set": "saunet", "scale": 1.0},
        # quantised activations of a dense block at 64 x 64 pixels, batch 32, through the bottleneck's 1 x 1 convolution (few output channels)
        {"name": "mm8_pixels_bf16", "op": "matmul_int8", "rows": 131072, "k": 256, "cols": 128, "dtype": "bf16", "bias": True, "relu": True},
        # odd everything: rows, depth and channels that fill no tile
        {"name": "mm8_ragged_f32", "op": "matmul_int8", "rows": 777, "k": 1001, "cols": 515, "dtype": "f32", "bias": True, "relu": False},
        # a large product, where the matrix cores are the bound
        {"name": "mm8_large_bf16", "op": "matmul_int8", "rows": 8192, "k": 4096, "cols": 4096, "dtype": "bf16", "bias": False, "relu": False},
        # one token through a square layer: the weight is read once and nothing else counts
        {"name": "lin8_token_bf16", "op": "linear_int8", "rows": 1, "k": 4096, "cols": 4096, "dtype": "bf16", "bias": True, "relu": False},
        # a handful of tokens through a wide layer, half precision
        {"name": "lin8_tokens_f16", "op": "linear_int8", "rows": 24, "k": 2048, "cols": 8192, "dtype": "f16", "bias": False, "relu": True},
        # floating-point pixels (16 x 16 map, batch 32, transition of the third dense block) quantised inside the call
        {"name": "lin8_pixels_bf16", "op": "linear_int8", "rows": 8192, "k": 1024, "cols": 512, "dtype": "bf16", "bias": True, "relu": True},
    ]


def _spread(rng, lo, hi):
    """a whole number between lo and hi, even over the logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["newton_schulz", "muon", "matmul_int8", "linear_int8"])
    if op == "newton_schulz":
        while True:
            c = {"op": op, "batch": rng.choice([1, 1, 2, 3, 7]), "rows": _spread(rng, 1, 4096), "cols": _spread(rng, 1, 14000),
                 "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
            if work(c)["flops"] <= work({"op": op, "batch": 1, "rows": 4096, "cols": 4096, "dtype": "f32"})["flops"]:
                return c
    if op == "muon":
        return {"op": op, "set": rng.choice(["layer", "saunet"]), "scale": rng.choice([0.3, 0.5, 0.7, 0.9]) + rng.random() * 0.1}
    big = 8192 * 4096 * 4096 if op == "matmul_int8" else 8192 * 1024 * 512
    while True:
        rows = rng.choice([_spread(rng, 1, 64), _spread(rng, 64, 150000)])
        c = {"op": op, "rows": rows, "k": _spread(rng, 8, 8192), "cols": _spread(rng, 1, 8192), "dtype": rng.choice(["bf16", "f16", "f32"]),
             "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}
        if rows * c["k"] * c["cols"] <= big and rows * (c["k"] + c["cols"]) <= 1 << 27:
            return c


def _shapes(case):
    if case["op"] == "newton_schulz":
        return [(case["rows"], case["cols"])] * case["batch"]
    s = case["scale"]
    return [(max(1, int(m * s)), max(1, int(n * s))) for m, n in SETS[case["set"]]]


def _ns_flops(m, n):
    """Least arithmetic of the iteration: m <= n.  Either every step forms the m x m Gram matrix (symmetric: m^2 n), its square (m^3) and the
    product with the matrix (2 m^2 n), or three and two steps are composed on the Gram matrix (14 symmetric m x m products in all)."""
    m, n = min(m, n), max(m, n)
    return min(NS_STEPS * (3 * m * m * n + m ** 3), 6 * m * m * n + 14 * m ** 3)


def work(case):
    op = case["op"]
    if op in ("newton_schulz", "muon"):
        elems = sum(m * n for m, n in _shapes(case))
        flops = sum(_ns_flops(m, n) for m, n in _shapes(case))
        if op == "muon":       # gradient read, momentum and parameter read and written
            return {"bytes": 20 * elems, "flops": flops + 8 * elems}
        return {"bytes": 2 * elems * (4 if case["dtype"] == "f32" else 2), "flops": flops}
    m, k, n = case["rows"], case["k"], case["cols"]
    size = 4 if case["dtype"] == "f32" else 2
    a = m * k if op == "matmul_int8" else m * k * size
    scales = 4 * n + (4 * m if op == "matmul_int8" else 0) + (4 * n if case["bias"] else 0)
    return {"bytes": a + n * k + m * n * size + scales, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _gradient(m, n, g):
    """what a weight gradient looks like: a few strong directions over a floor of noise, rows of different size"""
    r = max(1, min(m, n) // 16)
    low = torch.randn(m, r, generator=g, device="cuda") @ torch.randn(r, n, generator=g, device="cuda")
    x = low / math.sqrt(r) + 0.5 * torch.randn(m, n, generator=g, device="cuda")
    return 1e-3 * x * torch.exp(0.5 * torch.randn(m, 1, generator=g, device="cuda"))


def _activations(m, k, dtype, g):
    """normalised activations with a few channels that run hot"""
    hot = torch.exp(1.2 * torch.randn(1, k, generator=g, device="cuda"))
    return (torch.randn(m, k, generator=g, device="cuda") * hot).to(dtype)


def _quantised(x):
    """the definition of a quantised row in float64: scale = fl32(max |x| / 127), q = round-half-even(x / scale)"""
    top = x.abs().amax(1).to(torch.float32)
    scale = (top.double() / 127.0).to(torch.float32)
    scale = torch.where(scale < TINY, torch.zeros_like(scale), scale)
    q = torch.where(scale[:, None] > 0, (x.double() / scale.double()[:, None]).round(), torch.zeros((), dtype=torch.float64, device=x.device))
    return q.to(torch.int8), scale


def _inputs(case, seed):
    g = _gen(seed)
    op = case["op"]
    st = {"op": op}
    if op == "newton_schulz":
        dt = DTYPES[case["dtype"]]
        mats = torch.stack([_gradient(m, n, g).to(dt) for m, n in _shapes(case)])
        st["g"] = mats if case["batch"] > 1 else mats[0]
        return st
    if op == "muon":
        shapes = _shapes(case)
        # parameters and momentum live in one flat buffer each, every tensor on a 256-byte border, as a program with bucketed storage keeps them
        at = [0]
        for r, c in shapes:
            at.append(at[-1] + (r * c + 63) // 64 * 64)
        st["flat"] = torch.zeros(2, at[-1], device="cuda")
        st["params"], st["bufs"] = [], []
        for (r, c), o in zip(shapes, at):
            w, b = (f[o:o + r * c].view(r, c) for f in st["flat"])
            w.copy_(torch.randn(r, c, generator=g, device="cuda") * math.sqrt(2.0 / c))
            b.copy_(0.3 * _gradient(r, c, g))
            st["params"].append(torch.nn.Parameter(w))
            st["params"][-1].grad = _gradient(r, c, g)
            st["bufs"].append(b)
        return st
    m, k, n = case["rows"], case["k"], case["cols"]
    dt = DTYPES[case["dtype"]]
    x = _activations(m, k, dt, g)
    st["w"], st["ws"] = _quantised(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k))
    st["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
    st["relu"], st["dtype"] = case["relu"], dt
    if op == "matmul_int8":
        st["a"], st["as"] = _quantised(x)
    else:
        st["x"] = x
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own and st["op"] == "muon":
        from saunet_amd import optim
        st["opt"] = optim.FusedMuon(st["params"], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY)
        for p, b in zip(st["params"], st["bufs"]):
            st["opt"].state[p]["momentum_buffer"] = b
    elif own and "w" in st:
        from saunet_amd import functional as HF
        st["hw"] = HF.Int8Rows(st["w"], st["ws"])
        if "a" in st:
            st["ha"] = HF.Int8Rows(st["a"], st["as"])
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _orthogonalise(g, dtype):
    a, b, c = COEFF
    x = g.to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    norm = (x * x).sum(dim=(-2, -1), keepdim=True).sqrt()
    x = x / norm.clamp(min=NS_EPS)
    for _ in range(NS_STEPS):
        s = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.transpose(-2, -1).contiguous() if tall else x


def _muon_plain(st):
    for p, buf in zip(st["params"], st["bufs"]):
        w, g = p.data, p.grad
        buf.copy_(MOMENTUM * buf + (1 - MOMENTUM) * g)
        o = _orthogonalise((1 - MOMENTUM) * g + MOMENTUM * buf, torch.float32)
        rate = LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        w.copy_(w * (1 - LR * DECAY) - rate * o)


def _product_plain(a, sa, w, sw, bias, relu, dtype):
    y = torch.matmul(a.float(), w.float().t()) * sa[:, None] * sw[None, :]
    if bias is not None:
        y = y + bias
    return (y.clamp(min=0) if relu else y).to(dtype)


def run(st):
    op = st["op"]
    if own:
        from saunet_amd import functional as HF
        if op == "newton_schulz":
            return HF.newton_schulz(st["g"], steps=NS_STEPS, coefficients=COEFF, eps=NS_EPS)
        if op == "muon":
            st["opt"].step()
            return st["flat"]
        if op == "matmul_int8":
            return HF.matmul_int8(st["ha"], st["hw"], bias=st["bias"], relu=st["relu"], dtype=st["dtype"])
        return HF.linear_int8(st["x"], st["hw"], bias=st["bias"], relu=st["relu"])
    if op == "newton_schulz":
        return _orthogonalise(st["g"], torch.float32).to(st["g"].dtype)
    if op == "muon":
        _muon_plain(st)
        return st["flat"]
    if op == "matmul_int8":
        return _product_plain(st["a"], st["as"], st["w"], st["ws"], st["bias"], st["relu"], st["dtype"])
    q, scale = _quantised(st["x"])
    return _product_plain(q, scale, st["w"], st["ws"], st["bias"], st["relu"], st["dtype"])


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def _polar64(g):
    """p_k(s) applied to the singular values, written on the smaller Gram matrix: X <- X + ... as a polynomial in X X^T (or X^T X)"""
    a, b, c = COEFF
    x = g.double()
    x = x / max(float(torch.linalg.vector_norm(x)), NS_EPS)
    for _ in range(NS_STEPS):
        if x.shape[0] <= x.shape[1]:
            s = x @ x.T
            x = a * x + s @ (b * x + c * (s @ x))
        else:
            s = x.T @ x
            x = a * x + (b * x + c * (x @ s)) @ s
    return x


def _product64(q, sq, w, sw, bias, relu):
    out = torch.empty(q.shape[0], w.shape[0], dtype=torch.float64, device=q.device)
    wd = w.double().T
    for i in range(0, q.shape[0], 8192):
        out[i:i + 8192] = q[i:i + 8192].double() @ wd
    out *= sq.double()[:, None] * sw.double()
    if bias is not None:
        out += bias.double()
    return out.relu_() if relu else out


def exact(case, seed):
    st = _inputs(case, seed)
    op = case["op"]
    if op == "newton_schulz":
        return torch.stack([_polar64(x) for x in st["g"]]) if case["batch"] > 1 else _polar64(st["g"])
    if op == "muon":
        out = torch.zeros(st["flat"].shape, dtype=torch.float64, device="cuda")
        first = st["flat"].data_ptr()
        for p, b in zip(st["params"], st["bufs"]):
            w, g, b = p.detach().double(), p.grad.double(), b.double()
            b = b + (1 - MOMENTUM) * (g - b)
            o = _polar64(g + MOMENTUM * (b - g))
            at = (p.data_ptr() - first) // 4
            out[0, at:at + w.numel()] = (w - LR * DECAY * w - LR * max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * o).flatten()
            out[1, at:at + w.numel()] = b.flatten()
        return out
    if op == "matmul_int8":
        return _product64(st["a"], st["as"], st["w"], st["ws"], st["bias"], st["relu"])
    x = st["x"].double()
    scale = (x.abs().max(dim=1).values / 127).float()
    scale[scale < TINY] = 0
    q = torch.round(x / scale.double()[:, None])
    q[scale == 0] = 0
    return _product64(q, scale, st["w"], st["ws"], st["bias"], st["relu"])
