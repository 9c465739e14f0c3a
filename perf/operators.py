"""Measured cases of the decoder operators: group normalisation with an activation over channels-last feature
images, and the orthogonalised (Newton-Schulz) update of weight matrices with the optimizer step around it.

A feature image is what the rasteriser blends from ``custom_features``: ``[B, H, W, C]``, channels last.  A case is
a dict of plain values; ``run`` makes one pass through one operator, in its plain form or (``own``) through the
package's entry points.
"""
import math

import torch

own = False

NS = (3.4445, -4.775, 2.0315)     # coefficients of the quintic Newton-Schulz step
NS_STEPS = 5
NS_EPS = 1e-7
GN_EPS = 1e-5
LR, WEIGHT_DECAY, MOMENTUM = 0.02, 0.01, 0.95

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one tile of a feature image through one layer: only launch latency counts
        {"name": "gn_infer_16x16x64", "op": "group_norm", "train": False, "b": 1, "h": 16, "w": 16, "c": 64,
         "groups": 8, "act": "silu", "dtype": "bfloat16"},
        # one 1080p view with 32 features per pixel, rendered for display
        {"name": "gn_infer_1080p_c32", "op": "group_norm", "train": False, "b": 1, "h": 1080, "w": 1920, "c": 32,
         "groups": 8, "act": "silu", "dtype": "float16"},
        # a crop of odd size with 80 channels in five groups, trained in 32 bits
        {"name": "gn_train_2x67x119x80", "op": "group_norm", "train": True, "b": 2, "h": 67, "w": 119, "c": 80,
         "groups": 5, "act": "gelu", "dtype": "float32"},
        # a batch of eight views at an eighth of 1080p with wide features
        {"name": "gn_train_8x135x240x256", "op": "group_norm", "train": True, "b": 8, "h": 135, "w": 240, "c": 256,
         "groups": 32, "act": "silu", "dtype": "float16"},
        # a training batch of four 1080p feature images: the largest activation of a decoder
        {"name": "gn_train_4x1080p_c32", "op": "group_norm", "train": True, "b": 4, "h": 1080, "w": 1920, "c": 32,
         "groups": 8, "act": "silu", "dtype": "bfloat16"},
        # a 1x1 convolution of 64 features: the smallest matrix worth orthogonalising
        {"name": "ortho_64x64", "op": "orthogonalize", "batch": 1, "m": 64, "n": 64, "dtype": "float32"},
        # a stack of equal layers, tall matrices
        {"name": "ortho_8x2048x512_bf16", "op": "orthogonalize", "batch": 8, "m": 2048, "n": 512, "dtype": "bfloat16"},
        # a wide square layer in 32 bits, and the largest matrix in 16
        {"name": "ortho_2048x2048", "op": "orthogonalize", "batch": 1, "m": 2048, "n": 2048, "dtype": "float32"},
        {"name": "ortho_4096x4096_bf16", "op": "orthogonalize", "batch": 1, "m": 4096, "n": 4096, "dtype": "bfloat16"},
        # a four-layer decoder from 32 features per Gaussian to RGB, as wide as the renderer's own feature groups
        {"name": "muon_mlp_decoder", "op": "muon_step", "shapes": "64x32,64x64,64x64,3x64", "nesterov": True},
        # a convolutional decoder's filters (3x3, flattened), with odd input counts where view data is appended
        {"name": "muon_conv_decoder", "op": "muon_step",
         "shapes": "64x315,64x576,128x576,128x1152,256x1152,256x2304,128x2304,64x1152,3x576", "nesterov": True},
        # wide layers: the step is bound by its matrix products
        {"name": "muon_wide", "op": "muon_step", "shapes": "2048x2048,2048x2048,2048x2048,2048x2048,2048x8192,8192x2048",
         "nesterov": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "orthogonalize", "muon_step"])
    if op == "group_norm":
        groups = rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        c = groups * rng.choice([1, 2, 3, 4, 8, 10, 16])
        b = rng.randint(1, 8)
        pixels = _log(rng, 64, min(4 * 1080 * 1920, 4 * 1080 * 1920 * 32 // c) // b)
        h = max(1, int(math.sqrt(pixels) * rng.uniform(0.5, 1.0)))
        return {"op": op, "train": rng.random() < 0.5, "b": b, "h": h, "w": max(1, pixels // h), "c": c,
                "groups": groups, "act": rng.choice(["none", "silu", "gelu"]),
                "dtype": rng.choice(["float32", "bfloat16", "float16"])}
    if op == "orthogonalize":
        dtype = rng.choice(["float32", "bfloat16"])
        most = 2048 if dtype == "float32" else 4096
        m, n = _log(rng, 8, most), _log(rng, 8, most)
        batch = rng.randint(1, max(1, min(16, most ** 3 // (min(m, n) * m * n))))
        return {"op": op, "batch": batch, "m": m, "n": n, "dtype": dtype}
    count = rng.randint(1, 10)
    shapes = ",".join("%dx%d" % (_log(rng, 3, 1024), _log(rng, 16, 4096)) for _ in range(count))
    return {"op": op, "shapes": shapes, "nesterov": rng.random() < 0.7}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _gradient(gen, *size):
    """A weight gradient: a few strong directions (a sum of outer products of falling size) over a weak full-rank
    rest, of the size that a mean loss gives."""
    *lead, m, n = size
    rank = max(1, min(m, n) // 8)
    fall = torch.exp(-3.0 * torch.arange(rank, device="cuda") / rank)
    left = torch.randn(*lead, m, rank, generator=gen, device="cuda") * fall
    right = torch.randn(*lead, rank, n, generator=gen, device="cuda")
    return 1e-4 * (left @ right + 0.3 * torch.randn(*size, generator=gen, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "group_norm":
        b, h, w, c = (case[k] for k in "bhwc")
        dtype = DTYPES[case["dtype"]]
        # features have a mean and a spread of their own per channel; a tenth of the pixels is empty background
        spread = torch.rand(c, generator=gen, device="cuda") * 1.5 + 0.25
        mean = torch.randn(c, generator=gen, device="cuda")
        x = torch.randn(b, h, w, c, generator=gen, device="cuda").mul_(spread).add_(mean)
        x.mul_(torch.rand(b, h, w, 1, generator=gen, device="cuda") > 0.1)
        state = {"case": case, "x": x.to(dtype),
                 "weight": 1.0 + 0.2 * torch.randn(c, generator=gen, device="cuda"),
                 "bias": 0.2 * torch.randn(c, generator=gen, device="cuda")}
        if case["train"]:
            state["dy"] = (0.1 * torch.randn(b, h, w, c, generator=gen, device="cuda")).to(dtype)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_()
        return state
    if case["op"] == "orthogonalize":
        size = (case["m"], case["n"]) if case["batch"] == 1 else (case["batch"], case["m"], case["n"])
        return {"case": case, "update": _gradient(gen, *size).to(DTYPES[case["dtype"]])}
    shapes = _shapes(case)
    return {"case": case,
            "params": [torch.randn(m, n, generator=gen, device="cuda") / math.sqrt(n) for m, n in shapes],
            "grads": [_gradient(gen, m, n) for m, n in shapes],
            "buffers": [0.3 * _gradient(gen, m, n) for m, n in shapes]}


# ---- plain forms ---------------------------------------------------------------------------------------------
def _activation(u, act):
    if act == "silu":
        return u / (1 + torch.exp(-u))
    if act == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return u


def _activation_slope(u, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-u))
        return s * (1 + u * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    return torch.ones_like(u)


def _plain_group_norm(state, case):
    x = state["x"].detach()
    dtype, shape, g = x.dtype, x.shape, case["groups"]
    b, c = shape[0], shape[-1]
    x = x.float().reshape(b, -1, g, c // g)
    weight, bias = (state[k].detach().reshape(g, c // g) for k in ("weight", "bias"))
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + GN_EPS)
    xhat = centred * rstd
    u = xhat * weight + bias
    y = _activation(u, case["act"]).reshape(shape).to(dtype)
    if not case["train"]:
        return {"y": y}
    du = state["dy"].float().reshape(xhat.shape) * _activation_slope(u, case["act"])
    dxhat = du * weight
    dx = rstd * (dxhat - dxhat.mean((1, 3), keepdim=True) - xhat * (dxhat * xhat).mean((1, 3), keepdim=True))
    return {"y": y, "dx": dx.reshape(shape).to(dtype), "dweight": (du * xhat).sum((0, 1)).reshape(c),
            "dbias": du.sum((0, 1)).reshape(c)}


def _plain_orthogonalize(update):
    x = update.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=NS_EPS)
    a, b, c = NS
    for _ in range(NS_STEPS):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.transpose(-2, -1) if tall else x).to(update.dtype)


def _plain_muon(param, grad, buffer, nesterov):
    buffer.copy_(MOMENTUM * buffer + (1 - MOMENTUM) * grad)
    update = MOMENTUM * buffer + (1 - MOMENTUM) * grad if nesterov else buffer
    ratio = math.sqrt(max(1.0, param.shape[0] / param.shape[1]))
    param.copy_((1 - LR * WEIGHT_DECAY) * param - LR * ratio * _plain_orthogonalize(update))
    return param, buffer


def run(state):
    case = state["case"]
    if case["op"] == "group_norm":
        if own:
            from d3gs_research_b200 import group_norm_act
            y = group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], eps=GN_EPS, act=case["act"])
            if not case["train"]:
                return {"y": y}
            dx, dweight, dbias = torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["dy"])
            return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}
        return _plain_group_norm(state, case)
    if case["op"] == "orthogonalize":
        if own:
            from d3gs_research_b200 import orthogonalize
            return {"update": orthogonalize(state["update"], ns_coefficients=NS, eps=NS_EPS, ns_steps=NS_STEPS)}
        return {"update": _plain_orthogonalize(state["update"])}
    if own:
        from d3gs_research_b200 import muon_step
        muon_step(state["params"], state["grads"], state["buffers"], lr=LR, weight_decay=WEIGHT_DECAY,
                  momentum=MOMENTUM, nesterov=case["nesterov"], ns_coefficients=NS, eps=NS_EPS, ns_steps=NS_STEPS)
    else:
        for p, g, m in zip(state["params"], state["grads"], state["buffers"]):
            _plain_muon(p, g, m, case["nesterov"])
    return {"params": state["params"], "buffers": state["buffers"]}


def _ns_flops(m, n):
    m, n = min(m, n), max(m, n)
    # per step: the Gram matrix and its square are symmetric (half of each product), one full product applies them
    return NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)


def work(case):
    if case["op"] == "group_norm":
        size = 4 if case["dtype"] == "float32" else 2
        numel = case["b"] * case["h"] * case["w"] * case["c"]
        # x in, y out; in training dy in, dx out too (x is needed by both directions: read twice)
        return {"bytes": numel * size * (5 if case["train"] else 2) + 16 * case["c"],
                "flops": numel * (30 if case["train"] else 12)}
    if case["op"] == "orthogonalize":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * case["batch"] * case["m"] * case["n"] * size,
                "flops": case["batch"] * _ns_flops(case["m"], case["n"])}
    shapes = _shapes(case)
    # parameter and momentum in and out, gradient in
    return {"bytes": 20 * sum(m * n for m, n in shapes), "flops": sum(_ns_flops(m, n) + 8 * m * n for m, n in shapes)}


# ---- the definitions in 64 bits, written apart from the plain forms ------------------------------------------
def _exact_orthogonalize(update):
    """f(f(...f(X))) with f(X) = X (a I + S (b I + c S)), S = X^T X: the polynomial acts on the singular values, so
    the product may stand on either side; the shorter one is taken."""
    x = update.double()
    wide = x.shape[-1] > x.shape[-2]
    if wide:
        x = x.mT
    x = x / max(float(torch.linalg.vector_norm(x)), NS_EPS)
    eye = torch.eye(x.shape[-1], dtype=torch.float64, device=x.device)
    for _ in range(NS_STEPS):
        s = x.mT @ x
        x = x @ (NS[0] * eye + s @ (NS[1] * eye + NS[2] * s))
    return x.mT if wide else x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "group_norm":
        from torch.nn import functional as F
        xs = [state[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias")]
        rows = xs[0].flatten(1, 2).unflatten(2, (case["groups"], -1))
        var, mean = torch.var_mean(rows, (1, 3), correction=0, keepdim=True)
        u = ((rows - mean) * (var + GN_EPS).rsqrt()).flatten(2) * xs[1] + xs[2]
        y = {"none": lambda v: v, "silu": F.silu, "gelu": F.gelu}[case["act"]](u).reshape(xs[0].shape)
        if not case["train"]:
            return {"y": y}
        dx, dweight, dbias = torch.autograd.grad(y, xs, state["dy"].double())
        return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}
    if case["op"] == "orthogonalize":
        u = state["update"]
        return {"update": _exact_orthogonalize(u) if u.dim() == 2 else torch.stack([_exact_orthogonalize(v) for v in u])}
    params, buffers = [], []
    for p, g, m in zip(state["params"], state["grads"], state["buffers"]):
        m = torch.lerp(g.double(), m.double(), MOMENTUM)
        u = torch.lerp(g.double(), m, MOMENTUM) if case["nesterov"] else m
        rows, cols = p.shape
        params.append(p.double() * (1 - LR * WEIGHT_DECAY)
                      - LR * max(1.0, rows / cols) ** 0.5 * _exact_orthogonalize(u))
        buffers.append(m)
    return {"params": params, "buffers": buffers}
