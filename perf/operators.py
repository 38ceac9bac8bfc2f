"""Cases and plain forms of the operators that train deep multilayer perceptrons.

Four operators: layer norm with a fused activation, its backward pass, the
orthogonalisation of an update by Newton-Schulz products, and the optimiser
step around it (momentum, orthogonalisation, weight update).  Each case is a
dict of plain values; ``run`` computes the plain form in elementary torch
operations, or calls the framework's operators where ``own`` is true.
"""

import math

import torch

own = False

EPS = 1e-5                               # layer norm
STEPS, TINY = 5, 1e-7                    # Newton-Schulz
COEF = (3.4445, -4.7750, 2.0315)
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01   # optimiser step

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

MOST_ELEMENTS = 1_000_000 * 128          # of one layer norm case
MOST_PRODUCTS = 4 * 4096 ** 3            # of one Newton-Schulz step


def listed():
    return [
        # one micro-batch of the streaming scorer through a hidden layer: latency
        {"name": "norm micro-batch", "op": "norm", "rows": 256, "cols": 64,
         "dtype": "f32", "activation": "relu"},
        # the hidden layer of the 41-128-64-5 network over a shard of 1M flows
        {"name": "norm flow shard", "op": "norm", "rows": 1_000_000, "cols": 128,
         "dtype": "bf16", "activation": "relu"},
        # a wide hidden layer of odd sizes, full precision
        {"name": "norm wide odd", "op": "norm", "rows": 5003, "cols": 4099,
         "dtype": "f32", "activation": "none"},
        # backward of a small shard: latency of two dependent reductions
        {"name": "norm grad small", "op": "norm_grad", "rows": 1200, "cols": 64,
         "dtype": "f32", "activation": "sigmoid"},
        # backward of the 1M-flow shard's hidden layer
        {"name": "norm grad flow shard", "op": "norm_grad", "rows": 1_000_000,
         "cols": 128, "dtype": "bf16", "activation": "relu"},
        # backward of a wide layer, half precision, no activation
        {"name": "norm grad wide", "op": "norm_grad", "rows": 8192, "cols": 8192,
         "dtype": "f16", "activation": "none"},
        # the three weight gradients of the 41-128-64-5 network: latency
        {"name": "orthogonalise 41-128-64-5", "op": "orthogonalise",
         "shapes": "41x128 128x64 64x5", "dtype": "f32"},
        # one gradient of odd sizes in full precision
        {"name": "orthogonalise odd", "op": "orthogonalise", "shapes": "1001x777",
         "dtype": "f32"},
        # the largest: a square gradient in bfloat16
        {"name": "orthogonalise 4096", "op": "orthogonalise", "shapes": "4096x4096",
         "dtype": "bf16"},
        # a whole optimiser step of the 41-128-64-5 network
        {"name": "step 41-128-64-5", "op": "step", "shapes": "41x128 128x64 64x5",
         "dtype": "f32"},
        # an optimiser step of a wide network, both orientations, ragged ends
        {"name": "step 122-1024-4096-1024-5", "op": "step",
         "shapes": "122x1024 1024x4096 4096x1024 1024x5", "dtype": "f32"},
        # an optimiser step on one large matrix held in bfloat16
        {"name": "step 2048x4096", "op": "step", "shapes": "2048x4096",
         "dtype": "bf16"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _products(shapes):
    total = 0
    for r, c in shapes:
        m, n = min(r, c), max(r, c)
        total += 3 * m * m * n + m ** 3
    return total


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "orthogonalise", "step"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("norm", "norm_grad"):
        # hidden widths from 8 to 16384; rows from one to a whole shard
        cols = _log_uniform(rng, 8, 16384)
        rows = _log_uniform(rng, 1 if op == "norm" else 16, min(1_000_000, MOST_ELEMENTS // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype,
                "activation": rng.choice(["none", "relu", "sigmoid"])}
    # one matrix, or the chain of a network's layers
    while True:
        widths = [_log_uniform(rng, 1, 4096) for _ in range(rng.choice([2, 2, 3, 4]))]
        shapes = list(zip(widths, widths[1:]))
        if _products(shapes) <= MOST_PRODUCTS:
            break
    return {"op": op, "shapes": " ".join("%dx%d" % s for s in shapes), "dtype": dtype}


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def _gradient(r, c, g, dev):
    """A weight gradient: activations times deltas, summed over flows."""
    flows = 4 * max(r, c)
    act = torch.randn(flows, r, generator=g, device=dev).relu_()
    delta = torch.randn(flows, c, generator=g, device=dev)
    delta *= torch.rand(flows, 1, generator=g, device=dev) ** 2
    return act.T @ delta / flows ** 0.5


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    t = TYPES[case["dtype"]]
    s = {"op": case["op"]}
    if case["op"] in ("norm", "norm_grad"):
        n, d = case["rows"], case["cols"]
        s["activation"] = case["activation"]
        # pre-activations: columns of their own offset, rows of their own size
        x = torch.randn(n, d, generator=g, device=dev)
        x *= torch.rand(n, 1, generator=g, device=dev) * 2 + 0.5
        x += torch.randn(d, generator=g, device=dev) * 0.5
        s["x"] = x.to(t)
        del x
        s["weight"] = torch.rand(d, generator=g, device=dev) + 0.5
        s["bias"] = torch.randn(d, generator=g, device=dev) * 0.2
        if case["op"] == "norm_grad":
            # what the forward pass left: the output and the row statistics
            s["y"], s["mean"], s["rstd"] = _norm(s)
            s["dy"] = torch.randn(n, d, generator=g, device=dev).to(t)
        return s
    grads = [_gradient(r, c, g, dev) for r, c in _shapes(case)]
    s["grads"] = [x.to(t) for x in grads]
    if case["op"] == "step":
        s["weights"] = [(torch.randn(x.shape, generator=g, device=dev)
                         * (2.0 / x.shape[0]) ** 0.5).to(t) for x in grads]
        s["buffers"] = [2.0 * _gradient(x.shape[0], x.shape[1], g, dev) + x for x in grads]
    return s


def _norm(s):
    x = s["x"].float()
    d = x.shape[1]
    mean = x.sum(1) / d
    x = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((x * x).sum(1) / d + EPS)
    z = x * rstd[:, None] * s["weight"] + s["bias"]
    if s["activation"] == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif s["activation"] == "sigmoid":
        z = 1.0 / (1.0 + torch.exp(-z))
    return z.to(s["x"].dtype), mean, rstd


def _norm_grad(s):
    x, dz = s["x"].float(), s["dy"].float()
    d = x.shape[1]
    if s["activation"] == "relu":
        dz = torch.where(s["y"] > 0, dz, torch.zeros_like(dz))
    elif s["activation"] == "sigmoid":
        y = s["y"].float()
        dz = dz * (y * (1.0 - y))
    xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
    dweight, dbias = (dz * xh).sum(0), dz.sum(0)
    p = dz * s["weight"]
    dx = s["rstd"][:, None] * (p - (p.sum(1) / d)[:, None] - xh * ((p * xh).sum(1) / d)[:, None])
    return dx.to(s["x"].dtype), dweight, dbias


def _orthogonalise(g):
    """Plain Newton-Schulz of a matrix, in 32 bits; its norm in 64 (a long sum)."""
    x = g.float()
    x = x / x.double().square().sum().sqrt().clamp_min(TINY).float()
    if x.shape[0] > x.shape[1]:
        x = x.T.contiguous()
    a, b, c = COEF
    for _ in range(STEPS):
        p = x @ x.T
        x = a * x + (b * p + c * (p @ p)) @ x
    return x if g.shape[0] <= g.shape[1] else x.T


def _step(w, g, m):
    m.mul_(MOMENTUM).add_(g.float())
    o = _orthogonalise(g.float() + MOMENTUM * m)
    w.copy_((1.0 - LR * DECAY) * w.float() - LR * 0.2 * max(w.shape) ** 0.5 * o)


def run(state):
    s = state
    if own:
        from flowml import ops

        if s["op"] == "norm":
            return ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS,
                                  activation=s["activation"])
        if s["op"] == "norm_grad":
            return ops.layer_norm_grad(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"],
                                       y=s["y"], activation=s["activation"])
        if s["op"] == "orthogonalise":
            return ops.newton_schulz(s["grads"], steps=STEPS, coefficients=COEF, eps=TINY)
        ops.muon_update(s["weights"], s["grads"], s["buffers"], lr=LR, momentum=MOMENTUM,
                        weight_decay=DECAY, nesterov=True, steps=STEPS, coefficients=COEF,
                        eps=TINY)
        return s["weights"], s["buffers"]
    if s["op"] == "norm":
        return _norm(s)
    if s["op"] == "norm_grad":
        return _norm_grad(s)
    if s["op"] == "orthogonalise":
        return [_orthogonalise(g).to(g.dtype) for g in s["grads"]]
    for w, g, m in zip(s["weights"], s["grads"], s["buffers"]):
        _step(w, g, m)
    return s["weights"], s["buffers"]


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("norm", "norm_grad"):
        n, d = case["rows"], case["cols"]
        if case["op"] == "norm":
            return {"bytes": 2 * n * d * size + 8 * d + 8 * n, "flops": 8 * n * d}
        arrays = 3 if case["activation"] == "none" else 4
        return {"bytes": arrays * n * d * size + 12 * d + 8 * n, "flops": 14 * n * d}
    shapes = _shapes(case)
    values = sum(r * c for r, c in shapes)
    # read and write: a gradient and its result; or gradient, weight and buffer
    moved = values * (2 * size if case["op"] == "orthogonalise" else 3 * size + 8)
    # x x^T and its square are symmetric: half of their products are enough
    return {"bytes": moved, "flops": STEPS * _products(shapes)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_grad"):
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        if case["op"] == "norm":
            rstd = (var + EPS).rsqrt()
            z = (x - mean).mul_(rstd).mul_(s["weight"].double()).add_(s["bias"].double())
            if case["activation"] == "relu":
                z = z.clamp_min_(0.0)
            elif case["activation"] == "sigmoid":
                z = z.sigmoid_()
            return z, mean[:, 0], rstd[:, 0]
        # the row statistics are inputs, as the forward pass left them
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        x = x.sub_(mean).mul_(rstd)
        dz = s["dy"].double()
        if case["activation"] == "relu":
            dz = dz * (s["y"] > 0)
        elif case["activation"] == "sigmoid":
            y = s["y"].double()
            dz = dz.mul_(y - y * y)
        dbias = dz.sum(0)
        dweight = (dz * x).sum(0)
        p = dz.mul_(s["weight"].double())
        along = (p * x).mean(1, keepdim=True)
        dx = (p - p.mean(1, keepdim=True)).sub_(x.mul_(along)).mul_(rstd)
        return dx, dweight, dbias
    a, b, c = COEF
    eye = lambda k: torch.eye(k, dtype=torch.float64, device=s["grads"][0].device)  # noqa: E731

    def polar(u):
        # the same polynomial, multiplied from the shorter side
        u = u / max(float(torch.linalg.matrix_norm(u)), TINY)
        for _ in range(STEPS):
            if u.shape[0] <= u.shape[1]:
                k = u @ u.mT
                u = (a * eye(len(k)) + b * k + c * (k @ k)) @ u
            else:
                k = u.mT @ u
                u = u @ (a * eye(len(k)) + b * k + c * (k @ k))
        return u

    if case["op"] == "orthogonalise":
        return [polar(g.double()) for g in s["grads"]]
    weights, buffers = [], []
    for w, g, m in zip(s["weights"], s["grads"], s["buffers"]):
        m = m.double() * MOMENTUM + g.double()
        o = polar(g.double() + m * MOMENTUM)
        scale = 0.2 * math.sqrt(max(w.shape))
        weights.append(w.double() - LR * (DECAY * w.double() + scale * o))
        buffers.append(m)
    return weights, buffers
