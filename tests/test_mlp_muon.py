"""Layer norm and Muon together, as the MLP uses them."""

import math
import multiprocessing as mp
import os

import pytest
import torch

from flowml import FlowFrame, ops
from flowml.classification import MultilayerPerceptronClassifier
from flowml.classification.mlp import _flatten, _matrices, _unflatten, n_weights
from flowml.optim import Muon, muon

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LAYERS = [41, 128, 64, 5]


def network(layers, n, dtype=torch.float32, dev="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(n, layers[0], generator=g)
    y = torch.randint(0, layers[-1], (n,), generator=g)
    Ws = [torch.randn(o, i, generator=g) / i ** 0.5 for i, o in zip(layers, layers[1:])]
    bs = [0.1 * torch.randn(o, generator=g) for o in layers[1:]]
    norms = [(1 + 0.2 * torch.randn(o, generator=g), 0.2 * torch.randn(o, generator=g))
             for o in layers[1:-1]]
    return (X.to(dtype).to(dev), y.to(dev), [W.to(dtype).to(dev) for W in Ws],
            [b.to(dev) for b in bs], [(p.to(dev), q.to(dev)) for p, q in norms])


def reference(X, y, Ws, bs, norms, activation):
    """Loss and gradients in 64 bits, by autograd of the formulas."""
    to = lambda t: t.detach().cpu().double().requires_grad_()  # noqa: E731
    Ws, bs = [to(W) for W in Ws], [to(b) for b in bs]
    norms = [(to(p), to(q)) for p, q in norms]
    h = X.cpu().double()
    for i, (W, b) in enumerate(zip(Ws, bs)):
        h = h @ W.T + b
        if i < len(Ws) - 1:
            m = h.mean(1, keepdim=True)
            v = ((h - m) ** 2).mean(1, keepdim=True)
            h = (h - m) / torch.sqrt(v + 1e-5) * norms[i][0] + norms[i][1]
            h = torch.relu(h) if activation == "relu" else torch.sigmoid(h)
    loss = -(torch.log_softmax(h, 1)[torch.arange(len(y)), y.cpu()]).sum()
    loss.backward()
    return (loss.detach(), [W.grad for W in Ws], [b.grad for b in bs],
            [(p.grad, q.grad) for p, q in norms])


def far(a, b):
    return float((a.cpu().double() - b).norm() / b.norm())


@pytest.mark.parametrize("activation", ["relu", "sigmoid"])
@pytest.mark.parametrize("dtype,dev", [(torch.float32, "cpu")] + [
    pytest.param(t, "cuda", marks=pytest.mark.gpu) for t in (torch.float32, torch.bfloat16)])
def test_gradients(dtype, dev, activation):
    X, y, Ws, bs, norms = network(LAYERS, 700, dtype, dev)
    loss, gW, gB, gN = ops.mlp_grad(X, y, Ws, bs, activation=activation, norms=norms)
    rl, rW, rB, rN = reference(X, y, Ws, bs, norms, activation)
    # f32: sums of up to 700 in one order or another, three layers deep, and a
    # few relu borders crossed by a rounding (one of 700 * 128 values: 3e-3).
    # bf16: a rounding of half a step for each of the ten arrays on the way.
    tol = 3e-3 if dtype == torch.float32 else 10 * 2.0 ** -8
    assert abs(float(loss) - float(rl)) <= tol * abs(float(rl))
    for got, want in zip(gW + gB + [t for p in gN for t in p],
                         rW + rB + [t for p in rN for t in p]):
        assert got.shape == want.shape and far(got, want) <= tol


@pytest.mark.parametrize("dev", DEVICES)
def test_without_norms_nothing_changes(dev):
    X, y, Ws, bs, _ = network(LAYERS, 300, torch.float32, dev)
    assert len(ops.mlp_grad(X, y, Ws, bs)) == 3
    assert ops.mlp_forward(X, Ws, bs).shape == (300, 5)
    with pytest.raises(ValueError):
        ops.mlp_forward(X, Ws, bs, norms=[])
    with pytest.raises(ValueError):
        ops.mlp_grad(X, y, Ws, bs, norms=[(bs[0], bs[0])])


def test_flat_layout():
    for norm in (False, True):
        flat = torch.arange(n_weights(LAYERS, norm), dtype=torch.float32)
        Ws, bs, *norms = _unflatten(flat, LAYERS, norm)
        assert torch.equal(_flatten(Ws, bs, *norms), flat)
        for W, (off, r, c) in zip(Ws, _matrices(LAYERS, norm)):
            assert torch.equal(flat[off:off + r * c].view(r, c), W.T)


def steps_in_64_bits(f_grad, x, matrices, n, lr, momentum):
    """``muon`` from its definition."""
    x = x.double()
    mats = [slice(o, o + r * c) for o, r, c in matrices]
    rest = torch.ones(len(x), dtype=torch.bool)
    for s in mats:
        rest[s] = False
    bufs = [torch.zeros(r, c).double() for _, r, c in matrices]
    m1 = m2 = torch.zeros(int(rest.sum())).double()
    for t in range(1, n + 1):
        g = f_grad(x)[1]
        for i, (s, (_, r, c)) in enumerate(zip(mats, matrices)):
            G = g[s].view(r, c)
            bufs[i] = momentum * bufs[i] + G
            u = G + momentum * bufs[i]
            u = u / u.norm()
            for _ in range(5):
                k = u @ u.T
                u = 3.4445 * u + (-4.775 * k + 2.0315 * k @ k) @ u
            x[s] -= lr * 0.2 * math.sqrt(max(r, c)) * u.reshape(-1)
        m1 = 0.9 * m1 + 0.1 * g[rest]
        m2 = 0.999 * m2 + 0.001 * g[rest] ** 2
        x[rest] -= lr * (m1 / (1 - 0.9 ** t)) / ((m2 / (1 - 0.999 ** t)).sqrt() + 1e-8)
    return x


@pytest.mark.parametrize("dev", DEVICES)
def test_optimizer_steps(dev):
    matrices = [(3, 8, 20), (163, 30, 6), (350, 1, 9)]
    g = torch.Generator().manual_seed(0)
    target, curve = torch.randn(370, generator=g), torch.rand(370, generator=g) + 0.5
    x0 = torch.randn(370, generator=g)

    def f_grad(x):
        c, t = curve.to(x), target.to(x)
        return float((c * (x - t) ** 2).sum() / 2), c * (x - t)

    x, history = muon(f_grad, x0.to(dev), matrices, max_iter=4, lr=0.05, momentum=0.9)
    ref = steps_in_64_bits(f_grad, x0, matrices, 4, 0.05, 0.9)
    assert len(history) == 4 and history[0] == pytest.approx(f_grad(x0)[0], rel=1e-5)
    # four updates, each within 2^-10 of its size (Newton-Schulz in fp32: 1e-5)
    assert float((x.cpu().double() - ref).norm()) <= 2.0 ** -10 * float((ref - x0.double()).norm())
    for bad in ([(0, 8, 50)], [(-1, 2, 2)], [(0, 4, 4), (15, 2, 2)]):
        with pytest.raises(ValueError):
            muon(f_grad, x0.to(dev), bad)


def flows(n=500, f=9, k=3, dev="cpu"):
    g = torch.Generator().manual_seed(4)
    X = torch.randn(n, f, generator=g)
    y = (X @ torch.randn(f, k, generator=g)).argmax(1).double()
    return FlowFrame({"features": X.to(dev), "label": y.to(dev)})


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("solver,norm", [("muon", False), ("muon", True), ("l-bfgs", True),
                                         ("gd", True)])
def test_fit(solver, norm, dev, tmp_path):
    df = flows(dev=dev)
    est = MultilayerPerceptronClassifier(layers=[9, 24, 16, 3], maxIter=6, solver=solver, seed=2,
                                         layerNorm=norm, stepSize=0.02, tol=0.0)
    m = est.fit(df)
    assert m._weights.numel() == n_weights([9, 24, 16, 3], norm)
    assert torch.isfinite(m._weights).all() and len(m._objective_history) >= 6
    assert torch.equal(m._weights, est.fit(df)._weights)  # deterministic
    pred = m.transform(df)["prediction"]
    m.save(str(tmp_path / "m"))
    back = type(m).load(str(tmp_path / "m"))
    assert back.getLayerNorm() == norm and back.getSolver() == solver
    assert torch.equal(back.transform(df)["prediction"], pred)


def _worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.distributed.init_process_group("gloo", rank=rank, world_size=world)
    df = flows()
    half = len(df["label"]) // world
    part = FlowFrame({c: df[c][rank * half:(rank + 1) * half] for c in ("features", "label")})
    m = MultilayerPerceptronClassifier(layers=[9, 24, 3], maxIter=5, solver="muon", seed=2,
                                       layerNorm=True, stepSize=0.02).fit(part)
    q.put((rank, m._weights.numpy()))
    torch.distributed.destroy_process_group()


def test_two_ranks():
    """Two halves of the rows give the weights of the whole, on both ranks."""
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = 29411 + os.getpid() % 997
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
    whole = MultilayerPerceptronClassifier(layers=[9, 24, 3], maxIter=5, solver="muon", seed=2,
                                           layerNorm=True, stepSize=0.02).fit(flows())._weights
    a, b = torch.from_numpy(got[0]), torch.from_numpy(got[1])
    assert torch.equal(a, b)
    # sums of 500 rows in another order, through five steps of size 0.02
    assert float((a - whole).norm()) <= 1e-4 * float(whole.norm())


@pytest.mark.gpu
def test_training_step_in_a_graph():
    """Forward, backward and update, captured and replayed: the eager run's bits."""
    X, y, Ws, bs, norms = network(LAYERS, 2000, torch.bfloat16, "cuda")
    master = [W.float() for W in Ws]
    eager = Muon([W.clone() for W in master], lr=0.02)
    opt = Muon(master, lr=0.02)

    def step(o):
        ws = [W.to(torch.bfloat16) for W in o.weights]
        loss, gW, gB, gN = ops.mlp_grad(X, y, ws, bs, norms=norms)
        o.step([g.float() / len(X) for g in gW])
        return loss, gB, gN

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(Muon([W.clone() for W in master], lr=0.02))
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(opt)
    for turn in range(4):
        X.copy_(network(LAYERS, 2000, torch.bfloat16, "cuda", seed=9 + turn)[0])
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0])
        assert all(torch.equal(p, q) for p, q in zip(opt.weights + opt.buffers,
                                                     eager.weights + eager.buffers))
        assert all(torch.equal(p, q) for a, b in zip(out[2], want[2]) for p, q in zip(a, b))
