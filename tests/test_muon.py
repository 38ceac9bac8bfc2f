"""Newton-Schulz orthogonalisation and the optimiser step against 64 bits."""

import math

import pytest
import torch

from flowml import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
COEF = ops.NS_COEFFICIENTS


def gradient(kind, m, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if kind == "full":
        return rn(m, n)
    if kind == "low":  # rank r and a little noise
        r = max(1, min(m, n) // 16)
        return rn(m, r) @ rn(r, n) / r ** 0.5 + 0.01 * rn(m, n)
    if kind == "one":
        return rn(m, 1) @ rn(1, n)
    if kind == "offset":  # relu activations: one large singular value
        return (torch.relu(rn(4 * max(m, n), m)).T @ rn(4 * max(m, n), n)) / max(m, n)
    raise ValueError(kind)


def reference(G, steps=5, coef=COEF, eps=1e-7):
    """The definition in 64 bits, and the norms of the iterates."""
    a, b, c = coef
    x = G.double()
    x = x / max(float(x.norm()), eps)
    sizes = []
    for _ in range(steps):
        sizes.append(float(x.norm()))
        if x.shape[0] <= x.shape[1]:
            k = x @ x.T
            x = a * x + (b * k + c * k @ k) @ x
        else:
            k = x.T @ x
            x = a * x + x @ (b * k + c * k @ k)
    return x, sizes


def tolerance(G, sizes, dtype, coef=COEF):
    """Bound of the error's 2-norm.

    A step maps singular values by p; in the 2-norm its derivative is at most
    L = max |p'| over their range (the largest divided difference). What a step
    loses: pairs of fp16 hold 22 bits, and A, A^2, B and X are each rounded to
    them (16 half steps cover the polynomial's factors |b| and 2|c|), sums of K
    products in fp32 walk sqrt(K) quarters of that. It grows by L in each later
    step. bf16 results are rounded once (half a step, 2^-8), and their A and B
    are held in 11 bits: 5 steps of two such roundings, 2^-12 each as they are
    spread, on values that |p'| <= 1.6 no longer grows: under 2^-8.
    """
    a, b, c = coef
    s = torch.linspace(0, 1.2025, 2000).double()
    L = float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max())
    eta = 2.0 ** -22 * (16 + max(G.shape) ** 0.5)
    tol = sum(L ** (len(sizes) - 1 - k) * eta * v * 1.0 for k, v in enumerate(sizes))
    return tol


def check(G, got, steps=5, coef=COEF, eps=1e-7, dev="cpu"):
    ref, sizes = reference(G.to(dev), steps, coef, eps)
    off = float((got.to(dev).double() - ref).norm())
    tol = tolerance(G, sizes, G.dtype, coef)
    size = float(ref.norm())
    if G.dtype == torch.bfloat16:
        tol += (2.0 ** -8 + 2.0 ** -8) * size
    elif G.dtype == torch.float16:
        tol += 2.0 ** -11 * size + 2.0 ** -25 * G.numel() ** 0.5
    assert got.dtype == G.dtype and got.shape == G.shape and got.is_contiguous()
    assert off <= tol, (tuple(G.shape), G.dtype, off, tol, size)


SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (5, 3), (41, 128), (128, 64), (64, 5), (65, 64), (63, 200),
          (130, 257), (1, 3000), (2000, 3)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["full", "low", "one", "offset"])
def test_small(kind, dtype, dev):
    grads = [gradient(kind, m, n, seed=m + n).to(dtype).to(dev) for m, n in SHAPES]
    together = ops.newton_schulz(grads)
    for g, o in zip(grads, together):
        check(g, o)
    # alone or in company, a matrix gives the same result within the bound
    for g in grads[::4]:
        check(g, ops.newton_schulz(g))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n", [(255, 255), (256, 300), (300, 4000), (777, 1001), (1024, 512),
                                 (2048, 2050)])
def test_large(m, n, dtype):
    for kind in ("full", "low", "one", "offset"):
        G = gradient(kind, m, n, seed=3).to(dtype).cuda()
        got = ops.newton_schulz(G)
        check(G, got)
        assert torch.equal(got, ops.newton_schulz(G))  # one order of sums


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(1600, 1500), (2000, 4100), (4096, 4096), (5632, 5640)])
def test_tiles(m, n, dtype):
    """Sizes that take tiles of every side; the reference on the GPU in 64 bits."""
    G = gradient("full", m, n, seed=1).to(dtype).cuda()
    got = ops.newton_schulz(G)
    check(G, got, dev="cuda")
    assert torch.equal(got, ops.newton_schulz(G))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes", [[(65, 9001)], [(520, 4100)], [(1000, 4000)], [(4100, 1030)],
                                    [(16, 40001)], [(3001, 17)],
                                    [(1000, 4000), (300, 256), (12, 5000), (4000, 1000), (70, 300)]])
def test_long(shapes, dtype):
    """One axis much longer than the other: sums over it are shared out."""
    for kind in ("full", "one"):
        grads = [gradient(kind, m, n, seed=m).to(dtype).cuda() for m, n in shapes]
        out = ops.newton_schulz(grads)
        for g, o, again in zip(grads, out, ops.newton_schulz(grads)):
            check(g, o)
            assert torch.equal(o, again)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(2, 3000001), (2100001, 17)])
def test_very_long(m, n):
    G = gradient("full", m, n, seed=5).cuda()
    check(G, ops.newton_schulz(G), dev="cuda")


@pytest.mark.gpu
def test_too_large():
    """Refused before anything is launched."""
    G = torch.empty(33000, 33000, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="too large"):
        ops.newton_schulz([G.new_zeros(3, 3), G])


@pytest.mark.gpu
def test_many_matrices():
    """More than one table of matrices, of one shape and of several."""
    stack = torch.stack([gradient("full", 70, 33, seed=k) for k in range(53)]).cuda()
    out = ops.newton_schulz(stack)
    assert out.shape == stack.shape
    for g, o in zip(stack, out):
        check(g, o)
    mixed = [gradient("full", 1 + 13 * (k % 17), 1 + 29 * (k % 11), seed=k).cuda() for k in range(60)]
    for g, o in zip(mixed, ops.newton_schulz(mixed)):
        check(g, o)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("coef,steps", [((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 9), (COEF, 1),
                                        ((0.5, 0.0, 0.0), 2)])
def test_other_polynomials(coef, steps, dev):
    for m, n in ((30, 50), (200, 90)):
        G = gradient("offset", m, n).to(dev)
        check(G, ops.newton_schulz(G, steps=steps, coefficients=coef), steps, coef)
    if steps > 8:  # these converge: the result is orthogonal
        G = torch.eye(20, 30) + 0.1 * gradient("full", 20, 30)
        o = ops.newton_schulz(G.to(dev), steps=steps, coefficients=coef).cpu()
        assert (o @ o.T - torch.eye(20)).abs().max() < 1e-4


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("m,n", [(40, 70), (70, 7), (9, 3000), (130, 90), (300, 300)])
def test_special_values(m, n, dev):
    z = torch.zeros(m, n, device=dev)
    assert torch.equal(ops.newton_schulz(z), z)
    # norms below eps are divided by eps; very small and very large ones keep
    # their digits
    G = gradient("full", m, n).to(dev)
    G = G / G.norm()
    check(G * 1e-9, ops.newton_schulz(G * 1e-9))
    check(G * 1e-3, ops.newton_schulz(G * 1e-3, eps=1e-2), eps=1e-2)
    check(G * 1e30, ops.newton_schulz(G * 1e30))
    check(G * 1e-28, ops.newton_schulz(G * 1e-28, eps=1e-30), eps=1e-30)
    for bad in (float("nan"), float("inf")):
        H = G.clone()
        H[3, 5] = bad
        other = ops.newton_schulz([H, G])
        assert other[0].isnan().all()
        check(G, other[1])
    # empty matrices, an empty stack, an empty sequence
    outs = ops.newton_schulz([G, G[:0], G[:, :0]])
    check(G, outs[0])
    assert outs[1].shape == (0, n) and outs[2].shape == (m, 0)
    assert ops.newton_schulz(G[None][:0]).shape == (0, m, n)
    assert ops.newton_schulz([]) == []


@pytest.mark.parametrize("dev", DEVICES)
def test_strides(dev):
    base = gradient("full", 90, 140).to(dev)
    for G in (base.T, base[::2, 3:77], base[:, ::3], base[:1].expand(30, 140)):
        check(G, ops.newton_schulz(G))


def step_reference(w, g, m, lr, mu, wd, nesterov, steps=5):
    m = mu * m.double() + g.double()
    u = g.double() + mu * m if nesterov else m
    o, sizes = reference(u, steps)
    s = lr * 0.2 * math.sqrt(max(w.shape))
    return (1 - lr * wd) * w.double() - s * o, m, u, sizes, s


SETS = {"small": [(41, 128), (128, 64), (64, 5), (0, 4), (1, 1)],
        "mixed": [(41, 128), (64, 5), (300, 290), (3, 2100), (129, 70)]}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("which", SETS)
@pytest.mark.parametrize("wtype,gtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.float32, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_update(wtype, gtype, nesterov, which, dev):
    shapes = SETS[which]
    ws = [gradient("full", *s, seed=1).to(wtype).to(dev) for s in shapes]
    ms = [gradient("offset", *s, seed=2).to(dev) if s[0] else torch.zeros(s, device=dev) for s in shapes]
    for turn in range(2):
        gs = [gradient("full", *s, seed=3 + turn).to(gtype).to(dev) for s in shapes]
        before = [(w.clone(), m.clone()) for w, m in zip(ws, ms)]
        ops.muon_update(ws, gs, ms, lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
        for (w0, m0), w, m, g in zip(before, ws, ms, gs):
            if not w.numel():
                continue
            ref, mref, u, sizes, s = step_reference(w0.cpu(), g.cpu(), m0.cpu(), 0.05, 0.9, 0.1, nesterov)
            # buffer: two roundings, and mu in fp32
            e = 2.0 ** -23 * ((0.9 * m0.cpu().double()).abs() + mref.abs())
            assert ((m.cpu().double() - mref).abs() <= e).all()
            tol = s * (tolerance(u, sizes, wtype) + 2.0 ** -22 * float(ref.norm()))
            tol += 2.0 ** -22 * float(ref.norm())
            if wtype != torch.float32:
                tol += torch.finfo(wtype).eps / 2 * float(ref.norm())
            if wtype == torch.bfloat16:
                tol += s * 2.0 ** -8 * math.sqrt(min(w.shape))
            assert float((w.cpu().double() - ref).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("shapes", [[(41, 128), (64, 5)], [(41, 128), (300, 500), (5, 1300)]])
def test_update_twice_the_same_and_in_a_graph(shapes):
    mk = lambda seed: [gradient("offset", *s, seed=seed).cuda() for s in shapes]  # noqa: E731
    ws, gs, ms = mk(1), mk(2), mk(3)

    def step(w, g, m):
        ops.muon_update(w, g, m, lr=0.02, weight_decay=0.01)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    we, me = [w.clone() for w in ws], [m.clone() for m in ms]
    with torch.cuda.stream(s):
        step([w.clone() for w in ws], gs, [m.clone() for m in ms])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(ws, gs, ms)
    for turn in range(4):
        for g, f in zip(gs, mk(10 + turn)):
            g.copy_(f)
        step(we, gs, me)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ws + ms, we + me))


@pytest.mark.parametrize("dev", DEVICES)
def test_parameters(dev):
    """A leaf that wants gradients is stepped, and no backward pass goes through
    what it was."""
    w = torch.randn(30, 40, device=dev, requires_grad=True)
    was = w.detach().clone()
    y = (w * w).sum()
    ops.muon_update([w], [torch.ones_like(was)], [torch.zeros_like(was)], lr=0.1)
    assert w.requires_grad and w.is_leaf and not torch.equal(w.detach(), was)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        v = torch.randn(30, 40, device=dev)
        ops.muon_update([v], [torch.ones_like(was)], [torch.zeros_like(was)], lr=0.1)


def test_refusals():
    w, g, m = torch.randn(6, 4), torch.randn(6, 4), torch.zeros(6, 4)
    step = lambda *a, **k: ops.muon_update(*a, lr=0.1, **k)  # noqa: E731
    flat = torch.zeros(40)
    bad = [
        lambda: ops.newton_schulz(g[0]),
        lambda: ops.newton_schulz(g.double()),
        lambda: ops.newton_schulz(g.double()[None]),
        lambda: ops.newton_schulz([g, g.bfloat16()]),
        lambda: ops.newton_schulz([g, g[0]]),
        lambda: ops.newton_schulz([g, 3.0]),
        lambda: ops.newton_schulz(g, steps=0),
        lambda: ops.newton_schulz(g, steps=1.5),
        lambda: ops.newton_schulz(g, steps=math.inf),
        lambda: ops.newton_schulz(g, eps=0.0),
        lambda: ops.newton_schulz(g, eps=float("nan")),
        lambda: ops.newton_schulz(g, eps=1e-35),
        lambda: ops.newton_schulz(g, coefficients=(3.0, 0.0, 0.0)),
        lambda: ops.newton_schulz(g, coefficients=(1.0, 2.0)),
        lambda: ops.newton_schulz(g, coefficients=(float("nan"), 0.0, 0.0)),
        lambda: step([w], [g], []),
        lambda: step([w], [g[:5]], [m]),
        lambda: step([w], [g], [m.bfloat16()]),
        lambda: step([w.double()], [g], [m]),
        lambda: step([w.T], [g.T], [m.T]),
        lambda: step([w, w], [g, g], [m, m.clone()]),
        lambda: step([w, w.clone()], [g, g], [m, m]),
        lambda: step([w], [g], [w]),
        lambda: step([w], [m], [m]),
        lambda: step([w], [w], [m]),
        lambda: step([flat[:24].view(6, 4)], [g], [flat[16:40].view(6, 4)]),
        lambda: step([w], [g], [m], momentum=1.0),
        lambda: step([w], [g], [m], momentum=-0.1),
    ]
    keep = [t.clone() for t in (w, g, m)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)
    assert all(torch.equal(p, q) for p, q in zip(keep, (w, g, m)))
    step([], [], [])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("shapes", [[(41, 128), (64, 5)], [(256, 300)], [(700, 310), (4, 900)],
                                    pytest.param([(2048, 4096)], marks=pytest.mark.gpu),
                                    pytest.param([(4096, 1500), (70, 30)], marks=pytest.mark.gpu)])
def test_bf16_is_rounded_once(shapes, dev):
    """Results in bf16 are those in fp32, rounded: nothing else is lost."""
    gs = [gradient("full", *s, seed=1).bfloat16().to(dev) for s in shapes]
    got, want = ops.newton_schulz(gs), ops.newton_schulz([g.float() for g in gs])
    assert all(torch.equal(o, w.bfloat16()) for o, w in zip(got, want))
    ws = [gradient("offset", *s, seed=2).bfloat16().to(dev) for s in shapes]
    ms = [gradient("low", *s, seed=3).to(dev) for s in shapes]
    wf, mf = [w.float() for w in ws], [m.clone() for m in ms]
    ops.muon_update(ws, gs, ms, lr=0.05, weight_decay=0.1)
    ops.muon_update(wf, [g.float() for g in gs], mf, lr=0.05, weight_decay=0.1)
    assert all(torch.equal(w, f.bfloat16()) for w, f in zip(ws, wf))
    assert all(torch.equal(p, q) for p, q in zip(ms, mf))


def hard(kind):
    """Matrices with singular values far below the largest, or none."""
    g = torch.Generator().manual_seed(11)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    if kind == "rows":  # logspaced row scales
        return rn(12, 12) * torch.logspace(0, -9, 12)[:, None]
    if kind == "graded":  # logspaced singular values
        q, r = torch.linalg.qr(rn(12, 12).double())[0], torch.linalg.qr(rn(12, 12).double())[0]
        return (q * torch.logspace(0, -9, 12).double() @ r).float()
    if kind == "one":
        return rn(8, 1) @ rn(1, 100)
    if kind == "half":
        return rn(16, 8) @ rn(8, 16)
    if kind == "softmax":  # a last layer's gradient: its columns sum to 0
        d = torch.softmax(rn(200, 5), 1) - torch.eye(5)[torch.randint(0, 5, (200,), generator=g)]
        return torch.relu(rn(200, 64)).T @ d
    if kind == "same":
        return torch.ones(8, 100)
    if kind == "long":
        return rn(9, 2) @ rn(2, 3000)
    raise ValueError(kind)


HARD = ["rows", "graded", "one", "half", "softmax", "same", "long"]
FP32 = lambda coef: tuple(torch.tensor(coef, dtype=torch.float32).double().tolist())  # noqa: E731


def tolerance64(G, sizes, coef):
    """As ``tolerance`` with 53 bits for 22, for the result and the reference both,
    and the result's rounding to fp32."""
    a, b, c = coef
    s = torch.linspace(0, 1.2025, 2000).double()
    L = max(1.0, float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()))
    eta = 2.0 ** -53 * (16 + max(G.shape) ** 0.5)
    return 2 * sum(L ** (len(sizes) - 1 - k) * eta * v for k, v in enumerate(sizes))


@pytest.mark.gpu
@pytest.mark.parametrize("coef,steps", [(COEF, 5), (COEF, 6), (COEF, 10), (COEF, 12), (COEF, 16),
                                        (COEF, 20), ((2.0, -1.5, 0.5), 30), ((1.5, -0.5, 0.0), 40)])
def test_thin_in_many_steps(coef, steps):
    """Shorter sides of 16 or less are computed in 64 bits, however many steps."""
    coef = FP32(coef)  # as the kernels have them
    grads = [hard(k).cuda() for k in HARD]
    for G, o, again in zip(grads, ops.newton_schulz(grads, steps=steps, coefficients=coef),
                           ops.newton_schulz(grads[::-1], steps=steps, coefficients=coef)[::-1]):
        ref, sizes = reference(G.cpu(), steps, coef)
        off, size = float((o.cpu().double() - ref).norm()), float(ref.norm())
        assert off <= tolerance64(G, sizes, coef) + 2.0 ** -24 * size, (tuple(G.shape), off, size)
        assert torch.equal(o, again)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("coef", [COEF, (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)])
@pytest.mark.parametrize("steps", [12, 20, 30, 100])
def test_many_steps_stay_bounded(steps, coef, dev):
    """No singular value leaves the polynomial's range, whatever the matrix and the
    way it goes: 1.2025 for the default one, 1 for the others."""
    grads = [hard(k).to(dev) for k in HARD]
    grads += [gradient(kind, m, n, seed=m).to(dev) for m, n in ((30, 50), (200, 90), (300, 260))
              for kind in ("low", "one")]
    for few in (grads[:-2], grads):  # with a large one all but the thin go its way
        for o in ops.newton_schulz(few, steps=steps, coefficients=coef):
            top = float(torch.linalg.matrix_norm(o.cpu().double(), 2))
            # a last step's roundings: 1 % is 2^17 of them
            assert top <= 1.01 * (1.2025 if coef is COEF else 1.0)


@pytest.mark.parametrize("dev", DEVICES)
def test_update_in_many_steps(dev):
    """The momentum moves on once, not once in every run of steps."""
    shapes = [(5, 64), (9, 3000), (16, 16), (40, 16)]
    ws, gs, ms = [[gradient("full", *s, seed=k).to(dev) for s in shapes] for k in (1, 2, 3)]
    w0, m0 = [[t.cpu().clone() for t in ts] for ts in (ws, ms)]
    ops.muon_update(ws, gs, ms, lr=0.05, momentum=0.9, weight_decay=0.1, steps=12)
    for w, g, m, wb, mb in zip(ws, gs, ms, w0, m0):
        ref, mref, u, sizes, s = step_reference(wb, g.cpu(), mb, 0.05, 0.9, 0.1, True, steps=12)
        e = 2.0 ** -23 * ((0.9 * mb.double()).abs() + mref.abs())
        assert ((m.cpu().double() - mref).abs() <= e).all()
        # full rank, singular values of 0.1 and more after the first step: 12 steps
        # in fp32 of the default polynomial, whose slope past that is 3.9 at most and
        # 1.4 on average, lose 2^-22 (16 + 64) 1.4^12 < 2^-9
        assert float((w.cpu().double() - ref).norm()) <= s * 2.0 ** -9 * float(min(w.shape)) ** 0.5 \
            + 2.0 ** -22 * float(ref.norm())


@pytest.mark.parametrize("dev", DEVICES)
def test_no_gradient_passes(dev):
    """The result has no autograd graph, on either device and in every form."""
    G = gradient("full", 4, 6).to(dev).requires_grad_()
    S = torch.stack([gradient("full", 20, 30, seed=k) for k in range(3)]).to(dev).requires_grad_()
    for leaf, outs in ((G, [ops.newton_schulz(G, steps=2)]), (G, ops.newton_schulz([G], steps=2)),
                       (S, [ops.newton_schulz(S, steps=2)])):
        for o in outs:
            assert not o.requires_grad and o.grad_fn is None
            assert torch.equal(o, ops.newton_schulz(leaf.detach(), steps=2))


@pytest.mark.parametrize("dev", DEVICES)
def test_steps_as_a_float(dev):
    """A whole number is one, whatever its type and whatever was called before."""
    G = gradient("full", 20, 30).to(dev)
    ops._ns_scale.cache_clear()
    first = ops.newton_schulz(G, steps=7.0)
    assert torch.equal(first, ops.newton_schulz(G, steps=7))
    ops._ns_scale.cache_clear()
    w, m = [torch.zeros_like(G)], [torch.zeros_like(G)]
    ops.muon_update(w, [G], m, lr=1.0, steps=3.0)
    v, m = [torch.zeros_like(G)], [torch.zeros_like(G)]
    ops.muon_update(v, [G], m, lr=1.0, steps=3)
    assert torch.equal(w[0], v[0])
    for steps in (2.5, "5", None, float("nan"), -1.0):
        with pytest.raises(ValueError):
            ops.newton_schulz(G, steps=steps)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("coef,steps", [((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 9), (COEF, 1),
                                        (COEF, 3), ((0.5, 0.0, 0.0), 2)])
def test_other_polynomials_of_thin_matrices(coef, steps, dev):
    for m, n in ((5, 64), (64, 5), (16, 16), (12, 12), (9, 3000), (257, 3), (1, 1)):
        G = gradient("offset", m, n).to(dev)
        check(G, ops.newton_schulz(G, steps=steps, coefficients=coef), steps, coef)


@pytest.mark.gpu
def test_many_steps_in_a_graph():
    """Runs of steps of long and short thin matrices, captured: the eager bits."""
    gs = [gradient("low", *s, seed=1).cuda() for s in ((5, 1300), (16, 16), (40, 60))]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.newton_schulz(gs, steps=13)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.newton_schulz(gs, steps=13)
    for turn in range(4):
        for g in gs:
            g.copy_(gradient("full", *g.shape, seed=20 + turn))
        eager = ops.newton_schulz(gs, steps=13)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(30, 50), (120, 100), (300, 400)])
@pytest.mark.parametrize("steps", [5, 10])
def test_rows_far_apart(m, n, steps):
    """Rows far below the others: off by what the pairs' last place comes to. X is held
    to 2^-39 of the norm; a step adds that again, and A's and B's last places (2^-39
    and 2^-38, times |b| + 2c < 9 and 1) times a column of X, which is 1 long at most
    and meets them with any signs: three times their half steps, 16 for all. A later
    step multiplies by a in these rows: 1 + 17 (1 / a + 1 / a^2 + ...) < 8 of the first.
    """
    G = gradient("full", m, n, seed=2) * torch.logspace(0, -9, m)[:, None]
    got = ops.newton_schulz(G.cuda(), steps=steps).cpu()
    check(G, got, steps)
    ref = reference(G, steps)[0]
    low = G.norm(dim=1) / G.norm() < 2.0 ** -24
    assert low.sum() >= m // 6
    worst = float((got.double() - ref)[low].abs().max())
    assert worst <= 8 * 2.0 ** -39 * COEF[0] ** steps
