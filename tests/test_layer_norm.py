"""Layer norm forward and backward against the formulas in 64 bits."""

import pytest
import torch

from flowml import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32

# Longest chain of fp32 additions in a row sum: at most 64 values per lane one
# after the other, 16 waves, 6 steps in a wave; rows beyond a block's registers
# add D / 1024 values per lane.
def chain(d):
    return 96 + d // 1024


def half_step(t):
    return torch.finfo(t).eps / 2


def make(n, d, dtype, seed=0, dev="cpu", affine=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, d, generator=g) * (torch.rand(n, 1, generator=g) * 3 + 0.1)
    x = (x + torch.randn(d, generator=g)).to(dtype)
    w = torch.randn(d, generator=g) if affine else None
    b = torch.randn(d, generator=g) if affine else None
    dy = torch.randn(n, d, generator=g).to(dtype)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return to(x), to(w), to(b), to(dy)


def act64(z, act):
    return z if act == "none" else z.clamp_min(0) if act == "relu" else torch.sigmoid(z)


def check_forward(x, w, b, eps, act, got):
    """Every element within what fp32 sums and one rounding can lose."""
    y, mean, rstd = [t.cpu() for t in got]
    x = x.cpu()
    x64 = x.double()
    n, d = x.shape
    w64 = torch.ones(d).double() if w is None else w.cpu().double()
    b64 = torch.zeros(d).double() if b is None else b.cpu().double()
    mu = x64.mean(1, keepdim=True)
    var = ((x64 - mu) ** 2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x64 - mu) * r
    ref = act64(xh * w64 + b64, act)
    k = chain(d)
    size = x64.abs().amax(1, keepdim=True)
    # mean: k roundings of at most mean|x|; var: as many, relative, and the
    # mean's own error; z: both, and a few roundings of its own
    e_mean = k * U * size
    e_var = 2 * k * U * var + e_mean ** 2
    e_r = r * (e_var / (2 * (var + eps)) + 4 * U)
    e_z = w64.abs() * (r * e_mean + xh.abs() * (e_r / r) + 4 * U * xh.abs()) + 2 * U * (
        (xh * w64).abs() + b64.abs())
    e_y = e_z + (8 * U if act == "sigmoid" else 0)
    tol = e_y + (half_step(y.dtype) * (ref.abs() + e_y) if y.dtype != torch.float32 else 0)
    if y.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # below the smallest normal a step is 2^-24
    assert y.dtype == x.dtype and y.shape == x.shape
    assert ((y.double() - ref).abs() <= tol).all()
    assert ((mean.double() - mu[:, 0]).abs() <= e_mean[:, 0] + U * mu[:, 0].abs()).all()
    assert ((rstd.double() - r[:, 0]).abs() <= e_r[:, 0] + U * r[:, 0]).all()


def check_backward(dy, x, y, mean, rstd, w, act, got):
    dx, dw, db = [t.cpu().double() for t in got]
    n, d = x.shape
    x64, dz = x.cpu().double(), dy.cpu().double()
    y64 = None if y is None else y.cpu().double()
    if act == "relu":
        dz = dz * (y64 > 0)
    elif act == "sigmoid":
        dz = dz * (y64 * (1 - y64))
    w64 = torch.ones(d).double() if w is None else w.cpu().double()
    mu, r = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    xh = (x64 - mu) * r
    p = dz * w64
    s, q = p.mean(1, keepdim=True), (p * xh).mean(1, keepdim=True)
    ref = r * (p - s - xh * q)
    k = chain(d) + 8
    e = r * U * (k * (p.abs().mean(1, keepdim=True) + xh.abs() * (p * xh).abs().mean(1, keepdim=True))
                 + 8 * (p.abs() + s.abs() + (xh * q).abs()))
    tol = e + half_step(x.dtype) * (ref.abs() + e)
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got[0].dtype == x.dtype and ((dx - ref).abs() <= tol).all()
    # the longest chain over rows: one lane's share of them, groups and slabs
    k = min(n, 640) + 8
    assert ((dw - (dz * xh).sum(0)).abs() <= U * k * (dz * xh).abs().sum(0)).all()
    assert ((db - dz.sum(0)).abs() <= U * k * dz.abs().sum(0)).all()


SIZES = [(1, 1), (3, 1), (5, 2), (7, 3), (300, 5), (17, 8), (1000, 9), (129, 41), (64, 64),
         (257, 127), (4100, 128), (33, 129), (70, 511), (50, 1000), (19, 1025), (5, 2049),
         (9, 4099), (3, 8192), (2, 8193)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", SIZES)
def test_forward_and_backward(n, d, dtype, dev):
    for i, act in enumerate(["none", "relu", "sigmoid"]):
        x, w, b, dy = make(n, d, dtype, seed=n + d + i, dev=dev, affine=i != 0)
        out = ops.layer_norm(x, w, b, eps=1e-5, activation=act)
        check_forward(x, w, b, 1e-5, act, out)
        y, mean, rstd = out
        got = ops.layer_norm_grad(dy, x, mean, rstd, w, y=y, activation=act)
        check_backward(dy, x, y, mean, rstd, w, act, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "relu"])
def test_every_layout(act, dtype):
    """Row lengths at both sides of each change of lanes and pieces."""
    vec = 16 // dtype.itemsize
    for k in [1, 2, 4, 8, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256, 320, 512, 640, 1024, 1500, 2048,
              3000, 4096]:
        for d in (k * vec, k * vec + 1):
            n = 37 if d < 3000 else 5
            x, w, b, dy = make(n, d, dtype, seed=d, dev="cuda")
            out = ops.layer_norm(x, w, b, activation=act)
            check_forward(x, w, b, 1e-5, act, out)
            y, mean, rstd = out
            check_backward(dy, x, y, mean, rstd, w, act,
                           ops.layer_norm_grad(dy, x, mean, rstd, w, y=y, activation=act))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [16384, 16385, 40000, 100001])
def test_long_rows(d, dtype):
    x, w, b, dy = make(6, d, dtype, seed=d, dev="cuda")
    out = ops.layer_norm(x, w, b, activation="sigmoid")
    check_forward(x, w, b, 1e-5, "sigmoid", out)
    got = ops.layer_norm_grad(dy, x, out[1], out[2], w, y=out[0], activation="sigmoid")
    check_backward(dy, x, out[0], out[1], out[2], w, "sigmoid", got)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d", [(70_001, 64), (300_000, 8), (20_011, 500), (3001, 2048)])
def test_many_rows(n, d):
    x, w, b, dy = make(n, d, torch.bfloat16, seed=d, dev="cuda")
    out = ops.layer_norm(x, w, b, activation="relu")
    check_forward(x, w, b, 1e-5, "relu", out)
    got = ops.layer_norm_grad(dy, x, out[1], out[2], w, y=out[0], activation="relu")
    check_backward(dy, x, out[0], out[1], out[2], w, "relu", got)
    again = ops.layer_norm_grad(dy, x, out[1], out[2], w, y=out[0], activation="relu")
    assert all(torch.equal(p, q) for p, q in zip(got, again))  # one order of sums


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """The last rows of an array of over 2^32 bytes (and 2^31 values)."""
    n, d = (1 << 31) // 512 + 1000, 512
    x = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    x.fill_(1.0)
    tail = make(1000, d, torch.bfloat16, seed=3, dev="cuda")
    x[-1000:] = tail[0]
    y, mean, rstd = ops.layer_norm(x, tail[1], tail[2])
    check_forward(tail[0], tail[1], tail[2], 1e-5, "none", (y[-1000:], mean[-1000:], rstd[-1000:]))
    del y
    dx, dw, db = ops.layer_norm_grad(x, x, mean, rstd, tail[1])
    small = ops.layer_norm_grad(tail[0], tail[0], mean[-1000:], rstd[-1000:], tail[1])
    assert torch.equal(dx[-1000:], small[0])


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows(dev):
    x, w, b, dy = make(0, 7, torch.float32, dev=dev)
    y, mean, rstd = ops.layer_norm(x, w, b)
    assert y.shape == (0, 7) and mean.shape == rstd.shape == (0,)
    dx, dw, db = ops.layer_norm_grad(dy, x, mean, rstd, w)
    assert dx.shape == (0, 7) and (dw == 0).all() and (db == 0).all() and dw.shape == (7,)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype, dev):
    """Rows apart, columns apart, a row expanded, storage that starts odd."""
    x, w, b, dy = make(40, 90, dtype, seed=2, dev=dev)
    for xs, dys in ((x[:, 3:80], dy[:, 5:82]), (x[::2, :77], dy[1::2, 1:78]),
                    (x[:, ::2], dy[:, 1::2]), (x[:, 1:2].expand(40, 45).clone().T.contiguous().T, dy[:, :45]),
                    (x[:1, :45].expand(40, 45), dy[:1, 7:52].expand(40, 45))):
        d = xs.shape[1]
        out = ops.layer_norm(xs, w[:d], b[:d], activation="relu")
        check_forward(xs, w[:d], b[:d], 1e-5, "relu", out)
        flat = ops.layer_norm(xs.clone(memory_format=torch.contiguous_format), w[:d], b[:d], activation="relu")
        assert all(torch.equal(p, q) for p, q in zip(out, flat))
        ys = torch.empty(xs.shape[0], d + 3, dtype=dtype, device=dev)[:, 1:d + 1].copy_(out[0])
        got = ops.layer_norm_grad(dys, xs, out[1], out[2], w[:d], y=ys, activation="relu")
        check_backward(dys, xs, ys, out[1], out[2], w[:d], "relu", got)


@pytest.mark.parametrize("dev", DEVICES)
def test_special_values(dev):
    """Rows keep to themselves: a NaN or infinity spoils its own row, and the
    column sums that it enters; constant rows come out as the bias."""
    x, w, b, dy = make(8, 70, torch.float32, seed=4, dev=dev)
    x[1, 3] = float("nan")
    x[2, 60] = float("inf")
    x[3] = 4.0
    x[4] = 1e30      # the variance of 1e30's rounding noise is not a number's
    x[5] *= 1e-30
    y, mean, rstd = ops.layer_norm(x, w, b)
    assert y[1].isnan().all() and y[2].isnan().any() and mean[2] == float("inf")
    assert torch.equal(y[3], b) and rstd[3].item() == pytest.approx(1e-5 ** -0.5, rel=1e-6)
    for i in (0, 6, 7):
        check_forward(x[i:i + 1], w, b, 1e-5, "none", (y[i:i + 1], mean[i:i + 1], rstd[i:i + 1]))
    assert torch.allclose(y[5], b, atol=1e-6)
    r = ops.layer_norm(x, w, b, activation="relu")[0]
    assert r[1].isnan().all()
    dx, dw, db = ops.layer_norm_grad(dy, x, mean, rstd, w)
    keep = [0, 3, 5, 6, 7]
    ok = ops.layer_norm_grad(dy[keep], x[keep], mean[keep], rstd[keep], w)
    assert torch.equal(dx[keep], ok[0]) and dx[1].isnan().all()
    assert dw[3].isnan() and torch.isfinite(db).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_gradient_against_differences(act, dev):
    """<dL, v> against central differences of the formula in 64 bits."""
    x, w, b, dy = make(9, 33, torch.float32, seed=6, dev=dev)
    y, mean, rstd = ops.layer_norm(x, w, b, activation=act)
    dx, dw, db = [t.cpu().double() for t in
                  ops.layer_norm_grad(dy, x, mean, rstd, w, y=y, activation=act)]
    X, W, B, dY = [t.cpu().double() for t in (x, w, b, dy)]

    def loss(x, w, b):
        xh = (x - x.mean(1, keepdim=True)) / torch.sqrt(x.var(1, correction=0, keepdim=True) + 1e-5)
        return (act64(xh * w + b, act) * dY).sum()

    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        v = [torch.randn(t.shape, generator=g).double() for t in (X, W, B)]
        h = 1e-5
        num = (loss(*[t + h * u for t, u in zip((X, W, B), v)])
               - loss(*[t - h * u for t, u in zip((X, W, B), v)])) / (2 * h)
        ana = sum((t * u).sum() for t, u in zip((dx, dw, db), v))
        size = sum((t * u).abs().sum() for t, u in zip((dx, dw, db), v))
        # differences: h^2 and 2^-53 / h, both under 1e-9; fp32: 100 roundings
        assert abs(num - ana) <= 1e-7 * size + 100 * U * size


@pytest.mark.gpu
def test_stream_and_graph():
    """On a stream of its own, and captured: replays follow new inputs."""
    x, w, b, dy = make(500, 200, torch.bfloat16, seed=8, dev="cuda")

    def step():
        y, mean, rstd = ops.layer_norm(x, w, b, activation="relu")
        return (y, mean, rstd) + ops.layer_norm_grad(dy, x, mean, rstd, w, y=y, activation="relu")

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        fresh = make(500, 200, torch.bfloat16, seed=20 + seed, dev="cuda")
        x.copy_(fresh[0])
        dy.copy_(fresh[3])
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_refusals():
    x, w, b, dy = make(4, 6, torch.float32)
    y, mean, rstd = ops.layer_norm(x, w, b)
    bad = [
        lambda: ops.layer_norm(x[0]),
        lambda: ops.layer_norm(x[:, :0]),
        lambda: ops.layer_norm(x.double()),
        lambda: ops.layer_norm(x.to(torch.int32)),
        lambda: ops.layer_norm(x, w[:5]),
        lambda: ops.layer_norm(x, w, b[None]),
        lambda: ops.layer_norm(x, activation="tanh"),
        lambda: ops.layer_norm_grad(dy[:3], x, mean, rstd, w),
        lambda: ops.layer_norm_grad(dy.bfloat16(), x, mean, rstd, w),
        lambda: ops.layer_norm_grad(dy, x, mean[:3], rstd, w),
        lambda: ops.layer_norm_grad(dy, x, mean, rstd.double(), w),
        lambda: ops.layer_norm_grad(dy, x, mean, rstd, w, activation="relu"),
        lambda: ops.layer_norm_grad(dy, x, mean, rstd, w, y=y[:, :5], activation="relu"),
        lambda: ops.layer_norm_grad(dy, x, mean, rstd, w[:2]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("not refused:", i)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,dtype", [
    (70_001, 64, torch.float32), (20_011, 500, torch.float16), (9001, 1100, torch.float32),
    (3000, 4099, torch.float32), (3000, 4099, torch.float16), (4101, 8192, torch.float32),
    (2101, 16384, torch.float32), (2101, 16384, torch.float16)])
def test_many_rows_of_other_types(n, d, dtype):
    """More rows than the grid holds, so that blocks go through several, and (8192
    and 16384 columns of f32) results of over 128 MB."""
    x, w, b, dy = make(n, d, dtype, seed=d, dev="cuda")
    for act in ("relu", "none") if d < 4000 else ("relu",):
        y, mean, rstd = out = ops.layer_norm(x, w, b, activation=act)
        check_forward(x, w, b, 1e-5, act, out)
        got = ops.layer_norm_grad(dy, x, mean, rstd, w, y=y, activation=act)
        check_backward(dy, x, y, mean, rstd, w, act, got)
