"""Layer norm with the residual's addition against float64.

u = 2^-24 for an fp32 operation; r: rounding of a result to the tensors' type (2^-8 for bf16, 2 u for fp32); a: the mean of |h| of a row.
The mean is off by dmu = (n + 2) u a and a centred element by c = dmu + u (|h| + |mu|).  The mean of squares is off by 2 mean(|h - mu| c) + c^2
and (n + 4) u of itself, its inverse root by half of that relative to it, and 2 u more: di of itself.  xh = (h - mu) s by e = s c + |xh| (di + 2 u).
  y   : e |w| + 2 u (|xh w| + |b|) + r |y|
  dx  : with g = dy w, mg, mx the means of g and g xh: s (2 u |g| + (n + 2) u mean|g| + e |mx| + |xh| (mean(|g| e) + (n + 4) u mean|g xh|))
        + di |dx - dh| + 6 u s (|g| + |mg| + |xh mx|) + 2 u |dh| + r |dx|
  dw  : sum of |dy| e + (rows + 2) u sum |dy xh| + r |dw|;  db: (rows + 2) u sum |dy| + r |db|"""
import ctypes

import pytest
import torch

import spion_amd
from spion_amd import _lib
from spion_amd import norm as ln

pytestmark = pytest.mark.gpu
DEV, U, EPS = "cuda", 2.0 ** -24, 1e-5


@pytest.fixture(params=["node", "python"], autouse=True)
def both_nodes(request, monkeypatch):
    """Every test runs through the compiled node and through the Python function."""
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


def _close(name, got, value, bound):
    assert got.shape == value.shape and bool(torch.isfinite(got.float()).all()), name
    far = (got.detach().double() - value).abs() - bound
    assert float(far.max()) <= 1e-30, f"{name}: {float(far.max()):.3e} beyond its bound"


def _check(x, w, b, res, dy, dh, y, h, dx, dw, db, eps=EPS):
    bf = x.dtype == torch.bfloat16
    r = 2.0 ** -8 if bf else 2 * U
    n = x.shape[-1]
    X = x.detach().reshape(-1, n)
    H = X.double() if res is None else (X + res.detach().reshape(-1, n)).double()  # one rounding, to the type
    if res is not None:
        assert torch.equal(h.reshape(-1, n).double(), H)
    W = w.detach().double()
    Bi = torch.zeros_like(W) if b is None else b.detach().double()
    mean = lambda t: t.mean(1, keepdim=True)  # noqa: E731
    mu = mean(H)
    C = H - mu
    s = 1.0 / torch.sqrt(mean(C * C) + eps)
    xh = C * s
    c = (n + 2) * U * mean(H.abs()) + U * (H.abs() + mu.abs())
    di = (mean(C.abs() * c) + 0.5 * mean(c * c)) * s * s + (0.5 * (n + 4) + 2) * U
    e = s * c + xh.abs() * (di + 2 * U)
    Y = xh * W + Bi
    _close("y", y.reshape(-1, n), Y, e * W.abs() + 2 * U * ((xh * W).abs() + Bi.abs()) + r * Y.abs())
    if dy is None:
        return
    G = dy.double().reshape(-1, n)
    D = torch.zeros_like(G) if dh is None else dh.double().reshape(-1, n)
    g = G * W
    mg, mx = mean(g), mean(g * xh)
    dX = s * (g - mg - xh * mx)
    bound = s * (2 * U * g.abs() + (n + 2) * U * mean(g.abs()) + e * mx.abs() + xh.abs() * (mean(g.abs() * e) + (n + 4) * U * mean((g * xh).abs())))
    bound = bound + di * dX.abs() + 6 * U * s * (g.abs() + mg.abs() + (xh * mx).abs()) + 2 * U * D.abs()
    dX = dX + D
    _close("dx", dx.reshape(-1, n), dX, bound + r * dX.abs())
    rows = X.shape[0]
    dW = (G * xh).sum(0)
    _close("dw", dw, dW, (G.abs() * e).sum(0) + (rows + 2) * U * (G * xh).abs().sum(0) + r * dW.abs())
    if b is not None:
        dB = G.sum(0)
        _close("db", db, dB, (rows + 2) * U * G.abs().sum(0) + r * dB.abs())


def _train(x, w, b, res, dy, dh, eps=EPS):
    """y, h, dx, dw, db"""
    given = {n: t.detach().requires_grad_() for n, t in (("x", x), ("weight", w), ("bias", b), ("residual", res)) if t is not None}
    out = spion_amd.layer_norm(**given, eps=eps)
    if res is None:
        y, h, grads = out, None, torch.autograd.grad(out, list(given.values()), dy)
    else:
        (y, h), grads = out, torch.autograd.grad(out, list(given.values()), (dy, dh))
    grads = dict(zip(given, grads))
    if res is not None:
        assert torch.equal(grads["x"], grads["residual"])
    return y, h, grads["x"], grads["weight"], grads.get("bias")


def _inputs(seed, shape, dtype, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x, res, dy, dh = (torch.randn(shape, generator=g).to(DEV) for _ in range(4))
    w, b = (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(DEV), 0.5 * torch.randn(shape[-1], generator=g).to(DEV)
    return tuple(t.to(dtype) for t in (x + offset, w, b, res, dy, dh))


# every number of lanes and pieces to a row and their edges, rows past the registers, rows that do not start on 16 bytes
WIDTHS = [1, 2, 3, 7, 8, 31, 64, 65, 127, 128, 129, 256, 257, 511, 512, 520, 768, 1000, 1001, 1024, 1032, 2047, 2048, 2056, 4095, 4096, 4104, 5415,
          8192, 8200, 16383, 16384, 16392, 32768, 32770, 40001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", WIDTHS)
def test_widths(n, dtype):
    for rows in (1, 37):
        x, w, b, res, dy, dh = _inputs(n, (rows, n), dtype)
        _check(x, w, b, res, dy, dh, *_train(x, w, b, res, dy, dh))
        _check(x, w, None, None, dy, None, *_train(x, w, None, None, dy, None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(20000, 64), (5000, 129), (3, 1000, 256), (2, 3, 700, 48), (2500, 2048), (1500, 5000), (600, 20001)])
def test_many_rows(shape, dtype):
    """More rows than the work-groups take at once."""
    x, w, b, res, dy, dh = _inputs(1, shape, dtype)
    got = _train(x, w, b, res, dy, dh)
    _check(x, w, b, res, dy, dh, *got)
    for a, c in zip(got, _train(x, w, b, res, dy, dh)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 1000, 9000, 40000])
def test_a_mean_far_from_zero(n, dtype):
    """The variance is of the centred elements: a mean of 1000 deviations costs the rounding of the mean, not its square."""
    x, w, b, _, dy, _ = _inputs(7, (19, n), dtype, offset=1000.0)
    _check(x, w, b, None, dy, None, *_train(x, w, b, None, dy, None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_constant_rows(dtype):
    """No variance: y is the bias, and the gradient what eps leaves of it."""
    x, w, b, _, dy, _ = _inputs(8, (5, 96), dtype)
    x = x[:, :1].expand(5, 96)
    y, _, dx, dw, db = _train(x, w, b, None, dy, None)
    _check(x, w, b, None, dy, None, y, None, dx, dw, db)
    assert bool(((y.float() - b.float()).abs() < 0.01).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 1000, 9000])
def test_strides_and_alignments(n, dtype):
    g = torch.Generator().manual_seed(2)
    big = torch.randn(30, 2 * n + 3, generator=g).to(dtype).to(DEV)
    w, b = (torch.randn(2 * n, generator=g).to(dtype).to(DEV)[::2] for _ in range(2))
    for x, res, dy, dh in ((big[:, :n], big[:, n:2 * n], big[:, 1:n + 1], big[:, 3:n + 3]),
                           (big[:, :n].t().contiguous().t(), big[:1, :n].expand(30, n), big[::3, :n].repeat(3, 1), big[:, ::2][:, :n])):
        _check(x, w, b, res, dy, dh, *_train(x, w, b, res, dy, dh))


def test_one_gradient_of_two():
    x, w, b, res, dy, _ = _inputs(3, (50, 96), torch.float32)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, res)]
    y, h = spion_amd.layer_norm(*leaves)
    dx, dw, db, _ = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    _check(x, w, b, res, dy, None, y, h, dx, dw, db)
    dx, dw, db, dr = torch.autograd.grad(h, leaves, dy)
    assert torch.equal(dx, dy) and torch.equal(dr, dy) and not bool(dw.any()) and not bool(db.any())


def test_gradient_against_differences():
    """Central differences of <y, dy> + <h, dh> along each operand: fp32 results leave 2^-23 sqrt(n) |dy| |y| / step, curvature
    step^2 of the value."""
    x, w, b, res, dy, dh = _inputs(4, (40, 200), torch.float32)
    _, _, dx, dw, db = _train(x, w, b, res, dy, dh)
    g = torch.Generator().manual_seed(9)
    step = 2.0 ** -6
    for t, grad in ((x, dx), (res, dx), (w, dw), (b, db)):
        u = torch.randn(t.shape, generator=g).to(DEV)
        f = []
        for s in (step, -step):
            y, h = spion_amd.layer_norm(*(v + s * u if v is t else v for v in (x, w, b, res)))
            f.append(float((y.double() * dy).sum() + (h.double() * dh).sum()))
        size = float((grad.double() * u).abs().sum())
        noise = 4 * 2.0 ** -23 * (40 * 200) ** 0.5 * 16 / step
        assert abs((f[0] - f[1]) / (2 * step) - float((grad.double() * u).sum())) <= 1e-3 * size + noise


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16), (4, 0)])
def test_nothing_to_normalise(shape):
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    w, b = (torch.ones(shape[-1], device=DEV, requires_grad=True) for _ in range(2))
    y, h = spion_amd.layer_norm(x, w, b, x.detach())
    dx, dw, db = torch.autograd.grad((y.sum() + h.sum()), (x, w, b))
    assert y.shape == h.shape == dx.shape == torch.Size(shape) and not bool(dw.any()) and not bool(db.any())


def test_rows_of_infinities_and_nan_stay_their_own():
    x, w, b, _, dy, _ = _inputs(5, (40, 130), torch.float32)
    x[3, 7], x[11, 0], x[39, 129] = float("inf"), float("nan"), -float("inf")
    y, _, dx, _, _ = _train(x, w, b, None, dy, None)
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 11, 39]] = True
    assert torch.equal(~torch.isfinite(y).all(1), bad) and torch.equal(~torch.isfinite(dx).all(1), bad)


def test_streams_and_replays():
    x, w, b, res, dy, dh = _inputs(6, (500, 321), torch.float32)

    def step():
        return [t.detach() for t in _train(x, w, b, res, dy, dh)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(4):
        for i, t in enumerate((x, res, dy, dh)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * turn + i)))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.current_stream().wait_stream(side)
        for a, c in zip(outs, eager):
            assert torch.equal(a, c), turn


def test_c_entry_points_keep_to_their_buffers():
    for n in (64, 250, 9001):
        x, w, b, res, dy, dh = _inputs(6, (21, n), torch.float32)
        y, h, dx = (torch.full((25, n), 7.0, device=DEV) for _ in range(3))
        dw, db = (torch.full((n + 4,), 7.0, device=DEV) for _ in range(2))
        lib, stream = ln._layer_lib(), torch.cuda.current_stream().cuda_stream
        c = ln._LayerCall(x=x.data_ptr(), residual=res.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), y=y.data_ptr(), h=h.data_ptr(),
                          dy=dy.data_ptr(), dh=dh.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=db.data_ptr(), rows=21, width=n,
                          x_stride=n, residual_stride=n, dy_stride=n, dh_stride=n, eps=EPS)
        assert lib.spion_layer_norm_forward(ctypes.addressof(c), stream) == 0
        floats = lib.spion_layer_norm_workspace(ctypes.addressof(c))
        ws = torch.full((floats + 4,), 7.0, device=DEV)
        c.x, c.workspace, c.workspace_floats = h.data_ptr(), ws.data_ptr(), floats
        assert lib.spion_layer_norm_backward(ctypes.addressof(c), stream) == 0
        for t in (y, h, dx):
            assert bool((t[21:] == 7.0).all())
        for t in (dw, db):
            assert bool((t[n:] == 7.0).all())
        assert bool((ws[floats:] == 7.0).all())
        _check(x, w, b, res, dy, dh, y[:21], h[:21], dx[:21], dw[:n], db[:n])
        db.fill_(7.0)
        c.dbias = None
        assert lib.spion_layer_norm_backward(ctypes.addressof(c), stream) == 0
        assert bool((db == 7.0).all())
        c.workspace_floats = floats - 1
        assert lib.spion_layer_norm_backward(ctypes.addressof(c), stream) != 0
        with pytest.raises(_lib.SpionLibraryError, match="workspace"):
            _lib.check_error()


def test_module():
    mod = spion_amd.LayerNorm(64).to(DEV)
    x = torch.randn(2, 7, 64, device=DEV, dtype=torch.bfloat16)
    y, h = mod(x, x)
    (y.float().sum() + h.float().sum()).backward()
    assert mod.weight.grad.dtype == mod.bias.grad.dtype == torch.float32 and y.dtype == torch.bfloat16
    plain = spion_amd.LayerNorm(64, bias=False).to(DEV)
    assert torch.equal(plain(x), y.new_tensor(0) + spion_amd.layer_norm(x, plain.weight.detach().bfloat16()))


def test_a_second_derivative_is_refused():
    x = torch.randn(5, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV)
    y = spion_amd.layer_norm(x, w)
    (g,) = torch.autograd.grad(y, x, torch.randn_like(y).requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_traced_norm_computes(dtype, residual):
    """A traced norm gives on other inputs what the function gives."""
    def inputs(seed):
        return _inputs(seed, (37, 200), dtype)[:1] + _inputs(seed, (37, 200), dtype)[3:4]

    w, b = (torch.linspace(0.5, 1.5, 200, device=DEV).to(dtype) for _ in range(2))
    call = lambda x, r: spion_amd.layer_norm(x, w, b, r if residual else None)  # noqa: E731
    with torch.no_grad():
        traced = torch.jit.trace(call, inputs(1), check_trace=False)
        got, want = traced(*inputs(2)), call(*inputs(2))
    for a, c in zip(*(y if isinstance(y, tuple) else (y,) for y in (got, want))):
        assert torch.equal(a, c)


def test_calls_go_by_their_own_status():
    """What another call has left in the process-wide error slot neither fails a call nor is taken by it."""
    lib = _lib.core()
    x, w, b, _, dy, _ = _inputs(5, (5, 64), torch.float32)
    lib.spion_set_stream(None, None)  # a failure: no handle
    try:
        got = _train(x, w, b, None, dy, None)
        assert lib.spion_error_pending() == 1
    finally:
        lib.spion_clear_error()
    _check(x, w, b, None, dy, None, *got)


def test_rows_wider_than_a_launch_has_threads_for():
    """2^25 columns and more, twice for weight and bias: at 64 threads to a column their gradients would take 2^32 threads.  Elements of 1 and -1
    and a mean near 0: every element of a sum is exact, and the sums' roundings stay below 64 u of the magnitudes."""
    n = (1 << 25) + 5
    g = torch.Generator(device=DEV).manual_seed(1)
    x, dy = ((torch.randint(0, 2, (2, n), generator=g, device=DEV) * 2 - 1).float() for _ in range(2))
    w, b = torch.ones(n, device=DEV), torch.ones(n, device=DEV)
    y, _, dx, dw, db = _train(x, w, b, None, dy, None)
    X, G = x.double(), dy.double()
    C = X - X.mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt((C * C).mean(1, keepdim=True) + EPS)
    xh = C * inv
    assert float((y.detach().double() - xh - 1).abs().max()) <= 64 * U
    want = inv * (G - G.mean(1, keepdim=True) - xh * (G * xh).mean(1, keepdim=True))
    assert float((dx.double() - want).abs().max()) <= 64 * U
    assert float((dw.double() - (G * xh).sum(0)).abs().max()) <= 64 * U
    assert torch.equal(db.double(), G.sum(0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [769, 1026, 1159, 1535, 1536, 1537, 2500, 3071, 3073, 5000, 6143, 6144, 6145])
def test_three_pieces_a_lane(n, dtype):
    x, w, b, res, dy, dh = _inputs(n, (300, n), dtype)
    _check(x, w, b, res, dy, dh, *_train(x, w, b, res, dy, dh))
    _check(x, w, None, None, dy, None, *_train(x, w, None, None, dy, None))
