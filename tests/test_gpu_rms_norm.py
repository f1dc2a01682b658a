"""Root-mean-square norm with the residual's addition against float64.

u = 2^-24 for an fp32 operation; r: rounding of a result to the tensors' type (2^-8 for bf16, 2 u for fp32).  The mean of squares is
off by (n + 4) u of itself, its inverse root by half of that and 2 u more, y by two products: (n / 2 + 8) u + r of |y|.  Backward,
m = mean(dy w h inv): (2 n + 16) u of the mean of magnitudes; dx: (n + 16) u of inv (|dy w| + |h inv| mean|dy w h inv|) and of
|dh|, and the rounding; dw: a sum over the rows, (rows + n + 16) u of the magnitudes, and the rounding."""
import ctypes

import pytest
import torch

import spion_amd
from spion_amd import _lib
from spion_amd import norm as rn

pytestmark = pytest.mark.gpu
DEV, U, EPS = "cuda", 2.0 ** -24, 1e-6


@pytest.fixture(params=["node", "python"], autouse=True)
def both_nodes(request, monkeypatch):
    """Every test runs through the compiled node and through the Python function."""
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


def _close(name, got, value, bound):
    assert got.shape == value.shape and bool(torch.isfinite(got.float()).all()), name
    far = (got.detach().double() - value).abs() - bound
    assert float(far.max()) <= 1e-30, f"{name}: {float(far.max()):.3e} beyond its bound"


def _check(x, w, res, dy, dh, y, h, dx, dw, eps=EPS):
    bf = x.dtype == torch.bfloat16
    r = 2.0 ** -8 if bf else 2 * U
    n = x.shape[-1]
    X = x.detach().reshape(-1, n)
    H = X.double() if res is None else (X + res.detach().reshape(-1, n)).double()  # one rounding, to the type
    if res is not None:
        assert torch.equal(h.reshape(-1, n).double(), H)
    W = w.detach().double()
    inv = 1.0 / torch.sqrt((H * H).mean(1, keepdim=True) + eps)
    Y = H * inv * W
    _close("y", y.reshape(-1, n), Y, ((n / 2 + 8) * U + r) * Y.abs())
    if dy is None:
        return
    G = dy.double().reshape(-1, n)
    D = torch.zeros_like(G) if dh is None else dh.double().reshape(-1, n)
    gw, xh = G * W, H * inv
    dX = inv * (gw - xh * (gw * xh).mean(1, keepdim=True)) + D
    mag = inv * (gw.abs() + xh.abs() * (gw * xh).abs().mean(1, keepdim=True))
    _close("dx", dx.reshape(-1, n), dX, (2 * n + 32) * U * mag + 4 * U * D.abs() + r * dX.abs())
    dW = (G * xh).sum(0)
    _close("dw", dw, dW, (X.shape[0] + n + 16) * U * (G * xh).abs().sum(0) + r * dW.abs())


def _train(x, w, res, dy, dh):
    leaves = [t.detach().requires_grad_() for t in (x, w, res) if t is not None]
    out = spion_amd.rms_norm(*leaves)
    if res is None:
        return (out, None, *torch.autograd.grad(out, leaves, dy))
    y, h = out
    dx, dw, dr = torch.autograd.grad(out, leaves, (dy, dh))
    assert torch.equal(dx, dr)
    return y, h, dx, dw


# every number of lanes and pieces to a row and their edges, rows past the registers, rows that are not 16-byte aligned
WIDTHS = [1, 2, 3, 8, 31, 64, 65, 128, 129, 256, 257, 512, 520, 768, 1000, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 8200, 16384, 16392, 40000]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", WIDTHS)
def test_widths(n, dtype):
    g = torch.Generator().manual_seed(n)
    for rows in (1, 37):
        x, res, dy, dh = (torch.randn(rows, n, generator=g).to(dtype).to(DEV) for _ in range(4))
        w = (1 + 0.3 * torch.randn(n, generator=g)).to(dtype).to(DEV)
        _check(x, w, res, dy, dh, *_train(x, w, res, dy, dh))
        _check(x, w, None, dy, None, *_train(x, w, None, dy, None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(20000, 64), (5000, 129), (3, 1000, 256), (2, 3, 700, 48), (2500, 2048)])
def test_many_rows(shape, dtype):
    """More rows than the work-groups take at once."""
    g = torch.Generator().manual_seed(1)
    x, res, dy, dh = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(4))
    w = (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(dtype).to(DEV)
    got = _train(x, w, res, dy, dh)
    _check(x, w, res, dy, dh, *got)
    for a, b in zip(got, _train(x, w, res, dy, dh)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 1000, 9000])
def test_strides_and_alignments(n, dtype):
    g = torch.Generator().manual_seed(2)
    big = torch.randn(30, 2 * n + 3, generator=g).to(dtype).to(DEV)
    w = torch.randn(2 * n, generator=g).to(dtype).to(DEV)[::2]
    for x, res, dy, dh in ((big[:, :n], big[:, n:2 * n], big[:, 1:n + 1], big[:, 3:n + 3]),
                           (big[:, :n].t().contiguous().t(), big[:1, :n].expand(30, n), big[::3, :n].repeat(3, 1), big[:, ::2][:, :n])):
        _check(x, w, res, dy, dh, *_train(x, w, res, dy, dh))


def test_one_gradient_of_two():
    g = torch.Generator().manual_seed(3)
    x, res, dy = (torch.randn(50, 96, generator=g).to(DEV) for _ in range(3))
    w = torch.ones(96, device=DEV)
    leaves = [t.detach().requires_grad_() for t in (x, w, res)]
    y, h = spion_amd.rms_norm(*leaves)
    dx, dw, _ = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    _check(x, w, res, dy, None, y, h, dx, dw)
    dx, dw, dr = torch.autograd.grad(h, leaves, dy, allow_unused=True)
    assert torch.equal(dx, dy) and torch.equal(dr, dy) and not bool(dw.any())


def test_gradient_against_differences():
    """Central differences of <y, dy> + <h, dh> along each operand: fp32 results leave 2^-23 sqrt(n) |dy| |y| / step, curvature
    step^2 of the value."""
    g = torch.Generator().manual_seed(4)
    x, res, dy, dh = (torch.randn(40, 200, generator=g).to(DEV) for _ in range(4))
    w = (1 + 0.3 * torch.randn(200, generator=g)).to(DEV)
    _, _, dx, dw = _train(x, w, res, dy, dh)
    step = 2.0 ** -6
    for t, grad in ((x, dx), (res, dx), (w, dw)):
        u = torch.randn(t.shape, generator=g).to(DEV)
        f = []
        for s in (step, -step):
            y, h = spion_amd.rms_norm(*(v + s * u if v is t else v for v in (x, w, res)))
            f.append(float((y.double() * dy).sum() + (h.double() * dh).sum()))
        size = float((grad.double() * u).abs().sum())
        noise = 4 * 2.0 ** -23 * (40 * 200) ** 0.5 * 16 / step
        assert abs((f[0] - f[1]) / (2 * step) - float((grad.double() * u).sum())) <= 1e-3 * size + noise


def _e4m3(c):
    step = torch.exp2(torch.floor(torch.log2(c.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(c / step) * step, step


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 768), (37, 64), (5, 1000), (3, 257), (300, 4096), (2, 16384), (2, 40001)])
@pytest.mark.parametrize("residual", [False, True])
def test_fp8(rows, n, residual, dtype):
    g = torch.Generator().manual_seed(n)
    x = (torch.randn(rows, n, generator=g) * torch.exp(3 * torch.randn(rows, n, generator=g))).to(dtype).to(DEV)
    res = torch.randn(rows, n, generator=g).to(dtype).to(DEV) if residual else None
    w = torch.randn(n, generator=g).to(dtype).to(DEV)
    codes, scales, *h = spion_amd.rms_norm_fp8(x, w, res)
    H = x.double() if res is None else (x + res).double()
    if residual:
        assert torch.equal(h[0].double(), H)
    Y = H / torch.sqrt((H * H).mean(1, keepdim=True) + EPS) * w.double()
    S = Y.abs().amax(1) / 448
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scales.shape == (rows,)
    e = (n / 2 + 16) * U
    assert bool(((scales.double() - S).abs() <= e * S).all())
    # a code is the nearest to y / scale, as far as y and the scale are known: half a step, and their roundings
    c = codes.double()
    want, step = _e4m3(Y / S[:, None])
    assert bool(((c - Y / S[:, None]).abs() <= step / 2 * (1 + 1e-6) + 2 * e * (Y / S[:, None]).abs()).all())
    assert float((c != want).float().mean()) <= 1e-3 + 1 / c.numel()
    assert float(c.abs().max()) == 448


def test_fp8_of_unusual_rows():
    x = torch.ones(5, 100, device=DEV)
    x[0] = 0.0
    x[1] = 1e-42
    x[2, 7] = float("nan")
    x[3] *= 1e-30
    w = torch.ones(100, device=DEV)
    w[3] = 0.0
    codes, scales = spion_amd.rms_norm_fp8(x, w, eps=0.5)
    c = codes.float()
    assert not bool(c[0].any()) and float(scales[0]) == 2.0 ** -126
    assert bool(torch.isfinite(c[1]).all()) and bool(torch.isfinite(scales[1]))
    assert bool(torch.isnan(scales[2])) and bool(torch.isnan(c[2]).all())
    assert bool((c[3:, :3] == 448).all()) and bool((c[3:, 3] == 0).all())


def test_no_rows():
    for shape in ((0, 64), (3, 0, 8)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(shape[-1], device=DEV, requires_grad=True)
        y, h = spion_amd.rms_norm(x, w, x)
        dx, dw = torch.autograd.grad((y.sum() + h.sum()), (x, w))
        assert y.shape == h.shape == dx.shape == torch.Size(shape) and not bool(dw.any())
        with torch.no_grad():
            codes, scales = spion_amd.rms_norm_fp8(x, w)
        assert codes.shape == torch.Size(shape) and scales.shape == torch.Size(shape[:-1])


def test_streams_and_replays():
    g = torch.Generator().manual_seed(5)
    x, res, dy, dh = (torch.randn(500, 320, generator=g).to(DEV) for _ in range(4))
    w = torch.ones(320, device=DEV)

    def step():
        y, h, dx, dw = _train(x, w, res, dy, dh)
        with torch.no_grad():
            return [t.detach() for t in (y, h, dx, dw)] + [t.float() for t in spion_amd.rms_norm_fp8(x, w, res)]

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
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), turn


def test_c_entry_points_keep_to_their_buffers():
    for n in (64, 250):
        g = torch.Generator().manual_seed(6)
        x, res, dy, dh = (torch.randn(21, n, generator=g).to(DEV) for _ in range(4))
        w = torch.randn(n, generator=g).to(DEV)
        y, h, dx = (torch.full((25, n), 7.0, device=DEV) for _ in range(3))
        dw = torch.full((n + 4,), 7.0, device=DEV)
        codes, scales = torch.full((25, n), 7, dtype=torch.uint8, device=DEV), torch.full((25,), 7.0, device=DEV)
        lib, stream = rn._lib_typed(), torch.cuda.current_stream().cuda_stream
        c = rn._Call(x=x.data_ptr(), residual=res.data_ptr(), weight=w.data_ptr(), y=y.data_ptr(), h=h.data_ptr(), dy=dy.data_ptr(),
                     dh=dh.data_ptr(), dx=dx.data_ptr(), dweight=dw.data_ptr(), rows=21, width=n, x_stride=n, residual_stride=n,
                     dy_stride=n, dh_stride=n, eps=EPS)
        assert lib.spion_rms_norm_forward(ctypes.addressof(c), stream) == 0
        c.y, c.codes, c.scales = None, codes.data_ptr(), scales.data_ptr()
        assert lib.spion_rms_norm_forward(ctypes.addressof(c), stream) == 0
        floats = lib.spion_rms_norm_workspace(ctypes.addressof(c))
        ws = torch.full((floats + 4,), 7.0, device=DEV)
        c.x, c.workspace, c.workspace_floats = h.data_ptr(), ws.data_ptr(), floats
        assert lib.spion_rms_norm_backward(ctypes.addressof(c), stream) == 0
        for t in (y, h, dx, scales):
            assert bool((t[21:] == 7.0).all())
        assert bool((codes[21:] == 7).all()) and bool((dw[n:] == 7.0).all()) and bool((ws[floats:] == 7.0).all())
        _check(x, w, res, dy, dh, y[:21], h[:21], dx[:21], dw[:n])
        c.workspace_floats = floats - 1
        assert lib.spion_rms_norm_backward(ctypes.addressof(c), stream) != 0
        with pytest.raises(_lib.SpionLibraryError, match="workspace"):
            _lib.check_error()


def test_module():
    mod = spion_amd.RMSNorm(64).to(DEV)
    x = torch.randn(2, 7, 64, device=DEV, dtype=torch.bfloat16)
    y, h = mod(x, x)
    (y.float().sum() + h.float().sum()).backward()
    assert mod.weight.grad.dtype == torch.float32 and y.dtype == torch.bfloat16
    with torch.no_grad():
        codes, scales = mod.quantized(x)
    assert codes.shape == x.shape and scales.shape == (2, 7)


@pytest.mark.parametrize("width", [84, 768, 1000, 5415])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_codes_are_those_of_the_exact_quotient(dtype, residual, width):
    """1 / rms cancels in y / scale: a code is that of 448 h w / max|h w|.  bf16: the products are exact (16 bits), and a quotient that is not a
    midpoint of e4m3 is at least 2^-20 of itself away from one, further than its rounding to fp32: every code is the 64-bit
    quotient's, ties to even.  fp32: the product, 7 / 8 of it, the largest product and the quotient are rounded, 2^-24 each: a code
    may differ where the quotient lies within 4 * 2^-24 of a midpoint."""
    g = torch.Generator().manual_seed(width)
    x = torch.randn(2048, width, generator=g).to(dtype).to(DEV)
    res = (2.0 * torch.randn(2048, width, generator=g)).to(dtype).to(DEV) if residual else None
    w = (1.0 + 0.2 * torch.randn(width, generator=g)).to(dtype).to(DEV)
    codes = spion_amd.rms_norm_fp8(x, w, res)[0].double()
    hw = (x if res is None else x + res).double() * w.double()
    q = 448.0 * hw / hw.abs().amax(1, keepdim=True)
    want, step = _e4m3(q)  # (torch.round: ties to even)
    off = codes != want
    if dtype == torch.float32:
        to_midpoint = ((q / step).abs() % 1.0 - 0.5).abs() * step
        off &= to_midpoint > 4 * U * q.abs()
    assert int(off.sum()) == 0


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_traced_norms_compute(dtype, residual):
    """A traced norm, of either output, gives on other inputs what the function gives."""
    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return tuple(torch.randn(37, 200, generator=g).to(dtype).to(DEV) for _ in range(2))

    w = torch.linspace(0.5, 1.5, 200, device=DEV).to(dtype)
    for op in (spion_amd.rms_norm, spion_amd.rms_norm_fp8):
        call = lambda x, r: op(x, w, r if residual else None)  # noqa: E731, B023
        with torch.no_grad():
            traced = torch.jit.trace(call, inputs(1), check_trace=False)
            got, want = traced(*inputs(2)), call(*inputs(2))
        for a, b in zip(*(y if isinstance(y, tuple) else (y,) for y in (got, want))):
            assert torch.equal(a.float(), b.float())


def test_calls_go_by_their_own_status():
    """What another call has left in the process-wide error slot neither fails a call nor is taken by it."""
    lib = _lib.core()
    x, dy = torch.randn(5, 64, device=DEV), torch.ones(5, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    lib.spion_set_stream(None, None)  # a failure: no handle
    try:
        got = _train(x, w, None, dy, None)
        with torch.no_grad():
            spion_amd.rms_norm_fp8(x, w)
        assert lib.spion_error_pending() == 1
    finally:
        lib.spion_clear_error()
    _check(x, w, None, dy, None, *got)


def test_rows_wider_than_a_launch_has_threads_for():
    """2^26 columns and more: at 64 threads to a column the weight's gradient would take 2^32 threads.  Elements of 1 and -1 make every sum
    exact up to 2^24 and rounded by a few u beyond: 16 u of the magnitudes in each result."""
    n = (1 << 26) + 5
    g = torch.Generator(device=DEV).manual_seed(1)
    x, dy = ((torch.randint(0, 2, (2, n), generator=g, device=DEV) * 2 - 1).float() for _ in range(2))
    w = torch.ones(n, device=DEV)
    y, _, dx, dw = _train(x, w, None, dy, None)
    inv = 1.0 / (1.0 + EPS) ** 0.5
    m = inv * (x.double() * dy.double()).sum(1, keepdim=True) / n  # mean of dy w h inv
    assert float((y.detach().double() - x.double() * inv).abs().max()) <= 16 * U
    assert float((dx.double() - inv * (dy.double() - x.double() * inv * m)).abs().max()) <= 16 * U * (1 + float(m.abs().max()))
    want = (x.double() * dy.double()).sum(0) * inv
    assert float((dw.double() - want).abs().max()) <= 16 * U * 2
