"""Attention to keys of another length against float64 (cross_oracle.py)."""
import ctypes
import math
import threading

import pytest
import torch

import spion_amd
from cross_oracle import check, cross_reference
from spion_amd import _lib
from spion_amd import attention_cross as ac

pytestmark = pytest.mark.gpu
DEV = "cuda"
BOTH = [torch.float32, torch.bfloat16]


@pytest.fixture
def both_nodes(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


both = pytest.mark.parametrize("both_nodes", ["node", "python"], indirect=True)


def _inputs(B, H, G, Lq, Lk, d, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q, do = ((s * torch.randn(B, Lq, H, d, generator=g)).to(dtype).to(DEV).transpose(1, 2) for s in (scale, 1.0))
    kv = torch.randn(B, Lk, 2, G, d, generator=g).to(dtype).to(DEV)
    return q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), do


def _mask(kind, B, Lk, seed=0):
    """lengths: one sample without keys, one with a single one where there are enough samples; holes: any keys"""
    if kind is None:
        return None
    g = torch.Generator().manual_seed(seed)
    if kind == "lengths":
        lens = torch.randint(0, Lk + 1, (B, 1), generator=g)
        lens[0] = 0
        if B > 1:
            lens[1] = 1
        return (torch.arange(Lk)[None] < lens).float().to(DEV)
    m = (torch.rand(B, Lk, generator=g) < 0.4).float()
    if B > 1:
        m[B // 2] = 0
    return m.to(DEV)


def _train(q, k, v, do, mask=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = spion_amd.cross_attention(*leaves, mask)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))))


def _all(q, k, v, do, mask=None):
    got, want = _train(q, k, v, do, mask), cross_reference(q, k, v, mask, do)
    for name in want:
        check(name, got[name], want[name])
    with torch.no_grad():
        assert torch.equal(spion_amd.cross_attention(q, k, v, mask), got["out"])
    return got


SIZES = [(1, 1, 1, 1, 1), (2, 2, 2, 1, 31), (2, 3, 1, 1, 32), (1, 8, 2, 1, 1000), (3, 4, 4, 5, 33), (2, 6, 3, 7, 64), (1, 4, 1, 9, 129), (2, 2, 2, 32, 65),
         (2, 2, 1, 33, 96), (1, 3, 3, 100, 1), (2, 2, 2, 129, 257), (1, 6, 2, 47, 500), (2, 4, 2, 300, 40), (1, 2, 2, 1000, 70)]


@both
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradients(both_nodes, size, d, dtype):
    _all(*_inputs(*size, d, dtype, seed=sum(size)))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("kind", ["lengths", "holes"])
@pytest.mark.parametrize("size", [(3, 2, 2, 1, 40), (4, 4, 2, 3, 200), (3, 2, 1, 50, 130), (3, 2, 2, 200, 300), (2, 4, 4, 17, 1030)])
def test_key_masks(size, kind, d, dtype):
    q, k, v, do = _inputs(*size, d, dtype, seed=1)
    mask = _mask(kind, size[0], size[4], seed=2)
    got = _all(q, k, v, do, mask)
    empty = ~mask.bool().any(1)
    assert not bool(got["out"][empty].any()) and not bool(got["dq"][empty].any())
    for name in ("dk", "dv"):  # keys that are left out
        assert not bool(got[name].transpose(1, 2)[mask == 0].any())


@both
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("mask_type", [torch.bool, torch.float32, torch.int64, torch.uint8, torch.bfloat16])
def test_types_of_masks(both_nodes, mask_type, dtype):
    q, k, v, do = _inputs(3, 4, 2, 9, 77, 32, dtype)
    mask = _mask("holes", 3, 77)
    a, b = _train(q, k, v, do, mask), _train(q, k, v, do, mask.to(mask_type))
    for name in a:
        assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("size", [(3, 4, 2, 3, 200), (3, 2, 2, 140, 300), (2, 2, 2, 1, 3000), (40, 8, 8, 150, 130)])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan, 3.0e38])
def test_what_left_out_keys_hold_is_not_used(what, size, dtype):
    """Infinities, NaN and the types' largest values in keys that are left out change nothing."""
    q, k, v, do = _inputs(*size, 64, dtype, seed=3)
    mask = _mask("holes", size[0], size[4], seed=4)
    clean = _train(q, k, v, do, mask)
    k, v = k.clone(), v.clone()
    for t in (k, v):
        t.transpose(1, 2)[mask == 0] = what
    got = _train(q, k, v, do, mask)
    for name in clean:
        assert torch.equal(got[name], clean[name]), name


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,H,G,Lq,Lk,d", [
    (32, 8, 8, 200, 150, 64), (32, 16, 4, 150, 130, 32), (20, 8, 8, 257, 100, 128),  # strips that fill the machine
    (1, 4, 2, 700, 2000, 64), (2, 2, 2, 260, 3000, 32), (1, 2, 2, 200, 3001, 128),  # other sides in pieces
    (2, 8, 8, 3000, 77, 64), (1, 4, 1, 1500, 40, 32), (1, 4, 2, 1100, 65, 128),  # few keys
    (4, 8, 2, 4, 3000, 64), (16, 2, 2, 16, 1500, 32), (2, 4, 4, 1, 5000, 128), (64, 8, 8, 1, 300, 64)])  # few rows
@pytest.mark.parametrize("kind", [None, "lengths", "holes"])
def test_shapes_of_work(B, H, G, Lq, Lk, d, kind, dtype):
    q, k, v, do = _inputs(B, H, G, Lq, Lk, d, dtype, seed=5)
    _all(q, k, v, do, _mask(kind, B, Lk, seed=6))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("Lq,Lk", [(3, 17500), (40, 17000), (17000, 40)])
@pytest.mark.parametrize("kind", [None, "holes"])
def test_long_sides(Lq, Lk, kind, dtype):
    """More than one chunk of a key mask."""
    q, k, v, do = _inputs(2, 2, 1, Lq, Lk, 32, dtype, seed=7)
    _all(q, k, v, do, _mask(kind, 2, Lk, seed=8))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("Lq", [1, 200])
def test_large_logits(Lq, dtype):
    _all(*_inputs(2, 2, 2, Lq, 300, 64, dtype, seed=9, scale=30.0))


@both
@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("how", ["contiguous", "unaligned", "transposed", "one_sample", "one_head", "one_query", "one_key", "merged"])
def test_layouts(both_nodes, how, dtype):
    B, H, G, Lq, Lk, d = 2, 4, 2, 70, 90, 32
    q, k, v, do = (t.contiguous() for t in _inputs(B, H, G, Lq, Lk, d, dtype, seed=10))
    if how == "unaligned":
        q, k, v, do = (torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v, do))
    elif how == "transposed":
        q, k, v, do = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v, do))
    elif how == "one_sample":
        q, k, v, do = (t[:1].expand(B, -1, -1, -1) for t in (q, k, v, do))
    elif how == "one_head":
        q, k, v, do = (t[:, :1].expand(-1, t.shape[1], -1, -1) for t in (q, k, v, do))
    elif how == "one_query":
        q, do = (t[:, :, :1].expand(-1, -1, Lq, -1) for t in (q, do))
    elif how == "one_key":
        k, v = (t[:, :, :1].expand(-1, -1, Lk, -1) for t in (k, v))
    elif how == "merged":  # one projection's buffer for everything
        big = torch.randn(B, Lk, H + 2 * G, d, device=DEV).to(dtype)
        q, k, v = big[:, :Lq, :H].transpose(1, 2), big[:, :, H:H + G].transpose(1, 2), big[:, :, H + G:].transpose(1, 2)
    _all(q, k, v, do)


def test_gradients_of_shared_and_expanded_leaves():
    """One tensor as key and value, and states that several samples of queries share: the gradients of their uses add up."""
    q, k, _, do = _inputs(4, 4, 2, 20, 60, 32, torch.float32, seed=11)
    one = k[:1].contiguous().requires_grad_()
    out = spion_amd.cross_attention(q, one.expand(4, -1, -1, -1), one.expand(4, -1, -1, -1))
    (got,) = torch.autograd.grad(out, one, do)
    wide = one.detach().expand(4, -1, -1, -1)
    want = cross_reference(q, wide, wide, None, do)
    value, bound = (want["dk"][i].sum(0, keepdim=True) + want["dv"][i].sum(0, keepdim=True) for i in range(2))
    sums = 8 * 2.0 ** -24 * (want["dk"][0].abs().sum(0, keepdim=True) + want["dv"][0].abs().sum(0, keepdim=True))
    check("shared", got, (value, bound + sums))


@pytest.mark.parametrize("Lq,Lk", [(6, 50), (150, 100)])
def test_gradient_against_differences(Lq, Lk):
    """Central differences of <out, do> along each operand: fp32 results leave 2^-23 sqrt(n) |do| |out| / step, curvature step^2 of the
    value."""
    q, k, v, do = _inputs(2, 4, 2, Lq, Lk, 32, torch.float32, seed=12)
    mask = _mask("holes", 2, Lk, seed=13)
    got = _train(q, k, v, do, mask)
    g = torch.Generator().manual_seed(14)
    step = 2.0 ** -6
    for t, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        u = torch.randn(t.shape, generator=g).to(DEV)
        f = []
        for s in (step, -step):
            out = spion_amd.cross_attention(*(x + s * u if x is t else x for x in (q, k, v)), mask)
            f.append(float((out.double() * do).sum()))
        size = float((got[name].double() * u).abs().sum())
        noise = 4 * 2.0 ** -23 * out.numel() ** 0.5 * 16 / step
        assert abs((f[0] - f[1]) / (2 * step) - float((got[name].double() * u).sum())) <= 1e-3 * size + noise


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("size", [(3, 4, 2, 3, 2000, 64), (1, 2, 2, 300, 3000, 32), (64, 8, 8, 130, 200, 64), (2, 2, 1, 3000, 100, 128)])
def test_the_same_call_gives_the_same_bits(size, dtype):
    q, k, v, do = _inputs(*size, dtype, seed=15)
    a, b = _train(q, k, v, do), _train(q, k, v, do)
    for name in a:
        assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("B,H,G,Lq,Lk", [(2, 2, 2, 70, 90), (1, 2, 1, 3, 3000), (64, 4, 4, 200, 200), (2, 4, 2, 1500, 60)])
def test_a_nan_is_not_hidden(B, H, G, Lq, Lk, dtype):
    """A NaN in a key that takes part reaches every row of its head, one in a query its own row and the whole gradient of its keys."""
    q, k, v, do = _inputs(B, H, G, Lq, Lk, 64, dtype, seed=16)
    k2 = k.clone()
    k2[0, 0, Lk // 2, 5] = math.nan
    got = _train(q, k2, v, do)
    n = H // G
    assert bool(torch.isnan(got["out"][0, :n]).all()) and bool(torch.isfinite(got["out"][0, n:]).all())
    assert bool(torch.isnan(got["dv"][0, 0]).all()) and bool(torch.isfinite(got["dv"][0, 1:]).all())
    q2 = q.clone()
    q2[0, 0, Lq - 1, 3] = math.nan
    got = _train(q2, k, v, do)
    assert bool(torch.isnan(got["out"][0, 0, Lq - 1]).all()) and int(torch.isnan(got["out"]).any(-1).sum()) == 1
    assert bool(torch.isnan(got["dk"][0, 0]).all()) and bool(torch.isfinite(got["dk"][0, 1:]).all())


def test_states_past_32_bits_of_bytes():
    """K and V of 5.4 GB each: the last samples lie beyond 2^32 bytes."""
    B, G, Lk, d = 20, 8, 131072, 128
    g = torch.Generator(device=DEV).manual_seed(17)
    k, v = (torch.empty(B, Lk, G, d, dtype=torch.bfloat16, device=DEV).normal_(generator=g).transpose(1, 2) for _ in range(2))
    q = torch.randn(B, 16, 1, d, generator=g, device=DEV).bfloat16()
    with torch.no_grad():
        out = spion_amd.cross_attention(q, k, v)
    for b, h in ((0, 0), (B - 1, 0), (B - 1, 15), (B // 2, 7)):
        kk, vv = k[b, h // 2].double(), v[b, h // 2].double()
        p = torch.softmax(kk @ q[b, h, 0].double() / math.sqrt(d), 0)
        want = p @ vv
        # as in cross_oracle.py: weights and the output are rounded, sums are of 131072 terms
        u = 2.0 ** -24
        r = 2 * (d + 8) * u * float((kk.abs() @ q[b, h, 0].double().abs()).max()) / math.sqrt(d) + 2.0 ** -8 + 2 * Lk * u
        assert bool(((out[b, h, 0].double() - want).abs() <= r * (p @ vv.abs()) + 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("size", [(2, 4, 2, 1, 3000, 64), (2, 4, 2, 300, 700, 32)])
def test_streams_and_replays(size, dtype):
    q, k, v, do = _inputs(*size, dtype, seed=18)
    mask = _mask("holes", size[0], size[4], seed=19)

    def step():
        return list(_train(q, k, v, do, mask).values())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.cuda.graph(second):
        outs2 = step()
    for turn in range(4):
        for i, t in enumerate((q, k, v, do)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * turn + i)).to(dtype))
        mask.copy_(_mask("holes", size[0], size[4], seed=20 + turn))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            second.replay()  # at the same time: each has workspaces of its own
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a, b, c in zip(outs, outs2, eager):
            assert torch.equal(a, c) and torch.equal(b, c), turn


@both
@pytest.mark.parametrize("B,H,G,Lq,Lk", [(2, 4, 2, 5, 0), (2, 4, 2, 0, 5), (0, 4, 2, 5, 5), (2, 0, 0, 5, 5)])
def test_nothing_to_attend_to(both_nodes, B, H, G, Lq, Lk):
    q, k, v = (torch.randn(B, h, L, 32, device=DEV, requires_grad=True) for h, L in ((H, Lq), (G, Lk), (G, Lk)))
    out = spion_amd.cross_attention(q, k, v)
    assert out.shape == q.shape and not bool(out.any())
    for t, g in zip((q, k, v), torch.autograd.grad(out.sum(), (q, k, v))):
        assert g.shape == t.shape and not bool(g.any())


@both
def test_a_second_derivative_is_refused(both_nodes):
    q, k, v, do = _inputs(1, 2, 2, 5, 40, 32, torch.float32)
    q = q.detach().requires_grad_()
    (g,) = torch.autograd.grad(spion_amd.cross_attention(q, k, v), q, do.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@both
def test_a_mask_changed_before_the_backward_is_refused(both_nodes):
    q, k, v, do = _inputs(2, 2, 2, 5, 40, 32, torch.float32)
    mask = torch.ones(2, 40, device=DEV)
    out = spion_amd.cross_attention(q.detach().requires_grad_(), k, v, mask)
    mask[0, 3] = 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(do)


@both
def test_tangents_are_refused(both_nodes):
    import torch.autograd.forward_ad as fwd

    q, k, v, do = _inputs(1, 2, 2, 5, 40, 32, torch.float32)
    with fwd.dual_level(), torch.no_grad(), pytest.raises((NotImplementedError, RuntimeError)):
        spion_amd.cross_attention(fwd.make_dual(q.contiguous(), do.contiguous()), k, v)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("grad", [False, True])
def test_a_traced_call_computes(grad, dtype):
    a, b = (_inputs(2, 4, 2, 9, 130, 32, dtype, seed=s)[:3] for s in (21, 22))
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(lambda q, k, v: spion_amd.cross_attention(q, k, v), a, check_trace=False)
        assert torch.equal(traced(*b), spion_amd.cross_attention(*b))


def test_calls_go_by_their_own_status():
    """What another call has left in the process-wide error slot neither fails a call nor is taken by it."""
    lib = _lib.core()
    q, k, v, do = _inputs(1, 2, 2, 5, 40, 32, torch.float32)
    lib.spion_set_stream(None, None)  # a failure: no handle
    try:
        _all(q, k, v, do)
        assert lib.spion_error_pending() == 1
    finally:
        lib.spion_clear_error()


def test_two_threads_on_two_streams():
    inputs = [_inputs(2, 4, 2, 3, 4000, 64, torch.bfloat16, seed=23), _inputs(2, 4, 2, 200, 700, 64, torch.float32, seed=24)]
    want = [_train(*x) for x in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = _train(*inputs[i])
                stream.synchronize()
                wrong.extend(n for n in got if not torch.equal(got[n], want[i][n]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("Lq,Lk", [(3, 3000), (200, 70), (150, 1030)])
def test_c_entry_points_keep_to_their_buffers(Lq, Lk):
    B, H, G, d = 2, 4, 2, 64
    q, k, v, do = _inputs(B, H, G, Lq, Lk, d, torch.bfloat16, seed=25)
    lib, stream = ac._lib_typed(), torch.cuda.current_stream().cuda_stream

    def room(heads, L):  # rows in the middle of others
        big = torch.full((B, L + 4, heads, d), 7.0, dtype=torch.bfloat16, device=DEV)
        return big, big[:, 2:L + 2].transpose(1, 2)

    (Out, out), (DQ, dq), (DK, dk), (DV, dv) = room(H, Lq), room(H, Lq), room(G, Lk), room(G, Lk)
    lse = torch.full((B * H * Lq + 8,), 7.0, device=DEV)
    call = ac._call_of(q, k, v, out, lse, None)
    floats = lib.spion_cross_workspace(ctypes.addressof(call), 0)
    alone = torch.empty_like(out)
    ws = torch.full((floats + 4,), 7.0, device=DEV)
    if floats:  # without a workspace: in one piece
        plain = ac._call_of(q, k, v, alone, torch.empty_like(lse), None)
        assert lib.spion_cross_attention_forward(ctypes.addressof(plain), stream) == 0
        call.workspace, call.workspace_floats = ws.data_ptr(), floats
    assert lib.spion_cross_attention_forward(ctypes.addressof(call), stream) == 0
    assert bool((ws[floats:] == 7.0).all())
    floats = lib.spion_cross_workspace(ctypes.addressof(call), 1)
    ws = torch.full((floats + 4,), 7.0, device=DEV)
    call.workspace, call.workspace_floats = ws.data_ptr(), floats
    call.dO, call.dQ, call.dK, call.dV = (ac._heads(t) for t in (do, dq, dk, dv))
    assert lib.spion_cross_attention_backward(ctypes.addressof(call), stream) == 0
    assert bool((ws[floats:] == 7.0).all()) and bool((lse[B * H * Lq:] == 7.0).all())
    for big in (Out, DQ, DK, DV):
        assert bool((big[:, :2] == 7.0).all()) and bool((big[:, -2:] == 7.0).all())
    want = cross_reference(q, k, v, None, do)
    for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        check(name, t, want[name])
    if floats and lib.spion_cross_workspace(ctypes.addressof(call), 0):
        check("in one piece", alone, want["out"])


# ---------------------------------------------------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------------------------------------------------
def _plain_layer(layer, X, states, mask):
    """The layer in torch's operations, in the parameters' type."""
    if layer.norm is not None:
        X = torch.nn.functional.layer_norm(X, X.shape[-1:], layer.norm.weight, layer.norm.bias, layer.norm.eps)
    B, Lq, _ = X.shape
    n, d = layer.num_head // layer.num_key_head, layer.head_dim
    split = lambda t, heads: t.reshape(B, -1, heads, d).transpose(1, 2)  # noqa: E731
    q = split(layer.W_q(X), layer.num_head)
    k, v = (split(w(states), layer.num_key_head).repeat_interleave(n, 1) for w in (layer.W_k, layer.W_v))
    t = q @ k.transpose(-1, -2).contiguous() / math.sqrt(d)
    t = t.masked_fill((mask == 0)[:, None, None, :], -math.inf)
    return layer.ff((torch.softmax(t, -1) @ v).transpose(1, 2).reshape(B, Lq, -1))


@both
@pytest.mark.parametrize("key_heads", [4, 2])
def test_the_layer_against_torch(both_nodes, key_heads):
    """Norm, projections, attention and output projection with all their gradients, against the same in float64: each step adds a few
    roundings of fp32, 1e-4 of the largest value in all."""
    torch.manual_seed(0)
    layer = spion_amd.CrossAttention(dict(transformer_dim=96, head_dim=32, num_head=4, num_key_head=key_heads, states_dim=64, layer_norm=True))
    exact = spion_amd.CrossAttention(dict(transformer_dim=96, head_dim=32, num_head=4, num_key_head=key_heads, states_dim=64, layer_norm=True))
    exact.load_state_dict(layer.state_dict())
    layer, exact = layer.to(DEV), exact.to(DEV).double()
    X, states, dy = (torch.randn(3, L, n, device=DEV) for L, n in ((20, 96), (50, 64), (20, 96)))
    mask = (torch.arange(50, device=DEV)[None] < torch.tensor([[50], [17], [33]], device=DEV)).float()
    a, b = (t.clone().requires_grad_() for t in (X, states)), (t.double().requires_grad_() for t in (X, states))
    a, b = tuple(a), tuple(b)
    y, want = layer(*a, mask), _plain_layer(exact, *b, mask)
    params = list(layer.parameters()), list(exact.parameters())
    grads = torch.autograd.grad(y, (*a, *params[0]), dy), torch.autograd.grad(want, (*b, *params[1]), dy.double())
    for got, ref in zip((y, *grads[0]), (want, *grads[1])):
        assert float((got.double() - ref).abs().max()) <= 1e-4 * max(1e-2, float(ref.abs().max()))


@pytest.mark.parametrize("dtype", BOTH)
def test_token_by_token_over_kept_states(dtype):
    """A decoder block of norm with residual, cross attention and the next norm, for all tokens at once and for one after the other over
    states that are projected once."""
    torch.manual_seed(1)
    layer = spion_amd.CrossAttention(dict(transformer_dim=64, head_dim=32, num_head=4, num_key_head=2)).to(DEV).to(dtype)
    norms = [spion_amd.LayerNorm(64).to(DEV) for _ in range(2)]
    X, R = (torch.randn(3, 7, 64, device=DEV).to(dtype) for _ in range(2))
    states = torch.randn(3, 600, 64, device=DEV).to(dtype)
    mask = (torch.arange(600, device=DEV)[None] < torch.tensor([[600], [17], [333]], device=DEV)).float()
    with torch.no_grad():
        kept = layer.keys_values(states)

        def block(x, r):
            y, h = norms[0](x, r)
            return norms[1](layer.attend(y, kept, mask), h)[0]

        every = block(X, R)
        single = torch.cat([block(X[:, i:i + 1], R[:, i:i + 1]) for i in range(7)], 1)
    # the same sums in another order and, in bf16, roundings of five steps that may fall to the other side (2^-8 of values up to 4 each)
    tol = 1e-5 if dtype == torch.float32 else 5 * 2.0 ** -8 * 4
    assert float((every.float() - single.float()).abs().max()) <= tol


def test_the_layer_in_a_graph():
    torch.manual_seed(2)
    layer = spion_amd.CrossAttention(dict(transformer_dim=64, head_dim=32, num_head=2, layer_norm=True)).to(DEV)
    X, states, dy = (torch.randn(2, L, 64, device=DEV) for L in (1, 300, 1))
    mask = torch.ones(2, 300, device=DEV)
    with torch.no_grad():
        kept = layer.keys_values(states)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.attend(X, kept, mask)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.attend(X, kept, mask)
        for turn in range(4):
            X.copy_(torch.randn(X.shape, generator=torch.Generator().manual_seed(turn)))
            mask.copy_((torch.rand(2, 300, generator=torch.Generator().manual_seed(turn)) < 0.5).float())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, layer.attend(X, kept, mask)), turn


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
def test_the_layer_under_autocast(half):
    torch.manual_seed(3)
    layer = spion_amd.CrossAttention(dict(transformer_dim=64, head_dim=32, num_head=2, layer_norm=True)).to(DEV)
    X, states = (torch.randn(2, L, 64, device=DEV) for L in (9, 70))
    want = layer(X, states)
    for rows in (X, X.to(half)):
        with torch.autocast("cuda", dtype=half):
            y = layer(rows, states)
        y.float().sum().backward()
        assert y.dtype == half and float((y.float() - want).abs().max()) <= 0.1 * float(want.abs().max())


def test_the_encoder_layer_normalises_its_input():
    config = dict(transformer_dim=64, head_dim=32, num_head=2, max_seq_len=64, block_size=32, batch_size=2, attention_dropout=0.0, task="lra-image")
    torch.manual_seed(4)
    plain = spion_amd.Attention(config).to(DEV)
    normed = spion_amd.Attention(dict(config, layer_norm=True)).to(DEV)
    normed.load_state_dict(plain.state_dict(), strict=False)
    X = torch.randn(2, 64, 64, device=DEV)
    mask = torch.ones(2, 64, device=DEV)
    y = torch.nn.functional.layer_norm(X, (64,), eps=1e-5)
    a, b = normed(X, mask)[0], plain(y, mask)[0]
    assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
