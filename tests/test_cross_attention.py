"""What attention to keys of another length refuses, how it takes its operands and what it asks of a workspace, without a GPU."""
import ctypes
import math

import pytest
import torch

import spion_amd
from spion_amd import _lib
from spion_amd import attention_cross as ac


@pytest.fixture
def both_nodes(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


both = pytest.mark.parametrize("both_nodes", ["node", "python"], indirect=True)


def _ok():
    return dict(query=torch.zeros(2, 6, 5, 32), key=torch.zeros(2, 3, 7, 32), value=torch.zeros(2, 3, 7, 32))


def _huge(*shape):
    return torch.zeros(()).expand(*shape)  # no memory behind it


@both
@pytest.mark.parametrize("change,error", [
    (dict(query=torch.zeros(6, 5, 32)), ValueError), (dict(key=torch.zeros(2, 7, 32)), ValueError),
    (dict(key=torch.zeros(1, 3, 7, 32)), ValueError), (dict(key=torch.zeros(2, 3, 7, 64)), ValueError),
    (dict(value=torch.zeros(2, 3, 8, 32)), ValueError), (dict(value=torch.zeros(2, 3, 7)), ValueError),
    (dict(query=torch.zeros(2, 5, 5, 32)), ValueError), (dict(query=torch.zeros(2, 2, 5, 32)), ValueError),
    (dict(query=torch.zeros(2, 0, 5, 32)), ValueError), (dict(key=torch.zeros(2, 0, 7, 32), value=torch.zeros(2, 0, 7, 32)), ValueError),
    (dict(query=torch.zeros(2, 6, 5, 48), key=torch.zeros(2, 3, 7, 48), value=torch.zeros(2, 3, 7, 48)), ValueError),
    (dict(query=torch.zeros(2, 6, 5, 32).half()), TypeError), (dict(query=torch.zeros(2, 6, 5, 32).double()), TypeError),
    (dict(key_mask=torch.ones(2, 8)), ValueError), (dict(key_mask=torch.ones(7)), ValueError), (dict(), RuntimeError),
    (dict(key=_huge(2, 3, (1 << 32) + 7, 32), value=_huge(2, 3, (1 << 32) + 7, 32)), ValueError),  # 7 in 32 bits
    (dict(query=_huge(2, 6, (1 << 32) + 5, 32)), ValueError), (dict(query=_huge(2, 6, 1 << 29, 32)), ValueError)])
def test_refusals(both_nodes, change, error):
    with pytest.raises(error):
        spion_amd.cross_attention(**{**_ok(), **change})


def _call(at=16, **kw):
    c = ac._Call(Lse=at, workspace=at, workspace_floats=1 << 40, batch=2, heads=4, key_heads=2, q_len=5, k_len=7, head_dim=32)
    for n in ("Q", "K", "V", "Out", "dO", "dQ", "dK", "dV"):
        setattr(c, n, ac._Heads(at, 256, 64, 32))
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def test_c_entry_points_refuse_before_any_gpu_work():
    lib = ac._lib_typed()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16  # never read: every call below is refused
    h = ac._Heads
    sizes = [dict(batch=0), dict(heads=0), dict(key_heads=0), dict(q_len=0), dict(k_len=0), dict(heads=5), dict(heads=1), dict(head_dim=48),
             dict(k_len=(1 << 29) + 1), dict(q_len=(1 << 28) + 1), dict(batch=1 << 20, heads=1 << 11, key_heads=1 << 10),
             dict(batch=1 << 16, k_len=1 << 14), dict(key_mask=at, mask_bytes=2)]
    bad = sizes + [dict(Lse=None), dict(Q=h(None, 256, 64, 32)), dict(K=h(at + 4, 256, 64, 32)), dict(V=h(at, 2, 64, 32)),
                   dict(Q=h(at, 256, 64, -32)), dict(K=h(at, 256, 64, 1 << 23)), dict(V=h(at, 256, 64, 1 << 20), k_len=4096),
                   dict(Q=h(at, 256, 1 << 30, 32)), dict(Q=h(at, 256, 1 << 29, 32), heads=8), dict(Q=h(at, 256, 1 << 62, 32)),
                   dict(Q=h(at, 256, 64, 1 << 62)), dict(workspace=at + 4)]
    for kw in bad + [dict(Out=h(at, 256, 64, 0))]:
        assert lib.spion_cross_attention_forward(ctypes.addressof(_call(at, **kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_cross_attention_forward"):
            _lib.check_error()
    for kw in bad + [dict(dQ=h(at, 256, 64, 28)), dict(dO=h(None, 256, 64, 32)), dict(workspace=None), dict(workspace_floats=39),
                     dict(dK=h(at, 256, 64, 0)), dict(dV=h(at + 8, 256, 64, 32))]:
        assert lib.spion_cross_attention_backward(ctypes.addressof(_call(at, **kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_cross_attention_backward"):
            _lib.check_error()
    for kw in sizes:
        assert lib.spion_cross_workspace(ctypes.addressof(_call(at, **kw)), 1) == -1
    assert lib.spion_cross_attention_forward(None, None) != 0 and lib.spion_cross_attention_backward(None, None) != 0
    assert lib.spion_cross_workspace(None, 0) == -1
    _lib.core().spion_clear_error()
    assert lib.spion_cross_workspace(ctypes.addressof(_call(at)), 1) == 2 * 4 * 5


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("bf16", [0, 1])
def test_pieces_leave_a_bounded_workspace(bf16, d):
    """Work-groups of 128 rows, at most eight for each of 256 CUs where there is more than one piece; nothing but D for calls that fill the
    machine many times over."""
    def floats(backward, **kw):
        c = _call(16, head_dim=d, bf16=bf16, **kw)
        return ac._lib_typed().spion_cross_workspace(ctypes.addressof(c), backward)

    most = 8 * 256 * 4
    for B in (1, 3, 16, 64, 300, 1000):
        for H, G in ((1, 1), (8, 8), (8, 2), (6, 1)):
            for Lq in (1, 5, 33, 200, 1030, 5000):
                for Lk in (1, 90, 700, 3000, 40000):
                    kw = dict(batch=B, heads=H, key_heads=G, q_len=Lq, k_len=Lk)
                    assert floats(0, **kw) <= most * (32 * d + 64), kw
                    assert floats(1, **kw) <= B * H * Lq + 3 + most * 64 * d, kw
    assert floats(0, batch=131000, heads=4, key_heads=4, q_len=512, k_len=600) == 0
    assert floats(1, batch=131000, heads=4, key_heads=4, q_len=512, k_len=600) == 131000 * 4 * 512


def _aligned(*shape, dtype=torch.float32):
    x = torch.zeros(math.prod(shape) + 8, dtype=dtype)
    return x[(-x.data_ptr() % 16) // x.element_size():][: math.prod(shape)].view(shape)


def test_heads_are_copied_only_where_they_have_to_be(monkeypatch):
    views = _aligned(2, 40, 6, 32).transpose(1, 2), _aligned(2, 6, 40, 32), _aligned(2, 40, 2, 6, 32)[:, :, 1].transpose(1, 2), \
        _aligned(1, 6, 40, 32).expand(2, 6, 40, 32), _aligned(2, 1, 40, 32).expand(2, 6, 40, 32)
    off = _aligned(2 * 6 * 40 * 32 + 1)[1:].view(2, 6, 40, 32)  # contiguous, 4 bytes off
    turned = _aligned(2, 6, 32, 40).transpose(2, 3)
    copies = []
    contiguous, clone = torch.Tensor.contiguous, torch.Tensor.clone
    monkeypatch.setattr(torch.Tensor, "contiguous", lambda t, *a, **k: (copies.append("contiguous"), contiguous(t, *a, **k))[1])
    monkeypatch.setattr(torch.Tensor, "clone", lambda t, *a, **k: (copies.append("clone"), clone(t, *a, **k))[1])
    for t in views:
        for together in (1, 2, 6):
            assert ac._readable(t, together) is t
    assert copies == []
    for t, how in ((off, ["contiguous", "clone"]), (turned, ["contiguous"])):
        copies.clear()
        got = ac._readable(t, 2)
        assert copies == how and ac._fits(got, 2) and torch.equal(got, t)


def test_groups_that_lie_too_far_apart_are_copied():
    t = torch.empty(1, 4, 2, 32, device="meta").as_strided((1, 4, 2, 32), (0, 1 << 28, 32, 1))
    assert ac._fits(t, 1) and ac._fits(t, 2) and not ac._fits(t, 3) and not ac._fits(t, 4)


@pytest.mark.parametrize("dtype,H,L,d,interleaved", [
    (torch.float32, 64, (1 << 17) - 1, 64, True), (torch.float32, 64, 1 << 17, 64, False),  # 2^29 elements to a head's rows
    (torch.float32, 1 << 17, 2, 32, True), (torch.float32, (1 << 17) + 1, 2, 32, False),  # 2^24 bytes from row to row
    (torch.bfloat16, 1 << 16, 2, 128, True), (torch.bfloat16, (1 << 16) + 1, 2, 128, False)])
def test_outputs_lie_as_the_kernels_take_them(dtype, H, L, d, interleaved):
    for t in (torch.empty(1, L, H, d, dtype=dtype, device="meta").transpose(1, 2),
              torch.empty(1, 1, L, d, dtype=dtype, device="meta").expand(1, H, L, d)):
        out = ac._empty_like_heads(t)
        assert out.shape == t.shape and out.stride()[1:] == ((d, H * d, 1) if interleaved else (L * d, d, 1))
        assert ac._fits(out, 1)


def test_the_layer_refuses_what_its_core_does_not_take():
    ok = dict(transformer_dim=64, head_dim=32, num_head=4)
    assert spion_amd.CrossAttention(dict(ok, num_key_head=2, layer_norm=1e-6)).norm.eps == 1e-6
    for change in (dict(num_key_head=3), dict(num_key_head=0), dict(num_key_head=8), dict(head_dim=48)):
        with pytest.raises(ValueError):
            spion_amd.CrossAttention({**ok, **change})


@pytest.mark.parametrize("frozen", [(), (1, 2), (3, 4), (0,)])
def test_projections_of_keys_and_values_as_one(frozen):
    """The product of the stacked weights against the two products, in 64 bits; inputs without a gradient get none."""
    from spion_amd.attention_cross import _FusedKV

    g = torch.Generator().manual_seed(3)
    B, L, dim, G, d = 2, 5, 7, 3, 4
    states, wk, wv, bk, bv = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((B, L, dim), (G * d, dim), (G * d, dim), (G * d,), (G * d,)))
    ins = [t.requires_grad_(i not in frozen) for i, t in enumerate((states, wk, wv, bk, bv))]
    want = [(states @ w.t() + b).view(B, L, G, d).transpose(1, 2) for w, b in ((wk, bk), (wv, bv))]
    got = _FusedKV.apply(*ins, G, d)
    grads = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in want]
    leaves = [t for t in ins if t.requires_grad]
    for a, b in zip(got, want):
        assert torch.allclose(a, b, atol=1e-12)
    for a, b in zip(torch.autograd.grad(got, leaves, grads), torch.autograd.grad(want, leaves, grads)):
        assert torch.allclose(a, b, atol=1e-12)
