"""What the norm refuses, without a GPU."""
import ctypes

import pytest
import torch

import spion_amd
from spion_amd import _lib
from spion_amd import norm as rn


@pytest.fixture(params=["node", "python"], autouse=True)
def both_nodes(request, monkeypatch):
    """Every test runs through the compiled node and through the Python function."""
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


@pytest.mark.parametrize("change,error", [
    (dict(weight=torch.ones(7)), ValueError), (dict(weight=torch.ones(2, 4)), ValueError), (dict(residual=torch.ones(4, 8)), ValueError),
    (dict(x=torch.ones(3, 8).double()), TypeError), (dict(x=torch.ones(())), ValueError), (dict(eps=-1.0), ValueError),
    (dict(eps=float("nan")), ValueError), (dict(), RuntimeError)])
@pytest.mark.parametrize("op", ["rms_norm", "rms_norm_fp8"])
def test_refusals(op, change, error):
    with pytest.raises(error):
        getattr(spion_amd, op)(**{**dict(x=torch.ones(3, 8), weight=torch.ones(8)), **change})


def test_c_entry_points_refuse_before_any_gpu_work():
    lib = rn._lib_typed()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf)  # never read: every call below is refused

    def call(**kw):
        c = rn._Call(x=at, weight=at, y=at, dy=at, dx=at, dweight=at, workspace=at, workspace_floats=1 << 40, rows=4, width=8, x_stride=8,
                     dy_stride=8, eps=1e-6)
        for n, v in kw.items():
            setattr(c, n, v)
        return c

    sizes = [dict(rows=0), dict(width=0), dict(rows=(1 << 40) + 1), dict(width=(1 << 29) + 1), dict(x_stride=-8), dict(eps=-1.0),
             dict(eps=float("nan"))]
    for kw in sizes + [dict(x=None), dict(weight=None), dict(y=None), dict(residual=at), dict(codes=at), dict(codes=at, scales=at),
                       dict(y=None, codes=at)]:
        assert lib.spion_rms_norm_forward(ctypes.addressof(call(**kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_rms_norm_forward"):
            _lib.check_error()
    for kw in sizes + [dict(x=None), dict(weight=None), dict(dy=None), dict(dx=None), dict(dweight=None), dict(workspace=None),
                       dict(workspace_floats=4 * 8 - 1)]:
        assert lib.spion_rms_norm_backward(ctypes.addressof(call(**kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_rms_norm_backward"):
            _lib.check_error()
    assert lib.spion_rms_norm_forward(None, None) != 0 and lib.spion_rms_norm_backward(None, None) != 0
    assert lib.spion_rms_norm_workspace(ctypes.addressof(call(rows=0))) == -1
    _lib.core().spion_clear_error()


@pytest.mark.parametrize("op", ["rms_norm", "rms_norm_fp8"])
def test_rows_past_32_bits_are_refused(op):
    n = (1 << 32) + 64  # 64 in 32 bits
    x = torch.zeros(()).expand(2, n)
    with pytest.raises(ValueError, match="width"):
        getattr(spion_amd, op)(x, x[0])


@pytest.mark.parametrize("residual", [False, True])
def test_a_traced_call_in_8_bits_runs_again(residual, monkeypatch):
    """torch.jit.trace records the call, not the allocations inside it: every call of the traced function makes it anew."""
    made = []

    def forward(x, weight, residual, eps, fp8):
        made.append(x.shape[0])
        return (x * weight).to(torch.float8_e4m3fn), x.abs().amax(-1), None if residual is None else x + residual

    monkeypatch.setattr(rn, "_check", lambda *_: None)  # (the tensors here are not on a GPU)
    monkeypatch.setattr(rn, "_forward", forward)
    w = torch.arange(1.0, 9.0)
    x, y = torch.ones(3, 8), torch.full((3, 8), 2.0)
    traced = torch.jit.trace(lambda x, r: spion_amd.rms_norm_fp8(x, w, r if residual else None), (x, x), check_trace=False)
    got = traced(y, x)
    assert len(made) == 2 and len(got) == 2 + residual
    assert torch.equal(got[0].float(), (y * w).to(torch.float8_e4m3fn).float()) and torch.equal(got[1], y[:, 0])
    assert not residual or torch.equal(got[2], y + x)


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused_in_8_bits(grad, monkeypatch):
    """Forward-mode derivatives do not depend on grad mode: they are refused, not dropped."""
    import torch.autograd.forward_ad as fwd

    monkeypatch.setattr(rn, "_check", lambda *_: None)
    monkeypatch.setattr(rn, "_forward", lambda x, *_: (x.to(torch.float8_e4m3fn), x[:, 0], None))
    x = torch.ones(3, 8)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        assert spion_amd.rms_norm_fp8(x, x[0])[0].shape == x.shape
        with pytest.raises(NotImplementedError):
            spion_amd.rms_norm_fp8(fwd.make_dual(x, x), x[0])
        with pytest.raises(NotImplementedError):
            spion_amd.rms_norm_fp8(x, fwd.make_dual(x[0], x[0]))
