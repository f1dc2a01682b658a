"""What the layer norm refuses, without a GPU."""
import ctypes

import pytest
import torch

import spion_amd
from spion_amd import _lib
from spion_amd import norm as ln


@pytest.fixture(params=["node", "python"])
def both_nodes(request, monkeypatch):
    """Through the compiled node and through the Python function."""
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


@pytest.mark.parametrize("change,error", [
    (dict(weight=torch.ones(7)), ValueError), (dict(weight=torch.ones(2, 4)), ValueError), (dict(residual=torch.ones(4, 8)), ValueError),
    (dict(bias=torch.ones(7)), ValueError), (dict(bias=torch.ones(1, 8)), ValueError), (dict(x=torch.ones(3, 8).double()), TypeError),
    (dict(x=torch.ones(3, 8).half()), TypeError), (dict(x=torch.ones(())), ValueError), (dict(eps=-1.0), ValueError),
    (dict(eps=float("nan")), ValueError), (dict(), RuntimeError),
    (dict(x=torch.zeros(()).expand(2, (1 << 32) + 64), weight=torch.zeros(()).expand((1 << 32) + 64)), ValueError)])
def test_refusals(both_nodes, change, error):
    with pytest.raises(error):
        spion_amd.layer_norm(**{**dict(x=torch.ones(3, 8), weight=torch.ones(8)), **change})


def test_c_entry_points_refuse_before_any_gpu_work():
    lib = ln._layer_lib()
    buf = (ctypes.c_char * 4096)()
    at = ctypes.addressof(buf)  # never read: every call below is refused

    def call(**kw):
        c = ln._LayerCall(x=at, weight=at, bias=at, y=at, dy=at, dx=at, dweight=at, dbias=at, workspace=at, workspace_floats=1 << 40, rows=4,
                          width=8, x_stride=8, dy_stride=8, eps=1e-5)
        for n, v in kw.items():
            setattr(c, n, v)
        return c

    sizes = [dict(rows=0), dict(width=0), dict(rows=(1 << 40) + 1), dict(width=(1 << 29) + 1), dict(x_stride=-8), dict(eps=-1.0),
             dict(eps=float("nan"))]
    for kw in sizes + [dict(x=None), dict(weight=None), dict(y=None), dict(residual=at)]:
        assert lib.spion_layer_norm_forward(ctypes.addressof(call(**kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_layer_norm_forward"):
            _lib.check_error()
    for kw in sizes + [dict(x=None), dict(weight=None), dict(dy=None), dict(dx=None), dict(dweight=None), dict(workspace=None),
                       dict(workspace_floats=2 * 8 - 1)]:
        assert lib.spion_layer_norm_backward(ctypes.addressof(call(**kw)), None) != 0, kw
        with pytest.raises(_lib.SpionLibraryError, match="spion_layer_norm_backward"):
            _lib.check_error()
    assert lib.spion_layer_norm_forward(None, None) != 0 and lib.spion_layer_norm_backward(None, None) != 0
    assert lib.spion_layer_norm_workspace(ctypes.addressof(call(rows=0))) == -1
    _lib.core().spion_clear_error()


def test_the_module_has_the_parameters_of_torchs():
    mod, theirs = spion_amd.LayerNorm(48), torch.nn.LayerNorm(48)
    assert mod.load_state_dict(theirs.state_dict()) and list(mod.state_dict()) == list(theirs.state_dict())
    assert spion_amd.LayerNorm(48, bias=False).bias is None


def test_a_layer_has_one_norm():
    config = dict(transformer_dim=64, head_dim=32, num_head=2, max_seq_len=64, block_size=32, batch_size=1, attention_dropout=0.0,
                  task="lra-image", layer_norm=True)
    assert isinstance(spion_amd.Attention(config, inference=True).norm, spion_amd.LayerNorm)
    assert spion_amd.Attention(dict(config, layer_norm=1e-6), inference=True).norm.eps == 1e-6
    with pytest.raises(ValueError):
        spion_amd.Attention(dict(config, rms_norm=True), inference=True)
