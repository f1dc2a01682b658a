"""What the layer around the attention to an encoder's states hands to its core, without a GPU: the core is stated in torch's
operations here, and takes one type of heads as the kernels do."""
import pytest
import torch

import spion_amd
from spion_amd import attention_cross as ac


@pytest.fixture
def core(monkeypatch):
    """The types of the heads that the core was given, call by call."""
    seen = []

    def plain(query, key, value, key_mask=None):
        if not query.dtype == key.dtype == value.dtype:
            raise TypeError("heads of one type expected")
        if query.dtype not in (torch.float32, torch.bfloat16):
            raise TypeError("fp32 or bf16 heads expected")
        seen.append(query.dtype)
        n = query.shape[1] // key.shape[1]
        q, k, v = query.double(), key.double().repeat_interleave(n, 1), value.double().repeat_interleave(n, 1)
        t = q @ k.transpose(-1, -2) / q.shape[-1] ** 0.5
        if key_mask is not None:
            t = t.masked_fill((key_mask == 0)[:, None, None, :], float("-inf"))
        return (torch.softmax(t, -1) @ v).to(query.dtype)

    monkeypatch.setattr(ac, "cross_attention", plain)
    return seen


def _layer(**more):
    torch.manual_seed(0)
    return spion_amd.CrossAttention(dict(transformer_dim=48, head_dim=32, num_head=4, num_key_head=2, **more))


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("half", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kept_under", [False, True])
def test_states_kept_on_the_other_side_of_autocast(core, kept_under, half):
    """Keys and values that were projected outside autocast serve a call under it, and the other way round; they stay as they are where the
    core takes their type.  Off the fp32 layer by the roundings of a few values to the half type: 8 of them, of sums of sizes up to 4."""
    layer = _layer()
    X, states = _rand(1, 2, 3, 48), _rand(2, 2, 20, 48)
    want = layer(X, states)
    with torch.autocast("cpu", dtype=half, enabled=kept_under):
        # (the layer asks for the GPU's autocast: as it projects under that)
        kept = tuple(layer._split(w(states), 2) for w in (layer.W_k, layer.W_v))
    assert kept[0].dtype == (half if kept_under else torch.float32)
    core.clear()
    with torch.autocast("cpu", dtype=half, enabled=not kept_under):
        y = layer.attend(X, kept)
    assert core == [torch.float32 if half == torch.float16 else kept[0].dtype]
    assert y.dtype == (torch.float32 if kept_under else half)
    assert float((y.float() - want).detach().abs().max()) <= 8 * torch.finfo(half).eps / 2 * 4


def test_gradients_pass_the_change_of_type(core):
    layer = _layer()
    X, states = _rand(3, 2, 3, 48).requires_grad_(), _rand(4, 2, 20, 48)
    kept = layer.keys_values(states)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = layer.attend(X, kept)
    y.float().sum().backward()
    assert X.grad.dtype == torch.float32 and bool(X.grad.any()) and bool(layer.W_k.weight.grad.any())


class _Adapted(torch.nn.Linear):
    """A projection with a term of its own, and a ``weight`` that is only part of it."""

    def forward(self, x):
        return super().forward(x) + x.sum(-1, keepdim=True)


def _replaced(layer, how):
    """What a program does to a projection of keys or values; returns the projection."""
    old = layer.W_v
    if how == "adapter":
        layer.W_v = _Adapted(old.in_features, old.out_features)
    elif how == "no bias":
        layer.W_v = torch.nn.Linear(old.in_features, old.out_features, bias=False)
    elif how == "weight norm":
        torch.nn.utils.weight_norm(old)  # (its weight is made by a hook ahead of the module's forward)
        with torch.no_grad():
            old.weight_g.mul_(3.0)
    elif how == "parametrized":
        torch.nn.utils.parametrizations.orthogonal(old)
    elif how == "hook":
        old.register_forward_hook(lambda m, i, o: 2 * o)
    elif how == "own forward":
        old.forward = lambda x: torch.nn.functional.linear(x, old.weight) - 1
    return layer.W_v


@pytest.mark.filterwarnings("ignore:.*weight_norm.*")
@pytest.mark.parametrize("how", ["plain", "adapter", "no bias", "weight norm", "parametrized", "hook", "own forward"])
def test_projections_are_the_modules_own(how):
    """keys_values is what the layer's projections give, whatever a program has made of them (64-bit states: no rounding to speak of)."""
    layer = _layer().double()
    of_values = _replaced(layer, how).double()
    states = _rand(5, 2, 20, 48).double()
    k, v = layer.keys_values(states)
    for got, module in ((k, layer.W_k), (v, of_values)):
        assert torch.allclose(got, module(states).view(2, 20, 2, 32).transpose(1, 2), atol=1e-12)


def test_global_hooks_see_the_projections():
    layer = _layer()
    seen = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, i, o: seen.append(m) and None)
    try:
        layer.keys_values(_rand(6, 2, 20, 48))
    finally:
        handle.remove()
    assert layer.W_k in seen and layer.W_v in seen
