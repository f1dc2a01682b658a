"""The layer around the attention to an encoder's states in a program's hands, on the GPU."""
import pytest
import torch

import spion_amd

pytestmark = pytest.mark.gpu


def _rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _layer(**more):
    torch.manual_seed(0)
    return spion_amd.CrossAttention(dict(transformer_dim=64, head_dim=32, num_head=4, num_key_head=2, **more)).cuda()


@pytest.mark.parametrize("half", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kept_under", [False, True])
def test_states_kept_on_the_other_side_of_autocast(kept_under, half):
    """Keys and values projected outside autocast serve a call under it, and the other way round.  Off the fp32 layer by the roundings
    of a few values to the half type: 8 of them, of sums of magnitudes up to 4."""
    layer = _layer(layer_norm=True)
    X, states = _rand(1, 3, 2, 64), _rand(2, 3, 70, 64)
    mask = (torch.arange(70).cuda()[None] < torch.tensor([[70], [5], [33]]).cuda()).float()
    with torch.no_grad():
        want = layer(X, states, mask)
        with torch.autocast("cuda", dtype=half, enabled=kept_under):
            kept = layer.keys_values(states)
        with torch.autocast("cuda", dtype=half, enabled=not kept_under):
            y = layer.attend(X, kept, mask)
    assert kept[0].dtype == (half if kept_under else torch.float32) and y.dtype == (torch.float32 if kept_under else half)
    assert float((y.float() - want).abs().max()) <= 8 * torch.finfo(half).eps / 2 * 4
