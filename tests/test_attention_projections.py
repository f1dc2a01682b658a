"""The attention layer's projections, without a GPU: the core is replaced by one that keeps what it is given."""
import pytest
import torch

import spion_amd


class _Keeps(torch.nn.Module):
    def forward(self, q, k, v, mask):
        self.given = q, k, v
        return v, None


class _Adapted(torch.nn.Linear):
    """A projection with a term of its own, and a ``weight`` that is only part of it."""

    def forward(self, x):
        return super().forward(x) + x.sum(-1, keepdim=True)


def _layer():
    torch.manual_seed(0)
    layer = spion_amd.Attention(dict(transformer_dim=48, head_dim=32, num_head=2, max_seq_len=32, block_size=32, batch_size=2,
                                     attention_dropout=0.0, task="lra-image"), inference=True)
    layer.attn = _Keeps()
    return layer


@pytest.mark.filterwarnings("ignore:.*weight_norm.*")
@pytest.mark.parametrize("how", ["plain", "adapter", "no bias", "weight norm", "hook", "own forward"])
def test_heads_are_what_the_projections_give(how):
    """To 1e-4: two orders of 49 terms in fp32, of magnitudes that add up to 16 at most: 2 * 49 * 2^-24 * 16 = 9e-5."""
    layer = _layer()
    old = layer.W_k
    if how == "adapter":
        layer.W_k = _Adapted(48, 64)
    elif how == "no bias":
        layer.W_k = torch.nn.Linear(48, 64, bias=False)
    elif how == "weight norm":
        torch.nn.utils.weight_norm(old)  # (its weight is made by a hook ahead of the module's forward)
        with torch.no_grad():
            old.weight_g.mul_(3.0)
    elif how == "hook":
        old.register_forward_hook(lambda m, i, o: 2 * o)
    elif how == "own forward":
        old.forward = lambda x: torch.nn.functional.linear(x, old.weight) - 1
    X = torch.randn(2, 32, 48, generator=torch.Generator().manual_seed(1))
    layer(X, torch.ones(2, 32))
    for got, module in zip(layer.attn.given, (layer.W_q, layer.W_k, layer.W_v)):
        assert torch.allclose(got, layer.split_heads(module(X)), atol=1e-4, rtol=0)
