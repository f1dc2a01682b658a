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


@pytest.mark.parametrize("B,Lq,Lk,d", [(2, 40, 300, 32), (8, 700, 1000, 64)])
def test_a_training_step_in_a_graph(B, Lq, Lk, d):
    """Norm, projections, attention and all gradients, captured and replayed, with eager steps between the replays."""
    torch.manual_seed(1)
    layer = spion_amd.CrossAttention(dict(transformer_dim=64, head_dim=d, num_head=4, num_key_head=2, layer_norm=True)).cuda()
    params = list(layer.parameters())
    X, states, dy = _rand(3, B, Lq, 64), _rand(4, B, Lk, 64), _rand(5, B, Lq, 64)
    mask = (torch.arange(Lk).cuda()[None] < torch.randint(1, Lk, (B, 1), generator=torch.Generator().manual_seed(6)).cuda()).float()

    def step():
        leaves = [t.detach().requires_grad_() for t in (X, states)]
        y = layer(*leaves, mask)
        return [y.detach(), *torch.autograd.grad(y, [*leaves, *params], dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn in range(4):
        for i, t in enumerate((X, states, dy)):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * turn + i)))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), turn
