"""Calls of the attention to an encoder's states as programs make them, against float64 (cross_oracle.py)."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import spion_amd
from cross_oracle import check, cross_reference

pytestmark = pytest.mark.gpu
BOTH = [torch.float32, torch.bfloat16]


def _rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", BOTH)
def test_learned_queries_of_all_samples(dtype):
    """Pooling: one set of queries for every sample, read in place; its gradient is the sum over them."""
    B, H, Lq, Lk, d = 5, 4, 16, 300, 32
    own, k, v, do = _rand(1, H, Lq, d, dtype=dtype), *(_rand(i, B, H, Lk, d, dtype=dtype) for i in (2, 3)), _rand(4, B, H, Lq, d, dtype=dtype)
    own.requires_grad_()
    out = spion_amd.cross_attention(own.expand(B, H, Lq, d), k, v)
    want = cross_reference(own.detach().expand(B, H, Lq, d).contiguous(), k, v, None, do)
    check("out", out.detach(), want["out"])
    got, = torch.autograd.grad(out, own, do)
    value, bound = (t.sum(0) for t in want["dq"])
    check("dq", got, (value, bound + B * torch.finfo(dtype).eps * want["dq"][0].abs().sum(0)))  # a rounded partial sum for each sample


@pytest.mark.parametrize("dtype", BOTH)
def test_a_part_of_a_longer_cache(dtype):
    """Keys and values are the filled part of a buffer, whose rest holds NaN; the mask is one row for all samples."""
    B, H, G, n, room, d = 3, 8, 2, 77, 200, 64
    cache = torch.full((2, B, G, room, d), float("nan"), dtype=dtype, device="cuda")
    cache[:, :, :, :n] = _rand(5, 2, B, G, n, d, dtype=dtype)
    k, v = cache[0, :, :, :n], cache[1, :, :, :n]
    mask = (torch.arange(n, device="cuda") % 3 > 0)[None].expand(B, n)
    for Lq in (1, 40, 200):
        q = _rand(6, B, H, Lq, d, dtype=dtype)
        with torch.inference_mode():
            out = spion_amd.cross_attention(q, k, v, mask)
        check("out", out, cross_reference(q, k.contiguous(), v.contiguous(), mask)["out"])


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("L", [9, 150])
def test_one_tensor_in_all_places(L, dtype):
    x = _rand(7, 2, 3, L, 64, dtype=dtype).requires_grad_()
    out = spion_amd.cross_attention(x, x, x)
    got, = torch.autograd.grad(out.sum(), x)  # (a gradient of stride 0)
    want = cross_reference(x, x, x, None, torch.ones_like(out))
    check("out", out.detach(), want["out"])
    value = sum(want[n][0] for n in ("dq", "dk", "dv"))
    bound = sum(want[n][1] for n in ("dq", "dk", "dv")) + 2 * torch.finfo(dtype).eps * sum(want[n][0].abs() for n in ("dq", "dk", "dv"))
    check("dx", got, (value, bound))


@pytest.mark.parametrize("dtype", BOTH)
def test_recomputed_and_offloaded_steps(dtype):
    q, k, v, do = (_rand(i, 2, 4, n, 64, dtype=dtype) for i, n in ((8, 50), (9, 120), (10, 120), (11, 50)))

    def step(call):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(call(*leaves), leaves, do)

    plain = step(spion_amd.cross_attention)
    again = step(lambda *t: checkpoint(spion_amd.cross_attention, *t, use_reentrant=False))
    with torch.autograd.graph.save_on_cpu():
        away = step(spion_amd.cross_attention)
    for a, b, c in zip(plain, again, away):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_a_copied_layer_and_only_its_queries_trained():
    layer = spion_amd.CrossAttention(dict(transformer_dim=64, head_dim=32, num_head=4, num_key_head=2, layer_norm=True)).cuda()
    other = copy.deepcopy(layer)
    for p in (*other.W_k.parameters(), *other.W_v.parameters()):
        p.requires_grad_(False)
    x, states = _rand(12, 2, 20, 64), _rand(13, 2, 90, 64)
    for m in (layer, other):
        m(x, states).square().sum().backward()
    assert other.W_k.weight.grad is None and other.W_v.bias.grad is None
    for n in ("W_q", "ff", "norm"):
        assert torch.equal(getattr(layer, n).weight.grad, getattr(other, n).weight.grad), n
