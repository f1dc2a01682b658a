"""Calls of the attention to an encoder's states near the limits of sizes, some samples or heads of them against float64
(cross_oracle.py)."""
import pytest
import torch

import spion_amd
from cross_oracle import check, cross_reference
from spion_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _normal(seed, *shape):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)


def _some(B):
    return torch.tensor([0, 1, 2, B // 3, B // 2, B - 2, B - 1], device=DEV)


def test_one_token_of_many_samples_over_shared_states():
    """2^24 strips of 32 keys, of which a forward launches none."""
    B, G, Lk, d = 16384, 8, 4096, 32
    q, k, v = _normal(1, B, G, 1, d), _normal(2, 1, G, Lk, d).expand(B, G, Lk, d), _normal(3, 1, G, Lk, d).expand(B, G, Lk, d)
    mask = torch.arange(Lk, device=DEV)[None] < torch.randint(0, Lk + 1, (B, 1), device=DEV, generator=torch.Generator(device=DEV).manual_seed(4))
    with torch.no_grad():
        out = spion_amd.cross_attention(q, k, v, mask)
    i = _some(B)
    check("out", out[i], cross_reference(q[i], k[: len(i)], v[: len(i)], mask[i])["out"])
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("Lq,Lk", [(33, 2049), (2049, 33)])
def test_steps_of_more_strips_of_32_than_a_launch_holds(Lq, Lk):
    """2^24 strips of 32 and more on one side, which then goes in strips of 128.  That side is one sample's for all; its gradients, one for
    each sample, take 34 GB."""
    B, H, d = 1 << 17, 2, 32
    wide = lambda seed, L: (_normal(seed, 1, L, H, d).expand(B, L, H, d) if L > 33 else _normal(seed, B, L, H, d)).transpose(1, 2)  # noqa: E731
    q, k, v, do = wide(5, Lq), wide(6, Lk), wide(7, Lk), wide(8, Lq)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = spion_amd.cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    i = _some(B)
    want = cross_reference(q[i], k[i], v[i], None, do[i])
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        check(name, t[i], want[name])


@pytest.fixture(params=["node", "python"])
def both_nodes(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setitem(_lib._cache, "node", None)


def test_long_states_are_read_in_place(both_nodes):
    """K and V of 2^20 keys, 8 heads next to each other: 2^31 bytes each, of which no copy is made."""
    G, Lk, d = 8, 1 << 20, 128
    k, v = (_normal(seed, 1, Lk, G, d).transpose(1, 2) for seed in (9, 10))
    for Lq in (1, 50):
        q = _normal(11, 1, Lq, 2 * G, d).transpose(1, 2)
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        with torch.no_grad():
            out = spion_amd.cross_attention(q, k, v)
        assert torch.cuda.max_memory_allocated() - before < 1 << 28
        for h in (0, 2 * G - 1):
            want = cross_reference(q[:, h: h + 1], k[:, h // 2: h // 2 + 1], v[:, h // 2: h // 2 + 1])
            check("out", out[:, h: h + 1], want["out"])


@pytest.mark.parametrize("B,Lq", [(1, 3), (1, 127), (300, 127)])
def test_rows_as_far_apart_as_they_may_be(both_nodes, B, Lq):
    """Rows of 2^24 bytes: 127 of them reach 2^31 bytes.  (Samples share them.)"""
    far, L, d = 1 << 23, 127, 32
    big = _normal(12, L * far)

    def heads(at, H, n):
        return big.as_strided((B, H, n, d), (0, d, far, 1), at)

    q, do, k, v = heads(0, 4, Lq), heads(1000, 4, Lq), heads(2000, 2, L), heads(3000, 2, L)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = spion_amd.cross_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    want = cross_reference(q[:1], k[:1], v[:1], None, do[:1])
    for name, t in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        check(name, t[-1:], want[name])
