"""Calls of the attention to an encoder's states near the limits of sizes, some samples or heads of them against float64
(cross_oracle.py)."""
import pytest
import torch

import spion_amd
from cross_oracle import check, cross_reference

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
