"""Attention to keys of another length on seeded random shapes, masks and layouts of heads, against float64 (cross_oracle.py)."""
import random

import pytest
import torch

import spion_amd
from cross_oracle import check, cross_reference

pytestmark = pytest.mark.gpu
PAIRS = 1 << 22  # of queries and keys in all


def _log(rng, most):
    return int(round(2.0 ** rng.uniform(0, most)))


def _heads(g, how, B, H, L, d, dtype):
    t = torch.randn(B, L, H, d, generator=g).to(dtype).cuda()
    if how == "rows":  # [B, L, H, d], as a projection leaves them
        return t.transpose(1, 2)
    if how == "heads":
        return t.transpose(1, 2).contiguous()
    wide = torch.full((B, L + 3, H, d + 8), 7.0, dtype=dtype, device="cuda")  # part of a larger buffer
    wide[:, 2:L + 2, :, 8:] = t
    return wide[:, 2:L + 2, :, 8:].transpose(1, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seed", range(60))
def test_random_calls(seed, dtype):
    rng = random.Random(seed * 2 + (dtype == torch.bfloat16))
    d, G = rng.choice([32, 64, 128]), rng.randint(1, 4)
    H = G * rng.choice([1, 1, 2, 4, 7])
    Lq, Lk = _log(rng, rng.choice([0, 6, 11])), _log(rng, rng.choice([5, 9, 12]))
    Lq = max(1, min(Lq, PAIRS // (H * Lk)))
    B = max(1, min(_log(rng, 6), PAIRS // (H * Lq * Lk), (1 << 22) // (d * (H * Lq + 2 * G * Lk))))
    g = torch.Generator().manual_seed(seed)
    q, do = (_heads(g, rng.choice(["rows", "heads", "part"]), B, H, Lq, d, dtype) for _ in range(2))
    k, v = (_heads(g, rng.choice(["rows", "heads", "part"]), B, G, Lk, d, dtype) for _ in range(2))
    mask = None
    if rng.random() < 0.6:
        mask = (torch.rand(B, Lk, generator=g) < rng.choice([0.02, 0.5, 0.9])).cuda()
        if rng.random() < 0.5:
            mask[rng.randrange(B)] = False
    print(f"B {B} H {H} G {G} Lq {Lq} Lk {Lk} d {d} {dtype} mask {mask is not None}", flush=True)
    want = cross_reference(q, k, v, mask, do)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = spion_amd.cross_attention(*leaves, mask)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, do))))
    for name in want:
        check(name, got[name], want[name])
    with torch.no_grad():
        assert torch.equal(spion_amd.cross_attention(q, k, v, mask), got["out"])
