"""How far the bf16 attention to an encoder's states is off, in all: |got - exact| / |exact| over a whole tensor.

Where the header says that weights are taken as the sum of two bf16 numbers, what is left of their rounding is 2^-17 of them, and results are off by
the rounding of the results alone (and dQ, dK by what the rounded O leaves in D = dO . O).  The errors of both ways are formed here in
float64, ``two`` with the weights as they are and ``one`` with them rounded to bf16; a kernel that takes two numbers is nearer to the
former than to the latter, and no kernel is further off than the latter.  Either is a root of a mean over thousands of roundings and more, which
other roundings move by a few hundredths of it; the two differ by a tenth at least."""
import math

import pytest
import torch

import spion_amd

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bf16(x):
    return x.to(torch.bfloat16).double()


def _tr(x):
    return x.transpose(-1, -2).contiguous()


def _errors(q, k, v, mask, do):
    """{name: (exact, two, one)}"""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    B, H, Lq, d = q.shape
    G, Lk = k.shape[1:3]
    n = H // G
    scale = 1.0 / math.sqrt(d)
    k, v = (t.repeat_interleave(n, 1) for t in (k, v))
    t = q @ _tr(k) * scale
    if mask is not None:
        t = t.masked_fill((mask == 0)[:, None, None, :], -math.inf)
    e = torch.exp(t - t.amax(-1, keepdim=True))
    z = e.sum(-1, keepdim=True)
    p = e / z
    out = p @ v
    dp = do @ _tr(v)
    ds = p * (dp - (do * out).sum(-1, keepdim=True))
    ds_kernel = p * (dp - (do * _bf16(out)).sum(-1, keepdim=True))  # D of the output as it is stored

    def group(x):
        return x.reshape(B, G, n, Lk, d).sum(2)

    exact = {"out": out, "dq": scale * ds @ k, "dk": group(scale * _tr(ds) @ q), "dv": group(_tr(p) @ do)}
    two = {"out": out, "dq": scale * ds_kernel @ k, "dk": group(scale * _tr(ds_kernel) @ q), "dv": exact["dv"]}
    # (A kernel's weights are relative to a maximum that lies within 2^8 of the row's own and need not be it.  Relative to the row's own the
    # largest is 1 and has no rounding, which a few keys would show; P has no such scale.)
    one = {"out": _bf16(p) @ v, "dq": scale * _bf16(ds_kernel) @ k, "dk": group(scale * _tr(_bf16(ds_kernel)) @ q),
           "dv": group(_tr(_bf16(p)) @ do)}
    return {name: (x, _off(_bf16(two[name]), x), _off(_bf16(one[name]), x)) for name, x in exact.items()}


def _off(got, exact):
    return float((got.double() - exact).norm() / exact.norm())


ALL = ("out", "dq", "dk", "dv")


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("size,left,two_numbers", [
    # up to 32 rows that share a head of keys
    ((8, 8, 8, 1, 2048), None, ALL), ((4, 8, 2, 4, 700), 0.7, ALL), ((8, 4, 4, 16, 1500), 0.02, ALL), ((8, 8, 8, 3, 100), None, ALL),
    # up to 256 keys
    ((4, 8, 8, 600, 100), None, ("dq", "dk")), ((32, 8, 8, 1024, 100), 0.5, ("dq", "dk")), ((16, 8, 4, 512, 256), None, ("dq", "dk")),
    ((4, 8, 8, 500, 40), None, ("dq", "dk")),
    # more keys, of which a mask leaves a few; many of all
    ((8, 8, 8, 512, 2048), 0.01, ()), ((16, 8, 8, 512, 1024), None, ())])
def test_weights_as_two_numbers(size, left, two_numbers, d):
    B, H, G, Lq, Lk = size
    g = torch.Generator().manual_seed(d + Lq)
    q, do = (torch.randn(B, Lq, H, d, generator=g).bfloat16().to(DEV).transpose(1, 2) for _ in range(2))
    k, v = (torch.randn(B, Lk, G, d, generator=g).bfloat16().to(DEV).transpose(1, 2) for _ in range(2))
    mask = None
    if left is not None:
        mask = torch.rand(B, Lk, generator=g) < left
        mask[:, :2] = True  # (of one key alone dS is 0, and its errors have no measure)
        mask = mask.to(DEV)
    want = _errors(q, k, v, mask, do)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = spion_amd.cross_attention(*leaves, mask)
    for name, t in zip(ALL, (out.detach(), *torch.autograd.grad(out, leaves, do))):
        exact, two, one = want[name]
        off = _off(t, exact)
        print(f"{name}: off by {off:.5f}; two numbers {two:.5f}, one {one:.5f}", flush=True)
        assert one >= 1.1 * two, name
        assert off <= 1.05 * one, name
        if name in two_numbers:
            assert off <= (two + one) / 2, name
