"""64-bit statement of attention to keys of another length, and how far a kernel may be off it.

The bounds count roundings: u32 = 2^-24 for an fp32 operation, a bf16 value half a step of 2^-8.  A sum of n terms in fp32 is off by at
most n u32 of the sum of magnitudes.  With t the logits, P = exp(t) / Z, n the queries of all heads that share a head of keys:
  dt    = (d + 8) u32 |q|.|k| scale                            product, scale, subtraction of the maximum, exp2's argument
  rP    = 2 max_j dt + (Lk + 64) u32                           of numerator and denominator, exp2, the sum of the denominator
  out   : sum_j P |v| (rP + wP + Lk u32) + r |out|             wP: rounding of the weights P to bf16 in the product, r: of the output
  D     : dO.out of the output as rounded: sum_f |dO| (P |v|) (rP + wP + Lk u32) + (r + d u32) |dO|.|out|
  dS    : |dS| (rP + 4 u32) + P (d u32 |dO|.|v| + d(D))
  dQ    : scale sum_j (d(dS) + |dS| (wP + Lk u32)) |k| + r |dQ|
  dK    : scale sum_i (d(dS) + |dS| (wP + n u32)) |q| + r |dK|;  dV: sum_i P |dO| (rP + wP + n u32) + r |dV|
"""
import math

import torch

U32 = 2.0 ** -24


def _tr(x):
    return x.transpose(-1, -2).contiguous()


def cross_reference(q, k, v, mask=None, do=None):
    """Returns {"out", and with do "dq", "dk", "dv"}: each (value, bound) in float64 on the inputs' device."""
    bf = q.dtype == torch.bfloat16
    r, wP = (2.0 ** -8, 2.0 ** -8) if bf else (2 * U32, 2 * U32)
    q, k, v = (x.detach().double() for x in (q, k, v))
    B, H, Lq, d = q.shape
    G, Lk = k.shape[1:3]
    n = H // G
    scale = 1.0 / math.sqrt(d)
    there = torch.ones(B, Lk, dtype=torch.bool, device=q.device) if mask is None else mask != 0
    k, v = (torch.where(there[:, None, :, None], x, 0.0).repeat_interleave(n, 1) for x in (k, v))  # whatever lies in a key that is left out
    t = q @ _tr(k) * scale
    use = there[:, None, None, :]
    t = torch.where(use, t, -math.inf)
    top = t.amax(-1, keepdim=True) if Lk else torch.zeros_like(t[..., :1])
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(t - top)
    z = e.sum(-1, keepdim=True)
    p = torch.where(z > 0, e / z, 0.0)
    out = p @ v
    dt = torch.where(use & (p > 0), (d + 8) * U32 * (q.abs() @ _tr(k.abs()) * scale), 0.0)
    rP = 2 * dt.amax(-1, keepdim=True) + (Lk + 64) * U32
    pv = p @ v.abs()
    res = {"out": (out, pv * (rP + wP + Lk * U32) + r * out.abs())}
    if do is None:
        return res
    do = do.detach().double()
    dp = do @ _tr(v)
    D = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - D)
    ddp = d * U32 * (do.abs() @ _tr(v.abs()))
    dD = (do.abs() * pv).sum(-1, keepdim=True) * (rP + wP + Lk * U32) + (r + d * U32) * (do.abs() * out.abs()).sum(-1, keepdim=True)
    dds = ds.abs() * (rP + 4 * U32) + p * (ddp + dD)
    dq = scale * ds @ k
    res["dq"] = dq, scale * ((dds + ds.abs() * (wP + Lk * U32)) @ k.abs()) + r * dq.abs()

    def group(x):  # sums over the heads that share one
        return x.reshape(B, G, n, Lk, d).sum(2)

    dk = group(scale * _tr(ds) @ q)
    res["dk"] = dk, group(scale * (_tr(dds + ds.abs() * (wP + n * Lq * U32)) @ q.abs())) + r * dk.abs()
    dv = group(_tr(p) @ do)
    res["dv"] = dv, group(_tr(p * (rP + wP + n * Lq * U32)) @ do.abs()) + r * dv.abs()
    return res


def check(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), name
    far = (got.detach().double() - value).abs() - bound
    worst = float(far.max()) if far.numel() else 0.0
    assert worst <= 1e-30, f"{name}: {worst:.3e} beyond its bound at {int(far.argmax())}"
