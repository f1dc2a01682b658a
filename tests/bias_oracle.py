"""64-bit statement of attention with a relative position bias, and how far a kernel may be off it.

The bounds count roundings: u32 = 2^-24 for an fp32 operation, a bf16 value half a step of 2^-8.  A sum of n terms in fp32 is off by at
most n u32 of the sum of magnitudes.  With t the logits, P = exp(t) / Z:
  dt    = (d + 8) u32 (|q|.|k| scale + |bias|)                 product, scale, bias, subtraction of the maximum, exp2's argument
  rP    = 2 max_j dt + (Lk + 64) u32                           of numerator and denominator, exp2, the sum of the denominator
  out   : sum_j P |v| (rP + wP + Lk u32) + r |out|             wP: rounding of the weights P to bf16 in the product, r: of the output
  D     : for dQ dO.out of the output as rounded: sum_f |dO| (P |v|) (rP + wP + Lk u32) + (r + d u32) |dO|.|out|; for dK and dw the sum
          over the keys of P dP: (rP + (Lk + 8) u32) (sum_j P |dP| + |D|) + sum_j P d u32 |dO|.|v|
  dS    : |dS| (rP + 4 u32) + P (d u32 |dO|.|v| + d(D))
  dQ    : scale sum_j (d(dS) + |dS| (wP + Lk u32)) |k| + r |dQ|, dK alike; dV: sum_i P |dO| (rP + wP + Lq u32) + r |dV|
  dw    : sum over the bucket of d(dS) + |dS| (Lq + Lk + B) u32, + r |dw|
"""
import math

import torch

U32 = 2.0 ** -24


def bias_reference(q, k, v, w, buckets, mask=None, mat=None, block=0, offset=0, do=None):
    """Returns {"out", "p", and with do "dq", "dk", "dv", "dw"}: each (value, bound) in float64 on the inputs' device."""
    bf = q.dtype == torch.bfloat16
    r, wP = (2.0 ** -8, 2.0 ** -8) if bf else (2 * U32, 2 * U32)
    q, k, v, w = (x.detach().double() for x in (q, k, v, w))
    B, H, Lq, d = q.shape
    Lk = k.shape[2]
    dev = q.device
    scale = 1.0 / math.sqrt(d)
    R = buckets.shape[0] // 2
    rel = torch.arange(Lk, device=dev)[None, :] - torch.arange(Lq, device=dev)[:, None] - offset
    bucket = buckets.long().clamp(0, w.shape[0] - 1)[rel.clamp(-R, R) + R]
    there = torch.ones(B, Lk, dtype=torch.bool, device=dev) if mask is None else mask != 0
    k = torch.where(there[:, None, :, None], k, 0.0)  # whatever lies in a key that is left out
    v = torch.where(there[:, None, :, None], v, 0.0)
    inside = torch.ones(Lq, Lk, dtype=torch.bool, device=dev)
    if mat is not None:
        at = torch.arange(Lk, device=dev) // block
        inside = mat[at][:, at] != 0
    bias = w.t()[:, bucket]  # [H, Lq, Lk]
    t = q @ k.transpose(-1, -2).contiguous() * scale + bias
    use = there[:, None, None, :] & inside
    t = torch.where(use, t, -math.inf)
    off = (~inside).sum(-1).double()[:, None]  # logits of 0
    top = t.amax(-1, keepdim=True).clamp_min(0.0 if mat is not None else -math.inf)
    top = torch.where(torch.isinf(top), 0.0, top)
    e = torch.exp(t - top)
    z = e.sum(-1, keepdim=True) + off * torch.exp(-top)
    p = torch.where(z > 0, e / z, 0.0)
    out = p @ v
    fin = torch.where(torch.isinf(bias), 0.0, bias.abs())
    dt = (d + 8) * U32 * (q.abs() @ k.abs().transpose(-1, -2).contiguous() * scale + fin)
    dt = torch.where(use & (p > 0), dt, 0.0)
    rP = 2 * dt.amax(-1, keepdim=True) + (Lk + 64) * U32
    pv = p @ v.abs()
    res = {"out": (out, pv * (rP + wP + Lk * U32) + r * out.abs()), "p": (p, p * rP)}
    if do is None:
        return res
    do = do.detach().double()
    dp = do @ v.transpose(-1, -2).contiguous()
    D = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - D)
    ddp = d * U32 * (do.abs() @ v.abs().transpose(-1, -2).contiguous())
    dD = (do.abs() * pv).sum(-1, keepdim=True) * (rP + wP + Lk * U32) + (r + d * U32) * (do.abs() * out.abs()).sum(-1, keepdim=True)
    dds = ds.abs() * (rP + 4 * U32) + p * (ddp + dD)
    dq = scale * ds @ k
    res["dq"] = dq, scale * ((dds + ds.abs() * (wP + Lk * U32)) @ k.abs()) + r * dq.abs()
    dD = (rP + (Lk + 8) * U32) * ((p * dp.abs()).sum(-1, keepdim=True) + D.abs()) + (p * ddp).sum(-1, keepdim=True)
    dds = ds.abs() * (rP + 4 * U32) + p * (ddp + dD)
    tr = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dk = scale * tr(ds) @ q
    res["dk"] = dk, scale * (tr(dds + ds.abs() * (wP + Lq * U32)) @ q.abs()) + r * dk.abs()
    dv = tr(p) @ do
    res["dv"] = dv, tr(p * (rP + wP + Lq * U32)) @ do.abs() + r * dv.abs()
    sums = []
    for x in (ds, dds + ds.abs() * ((Lq + Lk + B) * U32)):
        sums.append(torch.zeros(w.shape[0], H, dtype=torch.float64, device=dev).index_add(
            0, bucket.reshape(-1), x.sum(0).reshape(H, -1).t()))
    res["dw"] = sums[0], sums[1] + r * sums[0].abs()
    return res


def check(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), name
    far = (got.detach().double() - value).abs() - bound
    worst = float(far.max()) if far.numel() else 0.0
    assert worst <= 1e-30, f"{name}: {worst:.3e} beyond its bound at {int(far.argmax())}"
