"""Performance cases of the operators around relative position: attention with a learned bias by buckets of relative
position, its mean score map, and the root-mean-square norm that takes the residual along.

A case is a dict of plain values:

  op          attention  ``relative_bias_attention``: softmax(q.k / sqrt(d) + w[bucket(position difference)]) v
              map        the same with the mean probability map of all samples and heads (what pattern discovery reads)
              norm       ``rms_norm`` with the residual's addition
              norm_fp8   ``rms_norm_fp8``: the same with an output in 8 bits and a scale for every row
  train       forward and backward (attention, norm); otherwise the forward without gradients
  dtype       float32 or bfloat16, of all tensors
  attention, map:  batch, heads, q_len, k_len, head_dim, buckets, distance (from which on all positions share a bucket),
              padded (with a key mask, samples half to completely full), block and density (0: every key; else block masks:
              keys outside the pattern count with a logit of 0, as in the other sparse modules)
  norm:       rows, width, residual (whether there is one)

``listed`` holds the fixed cases, ``draw`` gives others of the same ranges.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6


def _attention(name, dtype, train, batch, heads, q_len, k_len, head_dim, buckets=32, distance=128, padded=False, block=0,
               density=1.0, op="attention"):
    return {"name": name, "op": op, "train": train, "dtype": dtype, "batch": batch, "heads": heads, "q_len": q_len,
            "k_len": k_len, "head_dim": head_dim, "buckets": buckets, "distance": distance, "padded": padded,
            "block": block, "density": density}


def _norm(name, op, dtype, train, rows, width, residual=True):
    return {"name": name, "op": op, "train": train, "dtype": dtype, "rows": rows, "width": width, "residual": residual}


def listed():
    return [
        # One query a sample (a pooling or answer token) over the keys of a padded text sample.  Latency.
        _attention("bias_infer_token", "bfloat16", False, 8, 8, 1, 2048, 64, padded=True),
        # A training step of the fp32 layer's core at L = 1024 with a small batch.
        _attention("bias_train_short", "float32", True, 8, 2, 1024, 1024, 32),
        # The bf16 training step over padded text at a full batch: the largest dense call.
        _attention("bias_train_padded", "bfloat16", True, 16, 8, 2048, 2048, 64, padded=True),
        # fp32, sizes off the powers of two, wider heads, more and wider buckets.
        _attention("bias_train_ragged", "float32", True, 3, 4, 1000, 1000, 64, buckets=64, distance=500, padded=True),
        # The sparse phase in bf16: 8192 tokens, 64 x 64 blocks, a tenth of them kept.
        _attention("bias_train_sparse", "bfloat16", True, 2, 8, 8192, 8192, 64, block=64, density=0.10),
        # Evaluation of the fp32 layer in the sparse phase, padded, 32 x 32 blocks.
        _attention("bias_infer_sparse", "float32", False, 8, 2, 2048, 2048, 32, padded=True, block=32, density=0.08),
        # The dense phase ahead of discovery: the forward with the mean of its maps, as the image task runs it.
        _attention("map_image", "float32", False, 64, 2, 1024, 1024, 32, op="map"),
        # The same in bf16 over padded text of an odd length.
        _attention("map_padded", "bfloat16", False, 4, 8, 2000, 2000, 64, padded=True, op="map"),
        # The norms of a training step of the small encoder: many short rows.
        _norm("norm_train_tokens", "norm", "float32", True, 262144, 64),
        # Wide rows in bf16.
        _norm("norm_train_wide", "norm", "bfloat16", True, 8192, 4096),
        # Evaluation with 8-bit activations.
        _norm("norm_infer_8bit", "norm_fp8", "bfloat16", False, 16384, 1000),
        # One sample's pooled row.  Latency.
        _norm("norm_infer_8bit_row", "norm_fp8", "float32", False, 1, 768),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "map", "norm", "norm_fp8"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op in ("norm", "norm_fp8"):
        width = _log_int(rng, 16, 8192)
        rows = max(1, min(_log_int(rng, 1, 262144), (1 << 25) // width))
        c = _norm("", op, dtype, op == "norm" and rng.random() < 0.7, rows, width, rng.random() < 0.8)
    else:
        head_dim = rng.choice([32, 64])
        train = op == "attention" and rng.random() < 0.6
        length = _log_int(rng, 65, 2500 if op == "map" else 4096)
        heads = rng.randint(1, 8)
        room = (1 << 28) if dtype == "bfloat16" else (1 << 26)  # pairs of queries and keys in all
        batch = max(1, min(_log_int(rng, 1, 32), room // (length * length * heads)))
        block, density, q_len = 0, 1.0, length
        if op == "attention":
            kind = rng.choice(["dense", "sparse", "few"])
            if kind == "sparse" and length >= 128:
                block, density = rng.choice([32, 64, 128]), round(rng.uniform(0.05, 0.3), 3)
            elif kind == "few":  # the last few positions as queries
                q_len = _log_int(rng, 1, min(64, length))
        buckets = rng.choice([8, 16, 32, 64])
        distance = _log_int(rng, buckets, 800)
        c = _attention("", dtype, train, batch, heads, q_len, length, head_dim, buckets, distance, rng.random() < 0.5, block,
                       density, op)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _bucket_map(num_buckets, distance):
    """Bucket of every position difference -distance .. distance: half of the buckets for keys behind the query or on it, half
    for keys ahead; in each, one for every difference up to a half of them, then borders in a geometric row up to
    ``distance``.  Border k is the least n with (n / exact)^(half - exact) >= (distance / exact)^k, in whole numbers."""
    half = num_buckets // 2
    exact = half // 2
    logs = half - exact
    side = []
    k = 0
    for n in range(distance + 1):
        if n < exact:
            side.append(n)
            continue
        while k + 1 < logs and n ** logs * exact ** (k + 1) >= distance ** (k + 1) * exact ** logs:
            k += 1
        side.append(exact + k)
    return np.array([side[-r] if r <= 0 else half + side[r] for r in range(-distance, distance + 1)], dtype=np.int32)


def _block_mask(blocks, density, seed):
    """A band of three blocks and random ones up to the density."""
    r = np.random.default_rng(seed)
    i = np.arange(blocks)
    m = np.abs(i[:, None] - i[None, :]) <= 1
    off = np.flatnonzero(~m.ravel())
    want = int(round(density * blocks * blocks)) - int(m.sum())
    if want > 0:
        m.ravel()[r.choice(off, size=min(want, off.size), replace=False)] = True
    return m.astype(np.float32)


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = getattr(torch, case["dtype"])
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    s = dict(case)
    if case["op"] in ("norm", "norm_fp8"):
        rows, n = case["rows"], case["width"]
        s["x"] = normal(rows, n)
        s["res"] = normal(rows, n, scale=2.0) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(n, generator=g, device=dev)).to(dt)
        if case["train"]:
            s["dy"], s["dh"] = normal(rows, n), normal(rows, n) if case["residual"] else None
        return s
    B, H, Lq, Lk, d = (case[k] for k in ("batch", "heads", "q_len", "k_len", "head_dim"))
    # heads as a layer has them: views of its projections
    if Lq == Lk:
        qkv = normal(B, Lk, 3, H, d)
        s["q"], s["k"], s["v"] = (qkv[:, :, i].transpose(1, 2) for i in range(3))
    else:
        kv = normal(B, Lk, 2, H, d)
        s["q"] = normal(B, Lq, H, d).transpose(1, 2)
        s["k"], s["v"] = (kv[:, :, i].transpose(1, 2) for i in range(2))
    s["w"] = normal(case["buckets"], H, scale=0.7)
    s["map"] = torch.from_numpy(_bucket_map(case["buckets"], case["distance"])).to(dev)
    s["offset"] = Lk - Lq
    s["mask"] = None
    if case["padded"]:
        lens = torch.randint((Lk + 1) // 2, Lk + 1, (B, 1), generator=g, device=dev)
        s["mask"] = (torch.arange(Lk, device=dev)[None, :] < lens).to(torch.float32)
    s["mat"] = None
    if case["block"]:
        s["mat"] = torch.from_numpy(_block_mask(-(-Lk // case["block"]), case["density"], seed)).to(dev)
    if case["train"]:
        s["do"] = normal(B, Lq, H, d).transpose(1, 2)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return _plain_norm(s) if s["op"] in ("norm", "norm_fp8") else _plain_attention(s)


def _run_own(s):
    import spion_amd

    if s["op"] == "norm_fp8":
        return spion_amd.rms_norm_fp8(s["x"], s["w"], s["res"], EPS)
    if s["op"] == "norm":
        if not s["train"]:
            out = spion_amd.rms_norm(s["x"], s["w"], s["res"], EPS)
            return [out] if s["res"] is None else out
        leaves = [t.detach().requires_grad_() for t in (s["x"], s["w"], s["res"]) if t is not None]
        out = spion_amd.rms_norm(*leaves, eps=EPS)
        if s["res"] is None:
            return [out.detach(), *torch.autograd.grad(out, leaves, s["dy"])]
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (s["dy"], s["dh"]))]
    more = {"key_mask": s["mask"], "mat": s["mat"], "block_size": s["block"] or None, "offset": s["offset"]}
    if not s["train"]:
        with torch.no_grad():
            return spion_amd.relative_bias_attention(s["q"], s["k"], s["v"], s["w"], s["map"], score_map=s["op"] == "map", **more)
    leaves = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["v"], s["w"])]
    out = spion_amd.relative_bias_attention(*leaves, s["map"], **more)
    return [out.detach(), *torch.autograd.grad(out, leaves, s["do"])]


def _plain_norm(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    h = x if s["res"] is None else (x + s["res"].float()).to(dt).float()  # the stream as it is stored
    inv = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    xhat = h * inv
    y = xhat * w
    if s["op"] == "norm_fp8":
        scale = torch.clamp(y.abs().amax(-1) / 448.0, min=2.0 ** -126)
        out = [(y / scale[:, None]).to(torch.float8_e4m3fn), scale]
        return out if s["res"] is None else [*out, h.to(dt)]
    out = [y.to(dt)] if s["res"] is None else [y.to(dt), h.to(dt)]
    if not s["train"]:
        return out
    dy = s["dy"].float()
    dx = dy * w
    dh = inv * (dx - xhat * (dx * xhat).mean(-1, keepdim=True))
    dw = (dy * xhat).sum(0, dtype=torch.float64).to(dt)
    if s["res"] is None:
        return [*out, dh.to(dt), dw]
    dh = (dh + s["dh"].float()).to(dt)
    return [*out, dh, dw, dh]


def _plain_attention(s):
    dt = s["q"].dtype
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    B, H, Lq, d = q.shape
    Lk = k.shape[2]
    R = s["distance"]
    dev = q.device
    rel = torch.arange(Lk, device=dev)[None, :] - torch.arange(Lq, device=dev)[:, None] - s["offset"]
    bucket = s["map"].long()[rel.clamp(-R, R) + R]
    logits = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d)) + s["w"].float().t()[:, bucket]
    if s["mask"] is not None:
        logits = logits.masked_fill((s["mask"] == 0)[:, None, None, :], -math.inf)
    off = None
    if s["mat"] is not None:
        bs = s["block"]
        at = torch.arange(Lk, device=dev) // bs
        off = s["mat"][at][:, at] == 0
        logits = torch.where(off, 0.0, logits)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    if off is not None:
        p = p.masked_fill(off, 0.0)
    out = torch.matmul(p, v)
    if s["op"] == "map":
        return [out.to(dt), p.mean((0, 1))]
    if not s["train"]:
        return out.to(dt)
    do = s["do"].float()
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (do * out).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * (1.0 / math.sqrt(d))
    dk = torch.matmul(ds.transpose(-1, -2), q) * (1.0 / math.sqrt(d))
    # the table: sums of ds along its diagonals (rows turned over, each one place further to the right than the one
    # before), then over the diagonals of a bucket
    x = torch.nn.functional.pad(ds.sum(0, dtype=torch.float64).flip(1), (0, Lq)).reshape(H, -1)
    diag = x[:, : Lq * (Lq + Lk - 1)].reshape(H, Lq, Lq + Lk - 1).sum(1)
    far = torch.arange(Lq + Lk - 1, device=dev) - (Lq - 1) - s["offset"]
    dw = torch.zeros(s["buckets"], H, dtype=torch.float64, device=dev)
    dw = dw.index_add(0, s["map"].long()[far.clamp(-R, R) + R], diag.t())
    return [out.to(dt), dq.to(dt), dk.to(dt), dv.to(dt), dw.to(dt)]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] in ("norm", "norm_fp8"):
        rows, n, r = case["rows"], case["width"], int(case["residual"])
        out = rows * (n + 4) if case["op"] == "norm_fp8" else rows * n * e
        nbytes = rows * n * e * (1 + 2 * r) + out + n * e
        flops = 5 * rows * n
        if case["train"]:  # the stream and the gradients in, one gradient and the weight's out
            nbytes += rows * n * e * (3 + r) + 2 * n * e
            flops += 10 * rows * n
        return {"bytes": nbytes, "flops": flops}
    B, H, Lq, Lk, d = (case[k] for k in ("batch", "heads", "q_len", "k_len", "head_dim"))
    pairs = B * H * Lq * Lk * (0.75 if case["padded"] else 1.0)
    if case["block"]:
        nb = -(-Lk // case["block"])
        pairs *= max(case["density"], min(1.0, (3 * nb - 2) / nb ** 2))
    queries, keys = B * H * Lq * d * e, B * H * Lk * d * e
    nbytes = 2 * queries + 2 * keys + (B * Lk * 4 if case["padded"] else 0)
    flops = 4 * pairs * d
    if case["op"] == "map":
        nbytes += Lq * Lk * 4
        flops += 2 * pairs * d
    if case["train"]:
        nbytes += 4 * queries + 4 * keys + B * H * Lq * 8
        flops += 8 * pairs * d
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, a head at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_fp8"):
        return _exact_norm(s)
    B, H, Lq, d = s["q"].shape
    Lk = s["k"].shape[2]
    dev = s["q"].device
    R = s["distance"]
    d64 = {n: s[n].double() for n in ("q", "k", "v", "w", "do") if n in s}
    out = torch.zeros(B, H, Lq, d, dtype=torch.float64, device=dev)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(B, H, Lk, d, dtype=torch.float64, device=dev), None
    dv = torch.zeros_like(dk)
    dw = torch.zeros_like(d64["w"])
    mean = torch.zeros(Lq, Lk, dtype=torch.float64, device=dev)
    which = torch.arange(Lk, device=dev)[None, :] - (torch.arange(Lq, device=dev)[:, None] + s["offset"])
    which = s["map"].long()[(which + R).clamp(0, 2 * R)]
    inside = None
    if s["mat"] is not None:
        inside = (s["mat"] != 0).repeat_interleave(s["block"], 0).repeat_interleave(s["block"], 1)[:Lq, :Lk]
    of_bucket = [(which == i).to(torch.float64) for i in range(s["buckets"])] if case["train"] and which.numel() < 2 ** 21 else None
    ds_all = torch.zeros(H, Lq, Lk, dtype=torch.float64, device=dev) if case["train"] else None
    for b in range(B):
        there = torch.ones(Lk, dtype=torch.bool, device=dev) if s["mask"] is None else s["mask"][b] != 0
        for h in range(H):
            z = d64["q"][b, h] @ d64["k"][b, h].T.contiguous() / math.sqrt(d) + d64["w"][:, h][which]
            e = torch.exp(z) * there  # logits of some tens at most: no shift is needed in 64 bits
            if inside is not None:
                e = e * inside
                norm = e.sum(1) + (~inside).sum(1)
            else:
                norm = e.sum(1)
            p = e / norm[:, None].clamp_min(1e-300)
            out[b, h] = p @ d64["v"][b, h]
            if case["op"] == "map":
                mean += p
            if case["train"]:
                do = d64["do"][b, h]
                dv[b, h] = p.T @ do
                ds = p * (do @ d64["v"][b, h].T)
                ds = ds - p * ds.sum(1, keepdim=True)
                dq[b, h] = ds @ d64["k"][b, h] / math.sqrt(d)
                dk[b, h] = ds.T @ d64["q"][b, h] / math.sqrt(d)
                ds_all[h] += ds
    if case["op"] == "map":
        return [out, mean / (B * H)]
    if not case["train"]:
        return out
    if of_bucket is not None:
        for i, m in enumerate(of_bucket):
            dw[i] = (ds_all * m).sum((1, 2))
    else:
        for i in range(s["buckets"]):
            dw[i] = torch.stack([ds_all[h][which == i].sum() for h in range(H)])
    return [out, dq, dk, dv, dw]


def _exact_norm(s):
    x, w = s["x"].double(), s["w"].double()
    h = x
    if s["res"] is not None:
        h = (x + s["res"].double()).to(s["x"].dtype).double()  # the stream is stored in the tensors' type
    n = h.shape[1]
    rms = torch.sqrt(h.pow(2).sum(1, keepdim=True) / n + EPS)
    y = h / rms * w
    if s["op"] == "norm_fp8":
        scale = y.abs().max(1).values / 448.0
        # 8 bits: four of exponent, three of mantissa, by rounding to a multiple of the binade's step, ties to even
        c = y / scale[:, None]
        step = torch.exp2(torch.floor(torch.log2(c.abs().clamp_min(2.0 ** -6))) - 3)
        out = [torch.round(c / step) * step, scale]
        return out if s["res"] is None else [*out, h]
    out = [y] if s["res"] is None else [y, h]
    if not s["train"]:
        return out
    dy = s["dy"].double()
    dx = (dy * w) / rms - h * (dy * w * h).sum(1, keepdim=True) / (n * rms ** 3)
    dw = (dy * h / rms).sum(0)
    if s["res"] is None:
        return [*out, dx, dw]
    dx = dx + s["dh"].double()
    return [*out, dx, dw, dx]
