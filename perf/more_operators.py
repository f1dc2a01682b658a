"""Performance cases of the operators around an encoder's states: attention of other queries to them, and the layer norm that
takes the residual along.

A case is a dict of plain values:

  op          cross   ``cross_attention``: queries of one length over keys and values of another, heads of keys shared by
                      ``heads / key_heads`` heads of queries
              norm    ``layer_norm`` with weight and bias
  train       forward and backward; otherwise the forward without gradients
  dtype       float32 or bfloat16, of all tensors
  cross:      batch, heads, key_heads, q_len, k_len, head_dim, padded (with a key mask, samples half to completely full)
  norm:       rows, width, residual (whether there is one)

``listed`` holds the fixed cases, ``draw`` gives others of the same ranges.
"""
import math

import torch

own = False

EPS = 1e-5


def _cross(name, dtype, train, batch, heads, key_heads, q_len, k_len, head_dim, padded=False):
    return {"name": name, "op": "cross", "train": train, "dtype": dtype, "batch": batch, "heads": heads, "key_heads": key_heads,
            "q_len": q_len, "k_len": k_len, "head_dim": head_dim, "padded": padded}


def _norm(name, dtype, train, rows, width, residual=True):
    return {"name": name, "op": "norm", "train": train, "dtype": dtype, "rows": rows, "width": width, "residual": residual}


def listed():
    return [
        # One token of a decoder over the padded states of a text encoder.  Latency.
        _cross("cross_token", "bfloat16", False, 8, 8, 8, 1, 2048, 64, padded=True),
        # One token over long states whose key heads are shared by four heads each: K and V are read once.
        _cross("cross_token_grouped", "bfloat16", False, 4, 16, 4, 1, 32768, 128),
        # Pooling by sixteen learned queries over padded text in training, fp32 heads of the small encoder.
        _cross("cross_train_pool", "float32", True, 32, 2, 2, 16, 4096, 32, padded=True),
        # A training step of a short decoder over image tokens, fp32.
        _cross("cross_train_short", "float32", True, 32, 2, 2, 256, 1024, 32),
        # fp32, both lengths off the powers of two, wider heads, padded.
        _cross("cross_train_ragged", "float32", True, 3, 4, 4, 333, 1000, 64, padded=True),
        # The bf16 training step of a decoder over padded text at a full batch.
        _cross("cross_train_padded", "bfloat16", True, 16, 8, 8, 1024, 2048, 64, padded=True),
        # Long states, wide heads, shared key heads: the largest call.
        _cross("cross_train_grouped", "bfloat16", True, 2, 16, 4, 2048, 8192, 128),
        # Many queries over few states: image tokens over the hundred of a sentence.
        _cross("cross_train_few_keys", "bfloat16", True, 4, 8, 8, 4096, 100, 64),
        # The norms of a training step of the small encoder: many short rows.
        _norm("norm_train_tokens", "float32", True, 262144, 64),
        # Wide rows in bf16.
        _norm("norm_train_wide", "bfloat16", True, 8192, 4096),
        # Evaluation with rows of an odd width, no residual.
        _norm("norm_infer_odd", "bfloat16", False, 16384, 1001, residual=False),
        # One sample's pooled row.  Latency.
        _norm("norm_infer_row", "float32", False, 1, 768),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cross", "cross", "norm"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "norm":
        width = _log_int(rng, 16, 8192)
        rows = max(1, min(_log_int(rng, 1, 262144), (1 << 24) // width))
        c = _norm("", dtype, rng.random() < 0.6, rows, width, rng.random() < 0.7)
    else:
        head_dim = rng.choice([32, 64, 128])
        key_heads = rng.randint(1, 8)
        heads = key_heads * rng.choice([1, 1, 2, 4])
        kind = rng.choice(["token", "few", "rows", "rows"])
        if kind == "token":
            q_len, k_len, train = 1, _log_int(rng, 64, 32768), False
        else:
            q_len = _log_int(rng, 2, 64) if kind == "few" else _log_int(rng, 65, 4096)
            k_len, train = _log_int(rng, 16, 8192), rng.random() < 0.7
        room = (1 << 28) if dtype == "bfloat16" else (1 << 26)  # pairs of queries and keys in all
        cells = (1 << 26) if kind == "token" else (1 << 25)  # elements of K
        batch = max(1, min(_log_int(rng, 1, 32), room // (q_len * k_len * heads), cells // (k_len * key_heads * head_dim)))
        c = _cross("", dtype, train, batch, heads, key_heads, q_len, k_len, head_dim, rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    dt = getattr(torch, case["dtype"])
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    s = dict(case)
    if case["op"] == "norm":
        rows, n = case["rows"], case["width"]
        s["x"] = (normal(rows, n).float() + 0.5).to(dt)
        s["res"] = normal(rows, n, scale=2.0) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(n, generator=g, device=dev)).to(dt)
        s["b"] = normal(n, scale=0.3)
        if case["train"]:
            s["dy"], s["dh"] = normal(rows, n), normal(rows, n) if case["residual"] else None
        return s
    B, H, G, Lq, Lk, d = (case[k] for k in ("batch", "heads", "key_heads", "q_len", "k_len", "head_dim"))
    # heads as a layer has them: views of its projections, keys and values side by side
    kv = normal(B, Lk, 2, G, d)
    s["q"] = normal(B, Lq, H, d, scale=1.5).transpose(1, 2)
    s["k"], s["v"] = (kv[:, :, i].transpose(1, 2) for i in range(2))
    s["mask"] = None
    if case["padded"]:
        lens = torch.randint((Lk + 1) // 2, Lk + 1, (B, 1), generator=g, device=dev)
        s["mask"] = (torch.arange(Lk, device=dev)[None, :] < lens).to(torch.float32)
    if case["train"]:
        s["do"] = normal(B, Lq, H, d).transpose(1, 2)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return _plain_norm(s) if s["op"] == "norm" else _plain_cross(s)


def _run_own(s):
    import spion_amd

    if s["op"] == "norm":
        if not s["train"]:
            with torch.no_grad():
                out = spion_amd.layer_norm(s["x"], s["w"], s["b"], s["res"], EPS)
            return [out] if s["res"] is None else out
        leaves = [t.detach().requires_grad_() for t in (s["x"], s["w"], s["b"], s["res"]) if t is not None]
        out = spion_amd.layer_norm(*leaves, eps=EPS)
        if s["res"] is None:
            return [out.detach(), *torch.autograd.grad(out, leaves, s["dy"])]
        return [*(t.detach() for t in out), *torch.autograd.grad(out, leaves, (s["dy"], s["dh"]))]
    if not s["train"]:
        with torch.no_grad():
            return spion_amd.cross_attention(s["q"], s["k"], s["v"], s["mask"])
    leaves = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["v"])]
    out = spion_amd.cross_attention(*leaves, s["mask"])
    return [out.detach(), *torch.autograd.grad(out, leaves, s["do"])]


def _plain_norm(s):
    x, w, b, dt = s["x"].float(), s["w"].float(), s["b"].float(), s["x"].dtype
    h = x if s["res"] is None else (x + s["res"].float()).to(dt).float()  # the stream as it is stored
    centred = h - h.mean(-1, keepdim=True)
    inv = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * inv
    y = (xhat * w + b).to(dt)
    out = [y] if s["res"] is None else [y, h.to(dt)]
    if not s["train"]:
        return out
    dy = s["dy"].float()
    g = dy * w
    dx = inv * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    dw = (dy * xhat).sum(0, dtype=torch.float64).to(dt)
    db = dy.sum(0, dtype=torch.float64).to(dt)
    if s["res"] is None:
        return [*out, dx.to(dt), dw, db]
    dx = (dx + s["dh"].float()).to(dt)
    return [*out, dx, dw, db, dx]


def _plain_cross(s):
    dt = s["q"].dtype
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    B, H, Lq, d = q.shape
    G = k.shape[1]
    k, v = k.contiguous(), v.contiguous()
    q = q.reshape(B, G, H // G * Lq, d)  # the heads that share keys, one behind the other
    logits = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    if s["mask"] is not None:
        logits = logits.masked_fill((s["mask"] == 0)[:, None, None, :], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    out = torch.matmul(p, v)
    if not s["train"]:
        return out.reshape(B, H, Lq, d).to(dt)
    do = s["do"].float().reshape(B, G, H // G * Lq, d)
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, v.transpose(-1, -2))
    ds = p * (dp - (do * out).sum(-1, keepdim=True)) * (1.0 / math.sqrt(d))
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    return [out.reshape(B, H, Lq, d).to(dt), dq.reshape(B, H, Lq, d).to(dt), dk.to(dt), dv.to(dt)]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        rows, n, r = case["rows"], case["width"], int(case["residual"])
        nbytes = rows * n * e * (2 + 2 * r) + 2 * n * e
        flops = 8 * rows * n
        if case["train"]:  # the stream and the gradients in, one gradient and the parameters' out
            nbytes += rows * n * e * (3 + r) + 3 * n * e
            flops += 14 * rows * n
        return {"bytes": nbytes, "flops": flops}
    B, H, G, Lq, Lk, d = (case[k] for k in ("batch", "heads", "key_heads", "q_len", "k_len", "head_dim"))
    full = 0.75 if case["padded"] else 1.0
    pairs = B * H * Lq * Lk * full
    queries, keys = B * H * Lq * d * e, B * G * Lk * d * e * full
    nbytes = 2 * queries + 2 * keys + (B * Lk * 4 if case["padded"] else 0)
    flops = 4 * pairs * d
    if case["train"]:
        nbytes += 4 * queries + 2 * keys + 2 * B * G * Lk * d * e + B * H * Lq * 8
        flops += 8 * pairs * d
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, a head of queries at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    B, H, Lq, d = s["q"].shape
    G, Lk = s["k"].shape[1:3]
    dev = s["q"].device
    out = torch.zeros(B, H, Lq, d, dtype=torch.float64, device=dev)
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(B, G, Lk, d, dtype=torch.float64, device=dev) for _ in range(2))
    for b in range(B):
        keys = torch.arange(Lk, device=dev) if s["mask"] is None else torch.nonzero(s["mask"][b] != 0)[:, 0]
        for h in range(H):
            of = h // (H // G)
            q, k, v = s["q"][b, h].double(), s["k"][b, of].double()[keys], s["v"][b, of].double()[keys]
            p = torch.exp(q @ k.T.contiguous() / math.sqrt(d))  # logits of some tens at most: no shift is needed in 64 bits
            p = p / p.sum(1, keepdim=True).clamp_min(1e-300)
            out[b, h] = p @ v
            if case["train"]:
                do = s["do"][b, h].double()
                dv[b, of].index_add_(0, keys, p.T.contiguous() @ do)
                ds = p * (do @ v.T.contiguous())
                ds = ds - p * ds.sum(1, keepdim=True)
                dq[b, h] = ds @ k / math.sqrt(d)
                dk[b, of].index_add_(0, keys, ds.T.contiguous() @ q / math.sqrt(d))
    return [out, dq, dk, dv] if case["train"] else out


def _exact_norm(s):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    h = x
    if s["res"] is not None:
        h = (x + s["res"].double()).to(s["x"].dtype).double()  # the stream is stored in the tensors' type
    n = h.shape[1]
    mean = h.sum(1, keepdim=True) / n
    std = torch.sqrt((h - mean).pow(2).sum(1, keepdim=True) / n + EPS)
    xh = (h - mean) / std
    y = xh * w + b
    out = [y] if s["res"] is None else [y, h]
    if not s["train"]:
        return out
    dy = s["dy"].double()
    g = dy * w
    # d y / d h: through h itself, the mean and the deviation
    dx = g / std - g.sum(1, keepdim=True) / (n * std) - xh * (g * xh).sum(1, keepdim=True) / (n * std)
    dw, db = (dy * xh).sum(0), dy.sum(0)
    if s["res"] is None:
        return [*out, dx, dw, db]
    dx = dx + s["dh"].double()
    return [*out, dx, dw, db, dx]
