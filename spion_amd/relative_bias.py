"""Attention with a learned bias by buckets of relative position.

The reference's encoder knows positions from embeddings added to its input (models/model_transformer.py:17-52) and has no
such bias; here it enters the logits of both phases of the layer:

    v_ij = q_i . k_j / sqrt(d) + weight[bucket(j - i - offset), head],    out_i = sum_j softmax(v)_ij v_j

* ``relative_position_buckets(num_buckets, max_distance)`` is the usual division of the position differences: half of the buckets
  for keys behind the query (and on it), half for keys ahead, one bucket for every short difference, a geometric row of them
  from there to ``max_distance``, beyond which all differences share the last one.
* ``relative_bias_attention(query, key, value, weight, buckets, ...)`` is the operator with all its gradients, the table's
  among them.
* ``RelativeBiasAttention(config)`` is the module with the block modules' calling convention
  (models/attention_blockcuda_mask.py:21-103): ``forward(query, key, value, mask, mat=None) -> (out, 0)``; it owns the table.

fp32 and bf16 tensors, head dimension 32 or 64; softmax and sums in fp32; the probabilities are never written to memory.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib

MAX_DISTANCE = 1024


def relative_position_buckets(num_buckets: int = 32, max_distance: int = 128, device=None) -> torch.Tensor:
    """int32 [2 * max_distance + 1]: the bucket of each difference (key position - query position) from -max_distance to
    max_distance; what lies further out has the outermost buckets.  Border k of the geometric part is the least n with
    (n / exact)^(half - exact) >= (max_distance / exact)^k, found in whole numbers: no rounding moves a border."""
    if num_buckets < 4 or num_buckets % 4:
        raise ValueError("num_buckets: a positive multiple of 4 expected")
    half = num_buckets // 2
    exact = half // 2
    if not exact < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance {max_distance}: above {exact} and at most {MAX_DISTANCE} expected")
    logs = half - exact
    side, k = [], 0
    for n in range(max_distance + 1):
        if n < exact:
            side.append(n)
            continue
        while k + 1 < logs and n ** logs * exact ** (k + 1) >= max_distance ** (k + 1) * exact ** logs:
            k += 1
        side.append(exact + k)
    return torch.tensor([n for n in reversed(side[1:])] + [side[0]] + [half + n for n in side[1:]], dtype=torch.int32,
                        device=device)


class _Heads(ctypes.Structure):
    """``spion_heads``: a [B, H, L, d] tensor by its strides, in elements."""

    _fields_ = [("p", ctypes.c_void_p), ("batch_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong),
                ("row_stride", ctypes.c_longlong)]


class _Call(ctypes.Structure):
    """``spion_bias_attention``."""

    _fields_ = ([(n, _Heads) for n in ("Q", "K", "V", "Out", "dO", "dQ", "dK", "dV")]
                + [(n, ctypes.c_void_p) for n in ("weight", "dweight", "buckets", "key_mask", "mat", "Lse", "Mean", "workspace")]
                + [("workspace_floats", ctypes.c_longlong)]
                + [(n, ctypes.c_int) for n in ("batch", "heads", "q_len", "k_len", "head_dim", "bf16", "num_buckets",
                                               "max_distance", "offset", "block_size", "mask_bytes")])


def _lib_typed():
    lib = _lib.core()
    if not getattr(lib, "_spion_bias_typed", False):
        for name, res, args in (("spion_bias_workspace", ctypes.c_longlong, [ctypes.c_void_p, ctypes.c_int]),
                                ("spion_bias_attention_forward", ctypes.c_int, [ctypes.c_void_p] * 2),
                                ("spion_bias_attention_backward", ctypes.c_int, [ctypes.c_void_p] * 2)):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
        lib._spion_bias_typed = True
    return lib


def _heads(t):
    return _Heads(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _fits(t):
    return _lib.head_layout(t) is not None and t.stride(2) * t.element_size() <= 1 << 24


def _readable(t):
    """``t`` as the kernels read it: itself, or a contiguous copy where its strides or address are not theirs."""
    if _fits(t):
        return t
    c = t.contiguous()
    return c if _fits(c) else t.clone(memory_format=torch.contiguous_format)


def _empty_like_heads(t):
    """Uninitialised heads in the memory order of ``t``: [B, L, H, d] where the heads of a row lie next to each other, as a
    projection leaves them.  [B, H, L, d] where the kernels would not take that (rows 2^24 bytes apart, heads of 2^29 elements and
    more from their first row to their last): such a ``t`` is itself read from a copy."""
    B, H, L, d = t.shape
    if t.stride(1) < t.stride(2) and H * d * t.element_size() <= 1 << 24 and L * H * d < 1 << 29:
        return torch.empty((B, L, H, d), dtype=t.dtype, device=t.device).transpose(1, 2)
    return torch.empty((B, H, L, d), dtype=t.dtype, device=t.device)


def _call_of(q, k, weight, buckets, key_mask, mat, block_size, offset):
    B, H, Lq, d = q.shape
    c = _Call(weight=weight.data_ptr(), buckets=buckets.data_ptr(), batch=B, heads=H, q_len=Lq, k_len=k.shape[2], head_dim=d,
              bf16=int(q.dtype == torch.bfloat16), num_buckets=weight.shape[0], max_distance=buckets.shape[0] // 2,
              offset=offset, block_size=block_size)
    if key_mask is not None:
        c.key_mask, c.mask_bytes = key_mask.data_ptr(), key_mask.element_size()
    if mat is not None:
        c.mat = mat.data_ptr()
    return c


def _workspace(lib, call, backward, device):
    n = lib.spion_bias_workspace(ctypes.addressof(call), int(backward))
    _lib.check_call(n >= 0, "spion_bias_workspace")
    ws = torch.empty(n, dtype=torch.float32, device=device)
    call.workspace, call.workspace_floats = ws.data_ptr() if n else None, n
    return ws


class _RelativeBiasFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, weight, buckets, key_mask, mat, block_size, offset, score_map):
        dev, (B, H, Lq, d), Lk = query.device, query.shape, key.shape[2]
        lib = _lib_typed()
        q, k, v, w = _readable(query), _readable(key), _readable(value), weight.contiguous()
        out = _empty_like_heads(query)
        lse = torch.empty((B * H, Lq), dtype=torch.float32, device=dev)
        mean = torch.empty((Lq, Lk), dtype=torch.float32, device=dev) if score_map else None
        with torch.cuda.device(dev):
            call = _call_of(q, k, w, buckets, key_mask, mat, block_size, offset)
            call.Q, call.K, call.V, call.Out = (_heads(t) for t in (q, k, v, out))
            call.Lse = lse.data_ptr()
            if mean is not None:
                call.Mean = mean.data_ptr()
            ws = _workspace(lib, call, False, dev)
            _lib.check_call(lib.spion_bias_attention_forward(ctypes.addressof(call), _lib._raw_stream(dev.index)) == 0,
                            "spion_bias_attention_forward")
            del ws
        optional = {"key_mask": key_mask, "mat": mat}
        ctx.given = [n for n, t in optional.items() if t is not None]
        ctx.numbers = (block_size, offset)
        _lib.save_for_backward(ctx, q, k, v, w, out, lse, buckets, *(optional[n] for n in ctx.given))
        if mean is None:
            return out
        ctx.mark_non_differentiable(mean)
        return out, mean

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, *_):
        saved = _lib.saved_tensors(ctx)
        block_size, offset = ctx.numbers
        lse, buckets, w = saved[5].contiguous(), saved[6].contiguous(), saved[3].contiguous()
        q, k, v, out = (_readable(saved[i]) for i in (0, 1, 2, 4))
        rest = {n: t.contiguous() for n, t in zip(ctx.given, saved[7:])}
        dev = q.device
        lib = _lib_typed()
        go = grad_output if grad_output.dtype == q.dtype else grad_output.to(q.dtype)
        go = _readable(go)
        if q.dtype == torch.float32 and q.shape == k.shape and _lib.adjacent_head_views(q, k, v):
            dq, dk, dv = _lib.empty_adjacent_heads(*q.shape, dev)  # slices of one fused projection: the gradients likewise
        else:
            dq, dk, dv = (_empty_like_heads(t) for t in (q, k, v))
        dw = torch.empty(w.shape, dtype=w.dtype, device=dev)
        with torch.cuda.device(dev):
            call = _call_of(q, k, w, buckets, rest.get("key_mask"), rest.get("mat"), block_size, offset)
            call.Q, call.K, call.V, call.Out = (_heads(t) for t in (q, k, v, out))
            call.dO, call.dQ, call.dK, call.dV = (_heads(t) for t in (go, dq, dk, dv))
            call.Lse, call.dweight = lse.data_ptr(), dw.data_ptr()
            ws = _workspace(lib, call, True, dev)
            _lib.check_call(lib.spion_bias_attention_backward(ctypes.addressof(call), _lib._raw_stream(dev.index)) == 0,
                            "spion_bias_attention_backward")
            del ws
        return dq, dk, dv, dw, None, None, None, None, None, None


def _check(query, key, value, weight, buckets, key_mask, mat, block_size, offset, score_map):
    """The kernels take sizes, types and devices as they are told: anything else would be read past its end."""
    if query.dim() != 4 or key.dim() != 4:
        raise ValueError("heads [B, H, L, d] expected")
    B, H, Lq, d = query.shape
    Lk = key.shape[2]
    for name, t, shape in (("key", key, (B, H, Lk, d)), ("value", value, (B, H, Lk, d))):
        if tuple(t.shape) != shape:
            raise ValueError(f"{name} shape {tuple(t.shape)} does not match the query's {tuple(query.shape)}")
    if query.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"fp32 or bf16 heads expected, got {query.dtype}")
    if d not in (32, 64):
        raise ValueError(f"head dimension {d}: 32 or 64 expected")
    if weight.dim() != 2 or weight.shape[1] != H or weight.shape[0] < 1:
        raise ValueError(f"weight shape {tuple(weight.shape)}: [num_buckets, {H}] expected")
    if buckets.dim() != 1 or buckets.shape[0] % 2 == 0 or not 3 <= buckets.shape[0] <= 2 * MAX_DISTANCE + 1:
        raise ValueError(f"buckets: [2 R + 1] with R from 1 to {MAX_DISTANCE} expected, got {tuple(buckets.shape)}")
    if buckets.dtype != torch.int32:
        raise TypeError("buckets: int32 expected")
    if not -(1 << 29) <= int(offset) <= 1 << 29:
        raise ValueError("offset out of range")
    if key_mask is not None and tuple(key_mask.shape) != (B, Lk):
        raise ValueError(f"key mask shape {tuple(key_mask.shape)}: [{B}, {Lk}] expected")
    if mat is not None:
        if block_size is None or not 32 <= block_size <= 1 << 29 or block_size % 32:
            raise ValueError(f"block_size {block_size}: a multiple of 32 expected with a pattern")
        nb = -(-Lk // block_size)
        if tuple(mat.shape) != (nb, nb):
            raise ValueError(f"pattern shape {tuple(mat.shape)}: [{nb}, {nb}] expected")
        if Lq != Lk or offset != 0:
            raise ValueError("a pattern has as many queries as keys and no offset")
        if score_map:
            raise ValueError("the mean map is of the dense phase, without a pattern")
    if max(B, H, weight.shape[0]) >= 1 << 31 or max(Lq, Lk) > 1 << 29:  # (the library takes them in 32 bits)
        raise ValueError("sizes out of range")
    for t in (query, key, value, weight, buckets, key_mask, mat):
        if t is not None and (not t.is_cuda or t.device != query.device):
            raise RuntimeError("tensors on one GPU expected")
    for t in (key, value, weight):
        if t.dtype != query.dtype:
            raise TypeError("heads and weight of one type expected")


def relative_bias_attention(query, key, value, weight, buckets, key_mask=None, mat=None, block_size=None, offset: int = 0,
                            score_map: bool = False):
    """Attention with the bias ``weight[buckets[...], head]`` on its logits; gradients for query, key, value and weight.

    query [B, H, Lq, d], key and value [B, H, Lk, d]: fp32 or bf16, d 32 or 64, tensors or views (views of projections are read
    in place).  weight [num_buckets, H] of the same type.  buckets: int32 [2 R + 1], see ``relative_position_buckets``.
    key_mask [B, Lk]: keys with a 0 are left out (bool, or any type, compared with 0); a row without keys gives zeros.
    mat [nb, nb] with block_size: pairs in blocks that are 0 have probability 0 and count in the softmax with a logit of 0, as in
    the other sparse modules.  offset: query i stands at position i + offset (the last queries of a sequence: Lk - Lq).
    score_map: also return the mean of the probability maps over batch and heads, fp32 [Lq, Lk], without a gradient.

    An entry of weight that is -infinity (or the type's lowest value) takes its pairs out; a row that loses all of them gives zeros.
    Large finite entries do not serve for that: log2 Z is one fp32 number, and where all of a row's logits are near -1e9 it has no
    room for the sum: the row's gradients come out too large."""
    node = _lib.autograd_node()
    if node is not None and _lib.plain_autograd():  # csrc/operator_nodes.h: the same steps
        try:
            out = node.relative_bias_attention(query, key, value, weight, buckets, key_mask, mat, block_size or 0, offset, score_map)
        except RuntimeError as e:
            if str(e).startswith("spion_bias_"):
                raise _lib.SpionLibraryError(str(e)) from None
            raise
        return tuple(out) if score_map else out[0]
    _check(query, key, value, weight, buckets, key_mask, mat, block_size, offset, score_map)
    if key_mask is not None:
        if key_mask.dtype not in (torch.float32, torch.bool, torch.uint8):
            key_mask = key_mask != 0
        key_mask = key_mask.detach().contiguous()
    if mat is not None:
        mat = mat.detach().to(torch.float32).contiguous()
    if query.numel() == 0 or key.numel() == 0:  # nothing to attend to, or nobody to
        every = torch.ones((), dtype=torch.bool, device=query.device)
        q, *others = (t.masked_fill(every, 0.0) for t in (query, key, value, weight))
        out = q + sum(t.sum() for t in others)
        return (out, query.new_zeros((query.shape[2], key.shape[2]), dtype=torch.float32)) if score_map else out
    return _RelativeBiasFunction.apply(query, key, value, weight, buckets.contiguous(), key_mask, mat, int(block_size or 0),
                                       int(offset), bool(score_map))


class RelativeBiasAttention(nn.Module):
    """Attention core with a learned relative position bias, for either phase of a layer.

    ``config`` keys: head_dim, num_head, block_size (with patterns), relative_buckets (default 32), relative_max_distance
    (default 128).  ``forward(query, key, value, mask, mat=None) -> (out, 0)`` with ``query/key/value [B, H, L, d]``: dense without
    ``mat``, on the block pattern with it; batch and length come with the tensors.  ``mask`` ([B, L], 0 = padding) is used only when
    the module was built with ``key_mask=True``.  With ``emit_score_map`` set, a dense forward leaves the mean of its probability
    maps in ``score_map`` (what ``generate_pattern_*`` read).  ``weight`` [buckets, heads] is fp32; bf16 heads take it rounded."""

    def __init__(self, config, key_mask: bool = False):
        super().__init__()
        self.emb_dim = config["head_dim"]
        self.num_heads = config["num_head"]
        self.block_size = config.get("block_size")
        self.key_mask = bool(key_mask)
        num_buckets = config.get("relative_buckets", 32)
        _lib.core()  # raises when the HIP library has not been built: there is no fallback
        self.weight = nn.Parameter(torch.zeros(num_buckets, self.num_heads))
        self.register_buffer("buckets", relative_position_buckets(num_buckets, config.get("relative_max_distance", 128)),
                             persistent=False)
        self.emit_score_map = False
        self.score_map = None

    def forward(self, query, key, value, mask, mat=None):
        if query.dim() != 4 or query.shape[1] != self.num_heads or query.shape[3] != self.emb_dim:
            raise ValueError(f"query shape {tuple(query.shape)}: {self.num_heads} heads of {self.emb_dim} expected")
        weight = self.weight if self.weight.dtype == query.dtype else self.weight.to(query.dtype)
        emit = self.emit_score_map and mat is None
        out = relative_bias_attention(query, key, value, weight, self.buckets, mask if self.key_mask else None, mat,
                                      self.block_size if mat is not None else None, score_map=emit)
        if emit:
            out, self.score_map = out
        return out, 0
