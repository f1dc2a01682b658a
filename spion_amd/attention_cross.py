"""Attention of queries to an encoder's states of another length, and the layer around it.

The reference attends within one sequence (models/attention.py:79-103).  A decoder's tokens, a few pooling or answer tokens, or
another modality's, attend to the states that such an encoder leaves:

    out_i = sum_j softmax_j(q_i . k_j / sqrt(d)) v_j        over the keys j whose mask is not 0

* ``cross_attention(query, key, value, key_mask=None)`` is the operator, with gradients for query, key and value; several heads of
  queries may share a head of keys.
* ``CrossAttention(config)`` is the layer: projections, core, output projection, and on request the layer norm ahead of it.  Its
  ``keys_values(states)`` are computed once and kept by a program that answers token by token, and ``attend`` goes on from there.

fp32 and bf16 tensors, head dimension 32, 64 or 128; softmax and sums in fp32; the probabilities are never written to memory.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .attention import plain_projections
from .relative_bias import _Heads, _heads


class _Call(ctypes.Structure):
    """``spion_cross_attention``."""

    _fields_ = ([(n, _Heads) for n in ("Q", "K", "V", "Out", "dO", "dQ", "dK", "dV")]
                + [(n, ctypes.c_void_p) for n in ("key_mask", "Lse", "workspace")] + [("workspace_floats", ctypes.c_longlong)]
                + [(n, ctypes.c_int) for n in ("batch", "heads", "key_heads", "q_len", "k_len", "head_dim", "bf16", "mask_bytes")])


def _lib_typed():
    lib = _lib.core()
    if not getattr(lib, "_spion_cross_typed", False):
        for name, res, args in (("spion_cross_workspace", ctypes.c_longlong, [ctypes.c_void_p, ctypes.c_int]),
                                ("spion_cross_attention_forward", ctypes.c_int, [ctypes.c_void_p] * 2),
                                ("spion_cross_attention_backward", ctypes.c_int, [ctypes.c_void_p] * 2)):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
        lib._spion_cross_typed = True
    return lib


def _fits(t, together):
    """Whether the kernels read ``t`` in place (strides and address of 16 bytes, rows up to 2^24 bytes apart); ``together`` heads of it, within
    2^31 bytes, are reached from one address."""
    sb, sh, sl, sf = t.stride()
    e = t.element_size()
    if sf != 1 or t.data_ptr() % 16 or any(s < 0 or s * e % 16 for s in (sb, sh, sl)) or not t.shape[3] <= sl <= (1 << 24) // e:
        return False
    return ((together - 1) * sh + (t.shape[2] - 1) * sl + t.shape[3]) * e < 1 << 31


def _readable(t, together=1):
    """``t`` as the kernels read it: itself, or a contiguous copy where its strides or address are not theirs."""
    if _fits(t, together):
        return t
    c = t.contiguous()
    return c if _fits(c, together) else t.clone(memory_format=torch.contiguous_format)


def _empty_like_heads(t):
    """Uninitialised heads in the memory order of ``t``: [B, L, H, d] where the heads of a row lie next to each other, as a
    projection leaves them, and the kernels take that."""
    B, H, L, d = t.shape
    if t.stride(1) < t.stride(2) and H * d * t.element_size() <= 1 << 24 and L * H * d < 1 << 29:
        return torch.empty((B, L, H, d), dtype=t.dtype, device=t.device).transpose(1, 2)
    return torch.empty((B, H, L, d), dtype=t.dtype, device=t.device)


def _paired_views(k, v):
    """True when k, v ([B, G, L, d] views) are the two slices of one [B, L, 2, G, d] buffer, in this order."""
    B, G, L, d = k.shape
    strides = (L * 2 * G * d, d, 2 * G * d, 1)
    return k.stride() == strides and v.stride() == strides and v.data_ptr() - k.data_ptr() == G * d * k.element_size()


def _call_of(q, k, v, out, lse, key_mask):
    B, H, Lq, d = q.shape
    c = _Call(Q=_heads(q), K=_heads(k), V=_heads(v), Out=_heads(out), Lse=lse.data_ptr(), batch=B, heads=H, key_heads=k.shape[1],
              q_len=Lq, k_len=k.shape[2], head_dim=d, bf16=int(q.dtype == torch.bfloat16))
    if key_mask is not None:
        c.key_mask, c.mask_bytes = key_mask.data_ptr(), key_mask.element_size()
    return c


def _run(name, call, device):
    lib = _lib_typed()
    backward = name.endswith("backward")
    with torch.cuda.device(device):
        n = lib.spion_cross_workspace(ctypes.addressof(call), int(backward))
        _lib.check_call(n >= 0, "spion_cross_workspace")
        ws = torch.empty(n, dtype=torch.float32, device=device)
        call.workspace, call.workspace_floats = ws.data_ptr() if n else None, n
        _lib.check_call(getattr(lib, name)(ctypes.addressof(call), _lib._raw_stream(device.index)) == 0, name)


class _CrossAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, key_mask):
        q, k, v = _readable(query, query.shape[1] // key.shape[1]), _readable(key), _readable(value)
        out = _empty_like_heads(query)
        lse = torch.empty((query.shape[0] * query.shape[1], query.shape[2]), dtype=torch.float32, device=query.device)
        _run("spion_cross_attention_forward", _call_of(q, k, v, out, lse, key_mask), query.device)
        ctx.masked = key_mask is not None
        _lib.save_for_backward(ctx, q, k, v, out, lse, *([key_mask] if ctx.masked else []))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        saved = _lib.saved_tensors(ctx)
        each = saved[0].shape[1] // saved[1].shape[1]
        q, k, v, out = _readable(saved[0], each), _readable(saved[1]), _readable(saved[2]), _readable(saved[3], each)
        go = _readable(grad_output if grad_output.dtype == q.dtype else grad_output.to(q.dtype), each)
        dq = _empty_like_heads(q)
        if _paired_views(k, v):  # slices of one projection: the gradients likewise
            B, G, L, d = k.shape
            both = torch.empty((B, L, 2, G, d), dtype=k.dtype, device=k.device)
            dk, dv = (both[:, :, i].transpose(1, 2) for i in range(2))
        else:
            dk, dv = _empty_like_heads(k), _empty_like_heads(v)
        call = _call_of(q, k, v, out, saved[4].contiguous(), saved[5].contiguous() if ctx.masked else None)
        call.dO, call.dQ, call.dK, call.dV = (_heads(t) for t in (go, dq, dk, dv))
        _run("spion_cross_attention_backward", call, q.device)
        return dq, dk, dv, None


def _check(query, key, value, key_mask):
    """The kernels take sizes, types and devices as they are told: anything else would be read past its end."""
    if query.dim() != 4 or key.dim() != 4:
        raise ValueError("heads [B, H, L, d] expected")
    B, H, Lq, d = query.shape
    G, Lk = key.shape[1:3]
    if key.shape[0] != B or key.shape[3] != d:
        raise ValueError(f"key shape {tuple(key.shape)} does not match the query's {tuple(query.shape)}")
    if value.shape != key.shape:
        raise ValueError(f"value shape {tuple(value.shape)} does not match the key's {tuple(key.shape)}")
    if (G == 0) != (H == 0) or (G and H % G):
        raise ValueError(f"{H} heads over {G} heads of keys: a multiple expected")
    if query.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"fp32 or bf16 heads expected, got {query.dtype}")
    if d not in (32, 64, 128):
        raise ValueError(f"head dimension {d}: 32, 64 or 128 expected")
    if key_mask is not None and tuple(key_mask.shape) != (B, Lk):
        raise ValueError(f"key mask shape {tuple(key_mask.shape)}: [{B}, {Lk}] expected")
    if max(B, H) >= 1 << 31 or Lk > 1 << 29 or (G and H // G * Lq > 1 << 29):  # (the library takes them in 32 bits)
        raise ValueError("sizes out of range")
    for t in (query, key, value, key_mask):
        if t is not None and (not t.is_cuda or t.device != query.device):
            raise RuntimeError("tensors on one GPU expected")
    for t in (key, value):
        if t.dtype != query.dtype:
            raise TypeError("heads of one type expected")


def cross_attention(query, key, value, key_mask=None):
    """Attention of query [B, H, Lq, d] to key and value [B, G, Lk, d]; gradients for all three.

    fp32 or bf16, d 32, 64 or 128, lengths up to 2^29 (the header has the limits of a launch), tensors or views (views of projections, and
    expanded ones, are read in place).  H is a multiple of G: heads g H/G .. (g + 1) H/G - 1 of the query share head g of key and value.  key_mask [B, Lk]: keys with a 0 are
    left out, whatever they hold (bool, or any type, compared with 0); a row without keys gives zeros.  Infinities among fp32
    operands that take part, and values of 2^127 and more, give NaN."""
    node = _lib.autograd_node()
    if node is not None and _lib.plain_autograd():  # csrc/operator_nodes.h: the same steps
        try:
            return node.cross_attention(query, key, value, key_mask)
        except RuntimeError as e:
            if str(e).startswith("spion_cross_"):
                raise _lib.SpionLibraryError(str(e)) from None
            raise
    _check(query, key, value, key_mask)
    if key_mask is not None:
        if key_mask.dtype not in (torch.float32, torch.bool, torch.uint8):
            key_mask = key_mask != 0
        key_mask = key_mask.detach().contiguous()
    if query.numel() == 0 or key.numel() == 0:  # nothing to attend to, or nobody to
        every = torch.ones((), dtype=torch.bool, device=query.device)
        q, *others = (t.masked_fill(every, 0.0) for t in (query, key, value))
        return q + sum(t.sum() for t in others)
    return _CrossAttentionFunction.apply(query, key, value, key_mask)


class _FusedKV(torch.autograd.Function):
    """The projections of keys and values as one GEMM: states [B, L, dim] times the stacked weights gives one [B, L, 2, G, d] buffer
    whose slices are the heads.  The core reads them in place and hands back gradients that are slices of one buffer again, so the
    backward is one GEMM for the states and one for the stacked weights, without a copy."""

    @staticmethod
    def forward(ctx, states, wk, wv, bk, bv, G, d):
        B, L, dim = states.shape
        w = torch.cat((wk, wv), 0)
        X2 = states.reshape(B * L, dim)
        kv = torch.addmm(torch.cat((bk, bv), 0), X2, w.t()).view(B, L, 2, G, d)
        ctx.save_for_backward(X2, w)
        ctx.dims = (B, G, L, d, dim)
        return tuple(kv[:, :, i].transpose(1, 2) for i in range(2))

    @staticmethod
    @once_differentiable
    def backward(ctx, dk, dv):
        X2, w = ctx.saved_tensors
        B, G, L, d, dim = ctx.dims
        n = G * d
        if _paired_views(dk, dv):
            g2 = torch.as_strided(dk, (B * L, 2 * n), (2 * n, 1))
        else:
            g2 = torch.stack([g.transpose(1, 2) for g in (dk, dv)], 2).reshape(B * L, 2 * n)
        needs = ctx.needs_input_grad
        dX = (g2 @ w).view(B, L, dim) if needs[0] else None
        dW = (g2.t() @ X2).split(n) if needs[1] or needs[2] else (None, None)
        db = g2.sum(0).split(n) if needs[3] or needs[4] else (None, None)
        return dX, *dW, *db, None, None


class CrossAttention(nn.Module):
    """Attention layer of a sequence X [B, Lq, dim] over an encoder's states [B, Lk, states_dim].

    ``config`` keys: transformer_dim, head_dim, num_head; num_key_head (default num_head: every head has keys of its own), states_dim
    (default transformer_dim), layer_norm (True, or the eps: X is normalised first).

    ``forward(X, states, mask=None)`` -> [B, Lq, dim]; mask [B, Lk], 0 = padding.  A program that answers token by token keeps
    ``keys_values(states)`` and calls ``attend(X, keys_values, mask)``."""

    def __init__(self, config):
        super().__init__()
        self.dim = config["transformer_dim"]
        self.head_dim = config["head_dim"]
        self.num_head = config["num_head"]
        self.num_key_head = config.get("num_key_head", self.num_head)
        if self.num_key_head < 1 or self.num_head % self.num_key_head:
            raise ValueError(f"num_head {self.num_head}: a multiple of num_key_head {self.num_key_head} expected")
        if self.head_dim not in (32, 64, 128):
            raise ValueError(f"head_dim {self.head_dim}: 32, 64 or 128 expected")
        _lib.core()  # raises when the HIP library has not been built: there is no fallback
        states_dim = config.get("states_dim", self.dim)
        self.W_q = nn.Linear(self.dim, self.num_head * self.head_dim)
        self.W_k = nn.Linear(states_dim, self.num_key_head * self.head_dim)
        self.W_v = nn.Linear(states_dim, self.num_key_head * self.head_dim)
        self.ff = nn.Linear(self.num_head * self.head_dim, self.dim)
        self.norm = None
        if config.get("layer_norm"):
            from .norm import LayerNorm
            eps = config["layer_norm"]
            self.norm = LayerNorm(self.dim) if eps is True else LayerNorm(self.dim, eps)

    def _split(self, X, heads):
        return X.reshape(X.shape[0], X.shape[1], heads, self.head_dim).transpose(1, 2)

    def keys_values(self, states):
        """(key, value) [B, num_key_head, Lk, head_dim] of an encoder's states: one product where the projections are linear layers as they
        are, else what the modules give."""
        if plain_projections(self.W_k, self.W_v) and states.dtype == self.W_k.weight.dtype == self.W_v.weight.dtype \
                and not torch.is_autocast_enabled():
            return _FusedKV.apply(states, self.W_k.weight, self.W_v.weight, self.W_k.bias, self.W_v.bias, self.num_key_head, self.head_dim)
        return self._split(self.W_k(states), self.num_key_head), self._split(self.W_v(states), self.num_key_head)

    def attend(self, X, keys_values, mask=None):
        if self.norm is not None:  # (fp16 rows, as autocast leaves them, in fp32: what follows casts for itself)
            X = self.norm(X.float() if X.dtype == torch.float16 else X)
        q = self._split(self.W_q(X), self.num_head)
        heads = (q, *keys_values)
        if any(t.dtype == torch.float16 for t in heads):
            heads = tuple(t.float() for t in heads)
        # kept on the other side of autocast: the queries, which are the shorter, come to the type of the keys, and the output goes back
        with torch.autocast(device_type=X.device.type, enabled=False):
            out = cross_attention(heads[0].to(heads[1].dtype), *heads[1:], mask).to(q.dtype)
        return self.ff(out.transpose(1, 2).reshape(X.shape[0], X.shape[1], self.num_head * self.head_dim))

    def forward(self, X, states, mask=None):
        return self.attend(X, self.keys_values(states), mask)
