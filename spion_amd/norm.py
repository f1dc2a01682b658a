"""Root-mean-square norm with the residual's addition, for pre-norm layers around the attention core.

The reference's layer adds the residual in one operation and normalises with nn.LayerNorm in the next
(models/model_transformer.py:55-102).  Here one pass over the rows does both:

    h = x + residual,    y = h / sqrt(mean(h^2) + eps) * weight

* ``rms_norm(x, weight, residual=None, eps=1e-6)`` returns ``y``, or ``(y, h)`` with a residual, with gradients;
* ``rms_norm_fp8(...)`` returns ``y`` as 8-bit floats with a scale for every row, for inference;
* ``RMSNorm(dim)`` is the module.

fp32 and bf16 tensors of any width; ``h`` is rounded to the tensors' type before it is normalised, as if the addition were an
operation of its own; statistics and sums are fp32.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib


class _Call(ctypes.Structure):
    """``spion_rms_norm``."""

    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "residual", "weight", "y", "h", "codes", "scales", "dy", "dh", "dx", "dweight",
                                                "workspace")]
                + [(n, ctypes.c_longlong) for n in ("workspace_floats", "rows", "x_stride", "residual_stride", "dy_stride",
                                                    "dh_stride")]
                + [("width", ctypes.c_int), ("bf16", ctypes.c_int), ("eps", ctypes.c_float)])


def _lib_typed():
    lib = _lib.core()
    if not getattr(lib, "_spion_norm_typed", False):
        for name, res, args in (("spion_rms_norm_workspace", ctypes.c_longlong, [ctypes.c_void_p]),
                                ("spion_rms_norm_forward", ctypes.c_int, [ctypes.c_void_p] * 2),
                                ("spion_rms_norm_backward", ctypes.c_int, [ctypes.c_void_p] * 2)):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
        lib._spion_norm_typed = True
    return lib


def _rows(t):
    """``t`` as [rows, width] with its elements next to each other in a row: a view where its strides allow one."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 and t.stride(0) >= 0 else t.contiguous()


def _run(name, call, device):
    with torch.cuda.device(device):
        _lib.check_call(getattr(_lib_typed(), name)(ctypes.addressof(call), _lib._raw_stream(device.index)) == 0, name)


def _check(x, weight, residual, eps):
    if x.dim() < 1 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError(f"weight shape {tuple(weight.shape)} does not match rows of {tuple(x.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual shape {tuple(residual.shape)} does not match {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"fp32 or bf16 rows expected, got {x.dtype}")
    if x.shape[-1] > 1 << 29:  # (the library takes it in 32 bits)
        raise ValueError("width out of range")
    if not eps >= 0:
        raise ValueError("eps is not negative")
    for t in (x, weight, residual):
        if t is not None and (not t.is_cuda or t.device != x.device):
            raise RuntimeError("tensors on one GPU expected")
        if t is not None and t.dtype != x.dtype:
            raise TypeError("rows and weight of one type expected")


def _forward(x, weight, residual, eps, fp8):
    """(y or codes, scales or None, h or None) in the shape of ``x``."""
    dev = x.device
    out = torch.empty(x.shape, dtype=torch.float8_e4m3fn if fp8 else x.dtype, device=dev)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev) if fp8 else None
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if residual is not None else None
    if x.numel() == 0:
        if fp8:
            scales.fill_(2.0 ** -126)  # rows without elements
        return out, scales, h
    xr, w = _rows(x), weight.contiguous()
    call = _Call(x=xr.data_ptr(), weight=w.data_ptr(), rows=xr.shape[0], width=xr.shape[1], bf16=int(x.dtype == torch.bfloat16),
                 x_stride=xr.stride(0), eps=eps)
    if residual is not None:
        rr = _rows(residual)
        call.residual, call.residual_stride, call.h = rr.data_ptr(), rr.stride(0), h.data_ptr()
    if fp8:
        call.codes, call.scales = out.data_ptr(), scales.data_ptr()
    else:
        call.y = out.data_ptr()
    _run("spion_rms_norm_forward", call, dev)
    return out, scales, h


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, h = _forward(x, weight, residual, eps, False)
        ctx.eps, ctx.residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        _lib.save_for_backward(ctx, x if h is None else h, weight)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, w = _lib.saved_tensors(ctx)
        if dy is None and dh is None:
            return None, None, None, None
        dx, dw = torch.empty(h.shape, dtype=h.dtype, device=h.device), torch.empty(w.shape, dtype=w.dtype, device=h.device)
        if h.numel() == 0:
            return dx, dw.zero_(), dx if ctx.residual else None, None
        if dy is None:  # only the stream was used
            return dh, dw.zero_(), dh, None
        hr, w = _rows(h), w.contiguous()
        call = _Call(x=hr.data_ptr(), weight=w.data_ptr(), rows=hr.shape[0], width=hr.shape[1],
                     bf16=int(h.dtype == torch.bfloat16), x_stride=hr.stride(0), eps=ctx.eps, dx=dx.data_ptr(), dweight=dw.data_ptr())
        g = _rows(dy.to(h.dtype))
        call.dy, call.dy_stride = g.data_ptr(), g.stride(0)
        if dh is not None:
            d = _rows(dh.to(h.dtype))
            call.dh, call.dh_stride = d.data_ptr(), d.stride(0)
        floats = _lib_typed().spion_rms_norm_workspace(ctypes.addressof(call))
        _lib.check_call(floats >= 0, "spion_rms_norm_workspace")
        ws = torch.empty(floats, dtype=torch.float32, device=h.device)
        call.workspace, call.workspace_floats = ws.data_ptr(), floats
        _run("spion_rms_norm_backward", call, h.device)
        return dx, dw, dx if ctx.residual else None, None


class _RMSNormFp8Function(torch.autograd.Function):
    """Without a gradient.  A function all the same: torch.jit.trace records it as one operation (of the calls inside it, only the
    allocations), and forward-mode tangents and functorch transforms meet torch's refusal."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        out = tuple(t for t in _forward(x, weight, residual, eps, True) if t is not None)
        ctx.mark_non_differentiable(*out)
        return out


def _in_node(name, *args):
    """The compiled form (csrc/operator_nodes.h: the same steps), or None where Python's is asked for."""
    node = _lib.autograd_node()
    if node is None or not _lib.plain_autograd():
        return None
    try:
        return getattr(node, name)(*args)
    except RuntimeError as e:
        if str(e).startswith("spion_rms_norm"):
            raise _lib.SpionLibraryError(str(e)) from None
        raise


def rms_norm(x, weight, residual=None, eps: float = 1e-6):
    """``y``, or ``(y, h)`` where there is a residual: see the module's head.  x and residual [..., width], weight [width], of one
    type; gradients for all three."""
    out = _in_node("rms_norm", x, weight, residual, eps)
    if out is not None:
        return out[0] if residual is None else tuple(out)
    _check(x, weight, residual, eps)
    return _RMSNormFunction.apply(x, weight, residual, float(eps))


def rms_norm_fp8(x, weight, residual=None, eps: float = 1e-6):
    """``(codes, scales)``, or ``(codes, scales, h)`` where there is a residual: the norm as 8-bit floats (torch.float8_e4m3fn,
    [..., width]) times a scale for every row (fp32 [...]), max|y| / 448 and at least 2^-126.  For inference: it has no
    gradient and refuses tensors that ask for one."""
    out = _in_node("rms_norm_fp8", x, weight, residual, eps)
    if out is not None:
        return tuple(out)
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    return _RMSNormFp8Function.apply(x, weight, residual, float(eps))


class RMSNorm(nn.Module):
    """``forward(x, residual=None)`` is ``rms_norm`` with a weight of its own (initially ones), ``quantized(x, residual=None)``
    ``rms_norm_fp8``.  The weight is fp32; bf16 rows take it rounded."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        _lib.core()  # raises when the HIP library has not been built: there is no fallback
        self.weight = nn.Parameter(torch.ones(dim))

    def _weight(self, x):
        return self.weight if self.weight.dtype == x.dtype else self.weight.to(x.dtype)

    def forward(self, x, residual=None):
        return rms_norm(x, self._weight(x), residual, self.eps)

    def quantized(self, x, residual=None):
        return rms_norm_fp8(x, self._weight(x), residual, self.eps)
