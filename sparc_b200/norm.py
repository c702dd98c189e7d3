"""Layer norm over the last dimension, y = (x - mean) (var + eps)^(-1/2) weight + bias, forward and
backward with the weight's and bias's gradients, on the kernels of csrc/layer_norm.cu: the norm
the reference's networks put before each layer (sparc-impl/sparc/networks/sequence_classifier.py),
next to the RMSNorm of `stack.py`, whose stack takes either (``norm="layer"``).

x is float32 or bfloat16 with any leading dimensions (rows whose columns are adjacent are read in
place, others copied first); the statistics, the sums and the parameters are float32.
"""
from __future__ import annotations

import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib


def _check(x, weight, bias, eps):
    """Shape checks first (ValueError), then dtypes (TypeError), then the device (no CPU path)."""
    if x.dim() < 1 or weight.shape != x.shape[-1:]:
        raise ValueError("layer norm expects x [..., width] and weight [width]")
    if bias is not None and bias.shape != weight.shape:
        raise ValueError("layer norm expects bias [width]")
    if x.shape[-1] == 0:
        raise ValueError("layer norm expects at least one column")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    _lib.dtype_code(x.dtype)
    for name, t in (("x", x), ("weight", weight), ("bias", bias)):
        if t is not None:
            _lib.require_cuda(t, name)
            if t.device != x.device:
                raise RuntimeError(f"sparc_b200: {name} is on {t.device}, x on {x.device}")


def _rows(t):
    """t as [rows, width] with adjacent columns (a view where its strides allow one)."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _f32(t):
    return None if t is None else t.detach().to(torch.float32).contiguous()


def _forward(x, weight, bias, eps, shape, want_stats):
    L = _lib.lib()
    R, W = x.shape
    dev = x.device
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    stats = torch.empty((2, R), dtype=torch.float32, device=dev) if want_stats else None
    if R > 0:
        a = _lib.LayerNormFwdArgs(
            x.data_ptr(), weight.data_ptr(), _lib.ptr(bias), y.data_ptr(), _lib.ptr(stats),
            None if stats is None else stats.data_ptr() + 4 * R, x.stride(0), R, W, eps, _lib.dtype_code(x.dtype))
        with _lib.on_device(dev):
            _lib.check(L.sparc_layer_norm_forward(ctypes.byref(a), _lib.stream_handle(dev)),
                       "sparc_layer_norm_forward")
    return y, stats


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        rows, w = _rows(x), _f32(weight)
        y, stats = _forward(rows, w, _f32(bias), eps, x.shape, True)
        ctx.save_for_backward(rows, w, stats)
        ctx.dtypes = (weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        L = _lib.lib()
        x, w, stats = ctx.saved_tensors
        R, W = x.shape
        dev = x.device
        _, need_w, need_b, _ = ctx.needs_input_grad
        dx = torch.empty(dy.shape, dtype=x.dtype, device=dev)
        dw = torch.empty((W,), dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty((W,), dtype=torch.float32, device=dev) if need_b else None
        if R > 0:
            d = _rows(dy.to(x.dtype))
            nbytes = L.sparc_layer_norm_workspace_bytes(R, W) if need_w or need_b else 0
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None
            a = _lib.LayerNormBwdArgs(
                x.data_ptr(), d.data_ptr(), w.data_ptr(), stats.data_ptr(), stats.data_ptr() + 4 * R, dx.data_ptr(),
                _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes, x.stride(0), d.stride(0), R, W,
                _lib.dtype_code(x.dtype))
            with _lib.on_device(dev):
                _lib.check(L.sparc_layer_norm_backward(ctypes.byref(a), _lib.stream_handle(dev)),
                           "sparc_layer_norm_backward")
        else:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        return (dx, None if dw is None else dw.to(ctx.dtypes[0]), None if db is None else db.to(ctx.dtypes[1]), None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over x's last dimension, in x's dtype; differentiable (once) with respect to x,
    the weight and the bias."""
    _check(x, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNormFunction.apply(x, weight, bias, float(eps))
    return _forward(_rows(x), _f32(weight), _f32(bias), float(eps), x.shape, False)[0]


class LayerNorm(nn.Module):
    """Layer norm over the last dimension (parameters: weight, ones, and bias, zeros, unless bias
    is False), as torch.nn.LayerNorm's state dict has them."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
