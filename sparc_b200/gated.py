"""Gated linear recurrence h_t = a_t h_{t-1} + sqrt(1 - a_t^2) s(write_t) x_t with
a_t = exp(-exp(nu_log) s(retention_t)), s the logistic function: per channel a retention rate (as
SPARCMixer's nu_log) that every token's retention gate scales, and an input that its write gate
scales and sqrt(1 - a_t^2) keeps at the state's own variance. The scans of `real.py` take a and
b ready-made; here the gates are part of the kernels, and so are the gradients through them.

``gated_scan`` is the training and prefill form, ``gated_scan_step`` the one-token form for
decoding. x and the two gates are float32 or bfloat16 (one dtype), [B, T, D] with adjacent
channels in any batch and token strides: the three may be columns of one projection, and are read
in place. nu_log and the states are float32, and so is the arithmetic.

``segment_pos`` ([B, T] integers, as SPARCMixer's) restarts the recurrence at every token whose
position is 0 (packed sequences): nothing of the earlier segment is kept, not its infinities or
NaN either. The token's write keeps its factor sqrt(1 - a_t^2).
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_POS_DTYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8, torch.bool)


def _check(what, x, retention_gate, write_gate, nu_log, state, segment_pos, dim):
    """Shape checks first (ValueError), then dtypes (TypeError), then the device (no CPU path)."""
    if x.dim() != dim or retention_gate.shape != x.shape or write_gate.shape != x.shape:
        raise ValueError(f"{what} expects x, retention_gate and write_gate of one shape "
                         f"{'[batch, length, channels]' if dim == 3 else '[batch, channels]'}")
    B, D = x.shape[0], x.shape[-1]
    if nu_log.shape != (D,):
        raise ValueError("nu_log must have shape [channels]")
    if state is not None and state.shape != (B, D):
        raise ValueError("state must have shape [batch, channels]")
    if segment_pos is not None and segment_pos.shape != x.shape[:-1]:
        raise ValueError(f"segment_pos must have shape {tuple(x.shape[:-1])}")
    if 0 in x.shape:
        raise ValueError(f"{what} expects at least one row, token and channel, got {tuple(x.shape)}")
    _lib.dtype_code(x.dtype)
    if retention_gate.dtype != x.dtype or write_gate.dtype != x.dtype:
        raise TypeError(f"{what} expects x and its gates in one dtype, got {x.dtype}, {retention_gate.dtype}, "
                        f"{write_gate.dtype}")
    if segment_pos is not None and segment_pos.dtype not in _POS_DTYPES:
        raise TypeError(f"segment_pos must be an integer tensor, got {segment_pos.dtype}")
    for name, t in (("x", x), ("retention_gate", retention_gate), ("write_gate", write_gate), ("nu_log", nu_log),
                    ("state", state), ("segment_pos", segment_pos)):
        if t is not None:
            _lib.require_cuda(t, name)
            if t.device != x.device:
                raise RuntimeError(f"sparc_b200: {name} is on {t.device}, x on {x.device}")


def _rows(t):
    """t as the kernels read it: any strides but adjacent channels (copied where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _pos(segment_pos):
    """(dense positions, their size in bytes); only zero or not matters to the kernels."""
    return (None, 0) if segment_pos is None else (segment_pos.contiguous(), segment_pos.element_size())


def _f32(t):
    return None if t is None else t.detach().to(torch.float32).contiguous()


def _forward(x, r, w, nu_log, h0, pos, want_carry, want_last):
    """The kernel call on detached tensors: (y, last, carry)."""
    L = _lib.lib()
    B, T, D = x.shape
    dev = x.device
    y = torch.empty((B, T, D), dtype=x.dtype, device=dev)
    last = torch.empty((B, D), dtype=torch.float32, device=dev) if want_last else None
    carry = (torch.empty((B, L.sparc_gated_carry_chunks(T), D), dtype=torch.float32, device=dev) if want_carry
             else None)
    pos, pos_bytes = pos
    a = _lib.GatedFwdArgs(
        x.data_ptr(), r.data_ptr(), w.data_ptr(), nu_log.data_ptr(), _lib.ptr(h0), _lib.ptr(pos), pos_bytes,
        y.data_ptr(), _lib.ptr(last), _lib.ptr(carry), x.stride(0), x.stride(1), r.stride(0), r.stride(1),
        w.stride(0), w.stride(1), B, T, D, _lib.dtype_code(x.dtype))
    with _lib.on_device(dev):
        _lib.check(L.sparc_gated_scan_forward(ctypes.byref(a), _lib.stream_handle(dev)), "sparc_gated_scan_forward")
    return y, last, carry


class _GatedScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, retention_gate, write_gate, nu_log, state, segment_pos, want_last):
        x, r, w = _rows(x), _rows(retention_gate), _rows(write_gate)
        nu, h0, pos = _f32(nu_log), _f32(state), _pos(segment_pos)
        y, last, carry = _forward(x, r, w, nu, h0, pos, True, want_last)
        ctx.save_for_backward(x, r, w, nu, pos[0], carry)
        ctx.pos_bytes = pos[1]
        ctx.nu_dtype = nu_log.dtype
        ctx.state_dtype = None if state is None else state.dtype
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return (None,) * 7
        L = _lib.lib()
        x, r, w, nu, pos, carry = ctx.saved_tensors
        B, T, D = x.shape
        dev = x.device
        dy = torch.zeros((B, T, D), dtype=x.dtype, device=dev) if dy is None else _rows(dy.to(x.dtype))
        dlast = _f32(dlast)
        dx, dr, dw = (torch.empty((B, T, D), dtype=x.dtype, device=dev) for _ in range(3))
        dnu = torch.empty((D,), dtype=torch.float32, device=dev)
        dh0 = torch.empty((B, D), dtype=torch.float32, device=dev) if ctx.state_dtype is not None else None
        nbytes = L.sparc_gated_workspace_bytes(B, T, D)
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
        a = _lib.GatedBwdArgs(
            x.data_ptr(), r.data_ptr(), w.data_ptr(), nu.data_ptr(), dy.data_ptr(), carry.data_ptr(),
            _lib.ptr(dlast), _lib.ptr(pos), ctx.pos_bytes, dx.data_ptr(), dr.data_ptr(), dw.data_ptr(),
            dnu.data_ptr(), _lib.ptr(dh0), ws.data_ptr(), nbytes, x.stride(0), x.stride(1), r.stride(0), r.stride(1),
            w.stride(0), w.stride(1), dy.stride(0), dy.stride(1), B, T, D, _lib.dtype_code(x.dtype))
        with _lib.on_device(dev):
            _lib.check(L.sparc_gated_scan_backward(ctypes.byref(a), _lib.stream_handle(dev)),
                       "sparc_gated_scan_backward")
        return (dx, dr, dw, dnu.to(ctx.nu_dtype), None if dh0 is None else dh0.to(ctx.state_dtype), None, None)


def gated_scan(x: torch.Tensor, retention_gate: torch.Tensor, write_gate: torch.Tensor, nu_log: torch.Tensor,
               state: torch.Tensor | None = None, segment_pos: torch.Tensor | None = None,
               return_last: bool = False):
    """The recurrence over [B, T, D]: y [B, T, D] in x's dtype, or with `return_last` (y, last)
    with the state after the last token, float32 [B, D]. Starts from `state` ([B, D]) or zero.
    Differentiable (once) with respect to x, the gates, nu_log and the state, through y and last."""
    _check("gated scan", x, retention_gate, write_gate, nu_log, state, segment_pos, 3)
    if torch.is_grad_enabled() and (x.requires_grad or retention_gate.requires_grad or write_gate.requires_grad or
                                    nu_log.requires_grad or (state is not None and state.requires_grad)):
        y, last = _GatedScanFunction.apply(x, retention_gate, write_gate, nu_log, state, segment_pos, return_last)
    else:  # no gradient can be asked for: no carries are kept
        y, last, _ = _forward(_rows(x), _rows(retention_gate), _rows(write_gate), _f32(nu_log), _f32(state),
                              _pos(segment_pos), False, return_last)
    return (y, last) if return_last else y


@torch.no_grad()
def gated_scan_step(x: torch.Tensor, retention_gate: torch.Tensor, write_gate: torch.Tensor, nu_log: torch.Tensor,
                    state: torch.Tensor, segment_pos: torch.Tensor | None = None):
    """One token: x and the gates [B, D], the state [B, D]; returns (y [B, D] in x's dtype, the new
    state, float32). Without autograd, as ``sparc_decode_step``; a length-1 ``gated_scan`` with the
    state is the differentiable form. `segment_pos` ([B]) restarts the rows whose position is 0."""
    _check("gated scan step", x, retention_gate, write_gate, nu_log, state, segment_pos, 2)
    L = _lib.lib()
    x, r, w = _rows(x), _rows(retention_gate), _rows(write_gate)
    nu, h0 = _f32(nu_log), _f32(state)
    pos, pos_bytes = _pos(segment_pos)
    B, D = x.shape
    dev = x.device
    y = torch.empty((B, D), dtype=x.dtype, device=dev)
    new = torch.empty((B, D), dtype=torch.float32, device=dev)
    a = _lib.GatedStepArgs(x.data_ptr(), r.data_ptr(), w.data_ptr(), nu.data_ptr(), h0.data_ptr(), _lib.ptr(pos),
                           pos_bytes, y.data_ptr(), new.data_ptr(), x.stride(0), r.stride(0), w.stride(0), B, D,
                           _lib.dtype_code(x.dtype))
    with _lib.on_device(dev):
        _lib.check(L.sparc_gated_step(ctypes.byref(a), _lib.stream_handle(dev)), "sparc_gated_step")
    return y, new
