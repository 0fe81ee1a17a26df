"""The norms: RMSNorm with the reference's interface, and layer_norm and rms_norm with gradients.

Reference: specmoe/layers/layernorm.py:7-52. ``forward(x, residual=None)``: with a residual,
``residual = x + residual`` and ``x = rmsnorm(residual)`` are written in place and
``(x, residual)`` is returned (sglang's fused_add_rmsnorm, :31); without one, a new
normalized tensor is returned. The arithmetic is the reference's forward_native (:36-52):
fp32 sum, mean of squares, ``x * rsqrt(var + eps) * weight`` rounded once.

RMSNorm and add_rmsnorm_gate serve: they take no part in differentiation. ``layer_norm`` and ``rms_norm``
are the norms of a model that is trained (the reference has none). They write nothing in place, and
normalise the sum as it is kept, rounded to its type, so that their gradients are those of the values the
backward pass reads again.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch
from torch import nn

from .. import _lib
from ._torch import (address, dense, dtype_code, empty_rows, no_tangents, once, ptr, raw_stream, records_gradient,
                     require_gpu, rows_of, stream_of)


def add_rmsnorm_gate(hidden: torch.Tensor, residual: Optional[torch.Tensor],
                     norm_weight: torch.Tensor, eps: float,
                     gate_weight: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Residual add + RMSNorm (+ router gate) in one kernel. Writes the normalized states to
    ``out`` (default: ``hidden``, in place) and the sum to ``residual``; returns the router
    logits ``[T, E]`` when ``gate_weight`` ``[E, H]`` is given."""
    assert hidden.dim() == 2 and hidden.is_contiguous(), "hidden states must be [T, H] contiguous"
    T, H = hidden.shape
    require_gpu(hidden, residual, norm_weight, gate_weight, out)
    for t in (residual, norm_weight, gate_weight, out):
        if t is not None:
            assert t.dtype == hidden.dtype and t.is_contiguous(), "dtype/contiguity mismatch"
    assert norm_weight.numel() == H
    if residual is not None:
        assert residual.shape == hidden.shape
    out = hidden if out is None else out
    logits = None
    E = 0
    if gate_weight is not None:
        E = gate_weight.shape[0]
        assert gate_weight.shape == (E, H)
        logits = torch.empty((T, E), dtype=hidden.dtype, device=hidden.device)
    _lib.call("smx_add_rmsnorm_gate", ptr(hidden), ptr(residual), ptr(out), dtype_code(hidden.dtype),
              T, H, ptr(norm_weight), float(eps), ptr(gate_weight), E, ptr(logits), stream_of(hidden))
    return logits


class RMSNorm(nn.Module):
    def __init__(self, hidden_size: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(hidden_size))
        self.variance_epsilon = eps

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if x.device.type == "cuda":
            return self.forward_cuda(x, residual)
        return self.forward_native(x, residual)

    def forward_cuda(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None
                     ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        shape = x.shape
        x2 = x.view(-1, shape[-1])
        w = self.weight.data
        if w.dtype != x.dtype:
            w = w.to(x.dtype)
        if residual is not None:
            add_rmsnorm_gate(x2, residual.view(-1, shape[-1]), w, self.variance_epsilon)
            return x, residual
        out = torch.empty_like(x2)
        add_rmsnorm_gate(x2, None, w, self.variance_epsilon, out=out)
        return out.view(shape)

    def forward_native(self, *args, **kwargs):
        raise NotImplementedError("this build has no CPU RMSNorm path")


def _check_norm(x, weight, bias, eps, residual):
    """The call's sizes: (dtype code, columns), and the type of the parameters."""
    shape, dtype, device = x.shape, x.dtype, x.device
    if len(shape) < 1 or shape[-1] == 0:
        raise ValueError(f"x must be [..., H], got {tuple(shape)}")
    code = dtype_code(dtype)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    params = dtype
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is None:
            continue
        if t.shape != (shape if t is residual else shape[-1:]):
            raise ValueError(f"{name} must be {tuple(shape if t is residual else shape[-1:])}, got {tuple(t.shape)}")
        if t.device != device:
            raise ValueError(f"x is on {device}, {name} on {t.device}")
        if t.dtype != dtype and (t is residual or t.dtype != torch.float32):
            raise TypeError(f"dtype mismatch: x is {dtype}, {name} {t.dtype}")
        if t is not residual:
            params = t.dtype
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"dtype mismatch: weight is {weight.dtype}, bias {bias.dtype}")
    if not x.is_cuda:
        raise ValueError(f"expected a GPU tensor, got one on {device}")
    return code, shape[-1], params


@functools.lru_cache(maxsize=4096)
def _grad_workspace(*sizes: int) -> int:
    return _lib.lib().smx_norm_grad_workspace_size(*sizes)


def _norm_forward(kind, sizes, x, weight, bias, eps, residual, keep: bool):
    """y, the sum (None without a residual), and the rows' statistics where the gradient needs them."""
    index = x.device.index
    if index != torch.cuda.current_device():  # kernels are launched on the current device
        with torch.cuda.device(index):
            return _norm_forward(kind, sizes, x, weight, bias, eps, residual, keep)
    dtype, h, params = sizes
    xm, xs = rows_of(x)
    rows = xm.numel() // h
    y = empty_rows(x)
    rm = total = stats = rp = tp = sp = None
    rs = 0
    if residual is not None:
        rm, rs = rows_of(residual)
        total = torch.empty_like(y)
        rp, tp = rm.data_ptr(), total.data_ptr()
    if keep:
        stats = x.new_empty(rows if kind == _lib.SMX_NORM_RMS else 2 * rows, dtype=torch.float32)
        sp = stats.data_ptr()
    w, b = dense(weight), dense(bias)
    code = _lib.lib().smx_norm(kind, xm.data_ptr(), xs, rp, rs, dtype, rows, h, address(w), address(b),
                               dtype_code(params), eps, y.data_ptr(), tp, sp, raw_stream(index))
    if code:
        _lib.check("smx_norm", code)
    return y, total, stats


def _norm_backward(kind, sizes, dy, dsum, s, weight, stats, need):
    index = s.device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _norm_backward(kind, sizes, dy, dsum, s, weight, stats, need)
    need_x, need_w, need_b = need
    dtype, h, params = sizes
    if dy is None:  # only the sum was used
        return dsum if need_x else None, *(s.new_zeros(h, dtype=params) if n else None for n in (need_w, need_b))
    sm, ss = rows_of(s)
    dm, ds = rows_of(dy)
    rm, rs = (None, 0) if dsum is None else rows_of(dsum)
    rows = sm.numel() // h
    dx = dw = db = ws = xp = wp = bp = workp = None
    nbytes = 0
    if need_x:
        dx = empty_rows(s)
        xp = dx.data_ptr()
    if need_w:
        dw = s.new_empty(h, dtype=params)
        wp = dw.data_ptr()
    if need_b:
        db = s.new_empty(h, dtype=params)
        bp = db.data_ptr()
    if need_w or need_b:
        nbytes = _grad_workspace(kind, rows, h, dtype)
        ws = stats.new_empty(nbytes // 4)  # (fp32 partial sums)
        workp = ws.data_ptr()
    w = dense(weight)
    code = _lib.lib().smx_norm_grad(kind, dm.data_ptr(), ds, address(rm), rs, sm.data_ptr(), ss, dtype, rows, h, address(w),
                                    dtype_code(params), stats.data_ptr(), xp, wp, bp, workp, nbytes, raw_stream(index))
    if code:
        _lib.check("smx_norm_grad", code)
    return dx, dw, db


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, kind, eps, sizes):
        y, total, stats = _norm_forward(kind, sizes, x, weight, bias, eps, residual, True)
        ctx.save_for_backward(x if total is None else total, weight, stats)
        ctx.how = kind, sizes
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    def backward(ctx, dy, dsum=None):
        no_tangents("a norm", dy, dsum)
        if dy is None and dsum is None:
            return (None,) * 7
        kind, sizes = ctx.how
        s, weight, stats = ctx.saved_tensors  # as autograd hands them back: perhaps not at their old addresses
        x, w, b, r = ctx.needs_input_grad[:4]
        dx, dw, db = once("a norm", _norm_backward, (dy, dsum, s, weight), kind, sizes, dy, dsum, s, weight, stats,
                          (x or r, w, b))
        return dx if x else None, dw, db, dx if r else None, None, None, None


def _norm(kind, x, weight, bias, eps, residual):
    no_tangents("a norm", x, weight, bias, residual)
    eps = float(eps)
    sizes = _check_norm(x, weight, bias, eps, residual)
    if records_gradient(x, weight, bias, residual):
        return _Norm.apply(x, weight, bias, residual, kind, eps, sizes)
    y, total, _ = _norm_forward(kind, sizes, x, weight, bias, eps, residual, False)
    return y if total is None else (y, total)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None
               ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``(s - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (at most 16384 columns), of
    ``s = x``, or with a residual of ``s = x + residual``: then ``(y, s)`` is returned, s as it is kept.

    x and residual ``[..., H]`` in fp32, fp16 or bf16; weight and bias ``[H]`` in x's type or fp32, or None.
    Statistics and sums are fp32, y is rounded once. Differentiable once, in reverse mode, in x, weight,
    bias and residual; the gradients of weight and bias are summed in fp32, in a fixed order."""
    return _norm(_lib.SMX_NORM_LAYER, x, weight, bias, eps, residual)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
             residual: Optional[torch.Tensor] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``s / sqrt(mean(s^2) + eps) * weight``; otherwise as layer_norm."""
    return _norm(_lib.SMX_NORM_RMS, x, weight, None, eps, residual)
