"""The rows' way to the experts and back, with gradients.

``dispatch_rows`` copies each token's row to the places of its picks in the experts' order, where
``grouped_linear`` finds an expert's rows side by side; ``combine_rows`` adds a token's rows up again, by
weight. ``places`` is that of ``route_experts``. The fused SwiGLU path of ``stack_fused_moe`` does both inside
its kernels; these serve experts of other forms, and experts that are trained. The reference has no
counterpart.

    r = route_experts(logits, k)
    h = grouped_linear(dispatch_rows(x, r.places), w1, r.offsets, activation="swiglu")
    y = combine_rows(grouped_linear(h, w2, r.offsets), r.places, r.weights, residual=residual)
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from ._torch import address, dense, dtype_code, no_tangents, once, raw_stream, records_gradient, rows_of


def _check_places(places, tokens, device):
    if places.dtype != torch.int32 or places.dim() != 2 or not places.is_contiguous():
        raise TypeError("places must be a contiguous int32 matrix [T, k]")
    if places.device != device:
        raise ValueError(f"expected a GPU tensor, places is on {places.device}, the rows on {device}")
    if places.shape[1] == 0:
        raise ValueError("places holds no picks")
    if tokens is not None and places.shape[0] != tokens:
        raise ValueError(f"{tokens} rows of x, places of {places.shape[0]} tokens")


def _check_matrix(name, t):
    if t.dim() != 2 or t.shape[1] == 0:
        raise ValueError(f"{name} must be [rows, H], got {tuple(t.shape)}")
    dtype_code(t.dtype)


def _spread(x, places):
    index = x.device.index
    if index != torch.cuda.current_device():  # kernels are launched on the current device
        with torch.cuda.device(index):
            return _spread(x, places)
    (tokens, k), h = places.shape, x.shape[1]
    xm, xs = rows_of(x)
    rows = x.new_empty((tokens * k, h))
    code = _lib.lib().smx_dispatch_rows(xm.data_ptr(), xs, dtype_code(x.dtype), tokens, h, places.data_ptr(), k,
                                        rows.data_ptr(), raw_stream(index))
    if code:
        _lib.check("smx_dispatch_rows", code)
    return rows


def _gather(rows, places, weights, residual):
    index = rows.device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _gather(rows, places, weights, residual)
    (tokens, k), h = places.shape, rows.shape[1]
    m, stride = rows_of(rows)
    r, rs = (None, 0) if residual is None else rows_of(residual)
    w = dense(weights)
    y = rows.new_empty((tokens, h))
    code = _lib.lib().smx_combine_rows(m.data_ptr(), stride, dtype_code(rows.dtype), tokens, h, places.data_ptr(), k,
                                       address(w), address(r), rs, y.data_ptr(), raw_stream(index))
    if code:
        _lib.check("smx_combine_rows", code)
    return y


def _gather_backward(dy, rows, places, weights, shape, need_rows, need_w):
    index = dy.device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _gather_backward(dy, rows, places, weights, shape, need_rows, need_w)
    (tokens, k), h = places.shape, shape[1]
    d, ds = rows_of(dy)
    m, ms = (None, 0) if rows is None or not need_w else rows_of(rows)
    w = dense(weights)
    drows = dy.new_empty(shape) if need_rows else None
    dw = dy.new_empty((tokens, k), dtype=torch.float32) if need_w else None
    code = _lib.lib().smx_combine_rows_grad(
        d.data_ptr(), ds, address(m), ms, dtype_code(dy.dtype), tokens, h, places.data_ptr(), k, address(w),
        address(drows), address(dw), raw_stream(index))
    if code:
        _lib.check("smx_combine_rows_grad", code)
    return drows, dw


def _gather_once(dy, places):
    return (_gather(dy, places, None, None),)


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, places):
        ctx.save_for_backward(places)
        return _spread(x, places)

    @staticmethod
    def backward(ctx, dy):
        no_tangents("dispatch_rows", dy)
        places, = ctx.saved_tensors
        return *once("dispatch_rows", _gather_once, (dy,), dy, places), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, places, weights, residual):
        ctx.save_for_backward(rows if ctx.needs_input_grad[2] else None, places, weights)
        ctx.shape = rows.shape
        return _gather(rows, places, weights, residual)

    @staticmethod
    def backward(ctx, dy):
        no_tangents("combine_rows", dy)
        rows, places, weights = ctx.saved_tensors
        need_rows, _, need_w, need_r = ctx.needs_input_grad
        drows = dw = None
        if need_rows or need_w:
            drows, dw = once("combine_rows", _gather_backward, (dy, rows, weights), dy, rows, places, weights, ctx.shape,
                             need_rows, need_w)
        return drows, None, dw, dy if need_r else None


def dispatch_rows(x: torch.Tensor, places: torch.Tensor) -> torch.Tensor:
    """The rows of x ``[T, H]``, once per pick, in the experts' order: ``[T k, H]``, row ``places[t, j]`` of it x's row
    t. Rows of picks of nobody (negative places: at ``~places[t, j]``) are zeros. places int32 ``[T, k]``,
    k <= 16, holds each of the T k rows (or its complement) once, as from ``route_experts``; rows that it does not
    hold are left unwritten. Differentiable once, in reverse mode, in x."""
    no_tangents("dispatch_rows", x)
    _check_matrix("x", x)
    _check_places(places, x.shape[0], x.device)
    if not x.is_cuda:
        raise ValueError(f"expected a GPU tensor, got one on {x.device}")
    return _Dispatch.apply(x, places) if records_gradient(x) else _spread(x, places)


def combine_rows(rows: torch.Tensor, places: torch.Tensor, weights: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual[t] + sum over j of weights[t, j] * rows[places[t, j]]``: ``[T, H]``, summed in fp32 and rounded
    once. rows ``[T k, H]`` (fp32, fp16, bf16), weights fp32 ``[T, k]`` (None: 1), residual ``[T, H]`` of the
    rows' type. Picks of nobody (negative places) are left out, whatever their rows hold. Differentiable once, in
    reverse mode, in rows, weights and residual; places holds each row (or its complement) once."""
    no_tangents("combine_rows", rows, weights, residual)
    _check_matrix("rows", rows)
    _check_places(places, None, rows.device)
    tokens, k = places.shape
    if rows.shape[0] != tokens * k:
        raise ValueError(f"places of {tokens * k} picks, {rows.shape[0]} rows")
    if weights is not None:
        if weights.shape != places.shape:
            raise ValueError(f"weights must be {tuple(places.shape)}, got {tuple(weights.shape)}")
        if weights.dtype != torch.float32:
            raise TypeError(f"weights must be fp32, got {weights.dtype}")
    if residual is not None:
        if residual.shape != (tokens, rows.shape[1]):
            raise ValueError(f"residual must be {(tokens, rows.shape[1])}, got {tuple(residual.shape)}")
        if residual.dtype != rows.dtype:
            raise TypeError(f"dtype mismatch: rows are {rows.dtype}, residual {residual.dtype}")
    for name, t in (("weights", weights), ("residual", residual)):
        if t is not None and t.device != rows.device:
            raise ValueError(f"rows are on {rows.device}, {name} on {t.device}")
    if not rows.is_cuda:
        raise ValueError(f"expected a GPU tensor, got one on {rows.device}")
    if records_gradient(rows, weights, residual):
        return _Combine.apply(rows, places, weights, residual)
    return _gather(rows, places, weights, residual)
