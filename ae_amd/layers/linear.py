"""Matrix products with bias, activation and residual in one kernel, dense and grouped by expert.

``fused_linear`` is ``residual + act(x W^T + b)``; ``grouped_linear`` is the same with a weight
and a bias per group of consecutive rows, as rows sorted by expert have them
(``moe_align_block_size(topk_ids, 1, E)`` gives that order). Both are differentiable in x, weight,
bias and residual. They cover what the fused SwiGLU page of ``stack_fused_moe`` does not: experts
with biases or another activation, experts that are trained, dense MLPs and projections. The
reference has no counterpart: it leaves such products to torch.

Contract: everything runs on the current stream of x's device, without host synchronisation, so
the calls can be captured into a graph. A backward pass can be captured too, but not while an
autograd graph of the same leaves built outside the capture is still alive (torch's gradient
accumulation would join the capture from another stream): drop its outputs first.
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from ._torch import dtype_code, require_gpu, workspace


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t as a matrix of rows with adjacent elements, and their distance (a copy where needed)."""
    n = t.shape[-1]
    m = t if t.dim() == 2 else t.reshape(-1, n)
    if (m.stride(1) != 1 and n != 1) or (m.stride(0) < n and m.shape[0] > 1):
        m = m.contiguous()
    return m, (m.stride(0) if m.shape[0] > 1 else n)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _on(device: torch.device):
    """The device as the current one (kernels are launched on the current device)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _weight_strides(weight: torch.Tensor) -> tuple[int, int]:
    """Distances of a weight's rows and of the group's weights."""
    nw, k = weight.shape[-2:]
    row = weight.stride(-2) if nw > 1 else k
    group = 0
    if weight.dim() == 3:
        group = weight.stride(0) if weight.shape[0] > 1 else nw * row
    return row, group


class _Call:
    """Checked arguments of a product."""

    def __init__(self, x, weight, bias, activation, residual, offsets, slots, out):
        grouped = offsets is not None
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}; expected one of "
                             f"{[a for a in _lib.ACTIVATIONS if a]} or None")
        self.act = _lib.ACTIVATIONS[activation]
        self.dtype = dtype_code(x.dtype)
        if x.dim() < 1 or (grouped and x.dim() != 2):
            raise ValueError(f"x must be [{'rows' if grouped else '...'}, K], got {tuple(x.shape)}")
        if weight.dim() != (3 if grouped else 2):
            raise ValueError(f"weight must be [{'G, ' if grouped else ''}Nw, K], got {tuple(weight.shape)}")
        nw, k = weight.shape[-2:]
        if k != x.shape[-1]:
            raise ValueError(f"x has {x.shape[-1]} columns, weight {k}")
        if nw == 0 or k == 0:
            raise ValueError(f"empty weight {tuple(weight.shape)}")
        if self.act == _lib.ACTIVATIONS["swiglu"]:
            if nw % 2:
                raise ValueError(f"swiglu takes gate and up rows: {nw} weight rows are odd")
            self.n = nw // 2
        else:
            self.n = nw
        row, group = _weight_strides(weight)
        if (k > 1 and weight.stride(-1) != 1) or row < k:
            raise ValueError(f"weight rows must be apart, with adjacent elements: strides {weight.stride()}")
        shape = (*x.shape[:-1], self.n)
        for name, t, want in (("bias", bias, tuple(weight.shape[:-1])), ("residual", residual, shape),
                              ("out", out, shape)):
            if t is not None and tuple(t.shape) != want:
                raise ValueError(f"{name} must be {want}, got {tuple(t.shape)}")
        require_gpu(x, weight, bias, residual, offsets, slots, out)
        for t in (weight, bias, residual, out):
            if t is not None and t.dtype != x.dtype:
                raise TypeError(f"dtype mismatch: x is {x.dtype}, got {t.dtype}")
        for t in (weight, bias, residual, offsets, slots, out):
            if t is not None and t.device != x.device:
                raise ValueError(f"x is on {x.device}, got a tensor on {t.device}")
        self.groups = 0
        if grouped:
            if offsets.dtype != torch.int64 or offsets.dim() != 1 or not offsets.is_contiguous():
                raise TypeError("group_offsets must be a contiguous int64 vector")
            self.groups = offsets.numel() - 1
            if self.groups < 1:
                raise ValueError("group_offsets must hold at least two bounds")
            if slots is None and weight.shape[0] != self.groups:
                raise ValueError(f"{self.groups} groups, {weight.shape[0]} weights")
            if slots is not None:
                if slots.dtype != torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
                    raise TypeError("weight_slots must be a contiguous int64 vector")
                if slots.numel() != self.groups:
                    raise ValueError(f"{self.groups} groups, {slots.numel()} slots")
                if weight.shape[0] == 0:
                    raise ValueError("no weights")
        self.nw, self.k, self.shape = nw, k, shape
        self.wargs = (weight.data_ptr(), row)
        self.gargs = (group, weight.shape[0]) if grouped else ()
        self.offsets, self.slots = offsets, slots

    def workspace(self, query: str, rows: int, device: torch.device):
        n = getattr(_lib.lib(), query)(rows, self.k, self.n, self.groups, self.act, self.dtype)
        return (workspace(n, device) if n else None), n

    def forward(self, x, bias, residual, out, keep: bool):
        """y, and the fp32 pre-activations where the gradient needs them (kept in 32 bits: their rounding would
        weigh as much in the gradients as that of the gradients themselves)."""
        with _on(x.device):
            xm, xs = _rows(x)
            rows = xm.shape[0]
            fresh = out is None
            y = torch.empty(self.shape, dtype=x.dtype, device=x.device) if fresh else out
            ym = y if y.dim() == 2 else y.view(-1, self.n)
            ys = ym.stride(0) if rows > 1 else self.n
            rm, rs = (None, 0) if residual is None else _rows(residual)
            z = None
            if keep and self.act:
                z = torch.empty((rows, self.nw), dtype=torch.float32, device=x.device)
            ws, nbytes = self.workspace("smx_linear_workspace_size", rows, x.device)
            stream = torch.cuda.current_stream(x.device).cuda_stream
            head = (xm.data_ptr(), xs, self.dtype, rows, self.k, *self.wargs)
            tail = (ym.data_ptr(), ys, _ptr(z), _ptr(ws), nbytes, stream)
            if self.groups:
                _lib.call("smx_grouped_linear", *head, *self.gargs, self.n, _ptr(bias), self.act, _ptr(rm), rs,
                          self.offsets.data_ptr(), self.groups, _ptr(self.slots), int(fresh), *tail)
            else:
                _lib.call("smx_linear", *head, self.n, _ptr(bias), self.act, _ptr(rm), rs, *tail)
        return y, z

    def backward(self, dy, saved, need_x: bool, need_w: bool, need_b: bool):
        x, weight, z, offsets, slots = saved  # as autograd hands them back: perhaps not at their old addresses
        row, group = _weight_strides(weight)
        with _on(x.device):
            dm, ds = _rows(dy)
            xm, xs = _rows(x)
            rows = xm.shape[0]
            lead = (self.groups,) if self.groups else ()
            new = dict(dtype=x.dtype, device=x.device)
            dx = torch.empty(x.shape, **new) if need_x else None
            dw = torch.empty((*lead, self.nw, self.k), **new) if need_w else None
            db = torch.empty((*lead, self.nw), **new) if need_b else None
            ws, nbytes = self.workspace("smx_linear_grad_workspace_size", rows, x.device)
            stream = torch.cuda.current_stream(x.device).cuda_stream
            head = (dm.data_ptr(), ds, _ptr(z), xm.data_ptr(), xs, self.dtype, rows, self.k,
                    weight.data_ptr(), row)
            tail = (_ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), nbytes, stream)
            if self.groups:
                _lib.call("smx_grouped_linear_grad", *head, group, weight.shape[0], self.n, self.act,
                          offsets.data_ptr(), self.groups, _ptr(slots), *tail)
            else:
                _lib.call("smx_linear_grad", *head, self.n, self.act, *tail)
        return dx, dw, db


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, call):
        needs = ctx.needs_input_grad
        y, z = call.forward(x, bias, residual, None, any(needs[:3]))
        ctx.save_for_backward(x, weight, z, call.offsets, call.slots)
        call.offsets = call.slots = None
        ctx.call = call
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        grads = (None, None, None)
        if need_x or need_w or need_b:
            grads = ctx.call.backward(dy, ctx.saved_tensors, need_x, need_w, need_b)
        return (*grads, dy if need_r else None, None)


def _run(x, weight, bias, activation, residual, offsets, slots, out):
    call = _Call(x, weight, bias, activation, residual, offsets, slots, out)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        if out is not None:
            raise ValueError("out= takes no part in differentiation: call without it, or under torch.no_grad()")
        if slots is not None and (weight.requires_grad or (bias is not None and bias.requires_grad)):
            raise ValueError("weights reached through weight_slots have no gradient: several groups may share a "
                             "slot. Pass them detached, or index the weights first")
        return _Product.apply(x, weight, bias, residual, call)
    if out is not None and (out.stride(-1) != 1 and out.shape[-1] > 1 or not _viewable(out)):
        raise ValueError(f"out rows must be apart, with adjacent elements: strides {out.stride()}")
    return call.forward(x, bias, residual, out, False)[0]


def _viewable(out: torch.Tensor) -> bool:
    if out.dim() == 2:
        return out.shape[0] <= 1 or out.stride(0) >= out.shape[1]
    return out.is_contiguous()


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + act(x @ weight.T + bias)`` in one call.

    x ``[..., K]``, weight ``[Nw, K]`` (rows may be apart, elements adjacent), bias ``[Nw]``,
    residual ``[..., N]``; all of one type (fp32, fp16, bf16), summed in fp32, the result rounded
    once. ``activation``: None, "relu", "gelu" (erf), "gelu_tanh", "silu", or "swiglu", whose
    weight holds N gate rows and N up rows: ``silu(gate) * up``. Otherwise N = Nw. ``out`` receives
    the result where no gradient is recorded; it may be the residual. Differentiable once in x, weight,
    bias and residual."""
    return _run(x, weight, bias, activation, residual, None, None, out)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, group_offsets: torch.Tensor,
                   bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                   residual: Optional[torch.Tensor] = None,
                   weight_slots: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fused_linear with a weight per group of rows: rows ``group_offsets[g]`` to
    ``group_offsets[g + 1]`` of x ``[rows, K]`` use ``weight[g]`` and ``bias[g]``.

    weight ``[G, Nw, K]``, bias ``[G, Nw]``, group_offsets int64 ``[G + 1]`` on the GPU, not
    decreasing; groups may be empty, and their sizes need not be known on the host. With
    ``weight_slots`` (int64 ``[G]`` on the GPU) group g uses ``weight[weight_slots[g]]`` and
    ``bias[weight_slots[g]]``: the slot map of an expert pool, e.g. with the pages of
    stack_fused_moe ``pool[:, :2*I*H].unflatten(1, (2*I, H))`` (gate and up, for "swiglu") and
    ``pool[:, 2*I*H:].unflatten(1, (H, I))`` (down); such weights have no gradient.

    Rows outside every group, and rows of a group whose slot is not in the pool, have no product: their result is
    the residual's row, or zeros (with ``out`` they are left as they were), and x's gradient is zero there."""
    if group_offsets is None:
        raise TypeError("group_offsets must be a contiguous int64 vector")
    return _run(x, weight, bias, activation, residual, group_offsets, weight_slots, out)
