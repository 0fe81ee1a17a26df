"""Matrix products with bias, activation and residual in one kernel, dense and grouped by expert.

``fused_linear`` is ``residual + act(x W^T + b)``; ``grouped_linear`` is the same with a weight
and a bias per group of consecutive rows, as rows sorted by expert have them
(``moe_align_block_size(topk_ids, 1, E)`` gives that order). Both are differentiable (reverse mode) in x,
weight, bias and residual. They cover what the fused SwiGLU page of ``stack_fused_moe`` does not: experts
with biases or another activation, experts that are trained, dense MLPs and projections. The
reference has no counterpart: it leaves such products to torch.

Contract: everything runs on the current stream of x's device, without host synchronisation, so
the calls can be captured into a graph. A backward pass can be captured too, but not while an
autograd graph of the same leaves built outside the capture is still alive (torch's gradient
accumulation would join the capture from another stream): drop its outputs first. Traces (torch.jit.trace, make_fx,
torch.export), which would not see the kernels, are refused.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib
from ._torch import dtype_code, workspace


_ACTIVATIONS = _lib.ACTIVATIONS
_SWIGLU = _ACTIVATIONS["swiglu"]
_raw_stream = torch._C._cuda_getCurrentRawStream  # of a device index: the hipStream_t itself
_jit_trace, _modes, _mode = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack, torch._C._get_dispatch_mode
_TRACES = tuple(torch._C._TorchDispatchModeKey.__members__.values())  # (of make_fx, fake and functional tensors)


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t as a matrix of rows with adjacent elements, and their distance (a copy where needed)."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    m = t if t.dim() == 2 else t.reshape(-1, n)
    if (m.stride(1) != 1 and n != 1) or (m.stride(0) < n and m.shape[0] > 1):
        m = m.contiguous()
    return m, (m.stride(0) if m.shape[0] > 1 else n)


@functools.lru_cache(maxsize=4096)
def _workspace_size(query: str, *sizes: int) -> int:
    return getattr(_lib.lib(), query)(*sizes)


def _workspace(query: str, device: torch.device, *sizes: int) -> tuple[Optional[torch.Tensor], Optional[int], int]:
    """Scratch of a call from torch's caching allocator: the tensor, its address and its bytes."""
    n = _workspace_size(query, *sizes)
    if n == 0:
        return None, None, 0
    ws = workspace(n, device)
    return ws, ws.data_ptr(), n


def _weight_strides(weight: torch.Tensor) -> tuple[int, int]:
    """Distances of a weight's rows and of the groups' weights."""
    if weight.is_contiguous():
        k = weight.shape[-1]
        return k, (weight.shape[-2] * k if weight.dim() == 3 else 0)
    nw, k = weight.shape[-2:]
    row = weight.stride(-2) if nw > 1 else k
    if (k > 1 and weight.stride(-1) != 1) or row < k:
        raise ValueError(f"weight rows must be apart, with adjacent elements: strides {weight.stride()}")
    group = 0
    if weight.dim() == 3:
        group = weight.stride(0) if weight.shape[0] > 1 else nw * row
    return row, group


def _check(x, weight, bias, activation, residual, offsets, slots, out):
    """The call's sizes: (dtype code, activation code, K, N, weight rows, groups, y's shape), and the
    weight's strides."""
    try:
        act = _ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"unknown activation {activation!r}; expected one of "
                         f"{[a for a in _ACTIVATIONS if a]} or None") from None
    dtype = dtype_code(x.dtype)
    grouped = offsets is not None
    xshape, wshape = x.shape, weight.shape
    if len(xshape) < 1 or (grouped and len(xshape) != 2):
        raise ValueError(f"x must be [{'rows' if grouped else '...'}, K], got {tuple(xshape)}")
    if len(wshape) != (3 if grouped else 2):
        raise ValueError(f"weight must be [{'G, ' if grouped else ''}Nw, K], got {tuple(wshape)}")
    k, nw = xshape[-1], wshape[-2]
    if k != wshape[-1]:
        raise ValueError(f"x has {k} columns, weight {wshape[-1]}")
    if nw == 0 or k == 0:
        raise ValueError(f"empty weight {tuple(wshape)}")
    n = nw
    if act == _SWIGLU:
        if nw % 2:
            raise ValueError(f"swiglu takes gate and up rows: {nw} weight rows are odd")
        n = nw // 2
    shape = (*xshape[:-1], n)
    strides = _weight_strides(weight)
    device = x.device
    for name, t, want in (("weight", weight, None), ("bias", bias, wshape[:-1]), ("residual", residual, shape),
                          ("out", out, shape)):
        if t is None:
            continue
        if want is not None and t.shape != want:
            raise ValueError(f"{name} must be {tuple(want)}, got {tuple(t.shape)}")
        if t.dtype != x.dtype:
            raise TypeError(f"dtype mismatch: x is {x.dtype}, {name} {t.dtype}")
        if t.device != device:
            raise ValueError(f"x is on {device}, {name} on {t.device}")
    if not x.is_cuda:
        raise ValueError(f"expected a GPU tensor, got one on {device}")
    groups = 0
    if grouped:
        for name, t in (("group_offsets", offsets), ("weight_slots", slots)):
            if t is None:
                continue
            if t.dtype != torch.int64 or t.dim() != 1 or not t.is_contiguous():
                raise TypeError(f"{name} must be a contiguous int64 vector")
            if t.device != device:
                raise ValueError(f"expected a GPU tensor, {name} is on {t.device}, x on {device}")
        groups = offsets.shape[0] - 1
        if groups < 1:
            raise ValueError("group_offsets must hold at least two bounds")
        if slots is None and wshape[0] != groups:
            raise ValueError(f"{groups} groups, {wshape[0]} weights")
        if slots is not None and slots.shape[0] != groups:
            raise ValueError(f"{groups} groups, {slots.shape[0]} slots")
        if wshape[0] == 0:
            raise ValueError("no weights")
    return (dtype, act, k, n, nw, groups, shape), strides


def _forward(sizes, strides, x, weight, bias, residual, offsets, slots, out, keep: bool):
    """y, and the fp32 pre-activations where the gradient needs them (kept in 32 bits: their rounding would
    weigh as much in the gradients as that of the gradients themselves)."""
    dtype, act, k, n, nw, groups, shape = sizes
    device = x.device
    if device.index != torch.cuda.current_device():  # kernels are launched on the current device
        with torch.cuda.device(device):
            return _forward(sizes, strides, x, weight, bias, residual, offsets, slots, out, keep)
    row, group = strides
    xm, xs = _rows(x)
    rows = xm.numel() // k
    if out is None:
        y = torch.empty(shape, dtype=x.dtype, device=device)
        ys = n
    else:
        y = out
        ys = out.stride(0) if out.dim() == 2 and rows > 1 else n
    rm = rs = z = None
    if residual is not None:
        rm, rs = _rows(residual)
    if keep and act:
        z = torch.empty((rows, nw), dtype=torch.float32, device=device)
    ws, wp, nbytes = _workspace("smx_linear_workspace_size", device, rows, k, n, groups, act, dtype)
    head = (xm.data_ptr(), xs, dtype, rows, k, weight.data_ptr(), row)
    tail = (y.data_ptr(), ys, None if z is None else z.data_ptr(), wp, nbytes, _raw_stream(device.index))
    bm = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    bp = None if bm is None else bm.data_ptr()
    rp = None if rm is None else rm.data_ptr()
    if groups:
        code = _lib.lib().smx_grouped_linear(
            *head, group, weight.shape[0], n, bp, act, rp, rs or 0, offsets.data_ptr(), groups,
            None if slots is None else slots.data_ptr(), out is None, *tail)
    else:
        code = _lib.lib().smx_linear(*head, n, bp, act, rp, rs or 0, *tail)
    if code:
        _lib.check("smx_grouped_linear" if groups else "smx_linear", code)
    return y, z


def _backward(sizes, dy, saved, need_x: bool, need_w: bool, need_b: bool):
    dtype, act, k, n, nw, groups, _ = sizes
    x, weight, z, offsets, slots = saved  # as autograd hands them back: perhaps not at their old addresses
    device = x.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _backward(sizes, dy, saved, need_x, need_w, need_b)
    row, group = _weight_strides(weight)
    dm, ds = _rows(dy)
    xm, xs = _rows(x)
    rows = xm.numel() // k
    dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_x else None
    dw = torch.empty((groups, nw, k) if groups else (nw, k), dtype=x.dtype, device=device) if need_w else None
    db = torch.empty((groups, nw) if groups else (nw,), dtype=x.dtype, device=device) if need_b else None
    ws, wp, nbytes = _workspace("smx_linear_grad_workspace_size", device, rows, k, n, groups, act, dtype)
    head = (dm.data_ptr(), ds, None if z is None else z.data_ptr(), xm.data_ptr(), xs, dtype, rows, k,
            weight.data_ptr(), row)
    tail = (*(None if t is None else t.data_ptr() for t in (dx, dw, db)), wp, nbytes, _raw_stream(device.index))
    if groups:
        code = _lib.lib().smx_grouped_linear_grad(
            *head, group, weight.shape[0], n, act, offsets.data_ptr(), groups,
            None if slots is None else slots.data_ptr(), *tail)
    else:
        code = _lib.lib().smx_linear_grad(*head, n, act, *tail)
    if code:
        _lib.check("smx_grouped_linear_grad" if groups else "smx_linear_grad", code)
    return dx, dw, db


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, offsets, slots, sizes, strides):
        y, z = _forward(sizes, strides, x, weight, bias, residual, offsets, slots, None,
                        any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, weight, z, offsets, slots)
        ctx.sizes = sizes
        return y

    @staticmethod
    def backward(ctx, dy):
        if not torch.is_grad_enabled():
            return _gradients(ctx, dy)
        # a graph of the gradients themselves is recorded: they depend on dy, x and the weight in a way that it cannot
        # differentiate, and says so if it comes to that
        with torch.no_grad():
            grads = _gradients(ctx, dy)
        deps = (dy, *ctx.saved_tensors[:2])
        return (*(None if g is None else _Once.apply(g, *deps) for g in grads[:3]), *grads[3:])


class _Once(torch.autograd.Function):
    @staticmethod
    def forward(ctx, grad, *deps):
        return grad

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("fused_linear and grouped_linear are differentiable once")


def _gradients(ctx, dy):
    _check_plain(dy)
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    grads = (None, None, None)
    if need_x or need_w or need_b:
        grads = _backward(ctx.sizes, dy, ctx.saved_tensors, need_x, need_w, need_b)
    return (*grads, dy if need_r else None, None, None, None, None)


def _check_plain(*tensors) -> None:
    """Refuses traces, which would hold an empty result without its kernel, and forward-mode duals, whose tangents the
    kernels would drop."""
    if _jit_trace() is not None or (_modes() and any(_mode(key) is not None for key in _TRACES)):
        raise RuntimeError("fused_linear and grouped_linear cannot be traced")
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("fused_linear and grouped_linear have no forward-mode derivative")


def _run(x, weight, bias, activation, residual, offsets, slots, out):
    _check_plain(x, weight, bias, residual, out)
    sizes, strides = _check(x, weight, bias, activation, residual, offsets, slots, out)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        if out is not None:
            raise ValueError("out= takes no part in differentiation: call without it, or under torch.no_grad()")
        if slots is not None and (weight.requires_grad or (bias is not None and bias.requires_grad)):
            raise ValueError("weights reached through weight_slots have no gradient: several groups may share a "
                             "slot. Pass them detached, or index the weights first")
        return _Product.apply(x, weight, bias, residual, offsets, slots, sizes, strides)
    if out is not None:
        _check_out(out, residual, (x, weight, bias, offsets, slots))
        torch.autograd.graph.increment_version(out)  # a backward pass that has saved its old values says so
    return _forward(sizes, strides, x, weight, bias, residual, offsets, slots, out, False)[0]


def _check_out(out, residual, others):
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out= takes no part in differentiation: it may not require a gradient")
    if not out.is_contiguous():
        if out.dim() != 2 or (out.shape[1] > 1 and out.stride(1) != 1) or (
                out.shape[0] > 1 and out.stride(0) < out.shape[1]):
            raise ValueError(f"out rows must be apart, with adjacent elements: strides {out.stride()}")
    if residual is not None and (residual.data_ptr() != out.data_ptr() or residual.stride() != out.stride()):
        others = (*others, residual)
    if any(t is not None and _overlap(out, t) for t in others):
        raise ValueError("out may be the residual, but not overlap other operands")


def _span(t: torch.Tensor) -> tuple[int, int]:
    """The first byte of t's elements, and the byte behind the last."""
    first = t.data_ptr()
    return first, first + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _overlap(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether they share bytes. Of columns of one matrix (rows of the same pitch) only the columns count."""
    if out.numel() == 0 or t.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(out), _span(t)
    if a1 <= b0 or b1 <= a0:
        return False
    if out.dim() != 2 or t.dim() != 2 or out.dtype != t.dtype or out.stride(0) != t.stride(0) or t.stride(1) != 1:
        return True
    pitch, es = out.stride(0), out.element_size()
    if pitch < out.shape[1] or pitch < t.shape[1] or (b0 - a0) % es:
        return True
    d = (b0 - a0) // es % pitch  # t's first column, from out's
    return d < out.shape[1] or d + t.shape[1] > pitch


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + act(x @ weight.T + bias)`` in one call.

    x ``[..., K]``, weight ``[Nw, K]`` (rows may be apart, elements adjacent), bias ``[Nw]``,
    residual ``[..., N]``; all of one type (fp32, fp16, bf16), summed in fp32, the result rounded
    once. ``activation``: None, "relu", "gelu" (erf), "gelu_tanh", "silu", or "swiglu", whose
    weight holds N gate rows and N up rows: ``silu(gate) * up``. Otherwise N = Nw. ``out`` receives
    the result where no gradient is recorded; it may be the residual, but not overlap another
    operand. Differentiable once, in reverse mode, in x, weight, bias and residual."""
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
