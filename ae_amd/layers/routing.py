"""Routing with gradients: a token's experts, their weights, and the picks' order by expert.

``route_experts`` is to a block that is trained what ``select_experts`` is to one that serves: the same
choices of scores, groups and bias, with the gradient of the logits and with what ``grouped_linear``,
``dispatch_rows`` and ``combine_rows`` need. It serves as well, from one token on. The reference has no
counterpart.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional

import torch

from .. import _lib
from ._torch import dense, dtype_code, empty_rows, no_tangents, once, raw_stream, records_gradient, rows_of


class Routing(NamedTuple):
    weights: torch.Tensor  # fp32 [T, k]: the picks' weights
    ids: torch.Tensor      # int32 [T, k]: their experts, -1 for picks of nobody
    places: torch.Tensor   # int32 [T, k]: where each pick is in the experts' order (~ of it for picks of nobody)
    order: torch.Tensor    # int32 [T k]: the pick (token k + j) at each place (~ of it for picks of nobody)
    offsets: torch.Tensor  # int64 [E + 1]: the bounds of the experts' picks in that order


@functools.lru_cache(maxsize=4096)
def _workspace_size(t: int, e: int, k: int) -> int:
    return _lib.lib().smx_route_workspace_size(t, e, k)


def _check(logits, top_k, scoring, bias, num_groups, top_groups, scale):
    if logits.dim() != 2:
        raise ValueError(f"logits must be [T, E], got {tuple(logits.shape)}")
    dtype_code(logits.dtype)
    e = logits.shape[1]
    if scoring not in _lib.SCORINGS:
        raise ValueError(f"unknown scoring {scoring!r}; expected one of {list(_lib.SCORINGS)}")
    if num_groups < 1 or e % num_groups or not 1 <= top_groups <= num_groups:
        raise ValueError(f"{e} experts in {num_groups} groups, {top_groups} of them selectable")
    if not 1 <= top_k <= e // num_groups * top_groups:
        raise ValueError(f"top_k {top_k} of {e // num_groups * top_groups} selectable experts")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    if bias is not None:
        if bias.shape != (e,):
            raise ValueError(f"bias must be {(e,)}, got {tuple(bias.shape)}")
        if bias.device != logits.device:
            raise ValueError(f"logits are on {logits.device}, bias on {bias.device}")
        if not bias.is_floating_point():
            raise TypeError(f"unsupported dtype {bias.dtype} of bias")
        if bias.requires_grad and torch.is_grad_enabled():
            raise ValueError("bias moves the choice, not the weights: it has no gradient. Pass it detached")
    if not logits.is_cuda:
        raise ValueError(f"expected a GPU tensor, got one on {logits.device}")


def _forward(logits, k, scoring, bias, num_groups, top_groups, renormalize, scale):
    index = logits.device.index
    if index != torch.cuda.current_device():  # kernels are launched on the current device
        with torch.cuda.device(index):
            return _forward(logits, k, scoring, bias, num_groups, top_groups, renormalize, scale)
    t, e = logits.shape
    m, stride = rows_of(logits)
    weights = logits.new_empty((t, k), dtype=torch.float32)
    ids = torch.empty_like(weights, dtype=torch.int32)
    places = torch.empty_like(ids)
    order = ids.new_empty(t * k)
    offsets = ids.new_empty(e + 1, dtype=torch.int64)
    nbytes = _workspace_size(t, e, k)
    ws = workp = biasp = None
    if nbytes:
        ws = ids.new_empty(nbytes // 4)  # (counts)
        workp = ws.data_ptr()
    if bias is not None:
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.to(torch.float32).contiguous()
        biasp = bias.data_ptr()
    code = _lib.lib().smx_route(
        m.data_ptr(), stride, dtype_code(logits.dtype), t, e, k, scoring, biasp, num_groups, top_groups, renormalize,
        scale, weights.data_ptr(), ids.data_ptr(), places.data_ptr(), order.data_ptr(), offsets.data_ptr(), workp, nbytes,
        raw_stream(index))
    if code:
        _lib.check("smx_route", code)
    return weights, ids, places, order, offsets


def _backward(dw, logits, ids, scoring, renormalize, scale):
    index = logits.device.index
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            return _backward(dw, logits, ids, scoring, renormalize, scale)
    t, e = logits.shape
    m, stride = rows_of(logits)
    grad = empty_rows(logits)
    dw = dense(dw)
    code = _lib.lib().smx_route_grad(
        dw.data_ptr(), m.data_ptr(), stride, dtype_code(logits.dtype), t, e, ids.shape[1], scoring, renormalize, scale,
        ids.data_ptr(), grad.data_ptr(), raw_stream(index))
    if code:
        _lib.check("smx_route_grad", code)
    return (grad,)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, scoring, bias, num_groups, top_groups, renormalize, scale):
        out = _forward(logits, k, scoring, bias, num_groups, top_groups, renormalize, scale)
        ctx.save_for_backward(logits, out[1])
        ctx.how = (scoring, renormalize, scale)
        ctx.mark_non_differentiable(*out[1:])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    def backward(ctx, dw, *_):
        no_tangents("route_experts", dw)
        if dw is None:
            return (None,) * 8
        logits, ids = ctx.saved_tensors
        return *once("route_experts", _backward, (dw, logits), dw, logits, ids, *ctx.how), *(None,) * 7


def route_experts(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
                  num_groups: int = 1, top_groups: Optional[int] = None, renormalize: bool = True,
                  scale: float = 1.0) -> Routing:
    """The top_k experts of each token by the router's logits ``[T, E]`` (fp32, fp16, bf16; E <= 1024,
    top_k <= 16).

    Scores are the logits' softmax or sigmoid. A token's experts are those of the largest score + ``bias``
    (``[E]``, the bias that balances the experts' loads; it moves the choice only), in that order, ties to the
    lower expert, compared as exact scores would be. With ``num_groups`` > 1 only the ``top_groups`` best groups of
    consecutive experts are selectable (default: all): by their best expert, or with a bias by their two
    best. Weights are the scores, divided by their sum over the token's picks (``renormalize``), times
    ``scale``. An expert of logit -inf (or bias -inf) is never picked, and a token without enough experts (a padded
    row of -inf throughout) leaves picks of nobody: id -1, weight 0, no row.

    Differentiable once, in reverse mode, in the logits. An expert's load is ``offsets.diff()``."""
    no_tangents("route_experts", logits)
    top_groups = num_groups if top_groups is None else top_groups
    scale = float(scale)
    _check(logits, top_k, scoring, bias, num_groups, top_groups, scale)
    args = (logits, top_k, _lib.SCORINGS[scoring], bias, num_groups, top_groups, int(bool(renormalize)), scale)
    return Routing(*(_Route.apply(*args) if records_gradient(logits) else _forward(*args)))
