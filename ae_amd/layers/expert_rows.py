"""The rows' way to the experts and back, with gradients.

``dispatch_rows`` copies each token's row to the places of its picks in the experts' order, where
``grouped_linear`` finds an expert's rows side by side; ``combine_rows`` adds a token's rows up again, by
weight. ``places`` is that of ``route_experts``. The fused SwiGLU path of ``stack_fused_moe`` does both inside
its kernels; these serve experts of other forms, and experts that are trained. The reference has no
counterpart.

    r = route_experts(logits, k)
    h = grouped_linear(dispatch_rows(x, r.places), w1, r.offsets, activation="swiglu")
    y = combine_rows(grouped_linear(h, w2, r.offsets), r.places, r.weights, residual=residual)

Calls run on the current stream of their tensors' device, without host synchronisation, and can be captured into a graph; a
captured backward pass as fused_linear has it (no autograd graph of the same leaves from outside the capture alive).
Traces (torch.jit.trace, make_fx, torch.export) and torch.func's transforms, which would not see the kernels, are refused.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib


def dispatch_rows(x: torch.Tensor, places: torch.Tensor) -> torch.Tensor:
    """The rows of x ``[T, H]``, once per pick, in the experts' order: ``[T k, H]``, row ``places[t, j]`` of it x's row
    t. Rows of picks of nobody (negative places: at ``~places[t, j]``) are zeros. places int32 ``[T, k]``,
    k <= 16, holds each of the T k rows (or its complement) once, as from ``route_experts``; rows that it does not
    hold are left unwritten. Differentiable once, in reverse mode, in x."""
    return _lib.blocks().dispatch_rows(x, places)


def combine_rows(rows: torch.Tensor, places: torch.Tensor, weights: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual[t] + sum over j of weights[t, j] * rows[places[t, j]]``: ``[T, H]``, summed in fp32 and rounded
    once. rows ``[T k, H]`` (fp32, fp16, bf16), weights fp32 ``[T, k]`` (None: 1), residual ``[T, H]`` of the
    rows' type. Picks of nobody (negative places) are left out, whatever their rows hold. Differentiable once, in
    reverse mode, in rows, weights and residual; places holds each row (or its complement) once."""
    return _lib.blocks().combine_rows(rows, places, weights, residual)
