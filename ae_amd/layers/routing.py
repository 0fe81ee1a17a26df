"""Routing with gradients: a token's experts, their weights, and the picks' order by expert.

``route_experts`` is to a block that is trained what ``select_experts`` is to one that serves: the same
choices of scores, groups and bias, with the gradient of the logits and with what ``grouped_linear``,
``dispatch_rows`` and ``combine_rows`` need. It serves as well, from one token on. The reference has no
counterpart.

Calls run on the current stream of their tensors' device, without host synchronisation, and can be captured into a graph; a
captured backward pass as fused_linear has it (no autograd graph of the same leaves from outside the capture alive).
Traces (torch.jit.trace, make_fx, torch.export) and torch.func's transforms, which would not see the kernels, are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib


class Routing(NamedTuple):
    weights: torch.Tensor  # fp32 [T, k]: the picks' weights
    ids: torch.Tensor      # int32 [T, k]: their experts, -1 for picks of nobody
    places: torch.Tensor   # int32 [T, k]: where each pick is in the experts' order (~ of it for picks of nobody)
    order: torch.Tensor    # int32 [T k]: the pick (token k + j) at each place (~ of it for picks of nobody)
    offsets: torch.Tensor  # int64 [E + 1]: the bounds of the experts' picks in that order


def route_experts(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
                  num_groups: int = 1, top_groups: Optional[int] = None, renormalize: bool = True,
                  scale: float = 1.0) -> Routing:
    """The top_k experts of each token by the router's logits ``[T, E]`` (fp32, fp16, bf16; E <= 1024,
    top_k <= 16).

    Scores are the logits' softmax or sigmoid. A token's experts are those of the largest score + ``bias``
    (``[E]``, read in fp32, the bias that balances the experts' loads; it moves the choice only), in that order, ties to the
    lower expert, compared as exact scores would be. With ``num_groups`` > 1 only the ``top_groups`` best groups of
    consecutive experts are selectable (default: all): by their best expert, or with a bias by their two
    best. Weights are the scores, divided by their sum over the token's picks (``renormalize``), times
    ``scale``. An expert of logit -inf (or bias -inf) is never picked, and a token without enough experts (a padded
    row of -inf throughout) leaves picks of nobody: id -1, weight 0, no row.

    Differentiable once, in reverse mode, in the logits. An expert's load is ``offsets.diff()``."""
    return Routing._make(_lib.blocks().route_experts(logits, top_k, scoring, bias, num_groups, top_groups, renormalize,
                                                     scale))
