"""A router's choice of experts, tokens sorted by expert, and the experts' rows added
back to their tokens.

What lies between a router's scores, which ``balance_loss`` keeps balanced, and its
layer's output::

    routes = route_tokens(router_logits, RouteConfig(top_k=2), mask=attention_mask)
    order = expert_order(routes.experts, num_experts)
    rows = to_experts(x, order)                    # [tokens * 2, W], expert by expert
    ends = order.offsets.tolist()
    for e in range(num_experts):
        out[ends[e]:ends[e + 1]] = expert[e](rows[ends[e]:ends[e + 1]])
    y = from_experts(out, order, routes.weights)   # [..., W]

A token takes the ``top_k`` experts with the largest scores, the lowest first where
they are equal (NaN is above all), as ``balance_loss`` counts them.  Their weights are
the softmax over them, or with ``normalize=False`` over all experts.  A masked token
takes none: its experts are -1, its weights 0, its scores are not read, and its output
is 0.  Experts at -inf have weight 0.

A choice is dropped by a ``place`` of -1, for instance those beyond an expert's capacity
(without masked tokens, whose -1 is no index)::

    late = order.place - order.offsets[routes.experts] >= capacity
    order = order._replace(place=order.place.masked_fill(late, -1))

Rows without a choice, those behind the last (``order.offsets[-1]``) among them, are 0
in ``to_experts``; in ``from_experts`` they are not read (they may be NaN) and get a
gradient of 0.  Copies are exact; sums are float32, rounded once.

The calls and their backward nodes are C++ (``csrc/ace_autograd.cpp``).  They have no
forward-mode and no second derivative, and ``torch.func`` transforms do not know them;
``torch.compile`` breaks its graph at them.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from pydantic import BaseModel, ConfigDict, Field

from ace_kernels import _lib
from ace_kernels.balance import MAX_EXPERTS, MAX_TOP_K

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_EXPERT_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class RouteConfig(BaseModel):
    """Options of the choice of experts.

    top_k:     experts that a token takes (at most 16, and at most E).
    normalize: weights are the softmax over a token's own experts, which add up
               to 1; False: over all experts.
    """

    model_config = ConfigDict(frozen=True, extra="forbid")

    top_k: int = Field(ge=1, le=MAX_TOP_K)
    normalize: bool = True


class Routes(NamedTuple):
    """``experts`` (int64) and ``weights`` (float32, differentiable), both ``[...,
    top_k]``, the largest score's first."""

    experts: torch.Tensor
    weights: torch.Tensor


class ExpertOrder(NamedTuple):
    """``offsets`` ``[E + 1]``: expert e has the rows ``offsets[e]`` to ``offsets[e + 1]``;
    ``source`` ``[slots]``: which choice (token * top_k + j) each row is of, -1 behind the
    last; ``place`` ``[..., top_k]``: the row of each choice, -1 where there is none.  All
    int64."""

    offsets: torch.Tensor
    source: torch.Tensor
    place: torch.Tensor


def _check_route(logits: torch.Tensor, config: RouteConfig, mask: Optional[torch.Tensor]) -> None:
    if logits.dim() < 1:
        raise ValueError(f"logits must be [..., experts], got {tuple(logits.shape)}")
    experts = logits.shape[-1]
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"route_tokens takes 1 to {MAX_EXPERTS} experts, got {experts}")
    if config.top_k > experts:
        raise ValueError(f"top_k is {config.top_k}, but there are {experts} experts")
    if logits.device.type != "cuda":
        raise ValueError(f"route_tokens needs HIP ('cuda') tensors, got {logits.device}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if mask is not None:
        if mask.shape != logits.shape[:-1]:
            raise ValueError(f"mask must be {tuple(logits.shape[:-1])}, one per token, got {tuple(mask.shape)}")
        if mask.dtype != torch.bool:
            raise TypeError(f"mask must be bool (True: routed), got {mask.dtype}")
        if mask.device != logits.device:
            raise ValueError(f"mask is on {mask.device}, logits on {logits.device}")


def route_tokens(logits: torch.Tensor, config: RouteConfig, mask: Optional[torch.Tensor] = None) -> Routes:
    """The ``top_k`` experts of each token and their weights, from router scores ``[...,
    E]`` (float32, bfloat16 or float16).  ``mask`` ``[...]`` (bool): tokens that are
    routed.  Differentiable once in ``logits``, through ``weights``; for that the scores
    are kept, as they were, only with ``normalize=False``."""
    _check_route(logits, config, mask)
    return Routes(*_lib.autograd().route_tokens(logits, mask, config.top_k, config.normalize))


def expert_order(experts: torch.Tensor, num_experts: int) -> ExpertOrder:
    """The order of choices ``experts`` ``[..., top_k]`` (integers) by expert, those of one
    expert in their own order.  A number outside ``[0, num_experts)`` is no choice."""
    if experts.dim() < 1 or experts.shape[-1] < 1:
        raise ValueError(f"experts must be [..., top_k], got {tuple(experts.shape)}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"expert_order takes 1 to {MAX_EXPERTS} experts, got {num_experts}")
    if experts.device.type != "cuda":
        raise ValueError(f"expert_order needs HIP ('cuda') tensors, got {experts.device}")
    if experts.dtype not in _EXPERT_TYPES:
        raise TypeError(f"experts must be integers, got {experts.dtype}")
    return ExpertOrder(*_lib.autograd().expert_order(experts, num_experts))


def _check_rows(what: str, rows: torch.Tensor, order: ExpertOrder) -> None:
    _, source, place = order
    if rows.device.type != "cuda":
        raise ValueError(f"{what} needs HIP ('cuda') tensors, got {rows.device}")
    if rows.dtype not in _DTYPES:
        raise TypeError(f"{what} takes float32, bfloat16 or float16 rows, got {rows.dtype}")
    if source.dtype != torch.int64 or place.dtype != torch.int64:
        raise TypeError(f"the order must be int64, as expert_order gives it, got {source.dtype} and {place.dtype}")
    if source.device != rows.device or place.device != rows.device:
        raise ValueError(f"the rows are on {rows.device}, the order on {source.device} and {place.device}")
    if place.dim() < 1 or place.shape[-1] < 1 or source.shape != (place.numel(),):
        raise ValueError("the order must be expert_order's: source [slots] and place [..., top_k], got "
                         f"{tuple(source.shape)} and {tuple(place.shape)}")


def to_experts(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """Rows of tokens ``x`` ``[..., W]`` in expert order, ``[slots, W]``: each token's row at
    its ``top_k`` places, 0 where nothing is.  Differentiable once in ``x``."""
    _check_rows("to_experts", x, order)
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[:-1] != order.place.shape[:-1]:
        raise ValueError(f"x must be {(*order.place.shape[:-1], 'W')}, a row per token of the order, got {tuple(x.shape)}")
    return _lib.autograd().to_experts(x, order.source, order.place)


def from_experts(rows: torch.Tensor, order: ExpertOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each token's rows, of ``[slots, W]`` in expert order, added up with ``weights`` ``[...,
    top_k]`` (None: 1): ``[..., W]``.  Differentiable once in ``rows`` and ``weights``."""
    _check_rows("from_experts", rows, order)
    if rows.dim() != 2 or rows.shape[0] != order.place.numel() or rows.shape[1] < 1:
        raise ValueError(f"rows must be {(order.place.numel(), 'W')}, one per slot of the order, got {tuple(rows.shape)}")
    if weights is not None:
        if weights.shape != order.place.shape:
            raise ValueError(f"weights must be {tuple(order.place.shape)}, got {tuple(weights.shape)}")
        if weights.device != rows.device:
            raise ValueError(f"weights is on {weights.device}, rows on {rows.device}")
        if weights.dtype not in _DTYPES:
            raise TypeError(f"weights must be float32, bfloat16 or float16, got {weights.dtype}")
        if weights.dtype != torch.float32:
            weights = weights.float()
    return _lib.autograd().from_experts(rows, order.source, order.place, weights)
