"""The balance loss of an expert router, with the experts' token counts.

A router scores every token against E experts and the token takes the ``top_k``
largest; the balance loss pulls the experts' shares of the tokens together::

    out = balance_loss(router_logits, BalanceConfig(top_k=2), mask=attention_mask)
    (task_loss + 0.01 * out.loss).backward()
    out.counts  # tokens that take each expert

With p the softmax of a token's scores, n_e the counted tokens that take expert e
and M the counted tokens, the loss is ``E sum_e (n_e / (top_k M)) mean_t p_te``: 1
where all experts are taken alike.  The counts are constants to the gradient, as
they are in the definition.  Equal scores go to the lowest expert.

Leading dimensions are groups with a loss of their own: ``[layers, tokens, E]`` is
every layer's router of a step, ``[batch, tokens, E]`` a balance per sequence.  A
group without counted tokens has loss 0 and gradient 0.

The call and its backward node are C++ (``csrc/ace_autograd.cpp``).  They have no
forward-mode and no second derivative, and ``torch.func`` transforms do not know them;
``torch.compile`` breaks its graph at them.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Literal, NamedTuple, Optional

import torch
from pydantic import BaseModel, ConfigDict, Field

from ace_kernels import _lib
from ace_kernels.common import tickets
from ace_kernels.impls.hip_mi355x import _stream

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_REDUCTIONS = {"mean": _lib.RED_MEAN, "sum": _lib.RED_SUM, "none": _lib.RED_NONE}
MAX_EXPERTS = 512
MAX_TOP_K = 16


class BalanceConfig(BaseModel):
    """Options of the balance loss.

    top_k:     experts that a token takes (at most 16, and at most E).
    reduction: over the groups; "none" returns each group's loss.
    """

    model_config = ConfigDict(frozen=True, extra="forbid")

    top_k: int = Field(ge=1, le=MAX_TOP_K)
    reduction: Literal["mean", "sum", "none"] = "mean"


class BalanceLoss(NamedTuple):
    """``loss`` (float32; a scalar, or the leading dimensions with reduction
    "none") and ``counts`` (int64, leading dimensions and E)."""

    loss: torch.Tensor
    counts: torch.Tensor


def _check(logits: torch.Tensor, config: BalanceConfig, mask: Optional[torch.Tensor]) -> None:
    if logits.dim() < 2:
        raise ValueError(f"logits must be [..., tokens, experts], got {tuple(logits.shape)}")
    experts = logits.shape[-1]
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"balance_loss takes 1 to {MAX_EXPERTS} experts, got {experts}")
    if config.top_k > experts:
        raise ValueError(f"top_k is {config.top_k}, but there are {experts} experts")
    if math.prod(logits.shape[:-2]) < 1:
        raise ValueError(f"logits hold no group, got {tuple(logits.shape)}")
    if logits.device.type != "cuda":
        raise ValueError(f"balance_loss needs HIP ('cuda') tensors, got {logits.device}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if mask is not None:
        if mask.shape != logits.shape[:-1]:
            raise ValueError(f"mask must be {tuple(logits.shape[:-1])}, one per token, got {tuple(mask.shape)}")
        if mask.dtype != torch.bool:
            raise TypeError(f"mask must be bool (True: counted), got {mask.dtype}")
        if mask.device != logits.device:
            raise ValueError(f"mask is on {mask.device}, logits on {logits.device}")


@lru_cache(maxsize=256)
def _ticket_bytes(groups: int, tokens: int, experts: int) -> int:
    return _lib.lib().ace_balance_ticket_bytes(groups, tokens, experts)


def balance_loss(logits: torch.Tensor, config: BalanceConfig,
                 mask: Optional[torch.Tensor] = None) -> BalanceLoss:
    """The balance loss of router scores ``[..., tokens, E]`` (float32, bfloat16
    or float16) and the counts of tokens that take each expert.  ``mask``
    ``[..., tokens]`` (bool): tokens that count (the others' scores are not
    read).  Differentiable once in ``logits``."""
    _check(logits, config, mask)
    dev = logits.device
    tokens, experts = logits.shape[-2:]
    groups = math.prod(logits.shape[:-2])
    zeros = tickets(dev, _stream(dev), _ticket_bytes(groups, tokens, experts))
    return BalanceLoss(*_lib.autograd().balance_loss(logits, mask, groups, config.top_k,
                                                     _REDUCTIONS[config.reduction], zeros))
