"""Softmax cross entropy of hidden states against a large vocabulary, and the
confidences that the calibration loss takes.

``ace_loss`` calibrates up to 64 channels of given logits.  A language model's
head has tens of thousands of words and its logits are larger than everything
else of the step, so these losses take the hidden states and the head's weight
instead, and form the logits in pieces that are never kept (forward or
backward)::

    loss = vocab_loss(hidden, weight, labels)

    out = vocab_loss_confidence(hidden, weight, labels)
    keep = labels != -100
    ace = ace_loss(out.confidence[keep][None, None], out.correct[keep][None, None],
                   ACEConfig(activation="none"))
    (out.loss + ace).backward()

A token's confidence is the largest probability of its softmax, and ``correct``
says whether that word (the lowest index where several are equal) is the label:
the probability and the target of top-label calibration.  The confidence is
differentiable, so the calibration loss trains the model through it.

Tokens whose label is ``ignore_index``, or any number outside the vocabulary,
are not counted: their loss, confidence, correctness and gradients are 0 and
their hidden states are not read (they may be NaN).  The mean is over the counted
tokens, and 0 where there are none.  Logits and all sums are float32, and so are the
losses; the gradients have the inputs' type.  In bfloat16 and float16 the gradient of
each logit is rounded to that type before it is multiplied with the weight and the
hidden states (half a step: 2^-8, 2^-11), as a product in that type does.  In float16
it is scaled first, so that small probabilities count: for the hidden gradient by
each token's own upstream gradient (to within a factor of 64), for the weight's by the
tokens' largest, beside which entries below 2^-38 are lost.

The calls have no forward-mode and no second derivative, and ``torch.func`` transforms
do not know them; ``torch.compile`` breaks its graph at them.

The call and its backward node are C++ (``csrc/ace_autograd.cpp``).
"""

from __future__ import annotations

from typing import List, Literal, NamedTuple, Optional

import torch
from pydantic import BaseModel, ConfigDict, Field

from ace_kernels import _lib

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_REDUCTIONS = {"mean": _lib.RED_MEAN, "sum": _lib.RED_SUM, "none": _lib.RED_NONE}
_LABEL_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


class VocabConfig(BaseModel):
    """Options of the vocabulary losses.

    ignore_index: tokens with this label are not counted (nor are those whose
                  label is outside the vocabulary).
    reduction:    over the counted tokens: their mean, their sum, or "none" for
                  each token's loss.
    """

    model_config = ConfigDict(frozen=True, extra="forbid")

    ignore_index: int = Field(default=-100, ge=-(2**63), lt=2**63)  # an int64, as the labels are
    reduction: Literal["mean", "sum", "none"] = "mean"


_DEFAULT = VocabConfig()


class VocabScores(NamedTuple):
    """``loss`` as ``vocab_loss`` returns it, and per token, in the labels'
    shape, the ``confidence`` (differentiable) and ``correct`` (0 or 1)."""

    loss: torch.Tensor
    confidence: torch.Tensor
    correct: torch.Tensor


def _check(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor) -> None:
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError("hidden must be [..., H] and weight [V, H], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must have words and a hidden size, got {tuple(weight.shape)}")
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels must be {tuple(hidden.shape[:-1])}, one per token, got {tuple(labels.shape)}")
    if hidden.device.type != "cuda":
        raise ValueError(f"vocab_loss needs HIP ('cuda') tensors, got {hidden.device}")
    if weight.device != hidden.device or labels.device != hidden.device:
        raise ValueError(f"hidden is on {hidden.device}, weight on {weight.device}, labels on {labels.device}")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise TypeError("hidden and weight must both be float32, bfloat16 or float16, got "
                        f"{hidden.dtype} and {weight.dtype}")
    if labels.dtype not in _LABEL_TYPES:
        raise TypeError(f"labels must be integers, got {labels.dtype}")


def _call(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, config: Optional[VocabConfig],
          scores: bool) -> List[torch.Tensor]:
    _check(hidden, weight, labels)
    config = config or _DEFAULT
    out: List[torch.Tensor] = _lib.autograd().vocab_loss(hidden, weight, labels, config.ignore_index,
                                                         _REDUCTIONS[config.reduction], scores)
    return out


def vocab_loss(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
               config: Optional[VocabConfig] = None) -> torch.Tensor:
    """Cross entropy of ``softmax(hidden @ weight.T)`` against ``labels``.

    ``hidden`` is ``[..., H]`` and ``weight`` ``[V, H]``, both float32, bfloat16
    or float16; ``labels`` are integers of shape ``[...]``.  Returns a float32
    scalar, or one value per token with ``reduction="none"``.  Differentiable
    once in ``hidden`` and ``weight``.
    """
    return _call(hidden, weight, labels, config, False)[0]


def vocab_loss_confidence(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                          config: Optional[VocabConfig] = None) -> VocabScores:
    """``vocab_loss`` with each token's top-label confidence and correctness,
    from the same pass."""
    return VocabScores(*_call(hidden, weight, labels, config, True))
