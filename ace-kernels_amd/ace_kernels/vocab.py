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
tokens, and 0 where there are none.  Logits, sums and gradients accumulate in
float32; the gradients have the inputs' type, the losses are float32.
"""

from __future__ import annotations

from typing import Any, Literal, NamedTuple, Optional, Tuple

import torch
from pydantic import BaseModel, ConfigDict
from torch.autograd.function import once_differentiable

from ace_kernels import _lib
from ace_kernels.impls.hip_mi355x import _ptr, _stream

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
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

    ignore_index: int = -100
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


def _dense(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and starting at a multiple of 16 bytes."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                config: VocabConfig, scores: bool) -> Tuple[torch.Tensor, ...]:
        lib = _lib.lib()
        dev = hidden.device
        size = weight.shape[1]
        x, w = _dense(hidden.reshape(-1, size)), _dense(weight)
        y = labels.reshape(-1).to(torch.int64).contiguous()
        n = x.shape[0]
        reduction = _REDUCTIONS[config.reduction]
        dims = (n, size, weight.shape[0])
        code = _DTYPES[hidden.dtype]
        f32 = torch.float32
        loss = torch.empty(labels.shape if reduction == _lib.RED_NONE else (), dtype=f32, device=dev)
        confidence = torch.empty(labels.shape, dtype=f32, device=dev) if scores else None
        correct = torch.empty(labels.shape, dtype=f32, device=dev) if scores else None
        saved = torch.empty(lib.ace_vocab_saved_bytes(n), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            ws = torch.empty(lib.ace_vocab_workspace_bytes(code, *dims, 0), dtype=torch.uint8, device=dev)
            rc = lib.ace_vocab_forward(
                x.data_ptr(), w.data_ptr(), code, y.data_ptr(), *dims, config.ignore_index, reduction,
                saved.data_ptr(), loss.data_ptr(), _ptr(confidence), _ptr(correct),
                ws.data_ptr(), ws.numel(), _stream(dev))
        _lib.check(rc, "ace_vocab_forward")
        ctx.save_for_backward(hidden, weight, saved)
        ctx.call = (code, dims, reduction)
        ctx.set_materialize_grads(False)
        if not scores:
            return (loss,)
        ctx.mark_non_differentiable(correct)
        return loss, confidence, correct

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, grad_loss: Optional[torch.Tensor], grad_confidence: Optional[torch.Tensor] = None,
                 _correct: Optional[torch.Tensor] = None):
        hidden, weight, saved = ctx.saved_tensors
        code, dims, reduction = ctx.call
        lib = _lib.lib()
        dev = hidden.device
        if grad_loss is None and grad_confidence is None:
            return None, None, None, None, None
        go = None if grad_loss is None else grad_loss.to(torch.float32).contiguous()
        gc = None if grad_confidence is None else grad_confidence.to(torch.float32).contiguous()
        x, w = _dense(hidden.reshape(-1, dims[1])), _dense(weight)
        dx = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if ctx.needs_input_grad[1] else None
        with torch.cuda.device(dev):
            ws = torch.empty(lib.ace_vocab_workspace_bytes(code, *dims, 1), dtype=torch.uint8, device=dev)
            rc = lib.ace_vocab_backward(
                x.data_ptr(), w.data_ptr(), code, *dims, reduction, saved.data_ptr(), _ptr(go), _ptr(gc),
                _ptr(dx), _ptr(dw), ws.data_ptr(), ws.numel(), _stream(dev))
        _lib.check(rc, "ace_vocab_backward")
        return dx, dw, None, None, None


def vocab_loss(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
               config: Optional[VocabConfig] = None) -> torch.Tensor:
    """Cross entropy of ``softmax(hidden @ weight.T)`` against ``labels``.

    ``hidden`` is ``[..., H]`` and ``weight`` ``[V, H]``, both float32, bfloat16
    or float16; ``labels`` are integers of shape ``[...]``.  Returns a float32
    scalar, or one value per token with ``reduction="none"``.  Differentiable
    once in ``hidden`` and ``weight``.
    """
    _check(hidden, weight, labels)
    return _VocabLoss.apply(hidden, weight, labels, config or _DEFAULT, False)[0]


def vocab_loss_confidence(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                          config: Optional[VocabConfig] = None) -> VocabScores:
    """``vocab_loss`` with each token's top-label confidence and correctness,
    from the same pass."""
    _check(hidden, weight, labels)
    return VocabScores(*_VocabLoss.apply(hidden, weight, labels, config or _DEFAULT, True))
