"""Log probabilities of given tokens from a model's logits, with the entropy and
the largest alternatives of each.

Where the logits are there, as in serving and in a policy step, one pass over them
gives what a served model's calibration is measured on, and what a policy is trained
through::

    out = token_logprobs(logits, tokens, LogprobConfig(top=5, temperature=0.7))
    out.logprob       # log softmax(logits / temperature) at each token
    out.entropy       # of that softmax
    out.top_logprobs, out.top_tokens  # the five largest, in order

    out = token_logprobs(logits, tokens)
    ratio = torch.exp(out.logprob - old_logprob)
    (-(ratio * advantage) - 0.01 * out.entropy).mean().backward()

``vocab_loss`` (without logits, from the hidden states) is the one to train with
cross entropy.  ``exp(out.top_logprobs[..., 0])`` is a token's confidence, the
probability that ``ace_loss`` calibrates.

The alternatives are the largest logits, the lowest word first where they are equal;
NaN is above all.  Tokens that are ``ignore_index``, or any number outside the
vocabulary, are not counted: results and gradients are 0, ``top_tokens`` -1, and their
logits are not read (they may be NaN).  Words at -inf have probability 0 and add
nothing to the entropy; a row of nothing else has log probabilities of -inf, entropy
0 and gradient 0.  A row with NaN or +inf has NaN throughout.  Sums are float32, and
so are the results; the gradient has the logits' type.

The call and its backward node are C++ (``csrc/ace_autograd.cpp``).  They have no
forward-mode and no second derivative, and ``torch.func`` transforms do not know them;
``torch.compile`` breaks its graph at them.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch
from pydantic import BaseModel, ConfigDict, Field

from ace_kernels import _lib
from ace_kernels.common import tickets
from ace_kernels.impls.hip_mi355x import _stream

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_TOKEN_TYPES = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)
MAX_TOP = 32


class LogprobConfig(BaseModel):
    """Options of the token log probabilities.

    top:          alternatives that are returned (0: none; at most 32, and at most
                  the vocabulary).
    temperature:  the logits are divided by it.
    ignore_index: this token is not counted (nor is any outside the vocabulary).
    """

    model_config = ConfigDict(frozen=True, extra="forbid")

    top: int = Field(default=0, ge=0, le=MAX_TOP)
    temperature: float = Field(default=1.0, ge=1e-3, le=1e3)
    ignore_index: int = Field(default=-100, ge=-(2**63), lt=2**63)  # an int64, as the tokens are


_DEFAULT = LogprobConfig()


class TokenLogprobs(NamedTuple):
    """``logprob`` and ``entropy`` (float32, in the tokens' shape, differentiable);
    ``top_logprobs`` (float32) and ``top_tokens`` (int64), with a last dimension of
    ``top``, or None where it is 0."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor] = None
    top_tokens: Optional[torch.Tensor] = None


def _check(logits: torch.Tensor, tokens: torch.Tensor, config: LogprobConfig) -> None:
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., V], got {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must be {tuple(logits.shape[:-1])}, one per row of logits, got {tuple(tokens.shape)}")
    if config.top > logits.shape[-1]:
        raise ValueError(f"top is {config.top}, but there are {logits.shape[-1]} words")
    if logits.device.type != "cuda":
        raise ValueError(f"token_logprobs needs HIP ('cuda') tensors, got {logits.device}")
    if tokens.device != logits.device:
        raise ValueError(f"logits is on {logits.device}, tokens on {tokens.device}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if tokens.dtype not in _TOKEN_TYPES:
        raise TypeError(f"tokens must be integers, got {tokens.dtype}")


@lru_cache(maxsize=1024)
def _ticket_bytes(dtype: int, rows: int, vocab: int) -> int:
    return _lib.lib().ace_logprob_ticket_bytes(dtype, rows, vocab)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor,
                   config: Optional[LogprobConfig] = None) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under ``softmax(logits / temperature)``, its
    entropy, and the largest alternatives.

    ``logits`` is ``[..., V]`` (float32, bfloat16 or float16; rows may lie apart, as in a
    slice of a padded vocabulary, and are then read where they are), ``tokens`` integers
    of shape ``[...]``.  Differentiable once in ``logits``, through ``logprob`` and
    ``entropy``.
    """
    config = config or _DEFAULT
    _check(logits, tokens, config)
    dev = logits.device
    need = _ticket_bytes(_DTYPES[logits.dtype], tokens.numel(), logits.shape[-1])
    zeros = tickets(dev, _stream(dev), need) if need else None
    return TokenLogprobs(*_lib.autograd().token_logprobs(logits, tokens, config.ignore_index, config.temperature,
                                                         config.top, zeros))
