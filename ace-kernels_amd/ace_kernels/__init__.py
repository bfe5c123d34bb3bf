"""mL1-ACE calibration loss on MI355X (gfx950): the reference's API over HIP kernels.

Same public surface as the reference package (``src/ace_kernels/__init__.py``):
``ACEConfig``, ``ImplSpec``, ``ace_loss``, ``available_impls``, ``get_impl``.
Importing it registers ``hip_mi355x``; its kernels live in ``libace_hip.so``
(built by ``ace-kernels_amd/build.py``), loaded on first use.

Beside it, the losses of a language model's step that the calibration loss
joins there: ``vocab_loss`` and ``vocab_loss_confidence`` (``vocab.py``), and the
router's ``balance_loss`` (``balance.py``); the log probabilities of given tokens,
``token_logprobs`` (``logprobs.py``); and a router's way to its experts and back,
``route_tokens``, ``expert_order``, ``to_experts`` and ``from_experts`` (``experts.py``).
"""

from ace_kernels import impls
from ace_kernels.balance import BalanceConfig, BalanceLoss, balance_loss
from ace_kernels.config import ACEConfig
from ace_kernels.experts import (ExpertOrder, RouteConfig, Routes, expert_order, from_experts, route_tokens,
                                 to_experts)
from ace_kernels.logprobs import LogprobConfig, TokenLogprobs, token_logprobs
from ace_kernels.registry import ImplSpec, ace_loss, available_impls, get_impl
from ace_kernels.vocab import VocabConfig, VocabScores, vocab_loss, vocab_loss_confidence

__all__ = ["ACEConfig", "BalanceConfig", "BalanceLoss", "ExpertOrder", "ImplSpec", "LogprobConfig", "RouteConfig",
           "Routes", "TokenLogprobs", "VocabConfig", "VocabScores", "ace_loss", "available_impls", "balance_loss",
           "expert_order", "from_experts", "get_impl", "impls", "route_tokens", "to_experts", "token_logprobs",
           "vocab_loss", "vocab_loss_confidence"]
