"""mL1-ACE calibration loss on MI355X (gfx950): the reference's API over HIP kernels.

Same public surface as the reference package (``src/ace_kernels/__init__.py``):
``ACEConfig``, ``ImplSpec``, ``ace_loss``, ``available_impls``, ``get_impl``.
Importing it registers ``hip_mi355x``; its kernels live in ``libace_hip.so``
(built by ``ace-kernels_amd/build.py``), loaded on first use.

Beside it, the losses of a language model's step that the calibration loss
joins there: ``vocab_loss`` and ``vocab_loss_confidence`` (``vocab.py``), and the
router's ``balance_loss`` (``balance.py``).
"""

from ace_kernels import impls
from ace_kernels.balance import BalanceConfig, BalanceLoss, balance_loss
from ace_kernels.config import ACEConfig
from ace_kernels.registry import ImplSpec, ace_loss, available_impls, get_impl
from ace_kernels.vocab import VocabConfig, VocabScores, vocab_loss, vocab_loss_confidence

__all__ = ["ACEConfig", "BalanceConfig", "BalanceLoss", "ImplSpec", "VocabConfig", "VocabScores", "ace_loss",
           "available_impls", "balance_loss", "get_impl", "impls", "vocab_loss", "vocab_loss_confidence"]
