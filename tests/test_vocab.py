"""vocab_loss on the CPU: what it refuses, its options, and the library's own
argument checks (nothing is launched)."""

from __future__ import annotations

import pytest
import torch
from pydantic import ValidationError

from ace_kernels import VocabConfig, _lib, vocab_loss, vocab_loss_confidence

FAKE = 256  # non-null, aligned; never dereferenced


@pytest.mark.parametrize("call", [vocab_loss, vocab_loss_confidence])
def test_refusals(call) -> None:
    h, w, y = torch.randn(6, 8), torch.randn(10, 8), torch.zeros(6, dtype=torch.int64)
    with pytest.raises(ValueError, match="HIP"):
        call(h, w, y)
    with pytest.raises(ValueError, match="hidden must be"):
        call(h, torch.randn(10, 7), y)
    with pytest.raises(ValueError, match="hidden must be"):
        call(h, torch.randn(2, 10, 8), y)
    with pytest.raises(ValueError, match="hidden must be"):
        call(torch.tensor(1.0), w, y)
    with pytest.raises(ValueError, match="one per token"):
        call(h, w, y[:5])
    with pytest.raises(ValueError, match="one per token"):
        call(h, w, y[:, None])
    with pytest.raises(ValueError, match="must have words"):
        call(h, torch.randn(0, 8), y)
    with pytest.raises(ValueError, match="must have words"):
        call(torch.randn(6, 0), torch.randn(10, 0), y)


def test_type_refusals() -> None:
    """On fake ("meta" would be refused first) devices the types cannot be
    reached, so the check is called with tensors that claim a HIP device."""
    from ace_kernels import vocab

    class Claims:
        def __init__(self, t):
            self.t, self.dtype, self.shape, self.device = t, t.dtype, t.shape, torch.device("cuda", 0)

        def dim(self):
            return self.t.dim()

    h, w, y = Claims(torch.randn(6, 8)), Claims(torch.randn(10, 8)), Claims(torch.zeros(6, dtype=torch.int64))
    vocab._check(h, w, y)
    with pytest.raises(TypeError, match="must both be"):
        vocab._check(h, Claims(torch.randn(10, 8).half()), y)
    with pytest.raises(TypeError, match="must both be"):
        vocab._check(Claims(torch.randn(6, 8).double()), Claims(torch.randn(10, 8).double()), y)
    with pytest.raises(TypeError, match="integers"):
        vocab._check(h, w, Claims(torch.zeros(6)))
    with pytest.raises(ValueError, match="labels on"):
        vocab._check(h, w, torch.zeros(6, dtype=torch.int64))


def test_config() -> None:
    assert VocabConfig() == VocabConfig(ignore_index=-100, reduction="mean")
    with pytest.raises(ValidationError):
        VocabConfig(reduction="max")
    with pytest.raises(ValidationError):
        VocabConfig(smoothing=0.1)
    with pytest.raises(ValidationError):
        VocabConfig().reduction = "sum"


def _forward(**changed):
    a = dict(hidden=FAKE, weight=FAKE, dtype=_lib.BF16, labels=FAKE, tokens=4, size=8, vocab=100, ignore=-100,
             reduction=_lib.RED_MEAN, saved=FAKE, loss=FAKE, confidence=None, correct=None, ws=FAKE, nbytes=1 << 40)
    a.update(changed)
    return _lib.lib().ace_vocab_forward(*a.values(), None)


def _backward(**changed):
    a = dict(hidden=FAKE, weight=FAKE, dtype=_lib.BF16, tokens=4, size=8, vocab=100, reduction=_lib.RED_MEAN,
             saved=FAKE, gl=FAKE, gc=None, dh=FAKE, dw=FAKE, ws=FAKE, nbytes=1 << 40)
    a.update(changed)
    return _lib.lib().ace_vocab_backward(*a.values(), None)


BAD = [dict(hidden=None), dict(weight=None), dict(saved=None), dict(ws=None), dict(dtype=_lib.F64), dict(tokens=-1),
       dict(size=0), dict(vocab=0), dict(reduction=3), dict(hidden=FAKE + 2), dict(weight=FAKE + 8), dict(ws=FAKE + 4),
       dict(saved=FAKE + 4)]


@pytest.mark.parametrize("changed", BAD + [dict(labels=None), dict(loss=None)])
def test_forward_refuses_before_launch(changed) -> None:
    assert _forward(**changed) == _lib.EINVAL


@pytest.mark.parametrize("changed", BAD + [dict(dh=FAKE + 8), dict(dw=FAKE + 2)])
def test_backward_refuses_before_launch(changed) -> None:
    assert _backward(**changed) == _lib.EINVAL


@pytest.mark.parametrize("call", [_forward, _backward])
def test_limits_and_workspace(call) -> None:
    for too in (dict(tokens=(1 << 30) + 1), dict(vocab=(1 << 30) + 1), dict(size=(1 << 20) + 1)):
        assert call(**too) == _lib.EUNSUPPORTED
    need = _lib.lib().ace_vocab_workspace_bytes(_lib.BF16, 4, 8, 100, int(call is _backward))
    assert need > 0 and need % 256 == 0
    assert call(nbytes=need - 1) == 3  # ACE_EWORKSPACE


def test_workspace_is_bounded() -> None:
    """The logits are not kept: the backward of 8192 tokens over 131072 words
    takes far less than one copy of them."""
    lib = _lib.lib()
    logits = 8192 * 131072 * 2
    assert lib.ace_vocab_workspace_bytes(_lib.BF16, 8192, 1024, 131072, 1) < logits / 3
    assert lib.ace_vocab_workspace_bytes(_lib.BF16, 8192, 1024, 131072, 0) < logits / 50
    assert lib.ace_vocab_workspace_bytes(_lib.F64, 8, 8, 8, 0) == 0
    assert lib.ace_vocab_workspace_bytes(_lib.BF16, -1, 8, 8, 0) == 0
    assert lib.ace_vocab_saved_bytes(0) > 0 and lib.ace_vocab_saved_bytes(-1) == 0


def test_tangents_are_refused() -> None:
    """The call itself, under the checks of the Python side: a tensor with a
    tangent raises, where its loss would have had none."""
    import torch.autograd.forward_ad as fwd

    h, w, y = torch.randn(6, 8), torch.randn(10, 8), torch.zeros(6, dtype=torch.int64)
    with fwd.dual_level():
        for a, b in ((fwd.make_dual(h, torch.ones_like(h)), w), (h, fwd.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(NotImplementedError, match="vocab_loss has no forward-mode derivative"):
                _lib.autograd().vocab_loss(a, b, y, -100, _lib.RED_MEAN, False)


def test_ignore_index_is_an_int64() -> None:
    for good in (-(2 ** 63), -1, 0, 2 ** 63 - 1):
        assert VocabConfig(ignore_index=good).ignore_index == good
    for bad in (2 ** 63, -(2 ** 63) - 1, 2 ** 70):
        with pytest.raises(ValidationError):
            VocabConfig(ignore_index=bad)
