"""balance_loss on the CPU: what it refuses, its options, and the library's own
argument checks (nothing is launched)."""

from __future__ import annotations

import pytest
import torch
from pydantic import ValidationError

from ace_kernels import BalanceConfig, _lib, balance, balance_loss

FAKE = 256


def test_config() -> None:
    assert BalanceConfig(top_k=2).reduction == "mean"
    for bad in (dict(), dict(top_k=0), dict(top_k=17), dict(top_k=2, reduction="max"), dict(top_k=2, z=1)):
        with pytest.raises(ValidationError):
            BalanceConfig(**bad)


def test_refusals() -> None:
    cfg = BalanceConfig(top_k=4)
    with pytest.raises(ValueError, match="HIP"):
        balance_loss(torch.randn(5, 8), cfg)
    with pytest.raises(ValueError, match=r"\[..., tokens, experts\]"):
        balance_loss(torch.randn(8), cfg)
    with pytest.raises(ValueError, match="experts, got 513"):
        balance_loss(torch.randn(5, 513), cfg)
    with pytest.raises(ValueError, match="experts, got 0"):
        balance_loss(torch.randn(5, 0), cfg)
    with pytest.raises(ValueError, match="there are 3 experts"):
        balance_loss(torch.randn(5, 3), cfg)
    with pytest.raises(ValueError, match="no group"):
        balance_loss(torch.randn(0, 5, 8), cfg)


def test_type_and_mask_refusals() -> None:
    class Claims:
        def __init__(self, t):
            self.t, self.dtype, self.shape, self.device = t, t.dtype, t.shape, torch.device("cuda", 0)

        def dim(self):
            return self.t.dim()

    cfg, x = BalanceConfig(top_k=2), Claims(torch.randn(5, 8))
    balance._check(x, cfg, Claims(torch.ones(5, dtype=torch.bool)))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        balance._check(Claims(torch.randn(5, 8).double()), cfg, None)
    with pytest.raises(TypeError, match="must be bool"):
        balance._check(x, cfg, Claims(torch.ones(5)))
    with pytest.raises(ValueError, match="one per token"):
        balance._check(x, cfg, Claims(torch.ones(4, dtype=torch.bool)))
    with pytest.raises(ValueError, match="mask is on"):
        balance._check(x, cfg, torch.ones(5, dtype=torch.bool))


def _forward(**changed):
    a = dict(logits=FAKE, dtype=_lib.BF16, mask=None, groups=2, tokens=10, experts=8, top_k=2, reduction=_lib.RED_MEAN,
             loss=FAKE, counts=FAKE, share=FAKE, tickets=FAKE, ticket_bytes=1 << 30, ws=FAKE, nbytes=1 << 40)
    a.update(changed)
    return _lib.lib().ace_balance_forward(*a.values(), None)


def _backward(**changed):
    a = dict(logits=FAKE, dtype=_lib.BF16, mask=None, groups=2, tokens=10, experts=8, reduction=_lib.RED_MEAN,
             share=FAKE, grad=FAKE, d=FAKE)
    a.update(changed)
    return _lib.lib().ace_balance_backward(*a.values(), None)


BAD = [dict(logits=None), dict(dtype=_lib.F64), dict(groups=0), dict(tokens=-1), dict(experts=0), dict(reduction=3),
       dict(share=None)]


@pytest.mark.parametrize("changed", BAD + [dict(top_k=0), dict(top_k=9), dict(loss=None), dict(counts=None),
                                           dict(tickets=None), dict(ws=None), dict(ws=FAKE + 8), dict(tickets=FAKE + 2)])
def test_forward_refuses_before_launch(changed) -> None:
    assert _forward(**changed) == _lib.EINVAL


@pytest.mark.parametrize("changed", BAD + [dict(grad=None), dict(d=None)])
def test_backward_refuses_before_launch(changed) -> None:
    assert _backward(**changed) == _lib.EINVAL


def test_limits_and_workspace() -> None:
    lib = _lib.lib()
    assert _forward(experts=513) == _lib.EUNSUPPORTED and _backward(experts=513) == _lib.EUNSUPPORTED
    assert _forward(experts=64, top_k=17) == _lib.EUNSUPPORTED
    assert _forward(groups=(1 << 20) + 1) == _lib.EUNSUPPORTED
    need, tickets = lib.ace_balance_workspace_bytes(2, 10, 8), lib.ace_balance_ticket_bytes(2, 10, 8)
    assert need > 0 and tickets > 0
    assert _forward(nbytes=need - 1) == 3 and _forward(ticket_bytes=tickets - 1) == 3
    assert lib.ace_balance_workspace_bytes(0, 10, 8) == 0 and lib.ace_balance_ticket_bytes(0, 10, 8) == 0
    assert _backward(tokens=0, logits=None, share=None, grad=None, d=None) == 0  # nothing to do


def test_tangents_are_refused() -> None:
    """The call itself, under the checks of the Python side: scores with a tangent
    raise, where their loss would have had none."""
    import torch.autograd.forward_ad as fwd

    x = torch.randn(5, 8)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="balance_loss has no forward-mode derivative"):
        _lib.autograd().balance_loss(fwd.make_dual(x, torch.ones_like(x)), None, 1, 2, _lib.RED_MEAN,
                                     torch.zeros(4096, dtype=torch.uint8))
