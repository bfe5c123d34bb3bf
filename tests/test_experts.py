"""The experts' operators on the CPU: what they refuse, their options, and the
library's own argument checks (nothing is launched)."""

from __future__ import annotations

import pytest
import torch
from pydantic import ValidationError

from ace_kernels import ExpertOrder, RouteConfig, _lib, expert_order, experts, from_experts, route_tokens, to_experts
from test_logprobs import Claims

FAKE = 256
I64 = torch.int64


def test_config() -> None:
    assert RouteConfig(top_k=2).normalize is True
    for bad in (dict(), dict(top_k=0), dict(top_k=17), dict(top_k=2, normalize="x"), dict(top_k=2, z=1)):
        with pytest.raises(ValidationError):
            RouteConfig(**bad)


def test_route_refusals() -> None:
    cfg, x = RouteConfig(top_k=4), torch.randn(5, 8)
    with pytest.raises(ValueError, match="HIP"):
        route_tokens(x, cfg)
    with pytest.raises(ValueError, match=r"\[..., experts\]"):
        route_tokens(torch.tensor(1.0), cfg)
    with pytest.raises(ValueError, match="experts, got 513"):
        route_tokens(torch.randn(5, 513), cfg)
    with pytest.raises(ValueError, match="experts, got 0"):
        route_tokens(torch.randn(5, 0), cfg)
    with pytest.raises(ValueError, match="there are 3 experts"):
        route_tokens(torch.randn(5, 3), cfg)
    experts._check_route(Claims(x), cfg, Claims(torch.ones(5, dtype=torch.bool)))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        experts._check_route(Claims(x.double()), cfg, None)
    with pytest.raises(TypeError, match="must be bool"):
        experts._check_route(Claims(x), cfg, Claims(torch.ones(5)))
    with pytest.raises(ValueError, match="one per token"):
        experts._check_route(Claims(x), cfg, Claims(torch.ones(4, dtype=torch.bool)))
    with pytest.raises(ValueError, match="mask is on"):
        experts._check_route(Claims(x), cfg, torch.ones(5, dtype=torch.bool))


def test_order_refusals() -> None:
    e = torch.zeros(5, 2, dtype=I64)
    with pytest.raises(ValueError, match="HIP"):
        expert_order(e, 8)
    for bad in (0, -1, 513):
        with pytest.raises(ValueError, match="1 to 512 experts"):
            expert_order(e, bad)
    with pytest.raises(ValueError, match=r"\[..., top_k\]"):
        expert_order(torch.zeros(5, 0, dtype=I64), 8)
    with pytest.raises(ValueError, match=r"\[..., top_k\]"):
        expert_order(torch.tensor(1), 8)
    with pytest.raises(TypeError, match="must be integers"):
        expert_order(Claims(e.float()), 8)


def test_rows_refusals() -> None:
    order = ExpertOrder(*map(Claims, (torch.zeros(9, dtype=I64), torch.zeros(10, dtype=I64), torch.zeros(5, 2, dtype=I64))))
    order.place.numel = lambda: 10
    x, rows = torch.randn(5, 16), torch.randn(10, 16)
    with pytest.raises(ValueError, match="HIP"):
        to_experts(x, order)
    with pytest.raises(ValueError, match="HIP"):
        from_experts(rows, order)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16 rows"):
        to_experts(Claims(x.double()), order)
    for bad in (x[:4], torch.randn(5, 2, 16), torch.randn(5, 0), torch.tensor(1.0)):
        with pytest.raises(ValueError, match="a row per token"):
            to_experts(Claims(bad), order)
    for bad in (rows[:9], torch.randn(5, 2, 16), torch.randn(10, 0), torch.randn(10)):
        with pytest.raises(ValueError, match="one per slot"):
            from_experts(Claims(bad), order)
    for bad in (torch.randn(5, 3), torch.randn(10)):
        with pytest.raises(ValueError, match=r"weights must be \(5, 2\)"):
            from_experts(Claims(rows), order, Claims(bad))
    with pytest.raises(ValueError, match="weights is on"):
        from_experts(Claims(rows), order, torch.randn(5, 2))
    with pytest.raises(TypeError, match="weights must be"):
        from_experts(Claims(rows), order, Claims(torch.randn(5, 2).double()))
    with pytest.raises(TypeError, match="must be int64"):
        to_experts(Claims(x), order._replace(source=Claims(torch.zeros(10))))
    with pytest.raises(ValueError, match="the order on"):
        to_experts(Claims(x), order._replace(source=torch.zeros(10, dtype=I64)))
    for bad in (dict(source=Claims(torch.zeros(9, dtype=I64))), dict(source=Claims(torch.zeros(5, 2, dtype=I64)))):
        with pytest.raises(ValueError, match="expert_order's"):
            to_experts(Claims(x), order._replace(**bad))


def _route(**changed):
    a = dict(logits=FAKE, dtype=_lib.BF16, mask=None, tokens=10, experts=8, top_k=2, normalize=1, chosen=FAKE, weights=FAKE)
    a.update(changed)
    return _lib.lib().ace_route_forward(*a.values(), None)


def _route_back(**changed):
    a = dict(logits=FAKE, dtype=_lib.BF16, tokens=10, experts=8, top_k=2, normalize=1, chosen=FAKE, weights=FAKE, grad=FAKE,
             d=FAKE)
    a.update(changed)
    return _lib.lib().ace_route_backward(*a.values(), None)


BAD = [dict(logits=None), dict(dtype=_lib.F64), dict(tokens=-1), dict(experts=0), dict(top_k=0), dict(top_k=9),
       dict(chosen=None), dict(weights=None)]


@pytest.mark.parametrize("changed", BAD)
def test_route_refuses_before_launch(changed) -> None:
    assert _route(**changed) == _lib.EINVAL and _route_back(**changed) == _lib.EINVAL


def test_route_limits() -> None:
    assert _route_back(grad=None) == _lib.EINVAL and _route_back(d=None) == _lib.EINVAL
    for call in (_route, _route_back):
        assert call(experts=513) == _lib.EUNSUPPORTED
        assert call(experts=64, top_k=17) == _lib.EUNSUPPORTED
        assert call(tokens=(1 << 30) + 1) == _lib.EUNSUPPORTED
        assert call(tokens=0, logits=None, chosen=None, weights=None) == 0  # nothing to do


def _order(**changed):
    a = dict(chosen=FAKE, slots=100000, experts=8, offsets=FAKE, source=FAKE, place=FAKE, ws=FAKE, nbytes=1 << 40)
    a.update(changed)
    return _lib.lib().ace_expert_order(*a.values(), None)


@pytest.mark.parametrize("changed", [dict(chosen=None), dict(slots=-1), dict(experts=0), dict(offsets=None), dict(source=None),
                                     dict(place=None), dict(ws=None), dict(ws=FAKE + 2)])
def test_order_refuses_before_launch(changed) -> None:
    assert _order(**changed) == _lib.EINVAL


def test_order_limits() -> None:
    lib = _lib.lib()
    assert _order(experts=513) == _lib.EUNSUPPORTED and _order(slots=(1 << 30) + 1) == _lib.EUNSUPPORTED
    need = lib.ace_expert_order_workspace_bytes(100000, 8)
    assert need > 0 and _order(nbytes=need - 1) == 3
    assert lib.ace_expert_order_workspace_bytes(100, 8) == 0 and lib.ace_expert_order_workspace_bytes(0, 8) == 0
    assert lib.ace_expert_order_workspace_bytes(1 << 30, 512) <= 1 << 20


def _to(**changed):
    a = dict(x=FAKE, dtype=_lib.BF16, tokens=10, width=64, top_k=2, source=FAKE, place=FAKE, rows=FAKE)
    a.update(changed)
    return _lib.lib().ace_to_experts(*a.values(), None)


def _from(**changed):
    a = dict(x=FAKE, dtype=_lib.BF16, tokens=10, width=64, top_k=2, source=FAKE, place=FAKE, weights=FAKE, out=FAKE)
    a.update(changed)
    return _lib.lib().ace_from_experts(*a.values(), None)


def _from_back(**changed):
    a = dict(x=FAKE, grad=FAKE, dtype=_lib.BF16, tokens=10, width=64, top_k=2, source=FAKE, place=FAKE, weights=FAKE,
             d_rows=FAKE, d_weights=FAKE)
    a.update(changed)
    return _lib.lib().ace_from_experts_backward(*a.values(), None)


@pytest.mark.parametrize("changed", [dict(x=None), dict(dtype=_lib.F64), dict(tokens=-1), dict(width=0), dict(top_k=0),
                                     dict(source=None), dict(place=None)])
def test_rows_refuse_before_launch(changed) -> None:
    for call in (_to, _from, _from_back):
        assert call(**changed) == _lib.EINVAL


def test_last_block_stays_below_the_grid_limit() -> None:
    # four waves a block: 2^26 - 1 of them would round up to 2^32 threads
    for call in (_to, _from, _from_back):
        assert call(tokens=(1 << 26) - 1, top_k=1, width=1024) == _lib.EUNSUPPORTED
        assert call(tokens=(1 << 26) - 3, top_k=1, width=1024) == _lib.EUNSUPPORTED


def test_rows_limits() -> None:
    assert _to(rows=None) == _lib.EINVAL and _from(out=None) == _lib.EINVAL
    assert _from_back(grad=None) == _lib.EINVAL
    for call in (_to, _from, _from_back):
        assert call(width=(1 << 20) + 1) == _lib.EUNSUPPORTED
        assert call(tokens=1 << 25) == _lib.EUNSUPPORTED  # 2^26 slots
        assert call(tokens=1 << 20, width=1 << 20) == _lib.EUNSUPPORTED
        assert call(tokens=1 << 40, top_k=1 << 40) == _lib.EUNSUPPORTED
        assert call(tokens=0, x=None, source=None, place=None) == 0  # nothing to do
    assert _from_back(d_rows=None, d_weights=None) == 0


def test_tangents_are_refused() -> None:
    import torch.autograd.forward_ad as fwd

    mod, x = _lib.autograd(), torch.randn(5, 8)
    source, place = torch.zeros(5, dtype=I64), torch.zeros(5, 1, dtype=I64)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="route_tokens has no forward-mode derivative"):
            mod.route_tokens(dual, None, 2, True)
        with pytest.raises(NotImplementedError, match="to_experts has no forward-mode derivative"):
            mod.to_experts(dual, source, place)
        with pytest.raises(NotImplementedError, match="from_experts has no forward-mode derivative"):
            mod.from_experts(dual, source, place, None)
        with pytest.raises(NotImplementedError, match="from_experts has no forward-mode derivative"):
            mod.from_experts(x, source, place, fwd.make_dual(x[:, :1], torch.ones(5, 1)))
