"""The experts' operators on the GPU against their definitions in float64.

u = 2^-24.  A weight is an exponential over a sum: off relatively by 16 u (1 + the
scores' range) + 4 sqrt(E) u.  A float32 sum of k products is off by (k + 1) u of the
sum of their magnitudes, one over a row's width, added in width / 64 steps a lane and 6
across, by (width / 64 + 8) u of it.  Results of a 16-bit type are half a step off."""

from __future__ import annotations

import math

import pytest
import torch

from ace_kernels import (BalanceConfig, RouteConfig, balance_loss, expert_order, from_experts, route_tokens,
                         to_experts)
from gpu_helpers import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(seed, *shape):
    return torch.randn(shape, generator=_gen(seed), device="cuda")


def _scores(lead, experts, dtype, seed=0):
    return (1.5 * _normal(seed, *lead, experts) + _normal(seed + 1000, experts)).to(dtype)


def _mask(lead, share, seed=1):
    return torch.rand(lead, generator=_gen(seed), device="cuda") >= share


def _half(dtype, x):
    """Half a step of a result, also among the subnormals."""
    info = torch.finfo(dtype)
    return info.eps / 2 * x.abs() + info.tiny * info.eps / 2 * 1.01


# -------------------------------------------------------------------- route


def _route_exact(x, k, normalize, mask, up):
    s = x.detach().double()
    on = torch.ones(s.shape[:-1], dtype=torch.bool, device=s.device) if mask is None else mask
    s = torch.where(on[..., None], s, 0.0)
    order = torch.sort(torch.where(s.isnan(), math.inf, s), dim=-1, descending=True, stable=True).indices[..., :k]
    chosen = torch.zeros_like(s).scatter_(-1, order, 1.0)
    p = torch.softmax(torch.where(chosen > 0, s, -math.inf) if normalize else s, -1)
    w = p.gather(-1, order)
    spread = float(torch.where(s.isfinite(), s, 0.0).abs().amax()) * 2 if s.numel() else 0.0
    rel = 16 * U * (1 + spread) + 4 * math.sqrt(s.shape[-1]) * U
    u = up.double()
    pull, size = (w * u).sum(-1, keepdim=True), (w * u).abs().sum(-1, keepdim=True)
    d = torch.zeros_like(s).scatter_(-1, order, w * u) - p * pull
    near = torch.zeros_like(s).scatter_(-1, order, (w * u).abs()) + p * size
    keep = on[..., None]
    d = d * keep
    tol = (near * (2 * rel + (k + 4) * U)) * keep + _half(x.dtype, d) + u.abs().amax() * 2.0 ** -125 if s.numel() else near
    return torch.where(keep, order, -1), w * keep, rel * w * keep + 2.0 ** -126, d, tol


def _route(x, k, normalize=True, mask=None):
    up = _normal(7, *x.shape[:-1], k)
    order, w, tol, d, tol_d = _route_exact(x, k, normalize, mask, up)
    leaf = x.detach().requires_grad_(True)
    out = route_tokens(leaf, RouteConfig(top_k=k, normalize=normalize), mask)
    (grad,) = torch.autograd.grad(out.weights, leaf, up)
    assert out.experts.dtype == torch.int64 and out.weights.dtype == F32 and grad.dtype == x.dtype
    assert torch.equal(out.experts, order)
    assert ((out.weights.double() - w).abs() <= tol).all()
    err = (grad.double() - d).abs()
    assert (err <= tol_d).all(), f"gradient: worst {float((err / tol_d).max()):.3g} x bound"
    return out, grad


@TYPES
@pytest.mark.parametrize("experts", [1, 2, 3, 5, 7, 8, 9, 12, 16, 17, 31, 33, 60, 64, 65, 100, 128, 130, 250, 256, 257, 511, 512])
def test_route_experts(experts, dtype) -> None:
    say(f"route {experts} {dtype}")
    for k in sorted({1, min(2, experts), min(3, experts), min(6, experts), min(8, experts), min(16, experts)}):
        for normalize in (True, False):
            _route(_scores((133,), experts, dtype, seed=experts), k, normalize, _mask((133,), 0.2, seed=k))


@TYPES
@pytest.mark.parametrize("lead", [(), (1,), (2, 3, 5), (4097,), (100003,), (0,), (3, 0)])
def test_route_lengths(lead, dtype) -> None:
    for experts in (8, 24, 200):
        for normalize in (True, False):
            _route(_scores(lead, experts, dtype), 2, normalize)
            _route(_scores(lead, experts, dtype), 2, normalize, _mask(lead, 0.4))


@TYPES
@pytest.mark.parametrize("experts", [6, 40, 64, 200, 256, 400])
def test_route_ties_go_to_the_lowest_expert(experts, dtype) -> None:
    few = torch.randint(-1, 2, (300, experts), generator=_gen(experts), device="cuda").to(dtype)
    few[:100] = 0.0
    few[100:150] *= -0.0
    for k in (1, 2, 5):
        for normalize in (True, False):
            out, _ = _route(few, k, normalize)
            assert (out.experts[:100] == torch.arange(k, device="cuda")).all()


@TYPES
@pytest.mark.parametrize("normalize", [True, False])
def test_route_closed_experts(normalize, dtype) -> None:
    """Experts at -inf (or the type's lowest value) have weight 0 and no gradient,
    also where fewer are open than a token takes, and where none is."""
    x = _scores((200,), 30, dtype)
    for closed in (-math.inf, torch.finfo(dtype).min):
        y = x.clone()
        y[:, 7:20] = closed
        out, grad = _route(y, 4, normalize)
        assert not grad[:, 7:20].any()
        y[50:] = closed
        y[50:, 28] = 1.0
        up = _normal(7, 200, 4)
        leaf = y.requires_grad_(True)
        out = route_tokens(leaf, RouteConfig(top_k=4, normalize=normalize))
        (grad,) = torch.autograd.grad(out.weights, leaf, up)
        assert out.experts[50:].tolist() == [[28, 0, 1, 2]] * 150
        assert (out.weights[50:] == torch.tensor([1.0, 0, 0, 0], device="cuda")).all() and not grad[50:].any()
    y = x.clone()
    y[3] = -math.inf
    leaf = y.requires_grad_(True)
    out = route_tokens(leaf, RouteConfig(top_k=4, normalize=normalize))
    (grad,) = torch.autograd.grad(out.weights, leaf, _normal(7, 200, 4))
    assert out.experts[3].tolist() == [0, 1, 2, 3] and not out.weights[3].any() and not grad[3].any()
    assert torch.isfinite(out.weights).all() and torch.isfinite(grad).all()


@TYPES
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts", [8, 100])
def test_route_nan_and_masked_tokens(experts, normalize, dtype) -> None:
    x = _scores((90,), experts, dtype)
    mask = _mask((90,), 0.5)
    mask[0], mask[1] = True, False
    want, grad = _route(x, 3, normalize, mask)
    y = torch.where(mask[:, None], x, math.nan)
    y[0, 5] = math.nan
    leaf = y.requires_grad_(True)
    out = route_tokens(leaf, RouteConfig(top_k=3, normalize=normalize), mask)
    (got,) = torch.autograd.grad(out.weights, leaf, _normal(7, 90, 3))
    assert out.experts[0, 0] == 5 and out.weights[0].isnan().all() and got[0].isnan().any()
    for a, b in zip((*want, grad), (*out, got)):
        assert torch.equal(a[1:], b[1:])
    assert (out.experts[~mask] == -1).all() and not out.weights[~mask].any() and not got[~mask].any()


def test_route_agrees_with_the_balance_loss() -> None:
    for dtype in (F32, BF16):
        x = torch.randint(-3, 3, (1000, 48), generator=_gen(3), device="cuda").to(dtype)  # many ties
        mask = _mask((1000,), 0.2)
        out = route_tokens(x, RouteConfig(top_k=6), mask)
        counts = balance_loss(x, BalanceConfig(top_k=6), mask).counts
        assert torch.equal(torch.bincount(out.experts[mask].flatten(), minlength=48), counts)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_against_differences(normalize) -> None:
    x = _scores((60,), 12, F32)
    up = _normal(7, 60, 3)
    leaf = x.clone().requires_grad_(True)
    out = route_tokens(leaf, RouteConfig(top_k=3, normalize=normalize))
    (got,) = torch.autograd.grad(out.weights, leaf, up)
    way = _normal(8, 60, 12).double()

    def f(t):  # the choice is a constant
        w = torch.softmax(x.double() + t * way, 1).gather(1, out.experts)
        return float((up.double() * (w / w.sum(1, keepdim=True) if normalize else w)).sum())

    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(float((got.double() * way).sum()) - want) <= 1e-5 * (1 + abs(want))


@TYPES
def test_route_strides_and_offsets(dtype) -> None:
    x = _scores((2, 33), 21, dtype)
    mask = _mask((2, 33), 0.3)
    for normalize in (True, False):
        want, grad = _route(x, 2, normalize, mask)
        wide = torch.full((2, 33, 40), math.nan, dtype=dtype, device="cuda")
        wide[:, :, 5:26] = x
        flat = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
        flat[1:] = x.reshape(-1)
        masks = torch.zeros(33, 2, dtype=torch.bool, device="cuda").t()
        masks.copy_(mask)
        for y in (wide[:, :, 5:26], flat[1:].view(2, 33, 21), x.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
            for mm in (mask, masks):
                leaf = y.detach().requires_grad_(True)
                out = route_tokens(leaf, RouteConfig(top_k=2, normalize=normalize), mm)
                up = _normal(7, 2, 33, 2).transpose(0, 1).contiguous().transpose(0, 1)
                (got,) = torch.autograd.grad(out.weights, leaf, up)
                for a, b in zip((*want, grad), (*out, got)):
                    assert torch.equal(a, b)


def test_route_results_changed_in_place() -> None:
    leaf = _scores((20,), 8, F32).requires_grad_(True)
    out = route_tokens(leaf, RouteConfig(top_k=2))
    out.experts.clamp_(max=3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.weights.sum(), leaf)
    out = route_tokens(leaf, RouteConfig(top_k=2))
    doubled = out.weights.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(doubled.sum(), leaf)


def test_route_keeps_nothing_alive() -> None:
    """A result that nobody holds leaves no memory behind."""
    leaf = _scores((4000,), 256, F32).requires_grad_(True)
    route_tokens(leaf, RouteConfig(top_k=8))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        route_tokens(leaf, RouteConfig(top_k=8))
    assert torch.cuda.memory_allocated() == before


@pytest.mark.parametrize("normalize", [True, False])
def test_route_keeps_scores_only_where_they_are_read(normalize) -> None:
    """Normalised weights' gradient needs the weights alone: the scores' memory is free,
    and they may be changed, before the backward."""
    leaf = _scores((4000,), 256, F32).requires_grad_(True)
    cfg, up = RouteConfig(top_k=8, normalize=normalize), _normal(7, 4000, 8)
    (want,) = torch.autograd.grad(route_tokens(leaf, cfg).weights, leaf, up)
    scores = leaf * 1.0
    out = route_tokens(scores, cfg)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    del scores
    assert before - torch.cuda.memory_allocated() == (4000 * 256 * 4 if normalize else 0)
    assert torch.equal(torch.autograd.grad(out.weights, leaf, up)[0], want)
    scores = leaf * 1.0
    out = route_tokens(scores, cfg)
    scores.fill_(-math.inf)
    if normalize:
        assert torch.equal(torch.autograd.grad(out.weights, leaf, up)[0], want)
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out.weights, leaf, up)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_has_no_second_derivative_in_the_scores(normalize) -> None:
    leaf = _scores((20,), 8, F32).requires_grad_(True)
    for scores in (leaf, leaf * 1.0):
        out = route_tokens(scores, RouteConfig(top_k=2, normalize=normalize))
        (g,) = torch.autograd.grad(out.weights, leaf, torch.ones_like(out.weights), create_graph=True)
        with pytest.raises(RuntimeError, match="only once"):
            torch.autograd.grad(g.sum(), leaf)


# -------------------------------------------------------------------- order


def _order_exact(experts, count):
    flat = experts.reshape(-1).tolist()
    slots = sorted((s for s, e in enumerate(flat) if 0 <= e < count), key=lambda s: flat[s])
    place = [-1] * len(flat)
    for at, s in enumerate(slots):
        place[s] = at
    offsets = [0] * (count + 1)
    for s in slots:
        offsets[flat[s] + 1] += 1
    for e in range(count):
        offsets[e + 1] += offsets[e]
    return offsets, slots + [-1] * (len(flat) - len(slots)), place


def _choices(tokens, k, count, share=0.0, seed=0):
    e = torch.randint(count, (tokens, k), generator=_gen(seed), device="cuda")
    e = torch.minimum(e, torch.randint(count, (tokens, k), generator=_gen(seed + 1), device="cuda"))  # uneven
    return torch.where(torch.rand(tokens, k, generator=_gen(seed + 2), device="cuda") < share, -1, e)


@pytest.mark.parametrize("count", [1, 2, 3, 8, 64, 100, 511, 512])
@pytest.mark.parametrize("tokens,k", [(0, 2), (1, 1), (1, 7), (31, 2), (33, 2), (64, 1), (257, 4), (2047, 2), (2048, 2),
                                      (2049, 2), (4096, 2), (4097, 2), (5000, 3), (70001, 2)])
def test_order(tokens, k, count) -> None:
    for share in (0.0, 0.3, 1.0):
        e = _choices(tokens, k, count, share)
        got = expert_order(e, count)
        assert got.offsets.shape == (count + 1,) and got.place.shape == (tokens, k)
        for a, b in zip(got, _order_exact(e, count)):
            assert a.dtype == torch.int64 and a.flatten().tolist() == b


def test_order_of_a_whole_batch() -> None:
    """2^21 slots, more than the blocks take in one round each; one expert alone, and
    the same expert twice in a token."""
    for count, e in ((512, _choices(1 << 20, 2, 512, 0.1)), (7, torch.full((1 << 20, 2), 3, device="cuda"))):
        got = expert_order(e, count)
        flat = e.flatten()
        want = torch.sort(torch.where(flat >= 0, flat, count), stable=True).indices
        routed = int((flat >= 0).sum())
        assert got.offsets[-1] == routed and torch.equal(got.source[:routed], want[:routed])
        assert (got.source[routed:] == -1).all()
        assert torch.equal(got.offsets, torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"),
                                                   torch.bincount(flat[flat >= 0], minlength=count).cumsum(0)]))
        assert torch.equal(got.place.flatten()[got.source[:routed]], torch.arange(routed, device="cuda"))
        assert (got.place.flatten()[flat < 0] == -1).all()


def test_order_types_strides_and_strays() -> None:
    e = _choices(300, 4, 20, 0.2)
    want = expert_order(e, 20)
    odd = torch.where(e < 0, torch.tensor([-1, 20, 1 << 40, -(1 << 62)], device="cuda"), e)
    for other in (odd, e.int(), e.short(), e.to(torch.int8), torch.where(e < 0, 255, e).to(torch.uint8),
                  e.t().contiguous().t(), torch.stack([e, e], -1)[..., 0]):
        for a, b in zip(expert_order(other, 20), want):
            assert torch.equal(a, b)
    one = expert_order(torch.tensor([3, 1], device="cuda"), 4)
    assert one.offsets.tolist() == [0, 0, 1, 1, 2] and one.source.tolist() == [1, 0] and one.place.tolist() == [1, 0]


# --------------------------------------------------------------------- rows


def _rows_step(dtype, tokens, width, k, count, share=0.0, seed=0, weighted=True):
    """to_experts and from_experts with all gradients against the definitions."""
    order = expert_order(_choices(tokens, k, count, share, seed), count)
    routed, slots = int(order.offsets[-1]), tokens * k
    slot = order.source[:routed]
    token = slot // k
    x = _normal(seed, tokens, width).to(dtype).requires_grad_(True)
    rows = to_experts(x, order)
    assert rows.shape == (slots, width) and torch.equal(rows[:routed], x[token]) and not rows[routed:].any()
    g = _normal(seed + 1, slots, width).to(dtype)
    (dx,) = torch.autograd.grad(rows, x, g)
    zero = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
    want = zero.index_add(0, token, g[:routed].double())
    size = zero.index_add(0, token, g[:routed].double().abs())
    assert ((dx.double() - want).abs() <= (k + 1) * U * size + _half(dtype, want)).all()

    rows = _normal(seed + 2, slots, width).to(dtype)
    rows[routed:] = math.nan  # not read
    rows.requires_grad_(True)
    w = torch.rand(tokens, k, generator=_gen(seed + 3), device="cuda") if weighted else None
    flat = w.flatten()[slot].double()[:, None] if weighted else torch.ones(routed, 1, device="cuda").double()
    if weighted:
        w.requires_grad_(True)
    out = from_experts(rows, order, w)
    assert out.shape == (tokens, width) and out.dtype == dtype
    each = rows.detach()[:routed].double() * flat.detach()
    want, size = zero.index_add(0, token, each), zero.index_add(0, token, each.abs())
    assert ((out.double() - want).abs() <= (k + 1) * U * size + _half(dtype, want)).all()
    g = _normal(seed + 4, tokens, width).to(dtype)
    grads = torch.autograd.grad(out, (rows, w) if weighted else (rows,), g)
    want = g.double()[token] * flat.detach()
    assert ((grads[0][:routed].double() - want).abs() <= U * want.abs() + _half(dtype, want)).all()
    assert not grads[0][routed:].any()
    if weighted:
        each = rows.detach()[:routed].double() * g.double()[token]
        want = torch.zeros(slots, dtype=torch.float64, device="cuda").index_copy(0, slot, each.sum(1))
        size = torch.zeros(slots, dtype=torch.float64, device="cuda").index_copy(0, slot, each.abs().sum(1))
        assert grads[1].dtype == F32 and grads[1].shape == (tokens, k)
        assert ((grads[1].flatten().double() - want).abs() <= (width / 64 + 8) * U * size).all()
    return order


@TYPES
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 256, 511, 512, 513, 1000, 1023, 1024, 1025, 2047, 2048, 2049,
                                   4097, 8192, 20001])
def test_rows_widths(width, dtype) -> None:
    say(f"rows {width} {dtype}")
    _rows_step(dtype, 37, width, 3, 9, 0.3)
    _rows_step(dtype, 5, width, 1, 4)


@TYPES
@pytest.mark.parametrize("tokens,k,count", [(0, 2, 4), (1, 1, 1), (1, 16, 512), (2, 5, 7), (1000, 8, 64), (333, 13, 40), (20000, 2, 16)])
def test_rows_tokens(tokens, k, count, dtype) -> None:
    for share in (0.0, 0.3, 1.0):
        _rows_step(dtype, tokens, 72, k, count, share, seed=k)
        _rows_step(dtype, tokens, 72, k, count, share, seed=k, weighted=False)


@TYPES
@pytest.mark.parametrize("k", [63, 64, 65, 130])
def test_rows_of_many_choices(k, dtype) -> None:
    """More choices than a wave has lanes, the same expert many times among them."""
    _rows_step(dtype, 9, 200, k, 5, 0.2)
    _rows_step(dtype, 9, 200, k, 5, 0.2, weighted=False)


def test_a_wide_row() -> None:
    _rows_step(BF16, 3, 1 << 20, 2, 4)


@TYPES
def test_rows_beyond_the_caches(dtype) -> None:
    """More than 224 MB of rows, whose stores go past the caches; a row no whole number
    of pieces."""
    _rows_step(dtype, 45000, 1001, 2, 30, 0.1)
    _rows_step(dtype, 45000, 1001, 2, 30, 0.1, weighted=False)


@TYPES
def test_rows_strides_offsets_and_shapes(dtype) -> None:
    e = _choices(6, 2, 5, 0.2).view(2, 3, 2)
    order = expert_order(e, 5)
    assert order.place.shape == (2, 3, 2)
    x = _normal(0, 2, 3, 40).to(dtype)
    want = to_experts(x, order)
    assert torch.equal(want, to_experts(x.view(6, 40), expert_order(e.view(6, 2), 5)))
    flat = torch.empty(241, dtype=dtype, device="cuda")
    flat[1:] = x.flatten()
    turned = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    wide = torch.stack([x, x], -1)[..., 0]
    place = order.place.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    source = torch.stack([order.source, order.source], -1)[:, 0]
    for y in (flat[1:].view(2, 3, 40), turned, wide):
        leaf = y.detach().requires_grad_(True)
        rows = to_experts(leaf, order._replace(place=place, source=source))
        assert torch.equal(rows, want)
        g = _normal(1, 40, 12).to(dtype).t()
        (dx,) = torch.autograd.grad(rows, leaf, g)
        assert dx.shape == (2, 3, 40)
        assert torch.equal(dx, torch.autograd.grad(to_experts(z := x.clone().requires_grad_(True), order), z, g.contiguous())[0])
    w = torch.rand(2, 3, 2, generator=_gen(5), device="cuda")
    out = from_experts(want, order, w)
    assert out.shape == (2, 3, 40)
    assert torch.equal(out, from_experts(want.t().contiguous().t(), order, w.permute(2, 0, 1).contiguous().permute(1, 2, 0)))
    odd = torch.empty(481, dtype=dtype, device="cuda")
    odd[1:] = want.flatten()
    assert torch.equal(out, from_experts(odd[1:].view(12, 40), order, w))
    # weights of another type are taken to float32, and their gradient back
    half = w.bfloat16().requires_grad_(True)
    y = from_experts(want, order, half)
    assert torch.equal(y, from_experts(want, order, half.detach().float()))
    assert torch.autograd.grad(y.sum(), half)[0].dtype == BF16


def _consistent(order):
    """The slots that are at a row, and their rows, of any order."""
    place, source = order.place.flatten(), order.source
    n = len(source)
    at = torch.where((place >= 0) & (place < n), place, 0)
    there = (place >= 0) & (place < n) & (source[at] == torch.arange(n, device="cuda"))
    slots = there.nonzero()[:, 0]
    return slots, place[slots]


@TYPES
@pytest.mark.parametrize("kind", ["dropped", "capacity", "strays", "twice", "source"])
def test_orders_that_a_caller_has_changed(kind, dtype) -> None:
    """Places of -1, places outside the rows, the same place twice, sources that do not
    fit: a slot is at a row where both agree, every row that none is at is 0 and gets a
    gradient of 0, and nothing else is read."""
    tokens, k, count, width = 40, 3, 6, 72
    experts = _choices(tokens, k, count)
    order = expert_order(experts, count)
    place, source = order.place.clone(), order.source.clone()
    pick = torch.rand(tokens, k, generator=_gen(9), device="cuda") < 0.3
    if kind == "dropped":
        place[pick] = -1
    elif kind == "capacity":
        late = place - order.offsets[experts] >= 10
        assert late.any()
        place[late] = -1
    elif kind == "strays":
        place[pick] = torch.randint(-(1 << 40), 1 << 40, (int(pick.sum()),), generator=_gen(1), device="cuda")
    elif kind == "twice":
        place[pick] = 5
    else:
        source[::4] = torch.randint(-200, 200, (len(source[::4]),), generator=_gen(2), device="cuda")
    order = order._replace(place=place, source=source)
    slots, at = _consistent(order)
    assert 0 < len(slots) < tokens * k
    empty = torch.ones(tokens * k, dtype=torch.bool, device="cuda").index_fill(0, at, False)
    x = _normal(0, tokens, width).to(dtype).requires_grad_(True)
    rows = to_experts(x, order)
    assert torch.equal(rows[at], x[slots // k]) and not rows[empty].any()
    g = _normal(1, tokens * k, width).to(dtype)
    g[empty] = math.nan
    (dx,) = torch.autograd.grad(rows, x, g)
    zero = torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
    want, size = zero.index_add(0, slots // k, g[at].double()), zero.index_add(0, slots // k, g[at].double().abs())
    assert ((dx.double() - want).abs() <= (k + 1) * U * size + _half(dtype, want)).all()
    rows = rows.detach().masked_fill(empty[:, None], math.nan).requires_grad_(True)
    w = torch.rand(tokens, k, generator=_gen(3), device="cuda").requires_grad_(True)
    out = from_experts(rows, order, w)
    each = rows.detach()[at].double() * w.detach().flatten()[slots].double()[:, None]
    want, size = zero.index_add(0, slots // k, each), zero.index_add(0, slots // k, each.abs())
    assert ((out.double() - want).abs() <= (k + 1) * U * size + _half(dtype, want)).all()
    g = _normal(4, tokens, width).to(dtype)
    d_rows, d_w = torch.autograd.grad(out, (rows, w), g)
    want = g[slots // k].double() * w.detach().flatten()[slots].double()[:, None]
    assert ((d_rows[at].double() - want).abs() <= U * want.abs() + _half(dtype, want)).all() and not d_rows[empty].any()
    each = rows.detach()[at].double() * g[slots // k].double()
    want, size = torch.zeros(2, tokens * k, dtype=torch.float64, device="cuda")
    want, size = want.index_copy(0, slots, each.sum(1)), size.index_copy(0, slots, each.abs().sum(1))
    assert ((d_w.flatten().double() - want).abs() <= (width / 64 + 8) * U * size).all()


def test_one_gradient_alone() -> None:
    order = expert_order(_choices(50, 2, 6, 0.2), 6)
    rows, w = _normal(0, 100, 96).to(BF16), torch.rand(50, 2, generator=_gen(1), device="cuda")
    g = _normal(2, 50, 96).to(BF16)
    a, b = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(from_experts(a, order, b), (a, b), g)
    assert torch.equal(torch.autograd.grad(from_experts(a, order, w), a, g)[0], both[0])
    assert torch.equal(torch.autograd.grad(from_experts(rows, order, b), b, g)[0], both[1])
    assert torch.equal(torch.autograd.grad(from_experts(a, order, b), b, g)[0], both[1])


def test_rows_changed_in_place() -> None:
    order = expert_order(_choices(50, 2, 6), 6)
    leaf, w = _normal(0, 100, 32).requires_grad_(True), torch.rand(50, 2, device="cuda").requires_grad_(True)
    rows = leaf * 1.0
    out = from_experts(rows, order, w)
    rows.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.sum(), w)
    x = _normal(0, 50, 32).requires_grad_(True)
    y = to_experts(x, order)
    order.place.clamp_(max=3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


def test_derivatives_that_are_refused() -> None:
    import torch.autograd.forward_ad as fwd

    order = expert_order(_choices(20, 2, 6), 6)
    scores, x, rows = _scores((20,), 6, F32), _normal(0, 20, 16), _normal(1, 40, 16)
    w = torch.rand(20, 2, device="cuda")
    calls = [(lambda t: route_tokens(t, RouteConfig(top_k=2)).weights, scores), (lambda t: to_experts(t, order), x),
             (lambda t: from_experts(t, order, w), rows), (lambda t: from_experts(rows, order, t), w)]
    for call, t in calls:
        leaf = t.clone().requires_grad_(True)
        out = call(leaf)
        up = torch.ones_like(out).requires_grad_(True)
        (g,) = torch.autograd.grad(out, leaf, up, create_graph=True)
        with pytest.raises(RuntimeError, match="only once"):
            torch.autograd.grad(g.sum(), up, allow_unused=True)
        with fwd.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(fwd.make_dual(t, torch.ones_like(t)))
            out = call(leaf)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, fwd.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_negative_bit() -> None:
    def neg(t):
        return torch._neg_view(-t)

    scores = _scores((50,), 8, F32)
    want, _ = _route(scores, 2)
    assert all(torch.equal(a, b) for a, b in zip(want, route_tokens(neg(scores), RouteConfig(top_k=2))))
    order = expert_order(want.experts, 8)
    x = _normal(0, 50, 24)
    rows = to_experts(x, order)
    assert torch.equal(rows, to_experts(neg(x), order))
    leaf = neg(rows.clone()).requires_grad_(True)
    w = neg(want.weights.detach()).requires_grad_(True)
    g = _normal(3, 50, 24)
    out = from_experts(leaf, order, w)
    plain = [rows.clone().requires_grad_(True), want.weights.detach().clone().requires_grad_(True)]
    ref = from_experts(plain[0], order, plain[1])
    assert torch.equal(out, ref)
    for a, b in zip(torch.autograd.grad(out, (leaf, w), neg(g)), torch.autograd.grad(ref, plain, g)):
        assert torch.equal(a, b)


def test_rows_past_32_bit_offsets() -> None:
    """400000 tokens x 4096 to two experts each, 3.3 G elements: rows at the end are what
    they should be, in both directions."""
    tokens, width = 400000, 4096
    order = expert_order(_choices(tokens, 2, 16, 0.01), 16)
    routed = int(order.offsets[-1])
    x = torch.empty(tokens, width, dtype=BF16, device="cuda").normal_(generator=_gen(1)).requires_grad_(True)
    rows = to_experts(x, order)
    for part in (slice(0, 50), slice(524280, 524300), slice(routed - 50, routed)):
        assert torch.equal(rows[part], x[order.source[part] // 2])
    assert not rows[routed:].any()
    w = torch.rand(tokens, 2, generator=_gen(2), device="cuda").requires_grad_(True)
    out = from_experts(rows, order, w)
    for part in (slice(0, 50), slice(tokens - 50, tokens)):
        each = (x[part].double() * (w[part] * (order.place[part] >= 0)).sum(1, keepdim=True)).detach()
        assert ((out[part].double() - each).abs() <= 6 * U * each.abs() + _half(BF16, each)).all()
    d_x, d_w = torch.autograd.grad(out, (x, w), out.detach())
    for part in (slice(0, 50), slice(tokens - 50, tokens)):
        dots = (x[part].double() * out[part].double()).detach()
        want = dots.sum(1, keepdim=True) * (order.place[part] >= 0)
        assert ((d_w[part].double() - want).abs() <= 80 * U * dots.abs().sum(1, keepdim=True)).all()
        # two rounded halves: a step of bfloat16 in all
        want = (out[part].double() * (w[part] * (order.place[part] >= 0)).sum(1, keepdim=True)).detach()
        assert ((d_x[part].double() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-30).all()


# ------------------------------------------------------------------ together


class _Experts(torch.nn.Module):
    """A layer of experts between a router and the sum, one product per expert."""

    def __init__(self, width, count, k, mode) -> None:
        super().__init__()
        gen = torch.Generator().manual_seed(0)
        self.router = torch.nn.Parameter(torch.randn(width, count, generator=gen) * 0.3)
        self.expert = torch.nn.Parameter(torch.randn(count, width, width, generator=gen) * 0.1)
        self.k, self.mode = k, mode

    def forward(self, x, mask):
        scores = x @ self.router
        count = scores.shape[-1]
        if self.mode == "own":
            routes = route_tokens(scores, RouteConfig(top_k=self.k), mask)
            order = expert_order(routes.experts, count)
            rows = to_experts(x, order)
            ends = order.offsets.tolist()
            done = [torch.tanh(rows[ends[e]:ends[e + 1]] @ self.expert[e]) for e in range(count)]
            done.append(rows[ends[-1]:])
            return from_experts(torch.cat(done), order, routes.weights), scores
        at = torch.sort(scores, dim=-1, descending=True, stable=True).indices[..., :self.k]
        w = torch.softmax(scores.gather(-1, at), -1) * mask[..., None]
        all_w = torch.zeros_like(scores).scatter(-1, at, w)
        mixed = torch.stack([torch.tanh(x @ self.expert[e]) for e in range(count)], -1)
        return (mixed * all_w[..., None, :]).sum(-1), scores


@pytest.mark.parametrize("k,share", [(1, 0.0), (2, 0.3), (8, 0.1)])
def test_a_layer_of_experts(k, share) -> None:
    """Output and all gradients of a layer against plain float64: float32 products of 48
    terms and tanh lose less than 1e-5."""
    own, ref = _Experts(48, 8, k, "own").cuda(), _Experts(48, 8, k, "plain").cuda().double()
    x = _normal(0, 3, 70, 48)
    mask = _mask((3, 70), share)
    up = _normal(1, 3, 70, 48)
    a, b = x.clone().requires_grad_(True), x.double().requires_grad_(True)
    y, scores = own(a, mask)
    want, _ = ref(b, mask)
    assert float((y.detach().double() - want.detach()).norm()) <= 1e-5 * float(want.detach().norm())
    balance = balance_loss(scores, BalanceConfig(top_k=k), mask)
    assert int(balance.counts.sum()) == k * int(mask.sum())
    got = torch.autograd.grad(y, (a, own.router, own.expert), up)
    for g, w in zip(got, torch.autograd.grad(want, (b, ref.router, ref.expert), up.double())):
        assert float((g.double() - w).norm()) <= 1e-5 * float(w.norm()) + 1e-12


def test_streams_and_captured_steps() -> None:
    """The whole way with its gradients on other streams, and in two captured graphs
    whose replays, with eager calls between them, equal the eager result."""
    def leaves(seed):
        return [_scores((3000,), 20, F32, seed).requires_grad_(True), _normal(seed, 3000, 72).to(BF16).requires_grad_(True)]

    def step(ls):
        routes = route_tokens(ls[0], RouteConfig(top_k=3))
        order = expert_order(routes.experts, 20)
        rows = to_experts(ls[1], order)
        out = from_experts(rows, order, routes.weights)
        return [*order, routes.experts, rows.detach(), out.detach(), *torch.autograd.grad(out, ls, torch.ones_like(out))]

    sets = [leaves(1), leaves(2)]
    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, step(sets[i])))
    torch.cuda.synchronize()
    for i, out in got:
        for a, b in zip(out, want[i]):
            assert torch.equal(a, b)
    del got, want
    graphs, held = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            held.append(step(sets[i]))
    for r in range(4):
        for i in range(2):
            with torch.no_grad():
                for leaf, new in zip(sets[i], leaves(10 + 2 * r + i)):
                    leaf.copy_(new)
            graphs[i].replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in held[i]]
            for a, b in zip(kept, step(sets[i])):
                assert torch.equal(a, b), f"replay {r} of graph {i}"
