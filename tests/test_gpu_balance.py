"""balance_loss on the GPU against its definition in float64.

u = 2^-24.  p is off relatively by at most 16 u (1 + the scores' range) (the
rounded argument of the exponential, the exponential, the sum and the quotient),
the float32 sums over T tokens by 4 sqrt(T) u, and a float32 result by u.  The
gradient is a difference, q - sum q p: its bound is relative to q + sum q p, and
half a step of the scores' type on top."""

from __future__ import annotations

import math

import pytest
import torch

from ace_kernels import BalanceConfig, balance_loss
from gpu_helpers import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
U = 2.0 ** -24


def _scores(lead, tokens, experts, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = 1.5 * torch.randn(*lead, tokens, experts, generator=gen) + torch.randn(experts, generator=gen)
    return x.to(dtype).cuda()


def _mask(lead, tokens, share, seed=1):
    return (torch.rand(*lead, tokens, generator=torch.Generator().manual_seed(seed)) >= share).cuda()


def _exact(x, k, mask, reduction, up):
    """(loss, counts, gradient, bounds of loss and gradient)."""
    dtype = x.dtype
    lead, (t, e) = x.shape[:-2], x.shape[-2:]
    s = x.detach().double().reshape(-1, t, e)
    g = s.shape[0]
    on = torch.ones(g, t, dtype=torch.bool, device=x.device) if mask is None else mask.reshape(g, t)
    order = torch.sort(torch.where(s.isnan(), math.inf, s), dim=2, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, torch.arange(e, device=x.device).expand(g, t, e).contiguous())
    n = ((rank < k) & on[:, :, None]).sum(1)
    m = on.sum(1).clamp(min=1).double()
    p = torch.where(on[:, :, None], torch.softmax(torch.where(on[:, :, None], s, 0.0), 2), 0.0)
    q = e * n / (k * m * m)[:, None]
    loss = (q * p.sum(1)).sum(1)
    spread = float((torch.where(on[:, :, None], s, 0.0).abs().amax())) * 2 if s.numel() else 0.0
    rel = 16 * U * (1 + spread) + 4 * math.sqrt(max(1, t)) * U
    tol_loss = loss * rel
    if reduction == "none":
        w = up.reshape(g, 1, 1).double()
        loss, tol_loss = loss.reshape(lead), tol_loss.reshape(lead)
    else:
        w = up.double() * (1.0 / g if reduction == "mean" else 1.0)
        loss, tol_loss = loss.sum() * (1.0 / g if reduction == "mean" else 1), tol_loss.sum() * (1.0 / g if reduction == "mean" else 1)
    pull = (p * q[:, None]).sum(2, keepdim=True)
    grad = w * p * (q[:, None] - pull)
    half = torch.finfo(dtype).eps / 2
    tol = (w.abs() * p * (q[:, None] + pull)) * (2 * rel + 4 * math.sqrt(e) * U) + half * grad.abs() + torch.finfo(dtype).tiny * half
    return loss, n.reshape(*lead, e), grad.reshape(x.shape), tol_loss + U * loss, tol.reshape(x.shape)


def _compare(x, k, mask=None, reduction="mean", up=None):
    up = torch.tensor(0.7, device="cuda") if up is None else up
    want, n, d, tol, tol_d = _exact(x, k, mask, reduction, up)
    leaf = x.detach().clone().requires_grad_(True)
    out = balance_loss(leaf, BalanceConfig(top_k=k, reduction=reduction), mask)
    (got,) = torch.autograd.grad(out.loss, leaf, up)
    assert out.loss.dtype == F32 and out.counts.dtype == torch.int64 and got.dtype == x.dtype
    assert torch.equal(out.counts, n)
    assert ((out.loss.double() - want).abs() <= tol).all()
    err = (got.double() - d).abs()
    assert (err <= tol_d).all(), f"gradient: worst {float((err / tol_d).max()):.3g} x bound"
    return out, got


# every number of lanes a token and scores a lane, rows that end inside a piece
# and those shorter than one
@TYPES
@pytest.mark.parametrize("experts", [1, 2, 3, 5, 7, 8, 9, 12, 16, 17, 31, 33, 60, 64, 65, 100, 128, 130, 250, 256, 257, 511, 512])
def test_experts(experts, dtype) -> None:
    say(f"balance {experts} {dtype}")
    for k in sorted({1, min(2, experts), min(3, experts), min(6, experts), min(8, experts), min(16, experts)}):
        _compare(_scores((), 133, experts, dtype, seed=experts), k, _mask((), 133, 0.2, seed=k))


@TYPES
@pytest.mark.parametrize("lead,tokens", [((), 1), ((3,), 1), ((2, 3), 17), ((), 4097), ((5,), 1000), ((), 100003), ((300,), 40),
                                         ((33,), 2000), ((40, 40), 5)])
def test_groups_and_lengths(lead, tokens, dtype) -> None:
    x = _scores(lead, tokens, 24, dtype, seed=tokens)
    _compare(x, 2)
    mask = _mask(lead, tokens, 0.4)
    _compare(x, 2, mask)
    _compare(x, 2, mask, "sum")
    _compare(x, 2, mask, "none", torch.randn(lead, generator=torch.Generator().manual_seed(3)).cuda())


@TYPES
def test_empty_groups_and_no_tokens(dtype) -> None:
    x = _scores((3,), 50, 16, dtype)
    mask = _mask((3,), 50, 0.3)
    mask[1] = False
    out, grad = _compare(x, 2, mask, "none", torch.ones(3, device="cuda"))
    assert out.loss[1] == 0 and not grad[1].any() and not out.counts[1].any()
    out, grad = _compare(x, 2, torch.zeros_like(mask))
    assert out.loss == 0 and not grad.any()
    none = torch.empty(2, 0, 16, dtype=dtype, device="cuda", requires_grad=True)
    out = balance_loss(none, BalanceConfig(top_k=2))
    assert out.loss == 0 and not out.counts.any()
    assert torch.autograd.grad(out.loss, none)[0].shape == (2, 0, 16)


@TYPES
def test_masked_tokens_are_not_read(dtype) -> None:
    x = _scores((2,), 90, 20, dtype)
    mask = _mask((2,), 90, 0.5)
    want, grad = _compare(x, 3, mask)
    dirty = x.clone()
    dirty[~mask] = float("nan")
    dirty[0, int((~mask[0]).nonzero()[0])] = float("inf")
    leaf = dirty.requires_grad_(True)
    out = balance_loss(leaf, BalanceConfig(top_k=3), mask)
    assert torch.equal(out.loss, want.loss) and torch.equal(out.counts, want.counts)
    (got,) = torch.autograd.grad(out.loss, leaf, torch.tensor(0.7, device="cuda"))
    assert torch.equal(got, grad)


@TYPES
@pytest.mark.parametrize("experts", [6, 40, 64, 200, 256, 400])
def test_ties_go_to_the_lowest_expert(experts, dtype) -> None:
    gen = torch.Generator().manual_seed(experts)
    few = torch.randint(-1, 2, (300, experts), generator=gen).float()  # many equal scores
    few[:100] = 0.0
    few[100:150] *= -0.0
    for k in (1, 2, 5):
        out, _ = _compare(few.to(dtype).cuda(), k)
    same = torch.zeros(64, experts, dtype=dtype, device="cuda")
    out, _ = _compare(same, 5)
    assert (out.counts[:5] == 64).all() and not out.counts[5:].any()
    assert abs(float(out.loss) - 1) < 1e-6


@TYPES
def test_experts_at_minus_infinity(dtype) -> None:
    """Experts that are closed (-inf, or the type's lowest value) take nothing
    while others are open, and their gradient is 0."""
    for closed in (-math.inf, torch.finfo(dtype).min):
        x = _scores((), 200, 30, dtype)
        x[:, 7:20] = closed
        _, grad = _compare(torch.nan_to_num(x, neginf=torch.finfo(dtype).min) if closed == -math.inf else x, 4)
        leaf = x.clone().requires_grad_(True)
        out = balance_loss(leaf, BalanceConfig(top_k=4))
        (got,) = torch.autograd.grad(out.loss, leaf, torch.tensor(0.7, device="cuda"))
        assert not out.counts[7:20].any() and not got[:, 7:20].any() and torch.equal(got, grad)


@TYPES
def test_nan_stays_in_its_group(dtype) -> None:
    x = _scores((2,), 70, 16, dtype)
    x[1, 3, 5] = float("nan")
    out = balance_loss(x, BalanceConfig(top_k=2, reduction="none"))
    assert torch.isnan(out.loss[1]) and not torch.isnan(out.loss[0])
    assert out.counts[1].sum() == 140 and out.counts[1, 5] >= 1


def test_gradient_against_differences() -> None:
    x = _scores((2,), 60, 12, F32)
    mask = _mask((2,), 60, 0.2)
    leaf = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(balance_loss(leaf, BalanceConfig(top_k=2), mask).loss, leaf)
    n = balance_loss(x, BalanceConfig(top_k=2), mask).counts.double()
    m = mask.sum(1).double()
    way = torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).cuda().double()

    def f(t):  # the counts are constants
        p = torch.softmax(x.double() + t * way, 2) * mask[:, :, None]
        return float((12 * n / (2 * m * m)[:, None] * p.sum(1)).sum(1).mean())

    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(float((got.double() * way).sum()) - want) <= 1e-5 * (1 + abs(want))


@TYPES
def test_strides_and_offsets(dtype) -> None:
    x = _scores((2,), 33, 21, dtype)
    mask = _mask((2,), 33, 0.3)
    want, grad = _compare(x, 2, mask)
    wide = torch.full((2, 33, 40), float("nan"), dtype=dtype, device="cuda")
    wide[:, :, 5:26] = x
    flat = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
    flat[1:] = x.reshape(-1)
    masks = torch.zeros(33, 2, dtype=torch.bool, device="cuda").t()
    masks.copy_(mask)
    for y in (wide[:, :, 5:26], flat[1:].view(2, 33, 21), x.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        for mm in (mask, masks):
            leaf = y.detach().requires_grad_(True)
            out = balance_loss(leaf, BalanceConfig(top_k=2), mm)
            assert torch.equal(out.loss, want.loss) and torch.equal(out.counts, want.counts)
            (got,) = torch.autograd.grad(out.loss, leaf, torch.tensor(0.7, device="cuda"))
            assert torch.equal(got, grad)


def test_same_bits_again_and_streams() -> None:
    a, b = _scores((4,), 5000, 64, BF16, seed=1), _scores((), 30000, 256, F32, seed=2)
    cfg = BalanceConfig(top_k=6)
    want = [balance_loss(x, cfg) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got.append((i, balance_loss(x, cfg)))
    torch.cuda.synchronize()
    for i, o in got:
        assert torch.equal(o.loss, want[i].loss) and torch.equal(o.counts, want[i].counts)


def test_captured_steps_replay() -> None:
    """Two captured graphs with calls of several blocks, replayed in turn with
    eager calls in between; every replay equals the eager result."""
    cfg = BalanceConfig(top_k=4)
    leaves = [_scores((3,), 3000, 64, BF16, seed=i).requires_grad_(True) for i in range(2)]
    masks = [_mask((3,), 3000, 0.2, seed=i) for i in range(2)]

    def step(i):
        out = balance_loss(leaves[i], cfg, masks[i])
        return [out.loss, out.counts, *torch.autograd.grad(out.loss, leaves[i], torch.ones_like(out.loss))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, held = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            held.append(step(i))
    for r in range(4):
        for i in range(2):
            with torch.no_grad():
                leaves[i].copy_(_scores((3,), 3000, 64, BF16, seed=50 + 2 * r + i))
            graphs[i].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held[i]]
            for a, b in zip(got, step(i)):
                assert torch.equal(a, b), f"replay {r} of graph {i}"


def test_second_derivative_is_refused() -> None:
    leaf = _scores((), 20, 8, F32).requires_grad_(True)
    (g,) = torch.autograd.grad(balance_loss(leaf, BalanceConfig(top_k=2)).loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), leaf)


def test_forward_mode_is_refused() -> None:
    """In the call and in its backward: nothing comes back without its tangent."""
    import torch.autograd.forward_ad as fwd

    x, cfg = _scores((), 20, 8, F32), BalanceConfig(top_k=2)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            balance_loss(fwd.make_dual(x, torch.ones_like(x)), cfg)
        leaf = x.clone().requires_grad_(True)
        loss = balance_loss(leaf, cfg).loss
        up = fwd.make_dual(torch.ones_like(loss), torch.ones_like(loss))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(loss, leaf, up)


def test_second_derivative_in_the_upstream_gradient_is_refused() -> None:
    leaf = _scores((), 20, 8, F32).requires_grad_(True)
    loss = balance_loss(leaf, BalanceConfig(top_k=2)).loss
    up = torch.ones_like(loss).requires_grad_(True)
    (g,) = torch.autograd.grad(loss, leaf, up, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        torch.autograd.grad(g.sum(), up, allow_unused=True)


def test_scores_past_32_bit_offsets() -> None:
    """Five groups of 2^20 tokens and 512 experts, 2.7 G scores: each group is what it is
    alone, the last one's elements beyond 2^31."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(5, 1 << 20, 512, dtype=BF16, device="cuda").normal_(generator=gen)
    mask = torch.rand(5, 1 << 20, device="cuda", generator=gen) < 0.9
    cfg = BalanceConfig(top_k=4, reduction="none")
    leaf = x.requires_grad_(True)
    out = balance_loss(leaf, cfg, mask)
    up = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0], device="cuda") * 2.0 ** 20
    (grad,) = torch.autograd.grad(out.loss, leaf, up)
    for g in (0, 4):
        one = x[g].detach().requires_grad_(True)
        alone = balance_loss(one, cfg, mask[g])
        (want,) = torch.autograd.grad(alone.loss, one, up[g])
        assert torch.equal(out.counts[g], alone.counts)
        # blocks sum in another order: 4 sqrt(T) u each
        assert abs(out.loss[g].item() - alone.loss.item()) <= 8 * 1024 * U * alone.loss.item()
        assert torch.equal(grad[g], want)  # a token's gradient is its own: the counts are the same
    # the last group's last tokens, from the definition
    n, m = out.counts[4].double(), mask[4].sum().double()
    p = torch.softmax(x[4, -1000:].detach().double(), 1)
    q = 512 * n / (4 * m * m)
    pull = (p * q).sum(1, keepdim=True)
    want = float(up[4]) * p * (q - pull) * mask[4, -1000:, None]
    tol = float(up[4]) * p * (q + pull) * (2 * 16 * U * 12 + 4 * 512 ** 0.5 * U) + 2.0 ** -8 * want.abs()
    assert ((grad[4, -1000:].double() - want).abs() <= tol).all()


def test_negative_bit() -> None:
    """Scores whose memory holds the negatives of their values."""
    x = _scores((2,), 50, 16, F32)
    want, grad = _compare(x, 3)
    leaf = torch._neg_view(-x).requires_grad_(True)
    out = balance_loss(leaf, BalanceConfig(top_k=3))
    (got,) = torch.autograd.grad(out.loss, leaf, torch._neg_view(torch.tensor(-0.7, device="cuda")))
    assert torch.equal(out.loss, want.loss) and torch.equal(out.counts, want.counts) and torch.equal(got, grad)
