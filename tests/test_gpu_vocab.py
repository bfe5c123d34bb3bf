"""vocab_loss and vocab_loss_confidence on the GPU against their definition in
float64, with derived bounds (vocab_reference.py)."""

from __future__ import annotations

import pytest
import torch

from ace_kernels import VocabConfig, vocab_loss, vocab_loss_confidence
from gpu_helpers import say
from vocab_reference import U, exact, inputs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol)[bad].max()):.3g} x bound"


def _step(hidden, weight, labels, config, go=None, gc=None):
    """(scores, gradients) of one calibrated step."""
    h = hidden.detach().clone().requires_grad_(True)
    w = weight.detach().clone().requires_grad_(True)
    out = vocab_loss_confidence(h, w, labels, config)
    go = torch.ones_like(out.loss) if go is None else go
    gc = torch.zeros_like(out.confidence) if gc is None else gc
    return out, torch.autograd.grad((out.loss, out.confidence), (h, w), (go, gc))


def _compare(hidden, weight, labels, config=VocabConfig(), go=None, gc=None):
    want = exact(hidden, weight, labels, config.ignore_index, config.reduction, go, gc)
    out, (dh, dw) = _step(hidden, weight, labels, config, go, gc)
    assert dh.dtype == hidden.dtype and dw.dtype == weight.dtype and out.loss.dtype == F32
    if config.reduction == "none":
        tol = want.tol_nll + 2 * U * want.loss.abs()
    else:
        tol = (want.tol_nll + 2 * U * float(want.nll.abs().max() if want.nll.numel() else 0)) * (
            1 if config.reduction == "mean" else max(1, labels.numel()))
    _within(out.loss, want.loss, tol, "loss")
    _within(out.confidence, want.confidence, want.tol_confidence * want.confidence + 1e-30, "confidence")
    assert torch.equal(out.correct[want.sure].double(), want.correct[want.sure])
    if want.sure.all() or gc is None:  # else the confidence's gradient may be another word's
        _within(dh, want.d_hidden, want.tol_hidden + 1e-30, "d hidden")
        _within(dw, want.d_weight, want.tol_weight + 1e-30, "d weight")
    return out, (dh, dw)


# every tile and its borders; hidden sizes below, at and between a step of k,
# and those whose rows are no whole 16 bytes; vocabularies of one word and up
SIZES = [
    (1, 8, 1), (1, 64, 2), (3, 1, 5), (2, 7, 300), (17, 72, 129), (31, 128, 1000), (32, 100, 257), (33, 64, 128),
    (64, 200, 640), (65, 33, 1001), (128, 96, 384), (129, 512, 255), (255, 264, 2049), (300, 1000, 513),
    (520, 64, 70), (1030, 40, 33), (700, 136, 5003),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,size,v", SIZES)
def test_sizes(n, size, v, dtype) -> None:
    say(f"vocab {n}x{size}x{v} {dtype}")
    hidden, weight, labels = inputs(n, size, v, dtype, seed=n + v, ignored=0.2)
    gen = torch.Generator().manual_seed(5)
    go = torch.tensor(0.7, device="cuda")
    gc = (torch.randn(n, generator=gen) / n).cuda()
    _compare(hidden, weight, labels, VocabConfig(), go, gc)


def _drawn(seed):
    gen = torch.Generator().manual_seed(seed)

    def between(low, high):
        return int(round(low * (high / low) ** float(torch.rand((), generator=gen))))

    n, size, v = between(1, 3000), between(3, 700), between(2, 9000)
    if float(torch.rand((), generator=gen)) < 0.5:
        size = max(8, size // 8 * 8)
    share = [0.0, 0.3, 0.9][int(torch.randint(3, (), generator=gen))]
    return n, size, v, [F32, BF16, F16][seed % 3], share


@pytest.mark.parametrize("seed", range(48))
def test_drawn_sizes(seed) -> None:
    """Tiles, cuts of the work and edges that nobody thought of: the counted
    tokens' number is known on the device only."""
    n, size, v, dtype, share = _drawn(seed)
    say(f"vocab drawn {n}x{size}x{v} {dtype} ignored {share}")
    hidden, weight, labels = inputs(n, size, v, dtype, seed=seed, ignored=share)
    gc = (torch.randn(n, generator=torch.Generator().manual_seed(seed)) / n).cuda() if seed % 2 else None
    reduction = ["mean", "sum", "none"][seed // 3 % 3]
    _compare(hidden, weight, labels, VocabConfig(reduction=reduction), None, gc)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions(reduction, dtype) -> None:
    n = 150
    hidden, weight, labels = inputs(n, 128, 777, dtype, seed=3, ignored=0.3)
    gen = torch.Generator().manual_seed(6)
    go = torch.randn(n if reduction == "none" else (), generator=gen).cuda()
    _compare(hidden, weight, labels, VocabConfig(reduction=reduction), go, torch.randn(n, generator=gen).cuda())


@pytest.mark.parametrize("n,size,v", [(2100, 128, 8200), (6000, 64, 30000), (9000, 72, 1024), (70000, 40, 300),
                                      (3, 24, 200000), (40, 1024, 60000)])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_large_tiles_and_pieces(n, size, v, dtype) -> None:
    """The 256-wide tiles; 6000 x 30000 takes two pieces of the vocabulary;
    9000 tokens of a small head share out the tokens of the weight's gradient; 70000
    have more token tiles than blocks; few tokens of a long vocabulary have the
    hidden gradient in many partial tiles."""
    hidden, weight, labels = inputs(n, size, v, dtype, seed=8, ignored=0.4)
    _compare(hidden, weight, labels, VocabConfig(), torch.tensor(1.0, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_nothing_counted(dtype) -> None:
    hidden, weight, _ = inputs(40, 64, 100, dtype)
    for labels in (torch.full((40,), -100), torch.full((40,), 100), torch.full((40,), -1)):
        out, (dh, dw) = _step(hidden, weight, labels.cuda(), VocabConfig())
        assert out.loss.item() == 0 and not out.confidence.any() and not out.correct.any()
        assert not dh.any() and not dw.any()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_tokens(reduction) -> None:
    _, weight, _ = inputs(1, 64, 100, BF16)
    hidden = torch.empty(0, 64, dtype=BF16, device="cuda")
    out, (dh, dw) = _step(hidden, weight, torch.empty(0, dtype=torch.int64, device="cuda"), VocabConfig(reduction=reduction))
    assert out.loss.shape == ((0,) if reduction == "none" else ()) and not out.loss.any()
    assert dh.shape == (0, 64) and not dw.any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_ignored_tokens_are_not_read(dtype) -> None:
    """NaN and infinities in the hidden states of ignored tokens reach nothing,
    and the results are those of the counted tokens alone, bit for bit."""
    hidden, weight, labels = inputs(200, 96, 500, dtype, seed=4, ignored=0.5)
    gone = labels == -100
    hidden[gone] = float("nan")
    hidden[gone.nonzero()[0]] = float("inf")
    out, (dh, dw) = _compare(hidden.masked_fill(gone[:, None], 0), weight, labels)
    out2, (dh2, dw2) = _step(hidden, weight, labels, VocabConfig())
    for a, b in ((out.loss, out2.loss), (out.confidence, out2.confidence), (dh, dh2), (dw, dw2)):
        assert torch.equal(a, b)
    out3, (dh3, dw3) = _step(hidden[~gone], weight, labels[~gone], VocabConfig())
    assert torch.equal(out3.loss, out2.loss) and torch.equal(out3.confidence, out2.confidence[~gone])


def test_ignore_index_inside_the_vocabulary() -> None:
    hidden, weight, labels = inputs(90, 64, 50, F32, seed=2)
    _compare(hidden, weight, labels, VocabConfig(ignore_index=int(labels[0])))


def test_ties_go_to_the_lowest_word() -> None:
    """Equal rows of the weight give equal logits: the lowest index is the top
    label wherever the two lie (one lane, two lanes, two tiles, two blocks)."""
    hidden, weight, _ = inputs(40, 64, 3000, F32, seed=9)
    for low, high in ((5, 6), (5, 9), (5, 21), (5, 100), (5, 300), (100, 2999)):
        w = weight.clone()
        w[high] = w[low] = 20 * hidden[0] / hidden[0].norm()
        labels = torch.full((40,), low, device="cuda")
        top = (hidden.double() @ w.double().t()).argmax(1)
        assert vocab_loss_confidence(hidden, w, labels).correct[0] == 1
        labels.fill_(high)
        assert vocab_loss_confidence(hidden, w, labels).correct[0] == 0
        assert int(top[0]) in (low, high)


def test_nan_and_infinite_logits_stay_in_their_token() -> None:
    hidden, weight, labels = inputs(70, 64, 300, F32, seed=1)
    clean = vocab_loss(hidden, weight, labels, VocabConfig(reduction="none"))
    hidden[3, 5] = float("nan")
    hidden[40, 7] = float("inf")
    got = vocab_loss(hidden, weight, labels, VocabConfig(reduction="none"))
    assert torch.isnan(got[3]) and torch.isnan(got[40])
    keep = torch.ones(70, dtype=torch.bool, device="cuda")
    keep[[3, 40]] = False
    assert torch.equal(got[keep], clean[keep])


def test_words_at_minus_infinity() -> None:
    """A weight of the type's lowest value takes a word's probability to 0."""
    hidden, weight, labels = inputs(20, 64, 200, F32, seed=1)
    hidden[:, 0] = 1.0
    weight[150:, :] = 0.0
    weight[150:, 0] = torch.finfo(F32).min
    labels.clamp_(max=149)
    part = vocab_loss(hidden, weight[:150], labels)
    assert torch.allclose(vocab_loss(hidden, weight, labels), part, rtol=8 * U, atol=0)


def test_confident_tokens_keep_their_digits() -> None:
    """nll = log(1 + exp(-d)) of two words d apart, down to where it is below
    float32's step at the size of the logits."""
    d = torch.tensor([0.0, 1.0, 5.0, 10.0, 14.0], dtype=torch.float64)
    hidden = torch.zeros(5, 8)
    hidden[:, 0] = 1.0
    hidden[:, 1] = -d.float()
    hidden[:, 2] = 30.0
    weight = torch.zeros(2, 8)
    weight[:, 2] = 1.0
    weight[1, 1] = 1.0
    labels = torch.zeros(5, dtype=torch.int64)
    got = vocab_loss(hidden.cuda(), weight.cuda(), labels.cuda(), VocabConfig(reduction="none")).double().cpu()
    want = torch.log1p(torch.exp(-d))
    # the sum 1 + exp(-d) rounds at u; logits of 30 - d round at 16 u
    assert ((got - want).abs() <= 2 * U + 32 * U * torch.exp(-d)).all()


def test_gradient_against_differences() -> None:
    """A central difference of the float64 definition along a direction, at the
    kernels' own gradient."""
    hidden, weight, labels = inputs(60, 48, 211, F32, seed=12, ignored=0.2)
    gc = torch.randn(60, generator=torch.Generator().manual_seed(1)).cuda() / 60
    _, (dh, dw) = _step(hidden, weight, labels, VocabConfig(), None, gc)
    gen = torch.Generator().manual_seed(2)
    vh, vw = torch.randn(60, 48, generator=gen).cuda().double(), torch.randn(211, 48, generator=gen).cuda().double()

    def f(t):
        h, w = hidden.double() + t * vh, weight.double() + t * vw
        e = exact(h.double(), w.double(), labels)
        return float(e.loss + (gc.double() * e.confidence).sum())

    step = 1e-5
    want = (f(step) - f(-step)) / (2 * step)
    got = float((dh.double() * vh).sum() + (dw.double() * vw).sum())
    assert abs(got - want) <= 1e-5 * (1 + abs(want))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_strides_offsets_shapes_and_label_types(dtype) -> None:
    hidden, weight, labels = inputs(48, 72, 300, dtype, seed=7, ignored=0.2)
    want, (dh, dw) = _step(hidden, weight, labels, VocabConfig())
    wide = torch.full((48, 100), float("nan"), dtype=dtype, device="cuda")
    wide[:, 3:75] = hidden
    flat = torch.empty(300 * 72 + 3, dtype=dtype, device="cuda")
    flat[3:] = weight.reshape(-1)
    for h in (wide[:, 3:75], hidden.t().contiguous().t(), hidden):
        for w in (flat[3:].view(300, 72), weight.t().contiguous().t()):
            for y in (labels, labels.int(), labels.repeat_interleave(2)[::2]):
                out, (a, b) = _step(h, w, y, VocabConfig())
                assert torch.equal(out.loss, want.loss) and torch.equal(a, dh) and torch.equal(b, dw)
    out, (a, b) = _step(hidden.view(4, 12, 72), weight, labels.view(4, 12), VocabConfig(reduction="none"))
    assert out.loss.shape == out.confidence.shape == out.correct.shape == (4, 12) and a.shape == (4, 12, 72)
    one, (a, b) = _step(hidden[0], weight, labels[0], VocabConfig())
    assert one.loss.shape == one.confidence.shape == () and a.shape == (72,)


def test_float16_gradients_of_rare_words_survive() -> None:
    """Probabilities far below float16's smallest number, times a loss scale,
    still reach the weight's gradient."""
    n, size, v = 256, 64, 20000
    hidden, weight, labels = inputs(n, size, v, F16, seed=5)
    hidden = hidden + 12 * weight[labels]
    _compare(hidden, weight, labels, VocabConfig(), torch.tensor(65536.0, device="cuda"))


def test_one_gradient_alone_and_the_same_bits_again() -> None:
    hidden, weight, labels = inputs(200, 128, 3000, BF16, seed=6, ignored=0.1)
    _, (dh, dw) = _step(hidden, weight, labels, VocabConfig())
    h = hidden.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(vocab_loss(h, weight, labels), h)[0], dh)
    w = weight.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(vocab_loss(hidden, w, labels), w)[0], dw)
    h2, w2 = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = vocab_loss(h2, w2, labels)
    for _ in range(3):  # one graph, several backward passes
        a, b = torch.autograd.grad(loss, (h2, w2), retain_graph=True)
        assert torch.equal(a, dh) and torch.equal(b, dw)


def test_frozen_head_and_no_grad() -> None:
    hidden, weight, labels = inputs(30, 64, 100, BF16)
    assert not vocab_loss(hidden, weight, labels).requires_grad
    h = hidden.clone().requires_grad_(True)
    with torch.no_grad():
        assert not vocab_loss(h, weight, labels).requires_grad
    out = vocab_loss_confidence(h, weight, labels)
    assert out.confidence.requires_grad and not out.correct.requires_grad
    (only,) = torch.autograd.grad(out.confidence.sum(), h)
    want = exact(hidden, weight, labels, grad_loss=torch.zeros((), device="cuda"), grad_confidence=torch.ones(30, device="cuda"))
    assert want.sure.all()
    _within(only, want.d_hidden, want.tol_hidden + 1e-30, "d hidden")


def test_second_derivative_is_refused() -> None:
    hidden, weight, labels = inputs(10, 64, 50, F32)
    h = hidden.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(vocab_loss(h, weight, labels), h, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), h)


def test_changed_input_is_refused_in_backward() -> None:
    hidden, weight, labels = inputs(10, 64, 50, F32)
    w = weight.clone().requires_grad_(True)
    loss = vocab_loss(hidden, w, labels)
    with torch.no_grad():
        w += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_streams() -> None:
    """Calls on two streams at once do not share anything."""
    a = inputs(300, 128, 4000, BF16, seed=21)
    b = inputs(280, 128, 5000, BF16, seed=22)
    want = [_step(*x, VocabConfig()) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i] = _step(*x, VocabConfig())
    torch.cuda.synchronize()
    for (o, g), (o2, g2) in zip(want, got):
        assert torch.equal(o.loss, o2.loss) and torch.equal(g[0], g2[0]) and torch.equal(g[1], g2[1])


def test_captured_step_replays() -> None:
    """A captured step with its gradients: new inputs each replay, eager work in
    between, every replay compared with the eager result."""
    hidden, weight, labels = inputs(200, 128, 3000, BF16, seed=1, ignored=0.1)
    h, w, y = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True), labels.clone()

    def step():
        out = vocab_loss_confidence(h, w, y)
        return [out.loss, out.confidence, *torch.autograd.grad((out.loss, out.confidence), (h, w),
                                                               (torch.ones_like(out.loss), out.confidence.detach()))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        new = inputs(200, 128, 3000, BF16, seed=30 + i, ignored=0.3 * (i % 2))
        with torch.no_grad():
            h.copy_(new[0])
            w.copy_(new[1])
            y.copy_(new[2])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), f"replay {i}"


def test_forward_mode_is_refused() -> None:
    """In the call and in its backward: nothing comes back without its tangent."""
    import torch.autograd.forward_ad as fwd

    hidden, weight, labels = inputs(10, 64, 50, F32)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            vocab_loss_confidence(fwd.make_dual(hidden, torch.ones_like(hidden)), weight, labels)
        h = hidden.clone().requires_grad_(True)
        loss = vocab_loss(h, weight, labels)
        up = fwd.make_dual(torch.ones_like(loss), torch.ones_like(loss))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(loss, h, up)


def test_second_derivative_in_the_upstream_gradient_is_refused() -> None:
    hidden, weight, labels = inputs(10, 64, 50, F32)
    h = hidden.clone().requires_grad_(True)
    loss = vocab_loss(h, weight, labels)
    up = torch.ones_like(loss).requires_grad_(True)
    (g,) = torch.autograd.grad(loss, h, up, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        torch.autograd.grad(g.sum(), up, allow_unused=True)


def _compare_all(hidden, weight, labels, config=VocabConfig(), go=None, gc=None):
    """``_compare`` with both gradients always among it: tokens whose two largest
    logits are too close to tell which is the top label have no upstream gradient
    of their confidence, on which the top label bears."""
    if gc is not None:
        gc = torch.where(exact(hidden, weight, labels, config.ignore_index, config.reduction).sure, gc, 0.0)
    want = exact(hidden, weight, labels, config.ignore_index, config.reduction, go, gc)
    out, (dh, dw) = _compare(hidden, weight, labels, config, go, gc)
    _within(dh, want.d_hidden, want.tol_hidden + 1e-30, "d hidden")
    _within(dw, want.d_weight, want.tol_weight + 1e-30, "d weight")
    return out, (dh, dw)


def test_tiny_upstream_of_the_loss_beside_an_ordinary_one_of_the_confidence() -> None:
    """dS is held times the reciprocal of the loss's upstream gradient, unless that
    takes the confidence's part out of float32's range."""
    n, size, v = 300, 64, 500
    hidden, weight, labels = inputs(n, size, v, BF16, seed=31, ignored=0.1)
    gc = torch.randn(n, generator=torch.Generator().manual_seed(3)).cuda()
    for up in (1e-34, 1e-30, 1e-12, 1.0):
        for factor in (1.0, 1e5):
            _compare_all(hidden, weight, labels, VocabConfig(reduction="sum"), torch.tensor(up, device="cuda"), factor * gc)


def _by_size(hidden, weight, labels, config, go, gc, size_of, head):
    """The hidden gradient of tokens whose upstream gradients are of very different
    size, compared group by group: each group's bound knows only its own size.  float16
    holds dS of a token at 2^7 or more of what the group's reference allows for its
    subnormals (2^13), so that rounding is off by half a step, 2^-25, of that."""
    h = hidden.detach().clone().requires_grad_(True)
    leaves = (h,)
    w = weight.detach().clone().requires_grad_(not head)
    if not head:
        leaves = (h, w)
    out = vocab_loss_confidence(h, w, labels, config)
    grads = torch.autograd.grad((out.loss, out.confidence), leaves, (go, gc))
    counted = int(((labels >= 0) & (labels < weight.shape[0])).sum())
    for group in size_of.unique():
        at = size_of == group
        one = go[at] if config.reduction == "none" else (go / counted).expand(int(at.sum()))
        want = exact(hidden[at], weight, labels[at], reduction="none", grad_loss=one, grad_confidence=gc[at])
        most = float((one.abs() + gc[at].abs()).max())
        floor = 2.0 ** -25 / 2.0 ** 7 * most * weight.double().abs().sum(0)
        _within(grads[0][at], want.d_hidden, want.tol_hidden + floor, f"d hidden of group {int(group)}")
    return grads


@pytest.mark.parametrize("frozen_head", [False, True], ids=["both", "frozen head"])
@pytest.mark.parametrize("n,v", [(160, 20000), (2500, 60000)])  # one piece of the vocabulary, and two
def test_float16_hidden_gradients_of_tokens_with_small_upstream_gradients(n, v, frozen_head) -> None:
    """Upstream gradients over 2^-21..1 of a loss scale: each token's own hidden
    gradient is as good as if the token were alone.  The weight's rows share a mean,
    to which a token's many small probabilities add up."""
    size = 64
    hidden, weight, labels = inputs(n, size, v, F16, seed=17, ignored=0.1)
    hidden, weight = hidden / 8, weight + 0.5
    group = torch.arange(n, device="cuda") % 8
    size_of = torch.exp2(12.0 - 3 * group)
    gen = torch.Generator().manual_seed(2)
    sign = torch.sign(torch.randn(n, generator=gen)).cuda()
    # per-token weights of the loss
    grads = _by_size(hidden, weight, labels, VocabConfig(reduction="none"), size_of * sign, torch.zeros(n, device="cuda"), group,
                     frozen_head)
    want = exact(hidden, weight, labels, reduction="none", grad_loss=size_of * sign)
    _within(grads[0], want.d_hidden, want.tol_hidden, "d hidden")
    if not frozen_head:
        _within(grads[1], want.d_weight, want.tol_weight, "d weight")
    # and of the confidences beside a mean
    gc = torch.where(exact(hidden, weight, labels).sure, size_of * sign, 0.0)
    up = torch.tensor(2.0 ** -9 * n, device="cuda")
    _by_size(hidden, weight, labels, VocabConfig(), up, gc, group, frozen_head)
    # all alike, a few decades down, and tokens without any
    near = torch.exp2(-5.0 * (group % 2)) * sign * (group != 3)
    _by_size(hidden, weight, labels, VocabConfig(reduction="none"), near, torch.zeros(n, device="cuda"), group, frozen_head)


def test_float16_infinite_upstream_gradient_stays_in_its_token() -> None:
    n = 60
    hidden, weight, labels = inputs(n, 64, 3000, F16, seed=18)
    go = torch.exp2(-1.0 * (torch.arange(n, device="cuda") % 20))
    h = hidden.clone().requires_grad_(True)
    loss = vocab_loss(h, weight, labels, VocabConfig(reduction="none"))
    (want,) = torch.autograd.grad(loss, h, go, retain_graph=True)
    for wild in (float("inf"), float("nan")):
        go[7] = wild
        (got,) = torch.autograd.grad(loss, h, go, retain_graph=True)
        keep = torch.arange(n, device="cuda") != 7
        assert not torch.isfinite(got[7]).any()
        ref = exact(hidden[keep], weight, labels[keep], reduction="none", grad_loss=go[keep])
        _within(got[keep], ref.d_hidden, ref.tol_hidden, f"d hidden beside {wild}")
        assert torch.isfinite(want[keep]).all()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_weights_past_32_bit_offsets(dtype) -> None:
    """600000 words of 4096: the last words' elements are beyond 2^31.  Labels at both
    ends; gradients against the definition in float64, word by word at the ends."""
    n, size, v = 5, 4096, 600000
    gen = torch.Generator(device="cuda").manual_seed(7)
    weight = torch.empty(v, size, dtype=dtype, device="cuda").normal_(std=1 / 64, generator=gen)
    hidden = torch.randn(n, size, device="cuda", generator=gen).to(dtype)
    labels = torch.tensor([0, 1, v // 2, v - 2, v - 1], device="cuda")
    hidden = (hidden.float() + 5 * weight[labels].float() * 8).to(dtype).requires_grad_(True)
    w = weight.requires_grad_(True)
    out = vocab_loss_confidence(hidden, w, labels, VocabConfig(reduction="none"))
    up = torch.ones(n, device="cuda")
    dh, dw = torch.autograd.grad((out.loss, out.confidence), (hidden, w), (up, -0.5 * up))
    with torch.no_grad():
        h = hidden.double()
        s = torch.cat([h @ weight[i:i + 50000].double().t() for i in range(0, v, 50000)], 1)
        most = float(torch.stack([(h.abs() @ weight[i:i + 50000].double().abs().t()).max() for i in range(0, v, 50000)]).max())
        e = 2 * (4 * size ** 0.5 * U * most) + 16 * U * (1 + float(s.max() - s.min()))  # as in vocab_reference.py
        lse = torch.logsumexp(s, 1)
        here = torch.arange(n, device="cuda")
        _within(out.loss, lse - s[here, labels], e + 2 * U * lse, "loss")
        p = torch.exp(s - lse[:, None])
        best = s.argmax(1)
        conf = p[here, best]
        _within(out.confidence, conf, e * conf, "confidence")
        c = -0.5 * conf
        ds, size_ds = (1 - c)[:, None] * p, (1 + c.abs())[:, None] * p
        ds[here, labels] -= 1
        ds[here, best] += c
        size_ds[here, labels] += 1
        size_ds[here, best] += c.abs()
        half = torch.finfo(dtype).eps / 2
        rel = 3 * e + (half if dtype != F32 else 0)
        for words in (slice(0, 300), slice(v // 2 - 100, v // 2 + 100), slice(v - 300, v)):
            want, tol = ds[:, words].t() @ h, rel * (size_ds[:, words].t() @ h.abs())
            _within(dw[words], want, tol * (1 + half) + half * want.abs() + 1e-30, f"d weight {words}")
        want, tol = torch.zeros_like(h), torch.zeros_like(h)
        for i in range(0, v, 50000):
            part = weight[i:i + 50000].double()
            want += ds[:, i:i + 50000] @ part
            tol += (rel + 4 * v ** 0.5 * U) * (size_ds[:, i:i + 50000] @ part.abs())
        _within(dh, want, tol * (1 + half) + half * want.abs(), "d hidden")


def test_captured_float16_step_with_upstream_gradients_near_and_far_apart() -> None:
    """One graph: whether the rows of dS take scales of their own is the device's to
    say, anew in every replay."""
    n = 100
    hidden, weight, labels = inputs(n, 64, 3000, F16, seed=41, ignored=0.1)
    h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    go = torch.ones(n, device="cuda")

    def step():
        loss = vocab_loss(h, w, labels, VocabConfig(reduction="none"))
        return [loss, *torch.autograd.grad(loss, (h, w), go)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    far = torch.exp2(10.0 - 5.0 * (torch.arange(n, device="cuda") % 5))
    for up in (torch.ones(n, device="cuda"), far, 0.5 * torch.ones(n, device="cuda"), far.flip(0), torch.zeros(n, device="cuda")):
        go.copy_(up)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        want = exact(hidden, weight, labels, reduction="none", grad_loss=up)
        _within(got[1], want.d_hidden, want.tol_hidden, "d hidden")


def test_negative_bit() -> None:
    """Tensors whose memory holds the negatives of their values."""
    hidden, weight, labels = inputs(40, 64, 300, F32, seed=5)
    want, (dh, dw) = _step(hidden, weight, labels, VocabConfig(), torch.tensor(0.5, device="cuda"))
    h, w, y = (torch._neg_view(-t) for t in (hidden, weight, labels))
    assert h.is_neg() and h.is_contiguous() and y.is_neg()
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = vocab_loss(h, w, y)
    up = torch._neg_view(torch.tensor(-0.5, device="cuda"))
    a, b = torch.autograd.grad(loss, (h, w), up)
    assert torch.equal(loss, want.loss) and torch.equal(a, dh) and torch.equal(b, dw)
