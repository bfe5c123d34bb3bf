"""token_logprobs on the GPU against its definition in float64.

u = 2^-24.  An exponent z = (x - top) / t is off by 3 u |z| (difference, factor,
product), its exponential relatively by that and 2 u, a sum of V of them, added in
up to V / 64 steps a lane, by sqrt(V) u on top (roundings have no common sign); D is
the largest |z| that counts.  So a sum is off relatively by `rel` = (8 + 3 D +
sqrt(V)) u, log probabilities by that and 4 u (|z| + l), the entropy l + mean |z|, of
which the mean is a quotient of two sums, by 2 rel (1 + mean |z|) and 4 u (l + mean
|z|).  The gradient p (g + h (lp + H)) takes p's relative error, lp's and H's, and half
a step of its type."""

from __future__ import annotations

import math

import pytest
import torch

from ace_kernels import LogprobConfig, token_logprobs
from gpu_helpers import say

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
U = 2.0 ** -24


def _logits(lead, vocab, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = 2.0 * torch.randn(*lead, vocab, generator=gen, device="cuda")
    at = torch.randint(vocab, (*lead, 1), generator=gen, device="cuda")
    return x.scatter_add_(-1, at, 8.0 * torch.rand(*lead, 1, generator=gen, device="cuda")).to(dtype)


def _tokens(x, seed=1, ignored=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    y = torch.randint(x.shape[-1], x.shape[:-1], generator=gen, device="cuda")
    top = torch.nan_to_num(x.float(), nan=0.0).argmax(-1)
    y = torch.where(torch.rand(y.shape, generator=gen, device="cuda") < 0.5, top, y)
    return torch.where(torch.rand(y.shape, generator=gen, device="cuda") < ignored, -100, y)


def _upstream(y, seed=2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(y.shape, generator=gen, device="cuda") for _ in range(2)]


def _exact(x, y, t, top, up, ignore=-100):
    """(values, bounds) of logprob, entropy, top_logprobs and the gradient, and the
    top tokens.  Rows have a finite logit."""
    v = x.shape[-1]
    s, at = x.detach().double().reshape(-1, v), y.reshape(-1).long()
    on = (at >= 0) & (at < v) & (at != ignore)
    at = torch.where(on, at, 0)[:, None]
    s = torch.where(on[:, None], s, 0.0)
    z = (s - s.amax(1, keepdim=True)) / t
    far = torch.where(z.isinf(), 0.0, z).clamp(min=-200)  # a word further off has probability 0
    log_sum = torch.exp(z).sum(1, keepdim=True).log()
    lp = z - log_sum
    p = lp.exp()
    mean = -(p * torch.where(z.isinf(), 0.0, z)).sum(1, keepdim=True)
    h = log_sum + mean
    rel = U * (8 + 3 * -far.amin(1, keepdim=True) + math.sqrt(v))
    tol_lp = 4 * U * (-torch.where(z.isinf(), 0.0, z) + log_sum) + rel
    tol_h = 2 * rel * (1 + mean) + 4 * U * (log_sum + mean)
    best = torch.sort(s, dim=1, descending=True, stable=True).indices[:, :top]
    g, e = (u.double().reshape(-1, 1) for u in up)
    lp0 = torch.where(z.isinf(), 0.0, lp)
    d = -p * (g + e * (lp0 + h))
    tol_d = p * ((tol_lp + 4 * U) * (g + e * (lp0 + h)).abs() + e.abs() * (tol_lp + tol_h + 4 * U * (lp0.abs() + h)) + 3 * U * g.abs())
    d.scatter_add_(1, at, g)
    tol_d.scatter_add_(1, at, U * g.abs())
    half = torch.finfo(x.dtype).eps / 2
    d, tol_d = d / t, (tol_d + 4 * U * d.abs()) / t + half * d.abs() / t
    tol_d += torch.finfo(x.dtype).tiny * half * 1.01  # subnormals
    # p below 2^-126 is 0 in float32: there -lp <= 88 for what is just lost, and H <= log V <= 19, so
    # that p |g + h (lp + H)| <= 2^-126 (|g| + 107 |h|)
    tol_d += (g.abs() + 107 * e.abs()) / t * 2.0 ** -126
    keep = on[:, None].double()
    shape = y.shape
    values = [lp.gather(1, at) * keep, h * keep, torch.where(on[:, None], lp.gather(1, best), 0.0), d * keep]
    bounds = [tol_lp.gather(1, at) * keep, tol_h * keep, torch.where(on[:, None], tol_lp.gather(1, best), 0.0), tol_d * keep]
    shapes = [shape, shape, (*shape, top), x.shape]
    values = [a.reshape(b) for a, b in zip(values, shapes)]
    bounds = [a.reshape(b) for a, b in zip(bounds, shapes)]
    return values, bounds, torch.where(on[:, None], best, -1).reshape(*shape, top)


def _near(what, got, want, tol):
    same = (got.double() == want) | ((got.double() - want).abs() <= tol)
    assert same.all(), f"{what}: {int((~same).sum())} off, worst {float(((got.double() - want).abs() / tol)[~same].max()):.3g} x bound"


def _compare(x, y, top=0, t=1.0, up=None, want_of=None):
    config = LogprobConfig(top=top, temperature=t)
    up = _upstream(y) if up is None else up
    leaf = x.detach().requires_grad_(True)
    out = token_logprobs(leaf, y, config)
    (grad,) = torch.autograd.grad((out.logprob, out.entropy), leaf, up)
    assert out.logprob.dtype == out.entropy.dtype == F32 and grad.dtype == x.dtype and grad.shape == x.shape
    values, bounds, best = _exact(x if want_of is None else want_of, y, t, top, up)
    _near("logprob", out.logprob, values[0], bounds[0])
    _near("entropy", out.entropy, values[1], bounds[1])
    _near("gradient", grad, values[3], bounds[3])
    if top:
        assert out.top_tokens.dtype == torch.int64 and torch.equal(out.top_tokens, best)
        _near("top_logprobs", out.top_logprobs, values[2], bounds[2])
    else:
        assert out.top_logprobs is None and out.top_tokens is None
    return out, grad


# a lane's piece, a tile, a group, a wave's and four waves' first words, and one word
# to either side of them; rows that are cut into parts
SIZES = [1, 2, 3, 7, 8, 9, 15, 255, 256, 257, 511, 513, 1023, 1025, 2047, 2048, 2049, 4095, 4097, 8191, 8192, 8193, 16384,
         16385, 32000, 50257, 65537, 131072]


@TYPES
@pytest.mark.parametrize("vocab", SIZES)
def test_sizes(vocab, dtype) -> None:
    say(f"logprobs {vocab} {dtype}")
    x = _logits((5,), vocab, dtype, seed=vocab)
    for top in sorted({0, 1, min(vocab, 5), min(vocab, 20), min(vocab, 32)}):
        _compare(x, _tokens(x, seed=top), top)


# few rows are cut into parts, many are not, and many short ones share a block
@TYPES
@pytest.mark.parametrize("rows,vocab", [(1, 300000), (3, 40000), (130, 20000), (1100, 17000), (2500, 9001), (1023, 8000), (1024, 8000), (1024, 8193), (2047, 8000),
                                        (2048, 8000), (4099, 4000), (2500, 1000), (20001, 70), (300, 70)])
def test_rows(rows, vocab, dtype) -> None:
    say(f"logprobs {rows} x {vocab} {dtype}")
    x = _logits((rows,), vocab, dtype, seed=rows)
    y = _tokens(x, ignored=0.3)
    _compare(x, y, 0, 0.7)
    _compare(x, y, 7, 1.5)


@TYPES
def test_gradients_beyond_the_caches(dtype) -> None:
    """More than 224 MB of logits and gradients, whose stores go past the caches; rows
    no whole number of pieces."""
    x = _logits((1300,), 50257, dtype)
    _compare(x, _tokens(x, ignored=0.2))


@TYPES
@pytest.mark.parametrize("t", [0.001, 0.05, 1.0, 30.0, 1000.0])
def test_temperatures(t, dtype) -> None:
    x = _logits((2, 3), 5003, dtype)
    _compare(x, _tokens(x), 4, t)


@TYPES
def test_shapes_and_none(dtype) -> None:
    x = _logits((2, 3, 4), 100, dtype)
    _compare(x, _tokens(x), 3)
    one = _logits((), 100, dtype)
    out, _ = _compare(one, _tokens(one), 3)
    assert out.logprob.shape == () and out.top_tokens.shape == (3,)
    none = torch.empty(2, 0, 50, dtype=dtype, device="cuda", requires_grad=True)
    out = token_logprobs(none, torch.empty(2, 0, dtype=torch.int64, device="cuda"), LogprobConfig(top=3))
    assert out.logprob.shape == (2, 0) and out.top_tokens.shape == (2, 0, 3)
    assert torch.autograd.grad(out.logprob.sum(), none)[0].shape == none.shape
    for kind in (torch.int32, torch.int16, torch.int8, torch.uint8):
        y = _tokens(x).clamp(min=0)
        a, b = token_logprobs(x, y), token_logprobs(x, y.to(kind))
        assert torch.equal(a.logprob, b.logprob)


@TYPES
@pytest.mark.parametrize("rows,vocab", [(6, 20000), (2100, 500)])
def test_uncounted_rows_are_not_read(rows, vocab, dtype) -> None:
    x = _logits((rows,), vocab, dtype)
    y = _tokens(x, ignored=0.5)
    y[0], y[1], y[2], y[3] = vocab, -1, 1 << 40, -100
    want, grad = _compare(x, y, 4)
    dirty = torch.where(((y >= 0) & (y < vocab))[:, None], x, torch.nan)
    got, again = _compare(dirty, y, 4, want_of=x)
    for a, b in zip([*want, grad], [*got, again]):
        assert torch.equal(a, b)
    off = ~((y >= 0) & (y < vocab))
    assert not got.logprob[off].any() and not got.entropy[off].any() and not again[off].any()
    assert (got.top_tokens[off] == -1).all() and not got.top_logprobs[off].any()
    # a word of the vocabulary that is ignored
    word = int(y[~off][0])
    out = token_logprobs(x, y, LogprobConfig(ignore_index=word))
    assert not out.logprob[y == word].any()


@TYPES
@pytest.mark.parametrize("rows,vocab", [(6, 20000), (6, 300), (2100, 500)])
def test_equal_logits_go_to_the_lowest_word(rows, vocab, dtype) -> None:
    gen = torch.Generator(device="cuda").manual_seed(1)
    few = torch.randint(-1, 2, (rows, vocab), generator=gen, device="cuda").to(dtype)
    few[0] = 0.0
    few[1] *= -0.0  # 0 and -0 are equal
    few[2] = torch.finfo(dtype).min
    few[3] = torch.finfo(dtype).max
    for top in (1, 5, 32):
        out, _ = _compare(few, _tokens(few), top)
        for r in (0, 1, 2, 3):
            assert torch.equal(out.top_tokens[r].cpu(), torch.arange(top))


@TYPES
@pytest.mark.parametrize("rows,vocab", [(2, 70000), (3, 9000), (2100, 3000)])
def test_words_in_order(rows, vocab, dtype) -> None:
    """Ascending logits make every word a candidate; descending ones none after the
    first."""
    ramp = torch.linspace(-20, 20, vocab, device="cuda").to(dtype).expand(rows, vocab)
    for x in (ramp.contiguous(), ramp.flip(1).contiguous(), ramp):  # the last: rows with no distance
        _compare(x, _tokens(x), 20)
        _compare(x, _tokens(x), 32)


@TYPES
@pytest.mark.parametrize("rows,vocab", [(4, 30000), (2100, 600)])
def test_masked_words(rows, vocab, dtype) -> None:
    """Words at -inf, or at the type's lowest value: nothing of them in results and
    gradients; rows with one word, or fewer than the alternatives asked for."""
    x = _logits((rows,), vocab, dtype)
    y = _tokens(x)
    for low in (-math.inf, torch.finfo(dtype).min):
        masked = x.clone()
        masked[:, 1::2] = low
        masked[1, :] = low
        masked[1, 5] = 1.0
        masked[2, 3:] = low
        inside = torch.where(y % 2 == 1, y - 1, y)
        inside[1], inside[2] = 5, 0
        out, grad = _compare(masked, inside, 10)
        assert out.logprob[1] == 0 and out.entropy[1] == 0 and not grad[1].any()
        assert out.top_tokens[1, 0] == 5 and out.top_tokens[1, 1:].tolist() == [0, 1, 2, 3, 4, 6, 7, 8, 9]
        assert not grad[0, 1::2].any()
    # a token at -inf itself
    masked = x.clone()
    masked[0, 7] = -math.inf
    y[0] = 7
    up = [torch.ones_like(y, dtype=F32), torch.zeros_like(y, dtype=F32)]
    leaf = masked.requires_grad_(True)
    out = token_logprobs(leaf, y)
    (grad,) = torch.autograd.grad((out.logprob, out.entropy), leaf, up)
    assert out.logprob[0] == -math.inf and torch.isfinite(out.entropy).all() and torch.isfinite(grad).all()


@TYPES
@pytest.mark.parametrize("rows,vocab", [(4, 30000), (2100, 600)])
def test_rows_without_a_word_and_with_nan(rows, vocab, dtype) -> None:
    x = _logits((rows,), vocab, dtype)
    y = _tokens(x)
    clean, clean_grad = _compare(x, y, 5)
    x = x.clone()
    x[0] = -math.inf
    x[1, vocab - 1] = math.nan
    x[2, 3] = math.inf
    leaf = x.requires_grad_(True)
    out = token_logprobs(leaf, y, LogprobConfig(top=5))
    (grad,) = torch.autograd.grad((out.logprob, out.entropy), leaf, _upstream(y))
    assert out.logprob[0] == -math.inf and out.entropy[0] == 0 and not grad[0].any()
    assert (out.top_logprobs[0] == -math.inf).all() and out.top_tokens[0].tolist() == [0, 1, 2, 3, 4]
    for r in (1, 2):
        assert out.logprob[r].isnan() and out.entropy[r].isnan() and out.top_logprobs[r].isnan().all()
        assert grad[r].isnan().all()
    assert out.top_tokens[1, 0] == vocab - 1 and out.top_tokens[2, 0] == 3
    for a, b in zip([*clean, clean_grad], [*out, grad]):
        assert torch.equal(a[3:], b[3:])


@TYPES
def test_many_nans(dtype) -> None:
    x = torch.full((3, 20000), math.nan, dtype=dtype, device="cuda")
    x[1, ::2] = 1.0
    out = token_logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda"), LogprobConfig(top=8))
    assert out.top_tokens[0].tolist() == list(range(8)) and out.top_tokens[1].tolist() == list(range(1, 17, 2))


@TYPES
@pytest.mark.parametrize("rows,vocab", [(1024, 4096), (1, 1 << 20), (1024, 65536)])
def test_words_that_are_all_but_certain(rows, vocab, dtype) -> None:
    """The others' sum s is what the log probability of the largest word consists of, and
    each of them is far below a step of 1.  s is off by (3 |z| + 2) u s from its exponentials
    and by at most 32 u s, u for each word that a lane adds of a group; it meets the 1, and
    other lanes and waves, in float64; the logarithm adds 4 u of the result."""
    x = torch.full((rows, vocab), -18.0, dtype=dtype, device="cuda")  # each e^-18 = 2^-25.97
    y = (torch.arange(rows, device="cuda") * 7919 + vocab // 2) % vocab
    x[torch.arange(rows, device="cuda"), y] = 0.0
    out = token_logprobs(x, y, LogprobConfig(top=1))
    s = (vocab - 1) * math.exp(-18.0)
    tol = (3 * 18 / math.log(2.0) + 2 + 32) * U * s + 4 * U * math.log1p(s)
    for got in (out.logprob, out.top_logprobs[:, 0]):
        assert float((got.double() + math.log1p(s)).abs().max()) <= tol
    assert torch.equal(out.top_tokens[:, 0], y)


@TYPES
@pytest.mark.parametrize("t", [1.0, 0.5])
@pytest.mark.parametrize("rows,vocab,low", [(1024, 4096, -18.0), (1, 1 << 20, -18.0), (64, 32000, -26.0), (1300, 50257, -30.0),
                                            (5, 2, -9.0)])
def test_gradients_of_words_that_are_all_but_certain(rows, vocab, low, t, dtype) -> None:
    """g (1 - p) of the given word is what the others' p g add up to, s / (1 + s) of g, also
    where p rounds to 1.  The log probability is off relatively by the bound above over s,
    expm1 and the product by 4 u, an other word's p by (3 |z| + 6) u and what the sum is off; the
    entropy's term p (lp + H) = p |z| s / (1 + s) by twice that, lp and H each being small.  s
    meets the 1 in float64, in at most 16 steps across lanes, waves and parts."""
    z = low / t
    x = torch.full((rows, vocab), low, dtype=dtype, device="cuda")
    y = (torch.arange(rows, device="cuda") * 7919 + vocab // 2) % vocab
    here = torch.arange(rows, device="cuda")
    x[here, y] = 0.0
    s = (vocab - 1) * math.exp(z)
    rel = (3 * abs(z) / math.log(2.0) + 2 + 32 + 8) * U
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * half * 1.01 + 2.0 ** -125 + 3.0 / t * 16 * 2.0 ** -53
    g = torch.full((rows,), 3.0, device="cuda")
    for ups in ([g, torch.zeros_like(g)], [torch.zeros_like(g), g]):
        leaf = x.detach().requires_grad_(True)
        out = token_logprobs(leaf, y, LogprobConfig(temperature=t))
        (grad,) = torch.autograd.grad((out.logprob, out.entropy), leaf, ups)
        p, q = 1 / (1 + s), math.exp(z) / (1 + s)  # the given word's and each other's
        lp, lq = -math.log1p(s), z - math.log1p(s)
        h = math.log1p(s) - (vocab - 1) * q * z
        want = (3.0 * s * p / t, -3.0 * q / t) if ups[0] is g else (-3.0 * p * (lp + h) / t, -3.0 * q * (lq + h) / t)
        for got, value in ((grad[here, y], want[0]), (grad[here, (y + 1) % vocab], want[1])):
            err = float((got.double() - value).abs().max())
            assert err <= (3 * rel + half) * abs(value) + tiny, f"{err / abs(value):.3g} of {value:.3g}"


@TYPES
@pytest.mark.parametrize("rows", [1, 5, 1100])
@pytest.mark.parametrize("vocab", [1, 2, 257, 1025, 2049, 4097, 40001])
def test_rows_whose_largest_word_is_the_lowest_value(vocab, rows, dtype) -> None:
    """A type's lowest value is a word like any other where nothing else is open: all of a
    row at it, of which some sizes leave a wave one word, and one such word alone, in any lane."""
    low = torch.finfo(dtype).min
    x = torch.full((rows, vocab), low, dtype=dtype, device="cuda")
    y = (torch.arange(rows, device="cuda") * 7919 + vocab // 2) % vocab
    top = min(vocab, 5)
    out, _ = _compare(x, y, top)
    assert torch.equal(out.top_tokens, torch.arange(top, device="cuda").expand(rows, top))
    x = torch.full((rows, vocab), -math.inf, dtype=dtype, device="cuda")
    x[torch.arange(rows, device="cuda"), y] = low
    out, grad = _compare(x, y, top)
    assert not out.logprob.any() and not out.entropy.any() and not grad.any()
    assert torch.equal(out.top_tokens[:, 0], y) and not out.top_logprobs[:, 0].any()


@TYPES
@pytest.mark.parametrize("vocab", [501, 504, 9000])
def test_strides_and_offsets(vocab, dtype) -> None:
    """Rows that lie apart are read where they are; any other order is copied."""
    x = _logits((3, 4), vocab, dtype)
    y = _tokens(x)
    want, grad = _compare(x, y, 6)
    wide = torch.full((3, 4, vocab + 19), math.nan, dtype=dtype, device="cuda")
    wide[..., 3:3 + vocab] = x
    flat = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")
    flat[1:] = x.reshape(-1)
    padded = torch.full((3, 7, vocab), math.nan, dtype=dtype, device="cuda")
    padded[:, 2:6] = x
    turned = x.transpose(0, 1).contiguous().transpose(0, 1)
    for z in (wide[..., 3:3 + vocab], flat[1:].view(3, 4, vocab), padded[:, 2:6], turned,
              x.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        assert torch.equal(z, x)
        for yy in (y, y.t().contiguous().t()):
            leaf = z.detach().requires_grad_(True)
            out = token_logprobs(leaf, yy, LogprobConfig(top=6))
            (got,) = torch.autograd.grad((out.logprob, out.entropy), leaf, _upstream(y))
            for a, b in zip([*want, grad], [*out, got]):
                assert torch.equal(a, b)


def test_inference_mode_and_leading_dimensions() -> None:
    x = _logits((2, 5), 700, BF16)
    y = _tokens(x)
    want = token_logprobs(x, y, LogprobConfig(top=3))
    with torch.inference_mode():
        got = token_logprobs(x.clone(), y, LogprobConfig(top=3))
        flat = token_logprobs(x.view(10, 700), y.view(10), LogprobConfig(top=3))
    for a, b, c in zip(want, got, flat):
        assert torch.equal(a, b) and torch.equal(a.view(c.shape), c)
    assert not want.top_logprobs.requires_grad and want.logprob.grad_fn is None


def test_one_gradient_alone() -> None:
    x = _logits((4,), 900, F32)
    y = _tokens(x)
    up = _upstream(y)
    zero = torch.zeros_like(up[0])
    for i in range(2):
        leaf = x.clone().requires_grad_(True)
        out = token_logprobs(leaf, y)
        (got,) = torch.autograd.grad(out[i], leaf, up[i])
        both = [zero, zero]
        both[i] = up[i]
        _, want = _compare(x, y, 0, up=both)
        assert torch.equal(got, want)


def test_gradient_against_differences() -> None:
    x = _logits((3,), 400, F32)
    y = _tokens(x)
    up = _upstream(y)
    leaf = x.clone().requires_grad_(True)
    out = token_logprobs(leaf, y, LogprobConfig(temperature=0.8))
    (got,) = torch.autograd.grad((out.logprob, out.entropy), leaf, up)
    way = torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).cuda().double()

    def f(t):
        lp = torch.log_softmax((x.double() + t * way) / 0.8, 1)
        return float((up[0].double() * lp.gather(1, y[:, None])[:, 0]).sum() - (up[1].double() * (lp.exp() * lp).sum(1)).sum())

    want = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(float((got.double() * way).sum()) - want) <= 1e-5 * (1 + abs(want))


def test_same_bits_again_and_streams() -> None:
    """Cut rows on two streams at once: tickets and parts of their own."""
    xs = [_logits((3,), 100000, BF16, seed=1), _logits((40,), 30000, F32, seed=2)]
    ys = [_tokens(x) for x in xs]
    cfg = LogprobConfig(top=9)
    want = [token_logprobs(x, y, cfg) for x, y in zip(xs, ys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append((i, token_logprobs(xs[i], ys[i], cfg)))
    torch.cuda.synchronize()
    for i, o in got:
        for a, b in zip(o, want[i]):
            assert torch.equal(a, b)


def test_captured_steps_replay() -> None:
    """Two captured graphs with cut rows, replayed in turn with eager calls in
    between; every replay equals the eager result."""
    cfg = LogprobConfig(top=6)
    leaves = [_logits((5,), 40000, BF16, seed=i).requires_grad_(True) for i in range(2)]
    ys = [_tokens(x) for x in leaves]
    ups = [_upstream(y) for y in ys]

    def step(i):
        out = token_logprobs(leaves[i], ys[i], cfg)
        return [*(t.detach() for t in out), *torch.autograd.grad((out.logprob, out.entropy), leaves[i], ups[i])]

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
                leaves[i].copy_(_logits((5,), 40000, BF16, seed=50 + 2 * r + i))
            graphs[i].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held[i]]
            for a, b in zip(got, step(i)):
                assert torch.equal(a, b), f"replay {r} of graph {i}"


def test_changed_logits_and_results_in_place() -> None:
    leaf = _logits((4,), 300, F32).requires_grad_(True)
    y = _tokens(leaf)
    kept = leaf * 1.0
    out = token_logprobs(kept, y)
    kept.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.logprob.sum(), leaf)
    out = token_logprobs(leaf, y)
    want = torch.autograd.grad(out.logprob.sum(), leaf)[0]
    out = token_logprobs(leaf, y)
    doubled = out.logprob.mul_(2.0)  # the results may be changed: the backward keeps its own
    assert torch.equal(torch.autograd.grad(doubled.sum(), leaf, retain_graph=True)[0], 2 * want)


def test_derivatives_that_are_refused() -> None:
    import torch.autograd.forward_ad as fwd

    x = _logits((4,), 300, F32)
    y = _tokens(x)
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(token_logprobs(leaf, y).logprob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        torch.autograd.grad(g.sum(), leaf)
    out = token_logprobs(leaf, y)
    up = torch.ones_like(out.entropy).requires_grad_(True)
    (g,) = torch.autograd.grad(out.entropy, leaf, up, create_graph=True)
    with pytest.raises(RuntimeError, match="only once"):
        torch.autograd.grad(g.sum(), up, allow_unused=True)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            token_logprobs(fwd.make_dual(x, torch.ones_like(x)), y)
        lp = token_logprobs(leaf, y).logprob
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(lp, leaf, fwd.make_dual(torch.ones_like(lp), torch.ones_like(lp)))


def test_negative_bit() -> None:
    x = _logits((4,), 300, F32)
    y = _tokens(x)
    want, grad = _compare(x, y, 3)
    leaf = torch._neg_view(-x).requires_grad_(True)
    out = token_logprobs(leaf, y, LogprobConfig(top=3))
    up = [torch._neg_view(-u) for u in _upstream(y)]
    (got,) = torch.autograd.grad((out.logprob, out.entropy), leaf, up)
    for a, b in zip([*want, grad], [*out, got]):
        assert torch.equal(a, b)


def test_logits_past_32_bit_offsets() -> None:
    """35000 rows of 65536 words, 2.3 G logits: the last rows are what they are alone."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    leaf = torch.empty(35000, 65536, dtype=BF16, device="cuda").normal_(generator=gen).requires_grad_(True)
    y = torch.randint(65536, (35000,), generator=gen, device="cuda")
    up = _upstream(y)
    out = token_logprobs(leaf, y, LogprobConfig(top=4))
    (grad,) = torch.autograd.grad((out.logprob, out.entropy), leaf, up)
    for part in (slice(0, 40), slice(32760, 32780), slice(34960, 35000)):
        values, bounds, best = _exact(leaf[part].detach(), y[part], 1.0, 4, [u[part] for u in up])
        assert torch.equal(out.top_tokens[part], best)
        for a, v, b in zip((out.logprob, out.entropy, out.top_logprobs, grad), values, bounds):
            _near("part", a[part], v, b)


def test_a_long_row() -> None:
    """One row of 2^26 words, and its last word given."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(1, (1 << 26) + 3, dtype=BF16, device="cuda").normal_(generator=gen)
    y = torch.tensor([x.shape[1] - 1], device="cuda")
    _compare(x, y, 3)
