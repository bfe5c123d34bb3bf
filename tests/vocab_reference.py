"""The vocabulary losses in float64, from their definition, with the bounds that
float32 accumulation and the gradients' types put on the difference.

u = 2^-24 is float32's largest relative rounding error.  A float32 sum of n
products is off by at most c sqrt(n) u sum|a b| with c = 4 (rounding errors are
independent: four standard deviations of their sum), so every logit is within
e = 4 sqrt(H) u max_tv sum|h w|.  A softmax of such logits is within 2 e
relatively, and 16 u (1 + range of the logits) more for the exponential, whose
argument is rounded.  dS is stored in the inputs' type (half a step: eps / 2), and
multiplied with float32 sums over the vocabulary or the tokens; the gradient is
rounded to the inputs' type once more."""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

U = 2.0 ** -24


@dataclass
class Exact:
    loss: torch.Tensor
    nll: torch.Tensor
    confidence: torch.Tensor
    correct: torch.Tensor
    d_hidden: Optional[torch.Tensor]
    d_weight: Optional[torch.Tensor]
    tol_nll: float           # absolute
    tol_confidence: float    # relative
    tol_hidden: torch.Tensor
    tol_weight: torch.Tensor
    sure: torch.Tensor       # tokens whose two largest logits are further apart than 2 e


def exact(hidden, weight, labels, ignore_index=-100, reduction="mean", grad_loss=None, grad_confidence=None) -> Exact:
    """``grad_loss`` ([] or [N]) and ``grad_confidence`` ([N]) default to 1 and 0."""
    dtype = hidden.dtype
    h, w, y = hidden.detach().double(), weight.detach().double(), labels.long()
    n, size = h.shape
    v = w.shape[0]
    counted = (y != ignore_index) & (y >= 0) & (y < v)
    rows = counted.nonzero()[:, 0]
    hc, yc = h[rows], y[rows]
    s = hc @ w.t()
    f64 = {"dtype": torch.float64, "device": h.device}
    nll, conf, correct = (torch.zeros(n, **f64) for _ in range(3))
    d_h, d_w = torch.zeros_like(h), torch.zeros_like(w)
    tol_h, tol_w = torch.zeros_like(h), torch.zeros_like(w)
    sure = torch.ones(n, dtype=torch.bool, device=h.device)
    count = max(1, rows.numel())
    e, spread = 0.0, 0.0
    if rows.numel():
        here = torch.arange(rows.numel(), device=h.device)
        e = 4 * math.sqrt(size) * U * float((hc.abs() @ w.abs().t()).max())
        spread = float((s.amax(1) - s.amin(1)).max())
        lse = torch.logsumexp(s, 1)
        p = torch.exp(s - lse[:, None])
        # the lowest index of the largest logit
        best = (s == s.amax(1, keepdim=True)).double().argmax(1)
        if v > 1:
            two = s.topk(2, dim=1).values
            sure[rows] = (two[:, 0] - two[:, 1] > 2 * e) | (two[:, 0] == two[:, 1])
        nll[rows] = lse - s[here, yc]
        conf[rows] = p[here, best]
        correct[rows] = (best == yc).double()
        go = torch.ones((), **f64) if grad_loss is None else grad_loss.double()
        g = go.expand(n)[rows] if reduction == "none" else go.expand(rows.numel()) / (count if reduction == "mean" else 1)
        c = torch.zeros(rows.numel(), **f64) if grad_confidence is None else grad_confidence.double()[rows]
        c = c * conf[rows]
        ds = (g - c)[:, None] * p
        ds[here, yc] -= g
        ds[here, best] += c
        # the magnitudes that errors are relative to: before the cancellation at
        # the label and the best word
        size_ds = (g.abs() + c.abs())[:, None] * p
        size_ds[here, yc] += g.abs()
        size_ds[here, best] += c.abs()
        half = torch.finfo(dtype).eps / 2
        relative = 3 * (2 * e + 16 * U * (1 + spread)) + (half if dtype != torch.float32 else 0)
        if dtype == torch.float16:  # dS is scaled to 2^13 .. 2^14; steps of 2^-24 below its normal range
            size_ds = size_ds + 2.0 ** -24 / 2.0 ** 13 * float((g.abs() + c.abs()).max()) / relative
        d_h[rows] = ds @ w
        d_w = ds.t() @ hc
        tiny = torch.finfo(dtype).tiny * half
        tol_h[rows] = (relative + 4 * math.sqrt(v) * U) * (size_ds @ w.abs())
        tol_h = tol_h + half * d_h.abs() + tol_h * half + tiny
        tol_w = (relative + 4 * math.sqrt(count) * U) * (size_ds.t() @ hc.abs())
        tol_w = tol_w + half * d_w.abs() + tol_w * half + tiny
    loss = nll if reduction == "none" else nll.sum() / (count if reduction == "mean" else 1)
    return Exact(loss, nll, conf, correct, d_h, d_w, 2 * e + 16 * U * (1 + spread), 2 * e + 16 * U * (1 + spread),
                 tol_h, tol_w, sure)


def inputs(n, size, v, dtype, seed=0, ignored=0.0, device="cuda"):
    """Hidden states that each point at one word, most labels that word."""
    gen = torch.Generator().manual_seed(seed)
    weight = torch.randn(v, size, generator=gen) / math.sqrt(size)
    word = torch.randint(v, (n,), generator=gen)
    hidden = torch.randn(n, size, generator=gen) + (2 + 6 * torch.rand(n, 1, generator=gen)) * weight[word]
    other = torch.randint(v, (n,), generator=gen)
    labels = torch.where(torch.rand(n, generator=gen) < 0.7, word, other)
    labels = torch.where(torch.rand(n, generator=gen) < ignored, -100, labels)
    return hidden.to(device, dtype), weight.to(device, dtype), labels.to(device)
