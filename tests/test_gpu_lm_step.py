"""A language model's training step with all of its losses: cross entropy over
the vocabulary, the calibration of its confidences (``ace_loss``) and the
routers' balance loss, through one small model and one backward."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from ace_kernels import ACEConfig, BalanceConfig, VocabConfig, ace_loss, balance_loss, vocab_loss, vocab_loss_confidence
from oracle.reference import reference_ace

pytestmark = pytest.mark.gpu

LAYERS, WIDTH, EXPERTS, WORDS = 3, 64, 8, 500
ACE = ACEConfig(binning="soft", activation="none", num_bins=10)


class Tiny(nn.Module):
    """Embedding, residual layers that mix all experts by the router's softmax,
    and a head that is tied to the embedding."""

    def __init__(self) -> None:
        super().__init__()
        gen = torch.Generator().manual_seed(0)
        self.embed = nn.Parameter(torch.randn(WORDS, WIDTH, generator=gen) * 0.4)
        self.router = nn.Parameter(torch.randn(LAYERS, WIDTH, EXPERTS, generator=gen) * 0.3)
        self.expert = nn.Parameter(torch.randn(LAYERS, EXPERTS, WIDTH, WIDTH, generator=gen) * 0.1)

    def forward(self, words):
        x = self.embed[words]
        scores = []
        for i in range(LAYERS):
            s = x @ self.router[i]
            scores.append(s)
            mixed = torch.stack([x @ self.expert[i, e] for e in range(EXPERTS)], dim=-2)
            x = x + (torch.softmax(s, -1)[..., None] * torch.tanh(mixed)).sum(-2)
        return x, torch.stack(scores)


def _losses(hidden, weight, labels, scores, mask):
    out = vocab_loss_confidence(hidden, weight, labels)
    keep = labels != -100
    ace = ace_loss(out.confidence[keep][None, None], out.correct[keep][None, None], ACE)
    balance = balance_loss(scores, BalanceConfig(top_k=2), mask.expand(scores.shape[:-1]))
    return out.loss + 0.5 * ace + 0.01 * balance.loss, balance.counts


def _plain(hidden, weight, labels, scores, mask):
    """The same total in plain torch, differentiable, in the inputs' precision."""
    keep = labels != -100
    logits = hidden[keep] @ weight.t()
    ce = nn.functional.cross_entropy(logits, labels[keep])
    conf, at = torch.softmax(logits, 1).max(1)
    ace = reference_ace(conf[None, None].cpu(), (at == labels[keep]).to(conf.dtype)[None, None].cpu(), ACE).to(conf.device)
    p = torch.softmax(scores, -1) * mask[..., None]
    chosen = torch.sort(scores, dim=-1, descending=True, stable=True).indices[..., :2]
    n = (nn.functional.one_hot(chosen, EXPERTS).sum(-2) * mask[..., None]).sum((1, 2))
    m = mask.sum()
    balance = (EXPERTS * (n / (2 * m)) * (p.sum((1, 2)) / m)).sum(-1).mean()
    return ce + 0.5 * ace + 0.01 * balance, n


def _batch(seed):
    gen = torch.Generator().manual_seed(seed)
    words = torch.randint(WORDS, (4, 30), generator=gen).cuda()
    labels = words.roll(-1, 1).clone()
    labels[:, -1] = -100
    mask = torch.ones(4, 30, dtype=torch.bool, device="cuda")
    for b, length in enumerate((30, 17, 1, 25)):
        labels[b, max(0, length - 1):] = -100
        mask[b, length:] = False
    return words, labels, mask


def test_step_matches_plain_torch() -> None:
    """Loss within 1e-5 and gradients within 1e-4 of their norm of float64: the
    kernels' float32 sums are within 1e-6 (their own tests), and the calibration
    loss's soft bins pass them on with a factor below 2 K = 20."""
    model = Tiny().cuda()
    words, labels, mask = _batch(1)
    hidden, scores = model(words)
    scores = scores.flatten(1, 2)
    total, counts = _losses(hidden, model.embed, labels, scores, mask.flatten()[None])
    grads = torch.autograd.grad(total, list(model.parameters()))
    exact = Tiny().cuda().double()
    hidden, scores = exact(words)
    want, n = _plain(hidden, exact.embed, labels, scores, mask)
    want_grads = torch.autograd.grad(want, list(exact.parameters()))
    assert abs(float(total.detach()) - float(want.detach())) < 1e-5 * float(want.detach())
    assert torch.equal(counts, n)
    for a, b in zip(grads, want_grads):
        assert float((a.double() - b).norm()) <= 1e-4 * float(b.norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_runs(dtype) -> None:
    """A few optimiser steps, with the head in a lower precision than the
    parameters: everything stays finite and the tied weight gets both of its
    gradients."""
    model = Tiny().cuda()
    opt = torch.optim.AdamW(model.parameters(), lr=1e-2)
    for i in range(5):
        words, labels, mask = _batch(i)
        hidden, scores = model(words)
        total, counts = _losses(hidden.to(dtype), model.embed.to(dtype), labels, scores.flatten(1, 2), mask.flatten()[None])
        opt.zero_grad()
        total.backward()
        assert torch.isfinite(total) and all(torch.isfinite(p.grad).all() for p in model.parameters())
        assert int(counts.sum()) == 2 * LAYERS * int(mask.sum())
        opt.step()


def test_scoring_adds_up() -> None:
    """Each token's loss, their mean and their sum are of one piece, and a batch
    scored in two halves is the whole."""
    model = Tiny().cuda()
    words, labels, _ = _batch(3)
    with torch.no_grad():
        hidden, _ = model(words)
        each = vocab_loss(hidden, model.embed, labels, VocabConfig(reduction="none"))
        counted = int((labels != -100).sum())
        total = float(each.double().sum())
        # float32's rounding of the result
        assert abs(float(vocab_loss(hidden, model.embed, labels, VocabConfig(reduction="sum"))) - total) <= 1e-6 * total
        assert abs(float(vocab_loss(hidden, model.embed, labels)) - total / counted) <= 1e-6 * total / counted
        halves = [vocab_loss(hidden[i:i + 2], model.embed, labels[i:i + 2], VocabConfig(reduction="none")) for i in (0, 2)]
        assert torch.equal(torch.cat(halves), each)
