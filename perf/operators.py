"""Performance cases of the language-model losses: cross entropy over a large
vocabulary straight from the hidden states (``vocab_loss``), the same with
each token's top-label confidence (``vocab_loss_confidence``, what the
calibration loss takes) and the balance loss of an expert router
(``balance_loss``).

``listed()`` holds the named cases, ``draw(rng)`` gives more over the same
ranges.  ``run`` makes one pass: a training step's loss with its gradients, or
an evaluation pass without.  With ``own`` set it calls the package; otherwise
it computes the same from elementary torch operations in float32.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_IGNORE = -100
# tokens x hidden x vocabulary of the largest listed case, and tokens x experts
_MOST_HEAD = 8192 * 4096 * 65536
_MOST_ROUTER = 131072 * 256


def _head(name, mode, tokens, hidden, vocab, dtype, ignored=0.0):
    """mode: "train" (mean loss, both gradients), "calibrated" (that with the
    confidences and their upstream gradient), "score" (each token's loss, no
    gradient).  ignored: the share of tokens whose label is not counted."""
    case = {"op": "head", "mode": mode, "tokens": tokens, "hidden": hidden, "vocab": vocab, "dtype": dtype,
            "ignored": ignored}
    if name:
        case["name"] = name
    return case


def _router(name, groups, tokens, experts, top_k, dtype, masked=0.0):
    """groups: layers (or sequences) that each have a balance loss of their
    own; masked: the share of tokens that are padding."""
    case = {"op": "router", "groups": groups, "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "masked": masked}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # scoring a handful of tokens, as when one answer's last words are
        # graded: the weight is read once and little else happens
        _head("score bf16 7x512x32000", "score", 7, 512, 32000, "bf16"),
        # a unit-sized training step in float32 with an odd vocabulary
        _head("train f32 384x320x5003", "train", 384, 320, 5003, "f32", ignored=0.1),
        # a step of a small model: one short batch
        _head("train bf16 2048x1024x32768", "train", 2048, 1024, 32768, "bf16"),
        # instruction tuning under float16 with loss scaling: the prompt's
        # tokens are not counted, no size is a round one
        _head("train f16 1999x1000x50001", "train", 1999, 1000, 50001, "f16", ignored=0.4),
        # a whole batch of a mid-sized model
        _head("train bf16 8192x4096x65536", "train", 8192, 4096, 65536, "bf16", ignored=0.05),
        # perplexity of a long text over a large multilingual vocabulary
        _head("score bf16 4096x2048x131072", "score", 4096, 2048, 131072, "bf16"),
        # the calibrated step: cross entropy plus a loss of the confidences
        _head("calibrated bf16 4096x1024x32000", "calibrated", 4096, 1024, 32000, "bf16", ignored=0.1),
        # a calibrated step of few tokens: the weight and its gradient are
        # nearly all there is to move
        _head("calibrated f16 96x2048x50304", "calibrated", 96, 2048, 50304, "f16"),
        # one layer's router on a short batch: launches and host work
        _router("router f32 1x512x8 top 2", 1, 512, 8, 2, "f32"),
        # every layer's router of one step in one call
        _router("router bf16 32x4096x64 top 6", 32, 4096, 64, 6, "bf16", masked=0.1),
        # balance per sequence, odd lengths, padded
        _router("router bf16 16x8191x100 top 1", 16, 8191, 100, 1, "bf16", masked=0.3),
        # a wide router over a large global batch in float32
        _router("router f32 1x131072x256 top 8", 1, 131072, 256, 8, "f32", masked=0.05),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.4:
        experts = _log_between(rng, 4, 256)
        if rng.random() < 0.6:
            experts = max(4, experts // 8 * 8)
        groups = rng.choice([1, 1, _log_between(rng, 2, 64)])
        tokens = max(1, min(131072, _log_between(rng, 64, _MOST_ROUTER / 4) // (groups * experts)))
        return _router(None, groups, tokens, experts, rng.randint(1, min(8, experts)),
                       rng.choice(["f32", "bf16", "bf16", "f16"]), masked=rng.choice([0.0, 0.1, 0.5]))
    mode = rng.choice(["train", "train", "train", "calibrated", "score"])
    hidden = _log_between(rng, 64, 4096)
    if rng.random() < 0.75:
        hidden = max(64, hidden // 64 * 64)
    vocab = _log_between(rng, 1000, 131072)
    if rng.random() < 0.5:
        vocab = max(1024, vocab // 128 * 128)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    most = _MOST_HEAD // (32 if dtype == "f32" else 2)
    tokens = _log_between(rng, 1, max(2, min(8192, most // (hidden * vocab))))
    return _head(None, mode, tokens, hidden, vocab, dtype, ignored=rng.choice([0.0, 0.05, 0.4]))


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _head_inputs(case, seed):
    """Hidden states of a model that has learned something: each points at
    one word's weight, strongly or weakly, on top of noise; three quarters of
    the labels are that word.  Logits have unit noise."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, h, v, dtype = case["tokens"], case["hidden"], case["vocab"], _DTYPES[case["dtype"]]
    weight = _normal(gen, v, h) / math.sqrt(h)
    word = torch.randint(v, (n,), generator=gen, device="cuda")
    strength = 4.0 + (2.0 + math.log(v)) * _uniform(gen, n, 1)
    hidden = _normal(gen, n, h) + strength * weight[word]
    other = torch.randint(v, (n,), generator=gen, device="cuda")
    labels = torch.where(_uniform(gen, n) < 0.75, word, other)
    labels = torch.where(_uniform(gen, n) < case["ignored"], _IGNORE, labels)
    inputs = {"hidden": hidden.to(dtype), "weight": weight.to(dtype), "labels": labels}
    if case["mode"] == "calibrated":  # what a calibration loss hands back for each confidence
        inputs["conf_grad"] = 0.5 * _loss_scale(case) / n * torch.sign(_normal(gen, n))
    return inputs


def _router_inputs(case, seed):
    """Router scores of tokens with a shared preference for some experts."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g, t, e = case["groups"], case["tokens"], case["experts"]
    logits = 1.5 * _normal(gen, g, t, e) + _normal(gen, g, 1, e)
    mask = _uniform(gen, g, t) >= case["masked"] if case["masked"] else None
    return {"logits": logits.to(_DTYPES[case["dtype"]]), "mask": mask}


def _loss_scale(case):
    """What backward hands the loss: 1, or the scale that training in float16
    uses so that gradients do not underflow."""
    return 4096.0 if case["dtype"] == "f16" else 1.0


def prepare(case, seed):
    state = {"case": case}
    if case["op"] == "router":
        state.update(_router_inputs(case, seed))
        state["logits"].requires_grad_(True)
        state["grad"] = torch.tensor(0.01 * _loss_scale(case), device="cuda")
        return state
    state.update(_head_inputs(case, seed))
    if case["mode"] != "score":
        state["hidden"].requires_grad_(True)
        state["weight"].requires_grad_(True)
        state["grad"] = torch.tensor(_loss_scale(case), device="cuda")
    return state


def run(state):
    router = state["case"]["op"] == "router"
    if own:
        return _own_router(state) if router else _own_head(state)
    with torch.no_grad():
        return _plain_router(state) if router else _plain_head(state)


# ------------------------------------------------------------ the package's


def _package():
    path = str(Path(__file__).resolve().parent.parent / "ace-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ace_kernels

    return ace_kernels


def _own_head(state):
    ace = _package()
    hidden, weight, labels = state["hidden"], state["weight"], state["labels"]
    mode = state["case"]["mode"]
    if mode == "score":
        with torch.no_grad():
            return {"loss": ace.vocab_loss(hidden, weight, labels, ace.VocabConfig(reduction="none"))}
    if mode == "train":
        loss = ace.vocab_loss(hidden, weight, labels)
        grads = torch.autograd.grad(loss, (hidden, weight), state["grad"])
        return {"loss": loss, "hidden_grad": grads[0], "weight_grad": grads[1]}
    out = ace.vocab_loss_confidence(hidden, weight, labels)
    grads = torch.autograd.grad((out.loss, out.confidence), (hidden, weight), (state["grad"], state["conf_grad"]))
    return {"loss": out.loss, "confidence": out.confidence, "correct": out.correct,
            "hidden_grad": grads[0], "weight_grad": grads[1]}


def _own_router(state):
    ace = _package()
    out = ace.balance_loss(state["logits"], ace.BalanceConfig(top_k=state["case"]["top_k"]), mask=state["mask"])
    (grad,) = torch.autograd.grad(out.loss, state["logits"], state["grad"])
    return {"loss": out.loss, "counts": out.counts, "grad": grad}


# ---------------------------------------------------------- the plain forms


def _plain_head(state):
    mode, labels = state["case"]["mode"], state["labels"]
    hidden, weight = state["hidden"].float(), state["weight"].float()
    counted = labels != _IGNORE
    at = torch.where(counted, labels, 0)[:, None]
    logits = hidden @ weight.t()
    top, top_at = logits.max(1, keepdim=True)
    label_logit = logits.gather(1, at)
    p = logits.sub_(top).exp_()  # in place: the logits are not needed again
    total = p.sum(1, keepdim=True)
    nll = torch.where(counted, (total.log() + top - label_logit)[:, 0], 0.0)
    if mode == "score":
        return {"loss": nll}
    share = 1.0 / counted.sum().clamp(min=1)
    loss = (nll.double().sum() * share).float()
    p /= total
    confidence = torch.where(counted, 1.0 / total[:, 0], 0.0)
    row = torch.where(counted, state["grad"] * share, 0.0)[:, None]
    out = {"loss": loss}
    if mode == "calibrated":
        out["confidence"] = confidence
        out["correct"] = (counted & (top_at == at)[:, 0]).float()
        back = (state["conf_grad"] * confidence)[:, None]
        p *= row - back
        p.scatter_add_(1, top_at, back)
    else:
        p *= row
    p.scatter_add_(1, at, -row)
    out["hidden_grad"] = (p @ weight).to(state["hidden"].dtype)
    out["weight_grad"] = (p.t() @ hidden).to(state["weight"].dtype)
    return out


def _plain_router(state):
    case, mask = state["case"], state["mask"]
    logits = state["logits"].float()
    g, t, e = logits.shape
    k = case["top_k"]
    counted = torch.ones((g, t), dtype=torch.bool, device=logits.device) if mask is None else mask
    p = torch.exp(logits - logits.amax(2, keepdim=True))
    p = p / p.sum(2, keepdim=True)
    # a stable sort: ties go to the lowest index
    chosen = torch.sort(logits, dim=2, descending=True, stable=True).indices[:, :, :k]
    ones = counted[:, :, None].expand(g, t, k).long()
    counts = torch.zeros((g, e), dtype=torch.int64, device=logits.device)
    counts.scatter_add_(1, chosen.reshape(g, t * k), ones.reshape(g, t * k))
    tokens = counted.sum(1, keepdim=True).clamp(min=1)
    mean_p = (p * counted[:, :, None]).sum(1) / tokens
    share = counts / (k * tokens)
    loss = e * (share * mean_p).sum(1).mean()
    pull = (state["grad"] * e / g * share / tokens)[:, None, :]
    grad = p * (pull - (pull * p).sum(2, keepdim=True)) * counted[:, :, None]
    return {"loss": loss, "counts": counts, "grad": grad.to(state["logits"].dtype)}


# -------------------------------------------------------------------- sizes


def work(case):
    """Inputs read once, outputs written once.  A head: a product forward, two
    backward, about 5 operations a logit beside them.  A router: about 20
    operations a score."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "router":
        scores = case["groups"] * case["tokens"] * case["experts"]
        masks = case["groups"] * case["tokens"] if case["masked"] else 0
        return {"bytes": 2 * size * scores + masks + 8 * case["groups"] * case["experts"], "flops": 20 * scores}
    n, h, v = case["tokens"], case["hidden"], case["vocab"]
    counted = n * (1.0 - case["ignored"])
    if case["mode"] == "score":
        return {"bytes": size * (counted * h + v * h) + 12 * n, "flops": counted * v * (2 * h + 5)}
    extra = 12 * n if case["mode"] == "calibrated" else 0
    return {"bytes": size * ((counted + n) * h + 2 * v * h) + 8 * n + extra, "flops": counted * v * (6 * h + 5)}


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    return _exact_router(case, seed) if case["op"] == "router" else _exact_head(case, seed)


def _exact_head(case, seed):
    inputs = _head_inputs(case, seed)
    h, w, y = inputs["hidden"].double(), inputs["weight"].double(), inputs["labels"]
    rows = torch.nonzero(y >= 0)[:, 0]
    scores = torch.mm(h[rows], w.t())
    lse = torch.logsumexp(scores, 1)
    here = torch.arange(len(rows), device="cuda")
    nll = torch.zeros(len(y), dtype=torch.float64, device="cuda")
    nll[rows] = lse - scores[here, y[rows]]
    if case["mode"] == "score":
        return {"loss": nll}
    best = scores.argmax(1)
    d = torch.exp(scores.sub_(lse[:, None]))
    conf_rows = d[here, best]
    upstream = _loss_scale(case)
    d_nll = torch.full((len(rows),), upstream / max(1, len(rows)), dtype=torch.float64, device="cuda")
    out = {"loss": nll.sum() / max(1, len(rows))}
    weight_of_p = d_nll
    if case["mode"] == "calibrated":
        pull = inputs["conf_grad"].double()[rows] * conf_rows
        weight_of_p = d_nll - pull
        out["confidence"] = torch.zeros_like(nll).index_put_((rows,), conf_rows)
        out["correct"] = torch.zeros_like(nll).index_put_((rows,), (best == y[rows]).double())
    d.mul_(weight_of_p[:, None])
    d[here, y[rows]] -= d_nll
    if case["mode"] == "calibrated":
        d[here, best] += pull
    out["hidden_grad"] = torch.zeros_like(h).index_copy_(0, rows, torch.mm(d, w))
    out["weight_grad"] = torch.mm(d.t(), h[rows])
    return out


def _exact_router(case, seed):
    inputs = _router_inputs(case, seed)
    x, mask, k = inputs["logits"].double(), inputs["mask"], case["top_k"]
    g, t, e = x.shape
    keep = torch.ones((g, t), dtype=torch.float64, device="cuda") if mask is None else mask.double()
    p = torch.softmax(x, 2)
    # an expert is chosen when fewer than k others come before it
    order = torch.argsort(x, dim=2, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(2, order, torch.arange(e, device="cuda").expand(g, t, e).contiguous())
    counts = ((rank < k).double() * keep[:, :, None]).sum(1)
    m = keep.sum(1).clamp(min=1.0)[:, None]
    q = e * counts / (k * m * m)
    losses = (q * (p * keep[:, :, None]).sum(1)).sum(1)
    u = 0.01 * _loss_scale(case) / g
    grad = u * p * (q[:, None, :] - torch.matmul(p, q[:, :, None])) * keep[:, :, None]
    return {"loss": losses.mean(), "counts": counts.long(), "grad": grad}
