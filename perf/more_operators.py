"""Performance cases of what a language model's step has beside its losses: the
log probabilities of given tokens with the entropy and the top alternatives
(``token_logprobs``), the router's choice of experts with their weights
(``route_tokens``), tokens sorted by expert (``expert_order``, ``to_experts``) and
the experts' rows added back to their tokens (``from_experts``).

``listed()`` holds the named cases, ``draw(rng)`` gives more over the same
ranges.  ``run`` makes one pass: an operator with its gradients, or without them
when serving.  With ``own`` set it calls the package; otherwise it computes the
same from elementary torch operations in float32.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_IGNORE = -100
# the largest listed cases: tokens x vocabulary, tokens x experts, copies of
# tokens x width
_MOST_LOGITS = 8192 * 65536
_MOST_SCORES = 131072 * 256
_MOST_ROWS = 16384 * 4 * 4096


def _logprobs(name, mode, tokens, vocab, dtype, top=0, ignored=0.0, temperature=1.0):
    """mode: "score" (no gradient) or "train" (gradients of log probabilities and
    entropies).  top: alternatives asked for.  ignored: the share of tokens that
    are not counted."""
    case = {"op": "logprobs", "mode": mode, "tokens": tokens, "vocab": vocab, "dtype": dtype, "top": top,
            "ignored": ignored, "temperature": temperature}
    if name:
        case["name"] = name
    return case


def _route(name, mode, tokens, experts, top_k, dtype, normalize, masked=0.0):
    case = {"op": "route", "mode": mode, "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "normalize": normalize, "masked": masked}
    if name:
        case["name"] = name
    return case


def _rows(name, op, mode, tokens, width, top_k, experts, dtype, masked=0.0):
    """op: "to" (the order, and the tokens' rows in it) or "from" (rows back to
    their tokens, weighted).  masked: the share of tokens that take no expert."""
    case = {"op": op, "mode": mode, "tokens": tokens, "width": width, "top_k": top_k, "experts": experts,
            "dtype": dtype, "masked": masked}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the next token of one sequence, with five alternatives: latency
        _logprobs("logprobs bf16 1x131072 top 5", "score", 1, 131072, "bf16", top=5),
        # a batch of sequences at one decoding step, an odd vocabulary, sampled
        # at a temperature
        _logprobs("logprobs f16 48x50257 top 20", "score", 48, 50257, "f16", top=20, temperature=0.7),
        # scored prompts whose answer reports alternatives
        _logprobs("logprobs bf16 4096x32000 top 5", "score", 4096, 32000, "bf16", top=5, ignored=0.1),
        # a unit-sized policy step in float32 with an odd vocabulary
        _logprobs("logprobs train f32 384x5003", "train", 384, 5003, "f32", ignored=0.1),
        # a policy step of a mid-sized model: log probabilities and an entropy term
        _logprobs("logprobs train bf16 8192x65536", "train", 8192, 65536, "bf16", ignored=0.05),
        # one decoding step's router
        _route("route f32 64x8 top 2", "score", 64, 8, 2, "f32", True),
        # a training batch's router, padded
        _route("route train bf16 32768x64 top 6", "train", 32768, 64, 6, "bf16", True, masked=0.1),
        # a wide router over a large global batch, weights that are not normalised
        _route("route train f32 131072x256 top 8", "train", 131072, 256, 8, "f32", False),
        # one decoding step's tokens to their experts
        _rows("to bf16 33x2048 top 2 of 8", "to", "score", 33, 2048, 2, 8, "bf16"),
        # a training batch to its experts, and the gradient back
        _rows("to train bf16 16384x4096 top 4 of 64", "to", "train", 16384, 4096, 4, 64, "bf16", masked=0.05),
        # odd sizes under float16, padded
        _rows("from train f16 1999x1001 top 2 of 100", "from", "train", 1999, 1001, 2, 100, "f16", masked=0.3),
        # many small experts: rows back to the tokens, with all gradients
        _rows("from train bf16 8192x2048 top 8 of 256", "from", "train", 8192, 2048, 8, 256, "bf16"),
    ]


def _log_between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    masked = rng.choice([0.0, 0.1, 0.4])
    kind = rng.choice(["logprobs", "logprobs", "route", "to", "from"])
    mode = rng.choice(["train", "score"])
    if kind == "logprobs":
        vocab = _log_between(rng, 1000, 200000)
        if rng.random() < 0.5:
            vocab = max(1024, vocab // 128 * 128)
        tokens = _log_between(rng, 1, min(16384, _MOST_LOGITS // (4 if dtype == "f32" else 2) // vocab))
        top = rng.choice([0, 1, 5, 20]) if mode == "score" else 0
        return _logprobs(None, mode, tokens, vocab, dtype, top, masked, rng.choice([1.0, 1.0, 0.6, 1.3]))
    experts = _log_between(rng, 4, 256)
    if rng.random() < 0.6:
        experts = max(4, experts // 8 * 8)
    top_k = rng.randint(1, min(8, experts))
    if kind == "route":
        tokens = _log_between(rng, 1, min(131072, _MOST_SCORES // 2 // experts))
        return _route(None, mode, tokens, experts, top_k, dtype, rng.random() < 0.5, masked)
    width = _log_between(rng, 64, 8192)
    if rng.random() < 0.75:
        width = max(64, width // 64 * 64)
    tokens = _log_between(rng, 1, min(65536, _MOST_ROWS // (4 if dtype == "f32" else 2) // (top_k * width)))
    return _rows(None, kind, mode, tokens, width, top_k, experts, dtype, masked)


# ------------------------------------------------------------------- inputs


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _loss_scale(case):
    """What backward hands the loss: 1, or the scale that training in float16
    uses so that gradients do not underflow."""
    return 4096.0 if case["dtype"] == "f16" else 1.0


def _logprobs_inputs(case, seed):
    """Logits of a model that has learned something: unit noise times two, and
    one word that stands out strongly or weakly; three quarters of the given
    tokens are that word."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, v = case["tokens"], case["vocab"]
    word = torch.randint(v, (n,), generator=gen, device="cuda")
    logits = 2.0 * _normal(gen, n, v)
    logits[torch.arange(n, device="cuda"), word] += math.log(v) * (0.5 + _uniform(gen, n))
    other = torch.randint(v, (n,), generator=gen, device="cuda")
    tokens = torch.where(_uniform(gen, n) < 0.75, word, other)
    tokens = torch.where(_uniform(gen, n) < case["ignored"], _IGNORE, tokens)
    inputs = {"logits": logits.to(_DTYPES[case["dtype"]]), "tokens": tokens}
    if case["mode"] == "train":  # advantages of a policy step, and a share of the entropy
        inputs["logprob_grad"] = _loss_scale(case) / n * _normal(gen, n)
        inputs["entropy_grad"] = torch.full((n,), -0.01 * _loss_scale(case) / n, device="cuda")
    return inputs


def _route_inputs(case, seed):
    """Router scores of tokens with a shared preference for some experts."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, e, k = case["tokens"], case["experts"], case["top_k"]
    logits = 1.5 * _normal(gen, n, e) + _normal(gen, 1, e)
    inputs = {"logits": logits.to(_DTYPES[case["dtype"]]),
              "mask": _uniform(gen, n) >= case["masked"] if case["masked"] else None}
    if case["mode"] == "train":
        inputs["grad"] = _loss_scale(case) * _normal(gen, n, k)
    return inputs


def _rows_inputs(case, seed):
    """Tokens' choices of experts, some more popular than others; hidden states,
    or the experts' outputs in expert order with the weights and the order."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, w, k, e = case["tokens"], case["width"], case["top_k"], case["experts"]
    dtype, train = _DTYPES[case["dtype"]], case["mode"] == "train"
    experts = torch.topk(1.5 * _normal(gen, n, e) + _normal(gen, 1, e), k, dim=1).indices
    if case["masked"]:
        experts = torch.where(_uniform(gen, n, 1) < case["masked"], -1, experts)
    if case["op"] == "to":
        inputs = {"experts": experts, "x": _normal(gen, n, w).to(dtype)}
        if train:
            inputs["grad"] = _normal(gen, n * k, w).to(dtype)
        return inputs
    offsets, source, place = _plain_order(experts, e)
    inputs = {"rows": _normal(gen, n * k, w).to(dtype), "offsets": offsets, "source": source, "place": place,
              "weights": torch.softmax(_normal(gen, n, k), 1) * (experts >= 0)}
    if train:
        inputs["grad"] = _normal(gen, n, w).to(dtype)
    return inputs


_INPUTS = {"logprobs": _logprobs_inputs, "route": _route_inputs, "to": _rows_inputs, "from": _rows_inputs}
_LEAVES = {"logprobs": ("logits",), "route": ("logits",), "to": ("x",), "from": ("rows", "weights")}


def prepare(case, seed):
    state = {"case": case, **_INPUTS[case["op"]](case, seed)}
    if case["mode"] == "train":
        for name in _LEAVES[case["op"]]:
            state[name].requires_grad_(True)
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        with torch.set_grad_enabled(state["case"]["mode"] == "train"):
            return {"logprobs": _own_logprobs, "route": _own_route, "to": _own_to, "from": _own_from}[op](state)
    with torch.no_grad():
        return {"logprobs": _plain_logprobs, "route": _plain_route, "to": _plain_to, "from": _plain_from}[op](state)


# ------------------------------------------------------------ the package's


def _package():
    path = str(Path(__file__).resolve().parent.parent / "ace-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ace_kernels

    return ace_kernels


def _own_logprobs(state):
    ace, case = _package(), state["case"]
    config = ace.LogprobConfig(top=case["top"], temperature=case["temperature"], ignore_index=_IGNORE)
    out = ace.token_logprobs(state["logits"], state["tokens"], config)
    result = {"logprob": out.logprob, "entropy": out.entropy}
    if case["top"]:
        result["top_logprobs"], result["top_tokens"] = out.top_logprobs, out.top_tokens
    if case["mode"] == "train":
        upstream = (state["logprob_grad"], state["entropy_grad"])
        (result["grad"],) = torch.autograd.grad((out.logprob, out.entropy), state["logits"], upstream)
    return result


def _own_route(state):
    ace, case = _package(), state["case"]
    config = ace.RouteConfig(top_k=case["top_k"], normalize=case["normalize"])
    out = ace.route_tokens(state["logits"], config, mask=state["mask"])
    result = {"experts": out.experts, "weights": out.weights}
    if case["mode"] == "train":
        (result["grad"],) = torch.autograd.grad(out.weights, state["logits"], state["grad"])
    return result


def _own_to(state):
    ace = _package()
    order = ace.expert_order(state["experts"], state["case"]["experts"])
    rows = ace.to_experts(state["x"], order)
    result = {"offsets": order.offsets, "source": order.source, "place": order.place, "rows": rows}
    if state["case"]["mode"] == "train":
        (result["grad"],) = torch.autograd.grad(rows, state["x"], state["grad"])
    return result


def _own_from(state):
    ace = _package()
    order = ace.ExpertOrder(state["offsets"], state["source"], state["place"])
    out = ace.from_experts(state["rows"], order, state["weights"])
    result = {"out": out}
    if state["case"]["mode"] == "train":
        leaves = (state["rows"], state["weights"])
        result["rows_grad"], result["weights_grad"] = torch.autograd.grad(out, leaves, state["grad"])
    return result


# ---------------------------------------------------------- the plain forms


def _plain_logprobs(state):
    case, tokens = state["case"], state["tokens"]
    logits = state["logits"].float()
    n, v = logits.shape
    counted = (tokens >= 0) & (tokens < v) & (tokens != _IGNORE)
    at = torch.where(counted, tokens, 0)[:, None]
    out = {}
    if case["top"]:
        # the logits' bits in their order above the words' numbers: equal ones
        # go to the lowest number
        bits = (logits + 0.0).view(torch.int32)
        bits = bits ^ ((bits >> 31) & 0x7FFFFFFF)
        keys = (bits.long() << 32) | (v - 1 - torch.arange(v, device=logits.device))
        top_at = v - 1 - (torch.topk(keys, case["top"], dim=1).values & 0xFFFFFFFF)
        del bits, keys
    s = logits if case["temperature"] == 1.0 else logits / case["temperature"]
    s = s - s.amax(1, keepdim=True)
    s -= s.exp().sum(1, keepdim=True).log()  # log probabilities
    p = s.exp()
    entropy = -(p * s).sum(1)
    out["logprob"] = torch.where(counted, s.gather(1, at)[:, 0], 0.0)
    out["entropy"] = torch.where(counted, entropy, 0.0)
    if case["top"]:
        out["top_logprobs"] = torch.where(counted[:, None], s.gather(1, top_at), 0.0)
        out["top_tokens"] = torch.where(counted[:, None], top_at, -1)
    if case["mode"] == "train":
        g = torch.where(counted, state["logprob_grad"], 0.0)[:, None]
        h = torch.where(counted, state["entropy_grad"], 0.0)[:, None]
        d = s.add_(entropy[:, None]).mul_(h).add_(g).mul_(p).neg_()
        d.scatter_add_(1, at, g)
        out["grad"] = (d if case["temperature"] == 1.0 else d / case["temperature"]).to(state["logits"].dtype)
    return out


def _plain_route(state):
    case, mask = state["case"], state["mask"]
    k, logits = case["top_k"], state["logits"].float()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    # a stable sort: ties go to the lowest index
    experts = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    weights = p.gather(1, experts)
    total = weights.sum(1, keepdim=True)
    if case["normalize"]:
        weights = weights / total
    on = torch.ones_like(logits[:, :1], dtype=torch.bool) if mask is None else mask[:, None]
    out = {"experts": torch.where(on, experts, -1), "weights": torch.where(on, weights, 0.0)}
    if case["mode"] == "train":
        d = weights * state["grad"]
        if case["normalize"]:
            grad = torch.zeros_like(p).scatter_(1, experts, d - weights * d.sum(1, keepdim=True))
        else:
            grad = torch.zeros_like(p).scatter_(1, experts, d) - p * d.sum(1, keepdim=True)
        out["grad"] = torch.where(on, grad, 0.0).to(state["logits"].dtype)
    return out


def _plain_order(experts, count):
    """(offsets, source, place): a stable sort of the choices by expert, those
    without one last."""
    flat = experts.reshape(-1)
    routed = (flat >= 0) & (flat < count)
    source = torch.sort(torch.where(routed, flat, count), stable=True).indices
    per_expert = torch.zeros(count + 1, dtype=torch.int64, device=flat.device)
    per_expert.scatter_add_(0, torch.where(routed, flat, count), torch.ones_like(flat))
    offsets = torch.cat([per_expert.new_zeros(1), per_expert[:count].cumsum(0)])
    place = torch.empty_like(flat).scatter_(0, source, torch.arange(flat.numel(), device=flat.device))
    source = torch.where(torch.arange(flat.numel(), device=flat.device) < offsets[-1], source, -1)
    return offsets, source, torch.where(routed, place, -1).reshape(experts.shape)


def _plain_to(state):
    case, x = state["case"], state["x"]
    offsets, source, place = _plain_order(state["experts"], case["experts"])
    rows = torch.where((source >= 0)[:, None], x[source.clamp(min=0) // case["top_k"]], 0.0)
    out = {"offsets": offsets, "source": source, "place": place, "rows": rows}
    if case["mode"] == "train":
        back = torch.where((place >= 0)[:, :, None], state["grad"][place.clamp(min=0)], 0.0)
        out["grad"] = back.float().sum(1).to(x.dtype)
    return out


def _plain_from(state):
    rows, place, weights = state["rows"], state["place"], state["weights"]
    routed = (place >= 0)[:, :, None]
    mine = torch.where(routed, rows[place.clamp(min=0)], 0.0).float()
    out = {"out": (mine * weights[:, :, None]).sum(1).to(rows.dtype)}
    if state["case"]["mode"] == "train":
        grad = state["grad"].float()[:, None]
        out["weights_grad"] = (mine * grad).sum(2)
        back = torch.where(routed, weights[:, :, None] * grad, 0.0).to(rows.dtype)
        source = state["source"]
        back = back.reshape(rows.shape)[source.clamp(min=0)]
        out["rows_grad"] = torch.where((source >= 0)[:, None], back, 0.0)
    return out


# -------------------------------------------------------------------- sizes


def work(case):
    """Inputs read once, outputs written once.  Log probabilities: about 8
    operations a logit in each direction.  A router: about 20 operations a score.
    Rows: each token's once, each of its copies once."""
    size = 4 if case["dtype"] == "f32" else 2
    train, n = case["mode"] == "train", case["tokens"]
    if case["op"] == "logprobs":
        counted = n * (1.0 - case["ignored"])
        logits = counted * case["vocab"]
        moved = size * logits + 8 * n + 8 * n + 12 * case["top"] * n
        if train:
            moved += size * n * case["vocab"] + 8 * n
        return {"bytes": moved, "flops": (16 if train else 8) * logits}
    k = case["top_k"]
    on = 1.0 - case["masked"]
    if case["op"] == "route":
        scores = n * case["experts"]
        moved = size * on * scores + 12 * n * k + (n if case["masked"] else 0)
        if train:
            moved += size * scores + 4 * n * k
        return {"bytes": moved, "flops": (40 if train else 20) * on * scores}
    row = size * case["width"]
    copies, routed = n * k, on * n * k
    if case["op"] == "to":
        moved = 24 * copies + row * (on * n + copies)
        if train:
            moved += row * (routed + n)
        return {"bytes": moved, "flops": routed * case["width"] if train else 0}
    moved = 12 * copies + row * (routed + n)
    if train:
        moved += 4 * copies + row * (on * n + copies)
    return {"bytes": moved, "flops": (6 if train else 2) * routed * case["width"]}


# ------------------------------------------------------------------ 64 bits


def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    inputs = _INPUTS[case["op"]](case, seed)
    kind = {"logprobs": _exact_logprobs, "route": _exact_route, "to": _exact_to, "from": _exact_from}
    return kind[case["op"]](case, inputs)


def _exact_logprobs(case, inputs):
    y = inputs["tokens"]
    rows = torch.nonzero(y >= 0)[:, 0]
    x = inputs["logits"][rows].double()
    here = torch.arange(len(rows), device="cuda")
    lp = torch.log_softmax(x / case["temperature"], 1)
    p = lp.exp()
    h = -(p * lp).sum(1)

    def placed(values):
        return torch.zeros((len(y), *values.shape[1:]), dtype=values.dtype, device="cuda").index_copy_(0, rows, values)

    out = {"logprob": placed(lp[here, y[rows]]), "entropy": placed(h)}
    if case["top"]:
        best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_logprobs"] = placed(lp.gather(1, best))
        out["top_tokens"] = placed(best + 1) - 1
    if case["mode"] == "train":
        g, e = inputs["logprob_grad"].double()[rows], inputs["entropy_grad"].double()[rows]
        d = -p * (g[:, None] + e[:, None] * (lp + h[:, None]))
        d[here, y[rows]] += g
        out["grad"] = placed(d / case["temperature"])
    return out


def _exact_route(case, inputs):
    x, mask, k = inputs["logits"].double(), inputs["mask"], case["top_k"]
    n, e = x.shape
    on = torch.ones(n, 1, dtype=torch.float64, device="cuda") if mask is None else mask.double()[:, None]
    order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
    chosen = torch.zeros_like(x).scatter_(1, order, 1.0)
    p = torch.softmax(x if not case["normalize"] else torch.where(chosen > 0, x, -math.inf), 1)
    out = {"experts": torch.where(on > 0, order, -1), "weights": p.gather(1, order) * on}
    if case["mode"] == "train":
        up = torch.zeros_like(x).scatter_(1, order, inputs["grad"].double())
        out["grad"] = p * (up - (p * up).sum(1, keepdim=True)) * on
    return out


def _exact_order(experts, count):
    flat = experts.reshape(-1)
    numbers = torch.arange(flat.numel(), device=flat.device)
    # the place of a choice: all of lower experts, then those before it of its own
    key = torch.where(flat >= 0, flat, count) * flat.numel() + numbers
    ranked = torch.argsort(key)
    place = torch.empty_like(ranked)
    place[ranked] = numbers
    offsets = torch.searchsorted(key[ranked], torch.arange(count + 1, device=flat.device) * flat.numel())
    return offsets, torch.where(flat[ranked] >= 0, ranked, -1), torch.where(flat >= 0, place, -1).reshape(experts.shape)


def _exact_to(case, inputs):
    offsets, source, place = _exact_order(inputs["experts"], case["experts"])
    k, x = case["top_k"], inputs["x"].double()
    total = int(offsets[-1])
    rows = torch.zeros(len(source), case["width"], dtype=torch.float64, device="cuda")
    rows[:total] = x[torch.div(source[:total], k, rounding_mode="floor")]
    out = {"offsets": offsets, "source": source, "place": place, "rows": rows}
    if case["mode"] == "train":
        back = inputs["grad"][:total].double()
        token = torch.div(source[:total], k, rounding_mode="floor")
        out["grad"] = torch.zeros_like(x).index_add_(0, token, back)
    return out


def _exact_from(case, inputs):
    k, total = case["top_k"], int(inputs["offsets"][-1])
    slot = inputs["source"][:total]
    token = torch.div(slot, k, rounding_mode="floor")
    rows, weight = inputs["rows"][:total].double(), inputs["weights"].double().reshape(-1)[slot][:, None]
    out = {"out": torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")}
    out["out"].index_add_(0, token, rows * weight)
    if case["mode"] == "train":
        grad = inputs["grad"].double()[token]
        back = torch.zeros(case["tokens"] * k, case["width"], dtype=torch.float64, device="cuda")
        back[:total] = weight * grad
        per_slot = torch.zeros(case["tokens"] * k, dtype=torch.float64, device="cuda")
        per_slot[slot] = (rows * grad).sum(1)
        out["rows_grad"], out["weights_grad"] = back, per_slot.reshape(case["tokens"], k)
    return out
