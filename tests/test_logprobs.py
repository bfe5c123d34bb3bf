"""token_logprobs on the CPU: what it refuses, its options, and the library's own
argument checks (nothing is launched)."""

from __future__ import annotations

import pytest
import torch
from pydantic import ValidationError

from ace_kernels import LogprobConfig, _lib, logprobs, token_logprobs

FAKE = 256


class Claims:
    """A CPU tensor that says it is on the GPU, for the checks behind that one."""

    def __init__(self, t, index=0):
        self.t, self.dtype, self.shape, self.device = t, t.dtype, t.shape, torch.device("cuda", index)

    def dim(self):
        return self.t.dim()


def test_config() -> None:
    cfg = LogprobConfig()
    assert (cfg.top, cfg.temperature, cfg.ignore_index) == (0, 1.0, -100)
    for bad in (dict(top=-1), dict(top=33), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf")), dict(ignore_index=2**63), dict(z=1)):
        with pytest.raises(ValidationError):
            LogprobConfig(**bad)
    with pytest.raises(ValidationError):
        cfg.top = 3


def test_refusals() -> None:
    x, y = torch.randn(5, 8), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(ValueError, match="HIP"):
        token_logprobs(x, y)
    with pytest.raises(ValueError, match=r"\[..., V\]"):
        token_logprobs(torch.tensor(1.0), y)
    with pytest.raises(ValueError, match=r"\[..., V\]"):
        token_logprobs(torch.randn(5, 0), y)
    with pytest.raises(ValueError, match="one per row"):
        token_logprobs(x, y[:4])
    with pytest.raises(ValueError, match="there are 8 words"):
        token_logprobs(x, y, LogprobConfig(top=9))
    cfg = LogprobConfig()
    logprobs._check(Claims(x), Claims(y), cfg)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        logprobs._check(Claims(x.double()), Claims(y), cfg)
    with pytest.raises(TypeError, match="must be integers"):
        logprobs._check(Claims(x), Claims(y.float()), cfg)
    with pytest.raises(TypeError, match="must be integers"):
        logprobs._check(Claims(x), Claims(y.bool()), cfg)
    with pytest.raises(ValueError, match="tokens on cuda:1"):
        logprobs._check(Claims(x), Claims(y, 1), cfg)
    with pytest.raises(ValueError, match="tokens on cpu"):
        logprobs._check(Claims(x), y, cfg)


def _forward(**changed):
    a = dict(logits=FAKE, dtype=_lib.BF16, stride=1000, tokens=FAKE, rows=3, vocab=1000, ignore=-100, temperature=1.0,
             top=2, saved=FAKE, logprob=FAKE, entropy=FAKE, top_logprobs=FAKE, top_tokens=FAKE, tickets=FAKE,
             ticket_bytes=1 << 30, ws=FAKE, nbytes=1 << 40)
    a.update(changed)
    return _lib.lib().ace_logprob_forward(*a.values(), None)


def _backward(**changed):
    a = dict(logits=FAKE, dtype=_lib.BF16, stride=1000, rows=3, vocab=1000, temperature=1.0, saved=FAKE, gl=FAKE, ge=FAKE,
             d=FAKE)
    a.update(changed)
    return _lib.lib().ace_logprob_backward(*a.values(), None)


BAD = [dict(logits=None), dict(logits=FAKE + 1), dict(dtype=_lib.F64), dict(stride=-1), dict(rows=-1), dict(vocab=0),
       dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=1e4), dict(saved=None), dict(saved=FAKE + 8)]


@pytest.mark.parametrize("changed", BAD + [dict(tokens=None), dict(top=-1), dict(vocab=1, stride=1), dict(logprob=None),
                                           dict(entropy=None), dict(top_logprobs=None), dict(top_tokens=None)])
def test_forward_refuses_before_launch(changed) -> None:
    assert _forward(**changed) == _lib.EINVAL


@pytest.mark.parametrize("changed", BAD + [dict(d=None)])
def test_backward_refuses_before_launch(changed) -> None:
    assert _backward(**changed) == _lib.EINVAL


def test_last_block_stays_below_the_grid_limit() -> None:
    # four groups a block: 2^26 - 1 of them would round up to 2^32 threads
    call = dict(rows=8191, vocab=8193 * 2048, stride=8193 * 2048)
    assert call["rows"] * 8193 == (1 << 26) - 1
    assert _forward(**call) == _lib.EUNSUPPORTED and _backward(**call) == _lib.EUNSUPPORTED


def test_limits_and_workspace() -> None:
    lib = _lib.lib()
    for call in (_forward, _backward):
        assert call(rows=1 << 24) == _lib.EUNSUPPORTED
        assert call(vocab=(1 << 30) + 1) == _lib.EUNSUPPORTED
        assert call(rows=1 << 23, vocab=1 << 20) == _lib.EUNSUPPORTED
        assert call(rows=0, logits=None, saved=None) == 0  # nothing to do
    assert _forward(top=33) == _lib.EUNSUPPORTED
    wide = dict(vocab=131072, stride=131072)
    need = lib.ace_logprob_workspace_bytes(_lib.BF16, 3, 131072, 2)
    tickets = lib.ace_logprob_ticket_bytes(_lib.BF16, 3, 131072)
    assert need > 0 and tickets > 0
    assert _forward(**wide, nbytes=need - 1) == 3 and _forward(**wide, ticket_bytes=tickets - 1) == 3
    assert _forward(**wide, ws=None) == _lib.EINVAL and _forward(**wide, tickets=FAKE + 2) == _lib.EINVAL
    # rows that are not cut need neither
    assert lib.ace_logprob_workspace_bytes(_lib.BF16, 100000, 1000, 2) == 0
    assert lib.ace_logprob_ticket_bytes(_lib.BF16, 100000, 1000) == 0
    assert lib.ace_logprob_workspace_bytes(_lib.BF16, 0, 1000, 2) == 0
    assert lib.ace_logprob_saved_bytes(3) >= 48 and lib.ace_logprob_saved_bytes(0) > 0
    # tickets and parts fit what the stream's buffers hold at any size
    for rows in (1, 2, 31, 500, 2047, 2048):
        for vocab in (1, 5003, 32000, 131072, 1 << 20):
            for dtype in (_lib.F32, _lib.BF16):
                n, t = lib.ace_logprob_workspace_bytes(dtype, rows, vocab, 32), lib.ace_logprob_ticket_bytes(dtype, rows, vocab)
                assert (n == 0) == (t == 0) and n <= rows * 32 * 34 * 8 and t <= rows * 256


def test_tangents_are_refused() -> None:
    import torch.autograd.forward_ad as fwd

    x = torch.randn(5, 8)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="token_logprobs has no forward-mode derivative"):
        _lib.autograd().token_logprobs(fwd.make_dual(x, torch.ones_like(x)), torch.zeros(5, dtype=torch.int64), -100, 1.0,
                                       0, None)
