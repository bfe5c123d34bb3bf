"""vocab_loss and vocab_loss_confidence on the GPU at sizes that together take every
kernel that is built, each in one and in several pieces of the vocabulary where that
occurs (``test_vocab_plan.py`` checks that on the CPU), and both gradients at every size
of ``test_gpu_vocab.py``, whatever tokens have two top labels."""

from __future__ import annotations

import pytest
import torch

from ace_kernels import VocabConfig
from gpu_helpers import say
from test_gpu_vocab import SIZES, _compare_all, _drawn
from vocab_reference import inputs

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16

# tokens, hidden size, vocabulary, and what of the plan they are for (tiles by their
# token or word side).  Hidden sizes are ragged in all ways: no whole 16 bytes, no
# whole four values, or less than a step.
PLANS = {
    2: [
        (331, 150, 34567),   # score 128, dh and dw 256
        (1030, 520, 40003),  # all of 256, rows of whole 16 bytes
        (347, 141, 396103),  # all of 256, two pieces
        (14309, 134, 9294),  # dh 256 and dw by tokens, two pieces
        (419, 20, 331213),   # dh and dw 128, two pieces
        (470, 8, 288235),    # dh 128, dw 64, two pieces
        (75, 10, 1800003),   # score 128, two pieces
        (53, 12, 2600003),   # score and dh 64, two pieces
        (9, 12, 15200001),   # score and dh 32, two pieces
        (131, 12, 34511),    # score 256, dh and dw 64
        (70, 24, 52061),     # all of 128
        (3, 72, 66001),      # score and dw 64, dh 32
        (2, 13, 16483),      # dw 64
        (1300, 40, 700),     # dw by tokens
        (5, 88, 900),        # score and dw 32
    ],
    4: [
        (101, 20, 49547),    # score, dh and dw 128
        (35, 12, 67103),     # score and dh 64, dw 32
        (7321, 12, 9091),    # score 64, dw by tokens, two pieces
        (929, 9, 72263),     # score 128, dh and dw 64, two pieces
        (163, 10, 425147),   # dw 32, two pieces
        (20, 10, 3400003),   # dh 32, two pieces
        (207, 36, 331423),   # score 32, dw 128, two pieces
        (5621, 10, 11887),   # score and dh 128, two pieces
        (1111, 262, 20011),  # all of 128
        (1300, 40, 700),     # dw by tokens
        (5, 88, 900),        # score and dw 32
        (3, 7, 33001),       # dw 64
    ],
}
CASES = [(dtype, *sizes) for dtype in (BF16, F16, F32) for sizes in PLANS[4 if dtype is F32 else 2]]


@pytest.mark.parametrize("dtype,n,size,v", CASES)
def test_every_kernel(dtype, n, size, v) -> None:
    say(f"vocab plan {n}x{size}x{v} {dtype}")
    hidden, weight, labels = inputs(n, size, v, dtype, seed=n, ignored=0.2)
    gen = torch.Generator().manual_seed(v)
    gc = torch.randn(n, generator=gen).cuda()
    go = torch.randn(n, generator=gen).cuda()
    _compare_all(hidden, weight, labels, VocabConfig(), torch.tensor(0.7, device="cuda"), gc / n)
    _compare_all(hidden, weight, labels, VocabConfig(reduction="none"), go, gc)
    _compare_all(hidden, weight, labels, VocabConfig(reduction="sum"), torch.tensor(-1.5, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,size,v", SIZES)
def test_sizes_with_both_gradients(n, size, v, dtype) -> None:
    say(f"vocab {n}x{size}x{v} {dtype}")
    hidden, weight, labels = inputs(n, size, v, dtype, seed=n + v, ignored=0.2)
    gc = (torch.randn(n, generator=torch.Generator().manual_seed(5)) / n).cuda()
    _compare_all(hidden, weight, labels, VocabConfig(), torch.tensor(0.7, device="cuda"), gc)


@pytest.mark.parametrize("seed", range(48))
def test_drawn_sizes_with_both_gradients(seed) -> None:
    n, size, v, dtype, share = _drawn(seed)
    say(f"vocab drawn {n}x{size}x{v} {dtype} ignored {share}")
    hidden, weight, labels = inputs(n, size, v, dtype, seed=seed, ignored=share)
    gc = (torch.randn(n, generator=torch.Generator().manual_seed(seed)) / n).cuda()
    _compare_all(hidden, weight, labels, VocabConfig(reduction=["mean", "sum", "none"][seed // 3 % 3]), None, gc)
