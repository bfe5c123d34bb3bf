"""The plan of the vocabulary loss on the CPU (``ace_vocab_plan.hpp``, compiled here
with g++): the tiles that sizes lead to, and the workspace that they need."""

from __future__ import annotations

import ctypes
import random
import re
import subprocess
from collections import namedtuple
from pathlib import Path
from typing import Set, Tuple

import pytest

from ace_kernels import _lib
from test_vocab_isa import _code_objects

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "ace-kernels_amd" / "csrc"
Plan = namedtuple("Plan", "score dh dw dw_parts pieces pad piece dh_blocks dh_segs dw_blocks dw_segs score_blocks "
                          "dscore_blocks forward_bytes backward_bytes")


@pytest.fixture(scope="module")
def harness(tmp_path_factory) -> ctypes.CDLL:
    out = tmp_path_factory.mktemp("vocab") / "libvocab.so"
    subprocess.run(["g++", "-O2", "-shared", "-fPIC", "-std=c++17", f"-I{CSRC}", str(HERE / "vocab_harness.cpp"), "-o", str(out)],
                   check=True, capture_output=True)
    lib = ctypes.CDLL(str(out))
    ll, i = ctypes.c_longlong, ctypes.c_int
    lib.vocab_plan.argtypes = [i, ll, ll, ll, ctypes.POINTER(ll)]
    lib.vocab_plan.restype = None
    lib.vocab_parts.argtypes = [i] * 5
    lib.vocab_parts.restype = ll
    lib.vocab_score_parts.argtypes = [i, ll, ll, ll]
    lib.vocab_score_parts.restype = ll
    return lib


def plan_of(lib, es, n, h, v) -> Plan:
    out = (ctypes.c_longlong * 15)()
    lib.vocab_plan(es, n, h, v, out)
    return Plan(*out)


def shape(lib, tile) -> Tuple[int, int]:
    bm, bn = ctypes.c_int(), ctypes.c_int()
    lib.vocab_tile(tile, ctypes.byref(bm), ctypes.byref(bn))
    return bm.value, bn.value


def _sizes():
    """Tokens, hidden sizes and vocabularies over what a card holds."""
    for n in sorted({int(2 ** (i / 3)) for i in range(60)}):
        for h in (1, 8, 64, 200, 512, 1024, 4096, 16384):
            for v in sorted({int(2 ** (i / 2)) for i in range(42)}):
                if h * v < 2 ** 36:
                    yield n, h, v


def test_every_kernel_that_is_built_is_chosen_by_some_size(harness) -> None:
    chosen: Set[Tuple[str, str, int, int]] = set()
    for letter, es in (("f", 4), ("DF16_", 2), ("DF16b", 2)):
        for sizes in _sizes():
            p = plan_of(harness, es, *sizes)
            chosen |= {("score", letter, *shape(harness, p.score)), ("dscore", letter, *shape(harness, p.score)),
                       ("dh", letter, *shape(harness, p.dh)), ("dw", letter, *shape(harness, p.dw))}
    built = set()
    for elf in _code_objects(_lib.LIB_PATH):
        for m in re.finditer(rb"_ZN3ace5vocab\d+(score|dscore|grad)_kernelINS_3mma4TileI(f|DF16_|DF16b)Li(\d+)ELi(\d+)E([^\0]*?)\.kd", elf):
            kernel = m[1].decode()
            if kernel == "grad":
                kernel = "dw" if b"ELb1EEEv" in m[5] else "dh"
            built.add((kernel, m[2].decode(), int(m[3]), int(m[4])))
    assert built, "no kernels found"
    assert built == chosen, f"never chosen: {sorted(built - chosen)}; not built: {sorted(chosen - built)}"


def _kernels(p: Plan) -> Set[Tuple]:
    """What a call runs that the numerics could depend on: each kernel's tile, whether
    the weight's gradient is cut along the tokens, in one or several pieces of the
    vocabulary; rows padded or not."""
    many = p.pieces > 1
    return {("score", p.score, many), ("dh", p.dh, many), ("dw", p.dw, bool(p.dw_parts), many), ("padded", bool(p.pad), many)}


@pytest.mark.parametrize("es", [2, 4])
def test_gpu_cases_take_every_kernel(harness, es) -> None:
    from test_gpu_vocab_plans import PLANS

    chosen: Set[Tuple] = set()
    for sizes in [*_sizes(), *PLANS[es]]:
        chosen |= _kernels(plan_of(harness, es, *sizes))
    tested: Set[Tuple] = set()
    for sizes in PLANS[es]:
        tested |= _kernels(plan_of(harness, es, *sizes))
    assert tested == chosen, f"not tested: {sorted(chosen - tested, key=str)}"


@pytest.mark.parametrize("es", [2, 4])
def test_the_workspace_holds_the_parts(harness, es) -> None:
    """Whatever the number of counted tokens, which the device alone knows, and in
    the last, shorter piece of the vocabulary too."""
    rng = random.Random(es)
    step = 64 // es
    for _ in range(3000):
        n, h, v = (int(2 ** rng.uniform(0, top)) for top in (17, 13, 19))
        p = plan_of(harness, es, n, h, v)
        width = -(-h * es // 16) * 16 // es
        assert p.piece % 256 == 0 and (p.pieces - 1) * p.piece < v <= p.pieces * p.piece
        bm, bn = shape(harness, p.score)
        assert harness.vocab_score_parts(es, n, h, v) >= -(-n // bn)
        for count in {1, n, rng.randint(1, n), rng.randint(1, n)}:
            tts = -(-count // bn)
            assert harness.vocab_parts(0, es, tts, -(-v // bm), p.score_blocks) <= harness.vocab_score_parts(es, n, h, v)
            hm, hn = shape(harness, p.dh)
            units = -(-min(p.piece, v) // step)
            assert harness.vocab_parts(1, es, -(-width // hm) * -(-count // hn), units, p.dh_blocks) <= p.dh_segs
            if p.dw_parts:
                wm, wn = shape(harness, p.dw)
                for words in {min(p.piece, v), v - (p.pieces - 1) * p.piece}:
                    tiles = -(-width // wm) * -(-words // wn)
                    assert harness.vocab_parts(2, es, tiles, -(-count // step), p.dw_blocks) <= p.dw_segs


@pytest.mark.parametrize("es,n,h,v,cut", [
    (2, 512, 512, 4000, False), (2, 768, 320, 5003, False), (2, 1024, 1024, 1000, False), (2, 2048, 512, 4000, False),
    (2, 4096, 512, 4000, True), (2, 4096, 1024, 1000, True), (2, 9000, 320, 5003, True), (2, 2048, 64, 1000, True),
    (2, 512, 64, 1000, False), (2, 512, 128, 2000, False), (4, 512, 512, 4000, False), (4, 1024, 320, 5003, False),
    (4, 1024, 1024, 700, False), (4, 2048, 256, 12000, True), (4, 2048, 1024, 1000, True), (4, 1024, 64, 1000, True),
    (4, 1024, 128, 2000, True), (4, 350, 128, 2000, False), (4, 512, 256, 12000, False), (4, 1500, 256, 12000, True),
    (2, 2500, 256, 12000, False), (2, 5000, 1024, 3000, False), (2, 5000, 256, 9000, True), (4, 1024, 256, 9000, True)])
def test_the_weights_gradient_is_cut_along_the_tokens_where_that_was_measured_faster(harness, es, n, h, v, cut) -> None:
    assert bool(plan_of(harness, es, n, h, v).dw_parts) == cut
