"""Waits of the 8-bit kernels that give up.  No launch makes one give up, so the sources are held to the form that is safe: a wait's
outcome, and the flag that tells of one, reach a warp's lanes as one answer.  A lane that left a loop alone would leave the others at a vote, an
election or a load of tensor memory that is for all of them."""

import re
from pathlib import Path

import pytest

import llmserve_triton_kernels_b200

CSRC = Path(llmserve_triton_kernels_b200.__file__).parent / "csrc"
WAITING = ["attention8.cu", "gemm8_tcgen05.cu", "linear8_mid.cu", "linear8_scaled.cu", "linear8_waits.cuh"]


def statements(name):
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    return [" ".join(s.split()) for s in re.split(r"[;{}]", text)]


@pytest.mark.parametrize("name", WAITING)
def test_outcomes_are_voted_on(name):
    """A wait stands in a vote of the whole warp, or nobody asks for its outcome (copies and products that are waited for at the end)."""
    waits = [s for s in statements(name) if "mbar_wait(" in s]
    for s in waits:
        assert "(void)tma::mbar_wait(" in s or re.search(r"__all_sync\(0xffffffffu, .*mbar_wait\(", s), s
    assert waits


@pytest.mark.parametrize("name", WAITING)
def test_the_flag_is_voted_on(name):
    """One place reads the flag, and the two that ask it do so within a vote."""
    for s in statements(name):
        assert "(volatile int*)" not in s or name == "linear8_waits.cuh", s
        if "flag()" in s and "bool flag()" not in s:
            assert re.search(r"__(any|all)_sync\(0xffffffffu, !?(waits\.)?flag\(\)", s), s


def test_nothing_else_waits():
    """Every file whose kernels wait on barriers of the 8-bit products and attention is in the list above."""
    eight = {p.name for p in CSRC.iterdir() if re.search(r"8(_|\.)", p.name) and p.suffix in (".cu", ".cuh", ".h")}
    assert {n for n in eight if "mbar_wait(" in (CSRC / n).read_text()} == set(WAITING)
