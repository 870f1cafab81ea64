"""Rules on the CUDA sources that no run can show to be kept: a race may never come out wrong on a given machine."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[2] / "mia_train_b200" / "csrc"
# `x = ... mbar_wait(...)` or `x = mbar_test(...)`: one lane's view of an mbarrier
ANSWER = re.compile(r"\b(\w+) = mbar_(?:wait|test)\(")


def _shared_answers(source: str):
    """(line number, the code after it) of every shuffle or vote that hands one lane's view of a barrier to its warp."""
    code = re.sub(r"//[^\n]*", "", source)
    for name in set(ANSWER.findall(code)):
        for m in re.finditer(rf"__(?:shfl|reduce_or)_sync\(\w+, {name}\b[^;]*;", code):
            yield code[: m.start()].count("\n") + 1, code[m.end():].lstrip()


@pytest.mark.parametrize("path", sorted(CSRC.glob("*.cu*")), ids=lambda p: p.name)
def test_a_shuffled_wait_is_followed_by_a_warp_barrier(path):
    """Neither orders memory: what an mbarrier guards may be touched by the other lanes after `__syncwarp` only."""
    for line, rest in _shared_answers(path.read_text()):
        assert rest.startswith("__syncwarp();"), f"{path.name}:{line}"


def test_the_rule_sees_its_subject():
    assert len(list(_shared_answers((CSRC / "fp8_gemm.cu").read_text()))) == 3
