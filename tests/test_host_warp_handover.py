"""Hand-overs between the roles of the kernels, read from the sources. A warp whose lanes have read a stage of a ring gives
it back through one lane's arrival; without a warp barrier right before it the other lanes' reads are not ordered before
that arrival, and the stage may be refilled under them. Nothing can be measured there: a race shows when it likes."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "triton-gated-mlp_b200" / "csrc"
ARRIVAL = re.compile(r"if \(lane == 0\)\s*\{?\s*mbar_arrive\(")


def _statements(path):
    """Lines of a source without comments and blank lines: (number, text)."""
    text = re.sub(r"/\*.*?\*/", lambda m: "\n" * m.group().count("\n"), path.read_text(), flags=re.S)
    lines = ((i, re.sub(r"//.*", "", line).strip()) for i, line in enumerate(text.split("\n"), 1))
    return [(i, line) for i, line in lines if line]


@pytest.mark.parametrize("name", sorted(p.name for p in CSRC.glob("*.cuh")))
def test_one_lane_arrives_behind_a_warp_barrier(name):
    code = _statements(CSRC / name)
    for (_, before), (number, line) in zip(code, code[1:]):
        if ARRIVAL.search(line):
            assert before.endswith("__syncwarp();"), f"{name}:{number}: {line}"


def test_the_arrivals_are_found():
    found = sum(bool(ARRIVAL.search(line)) for p in CSRC.glob("*.cuh") for _, line in _statements(p))
    assert found >= 9
