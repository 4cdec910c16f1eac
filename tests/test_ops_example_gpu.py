"""examples/global_block.py: the operators together, on a potential's energies
per atom: the block learns, its forces follow the energy, and the row of one
moved atom alone is the one of the whole batch."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))

pytestmark = pytest.mark.gpu


def test_block_learns_and_its_gradients_hold():
    import global_block

    lines = []
    r = global_block.run(count=12, steps=60, log=lines.append)
    # targets have unit variance: the mean alone leaves a loss of 1
    assert r["losses"][-1] < 0.5 < r["losses"][0]
    # central differences of 32-bit energies: about 1e-6 of a sum of some hundred, over 2 h = 6e-3,
    # and h^2 times third derivatives of waves of up to four turns, (8 pi)^2 h^2 / 6 = 1e-3
    assert abs(r["slope"] - r["expected"]) < 1e-2 * abs(r["expected"]) + 5e-2
    # the same row summed in another order
    assert abs(r["alone"] - r["among"]) < 1e-4 * (1 + abs(r["among"]))
    assert len(lines) >= 4
