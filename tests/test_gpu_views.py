"""Views of values beside ops that could have kept those values to themselves: the
view's readers find its owner written (values of the oracle; unwritten buffers hold
whatever was there)."""

from __future__ import annotations

import numpy as np
import pytest

from metellus_amd.api import run
from metellus_amd.orchestrator import Operations
from oracle.ir_eval import evaluate
from tests.test_graph import _view_cases

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", _view_cases(), ids=lambda f: f.__name__)
def test_readers_of_a_view_find_its_owner_written(case):
    """16 terms a product of values within [0.5, e]: a few dozen roundings in all, and the
    device's exp (under 2 ulp); 1e-4 of a value is 800 times that."""
    rng = np.random.default_rng(1)
    ops = Operations()
    for name in "ab":
        ops.from_numpy(rng.uniform(0.5, 1.0, (16, 16)).astype(np.float32), name)
    case(ops)
    ops.elementwise("add", out="both", operands=("a", "b"))  # (not every case reads b)
    want = evaluate(ops)
    for _ in range(2):
        env = run(ops).env
        for name in ("X", "Y", "Z", "W", "V", "r"):
            if name in env and name in want:
                np.testing.assert_allclose(env[name], want[name], rtol=1e-4)
        assert "X" in env
