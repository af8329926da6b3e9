"""A search over branches against the definition of attention, output by output."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
def test_outputs_of_a_search(kind):
    """tests/paged_more_bounds_steps.py: every output within its own bound, which tokens left out,
    a missing mask or another child's tokens would break."""
    pytest.importorskip("torch")
    steps = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_more_bounds_steps.py")
    r = subprocess.run([sys.executable, "-u", steps, kind], timeout=100, text=True,
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
