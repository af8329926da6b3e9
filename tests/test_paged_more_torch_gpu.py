"""Rotary positions, forks, shared prompts and kept drafts together, on torch's tensors, streams
and graphs."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "e4m3", "int8"])
def test_a_search_over_branches(kind):
    """tests/paged_more_torch_steps.py: on torch's default stream, under torch.cuda.stream behind
    late inputs, and in two captured graphs that share a workspace, all with the same bits."""
    pytest.importorskip("torch")
    steps = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_more_torch_steps.py")
    r = subprocess.run([sys.executable, "-u", steps, kind], timeout=100, text=True,
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
