"""The paged-cache operators on torch's tensors, streams and graphs."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_streams_and_graphs_of_torch(kind):
    """tests/paged_torch_steps.py: steps on torch's default stream, under torch.cuda.stream
    behind late inputs, and captured by torch.cuda.graph, all with the same bits."""
    pytest.importorskip("torch")
    steps = os.path.join(os.path.dirname(os.path.abspath(__file__)), "paged_torch_steps.py")
    r = subprocess.run([sys.executable, "-u", steps, kind], timeout=100, text=True,
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout
