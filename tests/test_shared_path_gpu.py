"""Which kernels a batch with shared tokens runs on, told by the bits of its log-sum-exps: those of
``attend`` add the tokens up in another order."""

import numpy as np
import pytest

from pegaflow_amd.paged_cache import SHARE_ANYWAY
from pegaflow_amd.runtime import synchronize
from test_paged_cache_gpu import FORMS, LLAMA, device_array, device_rows, workspace  # noqa: F401
from test_shared_prefix_gpu import SharedBatch

pytestmark = pytest.mark.gpu


def attended(b, workspace):
    """Bits of ``attend``'s outputs and log-sum-exps."""
    n, heads, dim = b.q.shape
    q, _, _ = device_rows(b.q, b.strides, b.rows, offset=8)
    out, _, _ = device_rows(b.q, "contiguous", b.rows)
    lse = device_array(np.zeros((n, heads), np.float32), "fp32")
    b.dev.cache.attend(q, out, device_array(b.table, "int32"), device_array(b.lens, "int32"),
                       device_array(b.starts, "int32"), lse=lse, max_query_len=max(b.new),
                       workspace=workspace)
    synchronize()
    return (out.download().view(np.uint16).reshape(b.q.shape),
            lse.download().view(np.uint32).reshape(n, heads))


@pytest.mark.parametrize("form,group", [(LLAMA, 4), (FORMS[1], 1), (FORMS[2], 4), (FORMS[3], 4)],
                         ids=str)
@pytest.mark.parametrize("new", [1, 3, 5])
def test_small_batches_share_only_when_told(gpu, workspace, form, group, new):
    """Nothing is gained by 9 sequences behind 300 tokens: a hint as long, or any that is loose but
    shorter than SHARE_ANYWAY, leaves single tokens to attend; from there on they share."""
    b = SharedBatch([5, 3], [-(-300 // form[4]), -(-77 // form[4])],
                    [0, 40, 3, 129, 0, 64, 20, 0, 65], [new] * 9, form, group, seed=31)
    out, lse = attended(b, workspace)
    for hint in (300, 1 << 20, SHARE_ANYWAY - 1):
        got = b.run(workspace=workspace, max_shared_len=hint, max_own_len=b.table.size)
        b.check(*got)
        if new * group <= 16:
            assert np.array_equal(got[0], out) and np.array_equal(got[1].view(np.uint32), lse)
    for hint in (SHARE_ANYWAY, 1 << 40):
        got = b.run(workspace=workspace, max_shared_len=hint)
        b.check(*got)
        assert (got[1].view(np.uint32) != lse).mean() > 0.05
