"""Hints of calls on shared tokens, as they reach the library, without a GPU."""

import pytest

from pegaflow_amd import paged_cache
from test_paged_calls import Tensor, cache
from test_paged_more_calls import Library


def call(monkeypatch, **kw):
    fake = Library()
    c = cache()
    q = Tensor((5, 4, 64), "bf16")
    with monkeypatch.context() as patched:
        patched.setattr(paged_cache, "lib", lambda: fake)
        c.attend_shared(q, q, Tensor((2, 4), "int32"), Tensor((2,), "int32"),
                        Tensor((3,), "int32"), Tensor((2,), "int32"), Tensor((1,), "int32"), **kw)
    name, args = fake.calls[-1]
    assert name == "pf_kv_attend_shared"
    return args[1]._obj, args[2]._obj


@pytest.mark.parametrize("value", [0, 7, (1 << 32) - 1, 1 << 32, (1 << 63) - 1])
def test_the_longest_sequence_is_a_hint_as_for_attend(monkeypatch, value):
    a, s = call(monkeypatch, max_seq_len=value, max_query_len=3)
    assert a.max_seq_len == min(value, (1 << 32) - 1) and a.max_query_len == 3
    assert s.max_shared_len == s.max_own_len == 0
    assert call(monkeypatch)[0].max_seq_len == 0


def test_it_is_not_negative(monkeypatch):
    with pytest.raises(ValueError, match="not negative"):
        call(monkeypatch, max_seq_len=-1)
