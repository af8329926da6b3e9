"""Calls of rotary positions, layer-wide moves and shared tokens: names, shapes, frequencies and
bounds, without a GPU."""

import ctypes
import math

import numpy as np
import pytest

from pegaflow_amd import _lib, paged_cache
from pegaflow_amd.paged_cache import PagedLayers, RotaryPositions
from test_paged_calls import Tensor, cache


class Library:
    """Takes every call, and keeps its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    fake = Library()
    fake.cache = cache()
    monkeypatch.setattr(paged_cache, "lib", lambda: fake)
    return fake


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(_lib.SharedArgs) == 32
    assert ctypes.sizeof(_lib.ForkArgs) == 7 * 8 + 16
    assert ctypes.sizeof(_lib.CompactArgs) == 9 * 8 + 16


def test_frequencies(library):
    """Each scaling against its definition, in numpy."""
    for dim, base in ((128, 10000.0), (64, 500000.0), (20, 10000.0), (2, 10000.0)):
        i = np.arange(dim // 2)
        plain = base ** (-2 * i / dim)
        assert RotaryPositions(dim, base=base).frequencies == pytest.approx(plain, rel=1e-15)
        r = RotaryPositions(dim, base=base, scaling={"type": "linear", "factor": 4})
        assert r.frequencies == pytest.approx(plain / 4, rel=1e-15) and r.factor == 1
        r = RotaryPositions(dim, base=base, scaling={"type": "ntk", "factor": 4})
        wide = base * 4 ** (dim / (dim - 2)) if dim > 2 else base
        assert r.frequencies == pytest.approx(wide ** (-2 * i / dim), rel=1e-15)
        # By wavelength: within n / 4 as it is, beyond n stretched.
        n = 8192
        r = RotaryPositions(dim, base=base, scaling={
            "type": "llama3", "factor": 8, "original_max_position": n, "low_freq_factor": 1,
            "high_freq_factor": 4})
        wave = 2 * math.pi / plain
        smooth = (n / wave - 1) / 3
        want = np.where(wave < n / 4, plain,
                        np.where(wave > n, plain / 8, (1 - smooth) * plain / 8 + smooth * plain))
        assert r.frequencies == pytest.approx(want, rel=1e-14)
        # By index, with the values' own factor.
        r = RotaryPositions(dim, base=base, scaling={
            "type": "yarn", "factor": 16, "original_max_position": 4096})
        at = [dim * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (32, 1)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        assert r.frequencies == pytest.approx(plain / 16 * ramp + plain * (1 - ramp), rel=1e-14)
        assert r.factor == pytest.approx(0.1 * math.log(16) + 1)
    r = RotaryPositions(4, frequencies=[0.5, -0.25], factor=2)
    assert r.frequencies == [0.5, -0.25] and r.factor == 2
    name, args = library.calls[-1]
    assert name == "pf_rotary_create" and list(args[1]) == [0.5, -0.25]
    assert args[2:5] == (2, _lib.ROTARY_HALF, 2.0)


@pytest.mark.parametrize("args,kw", [
    ((0,), {}), ((7,), {}), ((-2,), {}), ((64,), {"layout": "pairs"}), ((64,), {"base": 0.0}),
    ((64,), {"scaling": {"type": "other"}}), ((64,), {"scaling": {"type": "linear"}}),
    ((64,), {"scaling": {"type": "linear", "factor": 0}}),
    ((64,), {"scaling": {"type": "linear", "factor": 2, "beta_fast": 3}}),
    ((64,), {"scaling": {"type": "llama3", "factor": 2}}),
    ((64,), {"scaling": {"type": "llama3", "factor": 2, "original_max_position": 0}}),
    ((64,), {"scaling": {"type": "llama3", "factor": 2, "original_max_position": 9,
                         "low_freq_factor": 4, "high_freq_factor": 4}}),
    ((64,), {"scaling": {"type": "yarn", "factor": 2, "original_max_position": 9, "beta_fast": 1}}),
    ((64,), {"base": 1.0, "scaling": {"type": "yarn", "factor": 2, "original_max_position": 9}}),
    ((64,), {"frequencies": [1.0]}), ((64,), {"factor": 2.0}),
    ((4,), {"frequencies": [1.0, 1.0], "scaling": {"type": "linear", "factor": 2}})], ids=str)
def test_bad_rotary_positions(library, args, kw):
    with pytest.raises(ValueError):
        RotaryPositions(*args, **kw)
    assert not library.calls


@pytest.mark.parametrize("value", [0, 7, (1 << 32) - 1, 1 << 32, (1 << 63) - 1])
def test_hints_past_32_bits_are_not_cut(library, value):
    c = library.cache
    q, one = Tensor((5, 4, 64), "bf16"), Tensor((1,), "int32")
    c.attend_shared(q, q, Tensor((2, 4), "int32"), Tensor((2,), "int32"), Tensor((3,), "int32"),
                    Tensor((2,), "int32"), one, max_shared_len=value, max_own_len=value,
                    max_query_len=value, window=value)
    want = min(value, (1 << 32) - 1)
    name, args = library.calls[-1]
    a, s = args[1]._obj, args[2]._obj
    assert name == "pf_kv_attend_shared"
    assert (a.window, a.max_query_len, s.max_shared_len, s.max_own_len) == (want,) * 4
    layers = PagedLayers([c])
    layers.compact(Tensor((2, 4), "int32"), Tensor((9,), "int32"), Tensor((3,), "int32"),
                   max_kept=value)
    assert library.calls[-1][1][1]._obj.max_kept == want


def test_shapes_that_do_not_fit(library):
    c = library.cache
    rotary = RotaryPositions(64)
    layers = PagedLayers([c])
    before = len(library.calls)
    rows, four, five = Tensor((5, 2, 64), "bf16"), Tensor((4,), "int64"), Tensor((5,), "int64")
    q, table = Tensor((5, 4, 64), "bf16"), Tensor((2, 4), "int32")
    two, three = Tensor((2,), "int32"), Tensor((3,), "int32")
    apart = Tensor((5, 2, 64), "bf16")
    apart.stride = lambda: (256, 128, 2)
    for call in (
            lambda: rotary.rotate(rows, q, five), lambda: rotary.rotate(rows, rows, four),
            lambda: rotary.rotate(rows, Tensor((4, 2, 64), "bf16"), five),
            lambda: rotary.rotate(apart, rows, five),
            lambda: rotary.rotate(Tensor((5, 2, 64), "fp32"), rows, five),
            lambda: c.write_rotated(q, q, rows, rows, four, five, rotary),
            lambda: c.write_rotated(q, q, rows, rows, five, four, rotary),
            lambda: c.write_rotated(q, rows, rows, rows, five, five, rotary),
            lambda: c.write_rotated(q, None, rows, rows, five, five, rotary),
            lambda: c.write_rotated(q, q, rows, q, five, five, rotary),
            lambda: c.write_rotated(q, q, rows, rows, Tensor((5,), "int32"), five, rotary),
            lambda: layers.copy_blocks(two, three),
            lambda: layers.fork(table, three, two, two, table),
            lambda: layers.fork(table, two, three, two, Tensor((3, 4), "int32")),
            lambda: layers.fork(table, two, two, two, Tensor((2, 5), "int32")),
            lambda: layers.compact(table, two, two),
            lambda: layers.compact(table, two, three, out_table=Tensor((2, 5), "int32")),
            lambda: layers.compact(table, two, three, out_lens=three),
            lambda: layers.compact(table, two, three, max_kept=-1),
            lambda: c.attend_shared(q, q, table, two, three, two, two),
            lambda: c.attend_shared(q, q, table, two, three, three, two, window=-1),
            lambda: c.attend_shared(q, q, table, two, three, three, two, max_own_len=-1)):
        with pytest.raises(ValueError):
            call()
    assert len(library.calls) == before
    with pytest.raises(ValueError):
        PagedLayers([])


def test_empty_torch_tensors_do_nothing():
    torch = pytest.importorskip("torch")
    c = cache()
    k = torch.empty(0, 2, 64, dtype=torch.bfloat16)
    none = torch.empty(0, dtype=torch.int64)

    memory = ctypes.create_string_buffer(64)

    class Rotary:
        handle = ctypes.addressof(memory)  # of no pairs: never read further

    c.write_rotated(k, k, k, k, none, none, Rotary)


def test_torch_tensors_run_on_torchs_current_stream(library, monkeypatch):
    torch = pytest.importorskip("torch")

    class OnDevice1(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 1

    def tensor(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice1)

    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 0x1230 + device,
                        raising=False)
    c, rotary = library.cache, RotaryPositions(64)
    layers = PagedLayers([c])
    k, q = tensor(5, 2, 64, dtype=torch.bfloat16), tensor(5, 4, 64, dtype=torch.bfloat16)
    at, table = tensor(5, dtype=torch.int64), tensor(2, 4)
    before = len(library.calls)
    rotary.rotate(q, q, at)
    c.write_rotated(q, q, k, k, at, at, rotary)
    layers.copy_blocks(tensor(3), tensor(3))
    layers.fork(table, tensor(2), tensor(2), tensor(2), tensor(2, 4))
    layers.compact(table, tensor(9), tensor(3))
    c.attend_shared(q, q, table, tensor(2), tensor(3), tensor(2), tensor(1))
    assert [args[-1] for _, args in library.calls[before:]] == [0x1231] * 6
