"""What the operators on 8-bit rows keep, and their memory while a step of an engine runs, without a GPU: the checks of devices are taken out, the library is a stand-in that
keeps the addresses it is given."""
import copy
import pickle

import pytest
import torch

from xeno_rt_amd.ops import hip
from xeno_rt_amd.parts.base import Runtime


class Library:
    """Products that want a workspace of `need` bytes."""

    def __init__(self, need):
        self.need, self.workspace = need, None

    def xrt_linear_int8_workspace(self, m, n, k, mode):
        return self.need

    def xrt_linear_int8(self, *arguments):
        self.workspace = arguments[10]
        return 0


@pytest.fixture
def ops(monkeypatch):
    monkeypatch.setattr(hip.HipOps, "_require", staticmethod(lambda *arguments, **named: None))
    monkeypatch.setattr(hip, "_current_device", lambda: -1)
    monkeypatch.setattr(hip, "_raw_stream", lambda index: 0)
    made = object.__new__(hip.HipOps)                           # (without a GPU there is no library to load)
    made.lib = Library(4096)
    return made


def stepped(ops, room=1 << 16):
    """A runtime whose steps have memory of their own already."""
    runtime = Runtime(ops, torch.bfloat16, "cpu")
    with runtime.step_memory():
        runtime.empty((room,), torch.uint8)
    with runtime.step_memory():
        pass
    assert runtime.arena.buffer is not None and runtime.arena.buffer.numel() >= room
    return runtime


def inside(runtime, address):
    begin = runtime.arena.buffer.data_ptr()
    return begin <= address < begin + runtime.arena.buffer.numel()


def test_rows_made_during_a_step_outlive_it(ops):
    runtime = stepped(ops)
    with runtime.step_memory():
        kept = ops.int8_rows(4, 100, "cpu")
        kept.values.fill_(55)
        kept.scales.fill_(2.0)
    with runtime.step_memory():                                 # the next step writes all of its memory
        runtime.empty((1 << 15,), torch.uint8).fill_(255)
    assert bool((kept.values == 55).all()) and bool((kept.scales == 2.0).all())
    assert not inside(runtime, kept.values.data_ptr()) and not inside(runtime, kept.scales.data_ptr())


def test_a_products_workspace_is_not_the_steps_memory(ops):
    runtime = stepped(ops)
    a = hip.Int8Rows(torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4), 100)
    w = hip.Int8Matrix(torch.zeros(32, 128, dtype=torch.int8), torch.zeros(32), 20, 100, False)
    with runtime.step_memory():
        ops.linear_int8(a, w, torch.zeros(4, 20))
        assert ops.lib.workspace and not inside(runtime, ops.lib.workspace)


def test_what_was_checked_stays_what_it_is(ops):
    """The calls take sizes from the rows and the matrix: larger ones, written over them, would be read behind the end of their tensors."""
    a = hip.Int8Rows(torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4), 100)
    w = hip.Int8Matrix(torch.zeros(32, 128, dtype=torch.int8), torch.zeros(32), 20, 100, False)
    before = a.shape, a.k, a.index, w.shape, w.gated, w.index
    for made, names in ((a, ("shape", "index", "values", "scales", "k", "_values", "_scales", "_k", "other")), (w, ("shape", "gated", "index", "data", "scales", "_data", "_scales"))):
        for name in names:
            with pytest.raises(AttributeError):
                setattr(made, name, (8, 100))
            with pytest.raises(AttributeError):
                delattr(made, name)
    assert (a.shape, a.k, a.index, w.shape, w.gated, w.index) == before


def test_rows_and_matrices_can_be_copied_and_kept_in_files(ops):
    a = hip.Int8Rows(torch.arange(512).to(torch.int8).view(4, 128), torch.rand(4), 100)
    w = hip.Int8Matrix(torch.ones(32, 128, dtype=torch.int8), torch.rand(32), 40, 100, True)
    for copied in (copy.copy, copy.deepcopy, lambda made: pickle.loads(pickle.dumps(made))):
        b, v = copied(a), copied(w)
        assert torch.equal(b.values, a.values) and torch.equal(b.scales, a.scales) and (b.shape, b.k, b.index) == (a.shape, a.k, a.index)
        assert torch.equal(v.data, w.data) and torch.equal(v.scales, w.scales) and (v.shape, v.gated, v.index) == (w.shape, w.gated, w.index)
    assert copy.deepcopy(a).values.data_ptr() != a.values.data_ptr()
