"""What the op_* calls refuse before anything is queued: no GPU is needed to see it."""

import ctypes as C

import numpy as np
import pytest
import torch

import npeff_ref_amd as d
from npeff_ref_amd import binding


class OnGpu:
    """What a tensor on a GPU tells about itself."""

    is_cuda, shape, dtype = True, (64,), torch.float32

    def __init__(self, device=0, dense=True):
        self.at, self.dense, self.device = device, dense, f"cuda:{device}"

    def get_device(self):
        return self.at

    def is_contiguous(self):
        return self.dense

    def data_ptr(self):
        return 4096

    def numel(self):
        return 64

    def element_size(self):
        return 4


def call_of(own):
    c = object.__new__(binding._Call)
    c.what, c.own, c.place, c.type, c.first = "op", own, -2 if own else 0, binding.F32, None
    return c


@pytest.fixture
def device0(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("bad", ["host", "host_bytes", "array", "number", "strided", "elsewhere", "freed"])
def test_a_workspace_is_looked_at(own, bad, device0):
    freed = object.__new__(d.DeviceArray)
    freed.shape, freed.dtype, freed.nbytes, freed.ptr = (64,), np.dtype(np.float32), 256, None
    w = {
        "host": torch.empty(64),
        "host_bytes": torch.empty(256, dtype=torch.uint8)[::2],
        "array": np.empty(64),
        "number": 4096,
        "strided": OnGpu(dense=False),
        "elsewhere": OnGpu(device=1),
        "freed": freed,
    }[bad]
    called = []
    with pytest.raises(d.DnpeffError, match="workspace"):
        call_of(own).run(lambda *a: called.append(a), (), 128, w, 7)
    assert not called


@pytest.mark.parametrize("own", [False, True])
def test_a_workspace_on_the_gpu_is_passed_on(own, device0):
    called = []
    call_of(own).run(lambda *a: called.append(a), (1, 2), 128, OnGpu(), 7)
    assert called == [(7, 1, 2, 4096, 256)]


def test_a_second_runtime_gets_no_workspace(device0, monkeypatch):
    monkeypatch.setattr(binding.lib, "without_torch", True)
    with pytest.raises(d.DnpeffError, match="torch was imported after"):
        call_of(True).run(lambda *a: 0, (), 128, OnGpu(), 7)


def test_views_of_memory_that_the_library_cannot_reach(device0, monkeypatch):
    assert d.DeviceArray.view(OnGpu()).ptr.value == 4096
    with pytest.raises(d.DnpeffError, match="current"):
        d.DeviceArray.view(OnGpu(device=1))
    monkeypatch.setattr(binding.lib, "without_torch", True)
    with pytest.raises(d.DnpeffError, match="torch was imported after"):
        d.DeviceArray.view(OnGpu())


def test_more_words_than_a_launch_dimension_holds():
    """Refused before anything is read or queued: the addresses are nobody's."""
    at, words = C.c_void_p(16), (1 << 31) - 100
    assert d.lib.dnpeff_vocab_loss(None, binding.BF16, 1, 8, words, at, 8, at, 8, at, at, at, at, 1 << 40) != 0
    assert b"too many for one launch" in d.lib.dnpeff_last_error()


def test_matrices_of_groups_that_share_elements():
    """As above: weights of groups that lie backwards, and gradients of theirs that overlap, are refused."""
    at, none, room = C.c_void_p(16), C.c_void_p(0), 1 << 40
    forward = d.lib.dnpeff_linear
    assert forward(None, binding.F32, 40, 8, 4, at, 8, at, 8, -32, none, 0, none, 0, at, 4, none, 0, 3, at, at, room) != 0
    assert b"matrices of W" in d.lib.dnpeff_last_error()
    backward = d.lib.dnpeff_linear_backward
    for lddw, dw_group in ((8, 31), (8, 0), (8, -64), (10, 32)):
        bad = backward(None, binding.F32, 40, 8, 4, at, 4, at, 8, at, 8, 32, none, 0, 0, at, 8, at, lddw, dw_group, none, 3, at, at, room)
        assert bad != 0 and b"matrices of dW" in d.lib.dnpeff_last_error()
