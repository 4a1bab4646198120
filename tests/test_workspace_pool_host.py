"""Which workspace a call gets, on a machine without a GPU: the pool with a fake library,
whose stream, capture and graph lifetimes the test sets."""

import contextlib
import ctypes

import pytest
import torch

CPU = torch.device("cpu")


class FakeLibrary:
    def __init__(self):
        self.capture, self.live, self.given, self.fail = 0, set(), [], 0
        self.words = {}  # address -> status word

    def cb_stream_capture_id(self, stream):
        return self.capture

    def cb_capture_workspace(self, stream, nbytes, out):
        if self.fail:
            return self.fail
        self.live.add(self.capture)
        self.given.append((self.capture, nbytes))
        out._obj.value = 0x10000000 * len(self.given)
        return 0

    def cb_capture_live(self, capture):
        return int(capture in self.live)

    def cb_status_str(self, code):
        return b"refused"

    def cb_workspace_status(self, address, out, stream):
        out._obj.value = self.words.pop(address, 0)
        return 11 if out._obj.value else 0


class FakeNative:
    def __init__(self):
        self.known = {}

    def set_workspace(self, device, stream, capture, address, nbytes):
        self.known[device, stream, capture] = (address, nbytes)

    def drop_workspace(self, device, stream, capture):
        del self.known[device, stream, capture]


@pytest.fixture
def world(monkeypatch):
    from cb200 import ops
    lib = FakeLibrary()
    stream = [7]
    monkeypatch.setattr(ops, "_stream", lambda device: stream[0])
    monkeypatch.setattr(ops.L, "load", lambda: lib)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    pool = ops.WorkspacePool()
    return lib, stream, pool


def test_streams_and_sizes(world):
    lib, stream, pool = world
    a = pool.get(10, CPU)
    assert a.numel() >= 10 and bool((a == 0).all()) and pool.get(100, CPU) is a
    stream[0] = 8
    assert pool.get(10, CPU) is not a
    stream[0] = 7
    big = pool.get(a.numel() + 1, CPU)
    assert big.numel() >= 2 * a.numel() and pool.get(10, CPU) is big


def test_captures_share_nothing(world):
    """Two graphs captured on one stream, and eager calls on it, have three workspaces."""
    lib, _, pool = world
    eager = pool.get(100, CPU)
    lib.capture = 1
    first = pool.get(100, CPU)
    assert first.data_ptr() != eager.data_ptr() and pool.get(100, CPU).data_ptr() == first.data_ptr()
    lib.capture = 2
    second = pool.get(100, CPU)
    assert second.data_ptr() not in (first.data_ptr(), eager.data_ptr())
    lib.capture = 0
    assert pool.get(100, CPU) is eager
    assert [c for c, _ in lib.given] == [1, 2]


def test_a_larger_request_leaves_earlier_buffers_alone(world):
    """Later and larger calls, captured or eager, replace no buffer that a graph or its status read still needs."""
    lib, _, pool = world
    eager = pool.get(100, CPU)
    lib.capture = 1
    small = pool.get(100, CPU)
    large = pool.get(5 << 20, CPU)
    assert large.numel() >= 5 << 20 and large.data_ptr() != small.data_ptr()
    lib.capture = 0
    pool.get(9 << 20, CPU)
    for buf in (eager, small, large):
        lib.words[buf.data_ptr()] = 2
        assert pool.check_status() == 2 and pool.check_status() == 0


def test_native_layer_follows(world):
    lib, _, pool = world
    native = FakeNative()
    pool.share(100, CPU, native)
    lib.capture = 5
    pool.share(100, CPU, native)
    assert set(native.known) == {(None, 7, 0), (None, 7, 5)}
    grown = pool.get(5 << 20, CPU)
    assert native.known[None, 7, 5] == (grown.data_ptr(), grown.numel())
    lib.live.clear()  # the graph is gone
    lib.capture = 6
    pool.share(100, CPU, native)
    assert set(native.known) == {(None, 7, 0), (None, 7, 6)}
    lib.live.clear()
    lib.capture = 0
    pool.check_status()
    assert set(native.known) == {(None, 7, 0)}


def test_refused_workspace_is_an_error(world):
    from cb200 import _lib as L
    lib, _, pool = world
    lib.capture, lib.fail = 3, L.CB_ERR_CUDA
    with pytest.raises(L.CbError):
        pool.get(100, CPU)


def test_outside_a_capture_the_library_refuses():
    from cb200 import _lib as L
    lib = L.load()
    p = ctypes.c_void_p()
    assert lib.cb_stream_capture_id(None) == 0
    assert lib.cb_capture_live(0) == 0 and lib.cb_capture_live(12345) == 0
    assert lib.cb_capture_workspace(None, 256, ctypes.byref(p)) == L.CB_ERR_INVALID_ARG
    assert lib.cb_capture_workspace(None, 0, ctypes.byref(p)) == L.CB_ERR_INVALID_ARG
    assert lib.cb_capture_workspace(None, 256, None) == L.CB_ERR_INVALID_ARG


def test_status_of_the_current_device(world, monkeypatch):
    """A device without an index is the current one, as everywhere in torch: its errors are seen."""
    lib, _, pool = world

    class Buffer:
        def __init__(self, address):
            self.data_ptr = lambda: address

    pool._bufs = {(0, 7, 0): [Buffer(0x100)], (1, 9, 0): [Buffer(0x200)]}
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    lib.words = {0x100: 1, 0x200: 2}
    assert pool.check_status(torch.device("cuda")) == 2
    assert pool.check_status(torch.device("cuda", 0)) == 1
    assert pool.check_status(torch.device("cuda")) == 0
    lib.words = {0x100: 1, 0x200: 2}
    assert pool.check_status() == 3
