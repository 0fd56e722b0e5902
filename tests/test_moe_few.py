"""Refusals of the layer for a few tokens, all before any device work, and the arithmetic of its workspace."""
import ctypes
import sys
import threading
import weakref

import pytest
import torch

from radeonflow_kernels_b200 import _lib, moe_few

A = 0x7000000                # aligned for everything; nothing stands behind it


def config(d=256, f=128, e=8, k=2, ns=1, wt=0):
    return _lib.RfMoeFewConfig(d, f, e, k, ns, wt)


@pytest.mark.parametrize("kw,status", [
    (dict(d=100), 1), (dict(d=0), 1), (dict(f=96), 1), (dict(f=192, wt=1), 1), (dict(d=192, wt=1), 1), (dict(ns=-1), 1), (dict(ns=65), 1),
    (dict(d=2 ** 21), 1), (dict(e=6), 7), (dict(e=512), 7), (dict(e=0), 7), (dict(k=0), 7), (dict(k=9), 7), (dict(e=2, k=4), 7), (dict(wt=2), 7)])
def test_config(rf_lib, kw, status):
    c, h = config(**kw), ctypes.c_void_p()
    assert rf_lib.rf_moe_few_create(ctypes.byref(c), A, None, A, A, A, A, A, A, ctypes.byref(h)) == status and not h
    assert rf_lib.rf_moe_few_workspace_bytes(ctypes.byref(c), 4) == 0


def test_pointers(rf_lib):
    h = ctypes.c_void_p()
    ptrs = lambda n, bad=None, at=0: (ctypes.c_void_p * n)(*[bad if i == at and bad is not None else A for i in range(n)])
    null = (ctypes.c_void_p * 9)(*[A] * 8, None)

    def create(router=A, bias=None, g=ptrs(9), u=ptrs(9), dn=ptrs(9), s=(None,) * 3, wt=0):
        c = config(wt=wt)
        return rf_lib.rf_moe_few_create(ctypes.byref(c), router, bias, g, u, dn, *s, ctypes.byref(h))

    assert create(router=None) == 2 and create(g=None) == 2 and create(u=None) == 2 and create(dn=null) == 2
    assert create(wt=1) == 2 and create(wt=1, s=(ptrs(9), ptrs(9), null)) == 2
    assert create(router=A + 8) == 3 and create(bias=A + 2) == 3 and create(g=ptrs(9, A + 8, 8)) == 3 and create(dn=ptrs(9, A + 4)) == 3
    assert create(wt=1, s=(ptrs(9), ptrs(9, A + 2, 3), ptrs(9))) == 3
    assert rf_lib.rf_moe_few_create(None, A, None, A, A, A, None, None, None, ctypes.byref(h)) == 2
    assert rf_lib.rf_moe_few_destroy(None) == 0
    assert rf_lib.rf_moe_few_forward(None, A, 1, A, A, 1 << 30, None) == 2


def test_workspace_bytes(rf_lib):
    c = config(d=7168, f=2048, e=256, k=8)
    for t in range(1, 33):
        n = rf_lib.rf_moe_few_workspace_bytes(ctypes.byref(c), t)
        # 8-byte words: partial sums of at least one K chunk each, and h
        assert n % 256 == 0 and n >= 8 * t * 9 * (2 * 2048 + 1024 + 7168)
    for t in (0, 33, -1):
        assert rf_lib.rf_moe_few_workspace_bytes(ctypes.byref(c), t) == 0


class Meta(torch.Tensor):
    """A tensor that says it lies on the GPU."""
    is_cuda = True


def test_python_weights(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)       # the index of the CPU's device
    t = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype).as_subclass(Meta)
    cfg = {"d_hidden": 128, "d_expert": 64, "n_routed_experts": 2, "n_experts_per_token": 1, "n_shared_experts": 1}
    good = {"router.weight": t(2, 128)}
    for p in ("experts.0", "experts.1", "shared_experts"):
        good.update({f"{p}.0.weight": t(128, 64), f"{p}.1.weight": t(128, 64), f"{p}.2.weight": t(64, 128)})
    for name, bad, match in (("router.weight", t(3, 128), "router"), ("experts.1.2.weight", t(128, 64), "experts.1.2"),
                             ("shared_experts.0.weight", t(128, 128), "shared_experts.0"),
                             ("experts.0.1.weight", t(128, 64, dtype=torch.float32), "fp16"),
                             ("experts.0.1.weight", t(64, 128).t(), "contiguous"),
                             ("experts.0.0.weight", torch.zeros(128, 64, dtype=torch.float16), "CUDA")):
        with pytest.raises(ValueError, match=match):
            moe_few.FewTokenMoE({**good, name: bad}, cfg)
    with pytest.raises(KeyError):
        moe_few.FewTokenMoE({k: v for k, v in good.items() if k != "experts.1.0.weight"}, cfg)
    with pytest.raises(ValueError, match="router_bias"):
        moe_few.FewTokenMoE(good, cfg, router_bias=t(2))
    f8 = torch.float8_e4m3fn
    cfg["d_expert"] = 128
    good8 = {"router.weight": t(2, 128), "experts.gate_up.weight": t(2, 256, 128, dtype=f8), "experts.gate_up.scale": t(2, 2, 1, dtype=torch.float32),
             "experts.down.weight": t(2, 128, 128, dtype=f8), "experts.down.scale": t(2, 1, 1, dtype=torch.float32),
             "shared_experts.gate_up.weight": t(256, 128, dtype=f8), "shared_experts.gate_up.scale": t(2, 1, dtype=torch.float32),
             "shared_experts.down.weight": t(128, 128, dtype=f8), "shared_experts.down.scale": t(1, 1, dtype=torch.float32)}
    for name, bad in (("experts.gate_up.scale", t(2, 1, 1, dtype=torch.float32)), ("experts.down.weight", t(2, 128, 128)),
                      ("shared_experts.down.scale", t(1, 1, 1, dtype=torch.float32))):
        with pytest.raises(ValueError, match=name.rsplit(".", 1)[0]):
            moe_few.FewTokenMoE({**good8, name: bad}, cfg)
    with pytest.raises(ValueError, match="multiples of 128"):
        moe_few.FewTokenMoE(good8, {**cfg, "d_expert": 64})


class FakeLibrary:
    """What `_workspace` asks of the library: a size for a number of tokens, a stream's capture."""

    def __init__(self, capture=0):
        self.capture = capture

    def rf_moe_few_workspace_bytes(self, config, n_tokens):
        return 1000 * n_tokens

    def rf_stream_capture_id(self, stream, out):
        out._obj.value = self.capture
        return 0


class FakeWorkspace:
    made = []

    def __init__(self, size):
        self.size = size
        FakeWorkspace.made.append(size)


@pytest.fixture
def bare_layer(monkeypatch):
    """A layer without weights, and its workspaces without a GPU."""
    library = FakeLibrary()
    monkeypatch.setattr(_lib, "lib", lambda: library)
    monkeypatch.setattr(moe_few, "_Workspace", FakeWorkspace)
    monkeypatch.setattr(moe_few, "_workspaces", weakref.WeakValueDictionary())
    FakeWorkspace.made.clear()

    def make():
        layer = moe_few.FewTokenMoE.__new__(moe_few.FewTokenMoE)
        layer._handle, layer.config, layer.device, layer._held, layer._sizes = None, config(), torch.device("cuda", 0), {}, {}
        return layer
    return make


def lines_of(fn):
    """How many lines of `_workspace` a call runs."""
    count = []
    code = moe_few.FewTokenMoE._workspace.__code__

    def trace(frame, event, arg):
        if frame.f_code is code:
            count.append(event == "line")
            return trace
        return None
    sys.settrace(trace)
    try:
        fn()
    finally:
        sys.settrace(None)
    return sum(count)


@pytest.mark.parametrize("first,second", [(4, 4), (4, 9), (9, 4)])
def test_two_threads_on_one_stream(bare_layer, first, second):
    """A thread is stopped in front of each line of `_workspace` in turn while another thread calls it, for the same stream."""
    code = moe_few.FewTokenMoE._workspace.__code__
    total = lines_of(lambda: bare_layer()._workspace(first, 7))
    assert total > 8
    stops = 0
    for stop in range(total):
        layer, got, left = bare_layer(), [], [stop]

        def other():
            try:
                got.append(layer._workspace(second, 7))
            except Exception as e:          # what the test is for
                got.append(e)

        thread = threading.Thread(target=other)

        def trace(frame, event, arg):
            if frame.f_code is not code:
                return None
            if event == "line":
                if left[0] == 0:
                    thread.start()
                    thread.join(0.1)        # (it may have to wait for this thread)
                left[0] -= 1
            return trace

        sys.settrace(trace)
        try:
            mine = layer._workspace(first, 7)
        finally:
            sys.settrace(None)
        if left[0] >= 0:            # fewer lines than before
            break
        thread.join(10)
        assert not thread.is_alive() and mine.size >= 1000 * first
        assert got and not isinstance(got[0], Exception) and got[0].size >= 1000 * second, (stop, got)
        stops += 1
        # the stream's calls to come share one
        assert layer._workspace(first, 7) is layer._workspace(second, 7) is layer._workspace(max(first, second), 7)
        del layer, mine, got
        moe_few._workspaces.clear()
    assert stops >= total - 2


def test_layers_share_a_streams_workspace(bare_layer):
    a, b = bare_layer(), bare_layer()
    one = a._workspace(4, 7)
    assert b._workspace(4, 7) is one and b._workspace(3, 7) is one and FakeWorkspace.made == [4096]
    large = b._workspace(5, 7)
    assert large.size == 8192 and a._workspace(4, 7) is one and a._workspace(5, 7) is large
    assert a._workspace(4, 8) is not one
    a.reset()
    assert a._workspace(4, 7) is not one


def test_captures_leave_nothing_with_the_layer(bare_layer, monkeypatch):
    """A capture's workspace is the graph's: layers share it while it is being captured and hold nothing of it."""
    class FakeCaptureWorkspace:
        def __init__(self, stream, capture, size):
            self.stream, self.capture, self.size = stream, capture, size

    library = FakeLibrary()
    monkeypatch.setattr(_lib, "lib", lambda: library)
    monkeypatch.setattr(moe_few, "_CaptureWorkspace", FakeCaptureWorkspace)
    monkeypatch.setattr(moe_few, "_captured", {})
    a, b = bare_layer(), bare_layer()
    eager = a._workspace(4, 7)
    for capture in range(1, 40):
        library.capture = capture
        one = a._workspace(4, 7)
        assert (one.stream, one.capture, one.size) == (7, capture, 4000)
        assert a._workspace(3, 7) is one and b._workspace(4, 7) is one
        assert b._workspace(4, 8) is not one            # a branch of the capture
        more = b._workspace(9, 7)
        assert more.size == 9000 and a._workspace(4, 7) is more
    library.capture = 0
    assert a._workspace(4, 7) is eager and len(moe_few._captured) == 2 and len(a._held) == 1 and not b._held


def test_captured_workspace_entry(rf_lib):
    assert rf_lib.rf_moe_few_workspace_alloc_captured(None, 100, None) == 2
    n = ctypes.c_size_t(5)
    assert rf_lib.rf_moe_few_workspace_reap(ctypes.byref(n)) == 0 and n.value == 0
    assert rf_lib.rf_moe_few_workspace_reap(None) == 0
