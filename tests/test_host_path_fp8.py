"""The native form of the grouped product's Python boundary: what it takes, what it hands to the library, what it leaves to the Python
code.  On the CPU, with objects that have a tensor's attributes and a stand-in for the library."""
import ctypes

import pytest
import torch

from radeonflow_kernels_b200 import _lib

FP8, F32, BF16, F16, I32 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.float16, torch.int32


class Fake:
    def __init__(self, shape, dtype, ptr=0x1000, is_cuda=True, contiguous=True, device=3):
        self.shape, self.dtype, self.is_cuda = torch.Size(shape), dtype, is_cuda
        self._ptr, self._contiguous, self._device = ptr, contiguous, device

    def is_contiguous(self):
        return self._contiguous

    def data_ptr(self):
        return self._ptr

    def get_device(self):
        return self._device


@pytest.fixture
def host(rf_lib):
    """The module with a stand-in that records its arguments and answers `status`; afterwards it is the library's again."""
    h = _lib.host()
    calls, status = [], [0]
    vp, ci = ctypes.c_void_p, ctypes.c_int
    fn = ctypes.CFUNCTYPE(ci, *[vp] * 6, *[ci] * 5, vp)(lambda *a: calls.append(a) or status[0])
    h.setup(ctypes.cast(rf_lib.run, vp).value, lambda: 3, lambda dev: 0x700 + dev, FP8, F32, BF16, F16)
    h.setup_grouped(ctypes.cast(fn, vp).value, I32)
    yield h, calls, status
    _lib._host = None
    _lib.host()


def _grouped(m=48, e=3, n=192, k=384, out=BF16):
    return [Fake((m, k), FP8, 0x10), Fake((e, n, k), FP8, 0x20), Fake((m, k // 128), F32, 0x30),
            Fake((e, (n + 127) // 128, k // 128), F32, 0x40), Fake((e + 1,), I32, 0x50), Fake((m, n), out, 0x60)]


@pytest.mark.parametrize("out,number", [(F16, 0), (BF16, 1)])
def test_grouped(host, out, number):
    h, calls, status = host
    assert h.grouped(*_grouped(out=out)) is True
    assert calls == [(0x10, 0x20, 0x30, 0x40, 0x50, 0x60, number, 48, 3, 192, 384, 0x703)]
    status[0] = 1
    assert h.grouped(*_grouped(out=out)) is False


@pytest.mark.parametrize("i", range(6))
@pytest.mark.parametrize("change", [dict(is_cuda=False), dict(contiguous=False), dict(dtype=torch.float64), dict(shape=(2,)), dict(device=1),
                                    dict(shape=(47, 384)), dict(shape=(4, 192, 384)), dict(shape=(5,))])
def test_grouped_leaves_every_other_form_alone(host, i, change):
    h, calls, _ = host
    ops = _grouped()
    ops[i] = Fake(**{"shape": ops[i].shape, "dtype": ops[i].dtype, **change})
    assert h.grouped(*ops) is False and calls == []


def test_exceptions_are_passed_on(host):
    h, calls, _ = host
    with pytest.raises(AttributeError):
        h.grouped(1, 2, 3, 4, 5, 6)
    ops = _grouped()
    ops[4].data_ptr = lambda: 1 / 0
    with pytest.raises(ZeroDivisionError):
        h.grouped(*ops)
    with pytest.raises(TypeError):
        h.setup_grouped(1)
    assert calls == []
