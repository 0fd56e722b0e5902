"""The native form of the FP8 quantisations' and the grouped product's Python boundary: what it takes, what it hands to the library,
what it leaves to the Python code.  On the CPU, with objects that have a tensor's attributes and stand-ins for the library."""
import ctypes

import pytest
import torch

from radeonflow_kernels_b200 import _lib

FP8, F32, BF16, F16, I32 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.float16, torch.int32


class Fake:
    def __init__(self, shape, dtype, ptr=0x1000, is_cuda=True, contiguous=True, device=3, stride=None):
        self.shape, self.dtype, self.is_cuda = torch.Size(shape), dtype, is_cuda
        self._ptr, self._contiguous, self._device = ptr, contiguous, device
        self._stride = stride or tuple(torch.empty(shape, device="meta").stride())
        self.made = []

    def is_contiguous(self):
        return self._contiguous

    def data_ptr(self):
        return self._ptr

    def stride(self):
        return self._stride

    def get_device(self):
        return self._device

    def new_empty(self, shape, dtype):
        t = Fake(shape, dtype, 0xFFFF000000000000 + len(self.made))
        self.made.append(t)
        return t


@pytest.fixture
def host(rf_lib):
    """The module with stand-ins that record their arguments and answer `status`; afterwards it is the library's again."""
    h = _lib.host()
    calls, status = [], [0]
    vp, ci, ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong

    def stand_in(*args):
        fn = ctypes.CFUNCTYPE(ci, *args)(lambda *a: calls.append(a) or status[0])
        keep.append(fn)
        return ctypes.cast(fn, vp).value

    keep = []
    h.setup(ctypes.cast(rf_lib.run, vp).value, lambda: 3, lambda dev: 0x700 + dev, FP8, F32, BF16, F16)
    h.setup_fp8(stand_in(vp, ci, ll, vp, ci, ci, ci, vp, vp, vp), stand_in(vp, ci, ll, ci, ci, vp, vp, vp),
                stand_in(vp, ci, ci, ci, ci, ll, ll, ll, vp, vp, vp), stand_in(*[vp] * 6, *[ci] * 5, vp), I32)
    yield h, calls, status
    _lib._host = None
    _lib.host()


Q, S = 0xFFFF000000000000, 0xFFFF000000000001


@pytest.mark.parametrize("dtype,number", [(F16, 0), (BF16, 1), (F32, 2)])
def test_quantize(host, dtype, number):
    h, calls, status = host
    x = Fake((5, 256), dtype, stride=(300, 1))
    q, s = h.quantize(x, None)
    assert x.made == [q, s] and (q.shape, q.dtype, s.shape, s.dtype) == ((5, 256), FP8, (5, 2), F32)
    rows = Fake((7,), I32, 0x2000)
    q, s = h.quantize(x, rows)
    assert (q.shape, s.shape) == ((7, 256), (7, 2))
    assert calls == [(0x1000, number, 300, None, 5, 5, 256, Q, S, 0x703), (0x1000, number, 300, 0x2000, 5, 7, 256, Q + 2, S + 2, 0x703)]
    status[0] = 3                           # refused: left to the Python code, which says why
    assert h.quantize(x, None) is None
    assert h.swiglu_quantize(Fake((5, 512), dtype, stride=(600, 1))) is None
    status[0] = 0
    q, s = h.swiglu_quantize(Fake((5, 512), dtype, stride=(600, 1)))
    assert calls[-1] == (0x1000, number, 600, 5, 256, Q, S, 0x703) and (q.shape, s.shape) == ((5, 256), (5, 2))


@pytest.mark.parametrize("shape,stride,want", [
    ((200, 384), (384, 1), (1, 200, 384, 0, 384, 1)), ((3, 200, 384), (9, 1, 201), (3, 200, 384, 9, 1, 201)), ((1, 128), (1, 1), (1, 1, 128, 0, 1, 1))])
def test_quantize_blocks(host, shape, stride, want):
    h, calls, _ = host
    q, s = h.quantize_blocks(Fake(shape, BF16, stride=stride))
    assert calls == [(0x1000, 1, *want, Q, S, 0x703)]
    assert tuple(q.shape) == shape and tuple(s.shape) == (*shape[:-2], (shape[-2] + 127) // 128, shape[-1] // 128)


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


@pytest.mark.parametrize("change", [dict(is_cuda=False), dict(dtype=torch.float64), dict(shape=(256,)), dict(shape=(5, 200)), dict(shape=(5, 0)),
                                    dict(shape=(1, 2, 3, 256)), dict(stride=(1, 5)), dict(device=0)])
def test_quantize_leaves_every_other_form_alone(host, change):
    h, calls, _ = host
    kw = {"shape": (5, 256), "dtype": F16, **change}
    x = Fake(**kw)
    assert h.quantize(x, None) is None and h.swiglu_quantize(x) is None and calls == [] and x.made == []
    if "stride" not in change:
        assert h.quantize_blocks(x) is None and calls == []


def test_rows_of_another_form(host):
    h, calls, _ = host
    x = Fake((5, 256), F16)
    for rows in (Fake((7,), torch.int64), Fake((7, 1), I32), Fake((7,), I32, contiguous=False), Fake((7,), I32, device=1),
                 Fake((7,), I32, is_cuda=False)):
        assert h.quantize(x, rows) is None
    assert h.quantize(Fake((0, 256), F16), Fake((7,), I32)) is None and calls == [] and x.made == []
    assert h.quantize_blocks(Fake((3, 256, 256), F16, stride=(1, 2, 768))) is None


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
        h.quantize(1, None)
    with pytest.raises(AttributeError):
        h.grouped(1, 2, 3, 4, 5, 6)
    x = Fake((5, 256), F16)
    x.new_empty = lambda *a, **k: 1 / 0
    with pytest.raises(ZeroDivisionError):
        h.quantize(x, None)
    x = Fake((5, 256), F16)
    x.data_ptr = lambda: 1 / 0
    with pytest.raises(ZeroDivisionError):
        h.quantize_blocks(x)
    assert calls == []
