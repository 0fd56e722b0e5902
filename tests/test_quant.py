"""Refusals of the FP8 quantisation, all before any device work."""
import ctypes

import pytest
import torch

from radeonflow_kernels_b200 import _lib, build, quant

A = 0x7000000                # aligned for everything; nothing stands behind it


def test_cpu_tensors_are_refused():
    for fn in (quant.fp8_quantize, quant.fp8_swiglu_quantize, quant.fp8_quantize_blocks):
        with pytest.raises(ValueError, match="CUDA"):
            fn(torch.zeros(4, 256))


@pytest.mark.parametrize("m,k,dtype,status", [(4, 100, 0, 1), (4, 0, 0, 1), (-1, 128, 0, 1), (4, 128, 3, 7), (4, 128, -1, 7),
                                              (2 ** 27, 2048, 0, 1)])
def test_rows_shapes(rf_lib, m, k, dtype, status):
    assert rf_lib.rf_fp8_quantize(A, dtype, k, None, 0, m, k, A, A, None) == status
    assert rf_lib.rf_fp8_swiglu_quantize(A, dtype, 2 * k, m, k, A, A, None) == status


def test_rows_pointers(rf_lib):
    q = lambda x=A, dtype=0, rows=None, src=0, q=A, s=A: rf_lib.rf_fp8_quantize(x, dtype, 128, rows, src, 4, 128, q, s, None)
    assert q(x=None) == 2 and q(q=None) == 2 and q(s=None) == 2
    assert q(x=A + 1) == 3 and q(x=A + 2, dtype=2) == 3 and q(q=A + 8) == 3 and q(s=A + 2) == 3 and q(rows=A + 2, src=4) == 3
    assert q(rows=A, src=0) == 1
    assert rf_lib.rf_fp8_quantize(None, 0, 128, None, 0, 0, 128, None, None, None) == 0         # nothing to do


def test_blocks(rf_lib):
    b = lambda w=A, dtype=0, e=1, n=64, k=128, sn=128, sk=1, q=A, s=A: rf_lib.rf_fp8_quantize_blocks(
        w, dtype, e, n, k, 0, sn, sk, q, s, None)
    assert b(k=64) == 1 and b(e=-1) == 1 and b(n=-1) == 1 and b(e=65536) == 1 and b(dtype=5) == 7
    assert b(sn=256, sk=2) == 7                            # neither axis contiguous
    assert b(w=None) == 2 and b(q=None) == 2 and b(s=None) == 2
    assert b(w=A + 1) == 3 and b(q=A + 4) == 3 and b(s=A + 1) == 3
    assert b(e=0) == 0 and b(n=0) == 0


class Meta(torch.Tensor):
    """A tensor that says it lies on the GPU."""
    is_cuda = True


def test_python_shapes(monkeypatch):
    monkeypatch.setattr(_lib, "_tensors", _lib._NoTensors)                    # the Python code's checks
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)       # the index of the CPU's device
    cuda = lambda *shape, dtype=torch.float16: torch.zeros(*shape, dtype=dtype).as_subclass(Meta)
    for x, match in ((cuda(4, 100), "multiple of 128"), (cuda(128), "multiple of 128"), (cuda(4, 0), "multiple of 128"),
                     (cuda(128, 4).t(), "contiguous"), (cuda(4, 128, dtype=torch.float64), "float16")):
        with pytest.raises(ValueError, match=match):
            quant.fp8_quantize(x)
    with pytest.raises(ValueError, match="multiple of 128"):
        quant.fp8_swiglu_quantize(cuda(4, 128))
    with pytest.raises(ValueError, match="contiguous"):
        quant.fp8_quantize_blocks(cuda(2, 256, 256)[:, ::2, ::2])
    for rows in (torch.zeros(3, dtype=torch.int64), torch.zeros(6, dtype=torch.int32)[::2], torch.zeros(1, 3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="rows"):
            quant.fp8_quantize(cuda(4, 128), rows=rows)
    with pytest.raises(ValueError, match="no rows"):
        quant.fp8_quantize(cuda(0, 128), rows=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="out's q"):
        quant.fp8_quantize(cuda(4, 128), out=(torch.zeros(4, 128), torch.zeros(4, 1)))


def test_the_extension_leaves_what_is_amiss_to_the_python_code(rf_lib):
    t = _lib.tensors()
    assert t is not _lib._NoTensors and t.__file__ == _lib.TENSORS_PATH
    for x in (1, None, torch.zeros(4, 128), torch.zeros(4, 128, dtype=torch.float64), cls_like()):
        assert t.quantize(x, None) is None and t.swiglu_quantize(x) is None and t.quantize_blocks(x) is None
    assert t.quantize(torch.zeros(4, 128)) is None and t.swiglu_quantize() is None
    with pytest.raises(TypeError):
        t.setup(1)


def cls_like():
    return torch.zeros(4, 128).as_subclass(Meta)


def test_without_the_extension(rf_lib, monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_tensors", None)
    monkeypatch.setattr(_lib, "TENSORS_PATH", str(tmp_path / "_tensors.so"))
    with pytest.warns(RuntimeWarning, match="cannot be used"):
        assert _lib.tensors() is _lib._NoTensors
    with pytest.raises(ValueError, match="CUDA"):
        quant.fp8_quantize(torch.zeros(4, 128))


def test_the_library_is_built_where_the_extension_cannot_be(rf_lib, monkeypatch, capsys):
    assert build.TENSORS_PATH == _lib.TENSORS_PATH and build.build_tensors() == build.TENSORS_PATH
    monkeypatch.setenv("CXX", "false")
    monkeypatch.setattr(build, "TENSORS_PATH", build.TENSORS_PATH + ".other")
    assert build.build() == build.LIB_PATH and "without its extension" in capsys.readouterr().err


def test_more_than_31_bits_of_a_size_are_refused(monkeypatch):
    """Sizes go to the library as 32-bit integers: 2^32 + 128 columns would count as 128.  (The memory is never touched.)"""
    monkeypatch.setattr(_lib, "_tensors", _lib._NoTensors)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    called = []
    monkeypatch.setattr(quant, "_outputs", lambda *a: called.append(a))
    cuda = lambda t: t.as_subclass(Meta)
    long = torch.empty(1, 2 ** 32 + 256, dtype=torch.float16)
    windows = torch.empty(2 ** 32 + 200, dtype=torch.float16).unfold(0, 128, 1)         # 2^32 + 73 rows
    for fn, x in ((quant.fp8_quantize, long), (quant.fp8_swiglu_quantize, long), (quant.fp8_quantize_blocks, long),
                  (quant.fp8_quantize_blocks, long.unsqueeze(0)), (quant.fp8_quantize, long[:, :2 ** 31]),
                  (lambda x: quant.fp8_quantize(x, rows=torch.zeros(3, dtype=torch.int32)), windows)):
        with pytest.raises(ValueError, match="2\\^31"):
            fn(cuda(x))
    assert not called
