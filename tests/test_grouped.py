"""Refusals of the grouped FP8 product, all before any device work."""
import pytest
import torch

from radeonflow_kernels_b200 import _lib, grouped

A = 0x7000000                # aligned for everything; nothing stands behind it


def call(lib, a=A, b=A, a_s=A, b_s=A, off=A, c=A, dtype=1, m=8, e=2, n=128, k=128):
    return lib.rf_fp8_grouped_gemm(a, b, a_s, b_s, off, c, dtype, m, e, n, k, None)


@pytest.mark.parametrize("kw,status", [
    (dict(n=100), 1), (dict(n=0), 1), (dict(k=64), 1), (dict(k=0), 1), (dict(m=-1), 1), (dict(e=0), 1), (dict(e=1025), 1),
    (dict(e=1024, n=64 * 2 ** 16), 1), (dict(m=2 ** 30, k=512), 1), (dict(dtype=2), 7), (dict(dtype=-1), 7),
    (dict(a=None), 2), (dict(b=None), 2), (dict(a_s=None), 2), (dict(b_s=None), 2), (dict(off=None), 2), (dict(c=None), 2),
    (dict(a=A + 8), 3), (dict(b=A + 8), 3), (dict(c=A + 8), 3), (dict(a_s=A + 2), 3), (dict(b_s=A + 2), 3), (dict(off=A + 2), 3),
    (dict(m=0, a=None), 0)])
def test_entry(rf_lib, kw, status):
    assert call(rf_lib, **kw) == status


class Meta(torch.Tensor):
    """A tensor that says it lies on the GPU."""
    is_cuda = True


def test_python(monkeypatch):
    monkeypatch.setattr(_lib, "_host", _lib._NoHost)                      # the Python code's checks
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)       # the index of the CPU's device
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype).as_subclass(Meta)
    f8 = torch.float8_e4m3fn
    good = dict(a=t(8, 256, dtype=f8), b=t(3, 192, 256, dtype=f8), a_scale=t(8, 2), b_scale=t(3, 2, 2),
                offsets=t(4, dtype=torch.int32), c=t(8, 192, dtype=torch.bfloat16))
    for kw, match in ((dict(a=t(8, 256)), "float8"), (dict(b=t(3, 192, 256, dtype=torch.uint8)), "float8"),
                      (dict(a=t(8, 128, dtype=f8)), r"\[m, k\]"), (dict(a_scale=t(8, 3)), "shape"), (dict(b_scale=t(3, 1, 2)), "shape"),
                      (dict(offsets=t(3, dtype=torch.int32)), "shape"), (dict(offsets=t(4, dtype=torch.int64)), "int32"),
                      (dict(c=t(8, 192)), "bfloat16"), (dict(c=t(192, 8, dtype=torch.bfloat16).t()), "contiguous"),
                      (dict(b=t(3, 100, 256, dtype=f8)), "n % 64"), (dict(b=t(0, 192, 256, dtype=f8)), "groups")):
        with pytest.raises(ValueError, match=match):
            grouped.fp8_grouped_mm(**{**good, **kw})
    with pytest.raises(ValueError, match="CUDA"):
        grouped.fp8_grouped_mm(**{**good, "c": torch.zeros(8, 192, dtype=torch.bfloat16)})
