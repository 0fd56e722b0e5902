"""Python boundary of the grouped FP8 block-scaled product: each group of rows by a weight of its own.

The experts of an MoE layer in FP8: rows sorted by expert (`rf_moe_permute`'s first_token_offset gives the offsets),
quantised by `quant.fp8_quantize`, times weights quantised by `quant.fp8_quantize_blocks`.  The reference has no counterpart
(its grouped GEMM is fp16, src/moe/gemm_thirdparty.cpp:65-115).
"""
import torch

from . import _lib

_OUT = {torch.float16: 0, torch.bfloat16: 1}       # RF_F16, RF_BF16
MAX_GROUPS = 1024


def fp8_grouped_mm(a, b, a_scale, b_scale, offsets, c):
    """c[r] = sum_kb a_scale[r, kb] * b_scale[g, :, kb] * (a[r] . b[g]^T)_kb for the rows r in offsets[g] .. offsets[g + 1] - 1.

    a [m, k] e4m3fn, b [groups, n, k] e4m3fn, a_scale [m, k/128] fp32, b_scale [groups, ceil(n/128), k/128] fp32, offsets
    [groups + 1] int32 on the device, ascending, in 0 .. m (others are clipped to that, and one below an earlier one counts as the
    earlier one); c [m, n] bf16 or fp16, returned.
    All contiguous, on the current device.  n % 64 == 0, k % 128 == 0, at most 1024 groups, which may be empty.  Rows in no
    group are left as they were.  The counts stay on the device: nothing is synchronised, and a captured call follows the
    offsets of its replay.
    """
    if (_lib._host or _lib.host()).grouped(a, b, a_scale, b_scale, offsets, c):     # (the checks and the call in native code)
        return c
    for name, t in (("a", a), ("b", b), ("a_scale", a_scale), ("b_scale", b_scale), ("offsets", offsets), ("c", c)):
        if not t.is_cuda:
            raise ValueError("fp8_grouped_mm: all tensors must be CUDA tensors (there is no CPU path)")
        if not t.is_contiguous():
            raise ValueError(f"fp8_grouped_mm: {name} must be contiguous")
        if t.device != a.device:
            raise ValueError("fp8_grouped_mm: all tensors must be on one device")
    if a.device.index != torch.cuda.current_device():
        raise ValueError("fp8_grouped_mm: the tensors must be on the current device")
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise ValueError("fp8_grouped_mm: a and b must be float8_e4m3fn")
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32 or offsets.dtype != torch.int32:
        raise ValueError("fp8_grouped_mm: scales must be float32 and offsets int32")
    if c.dtype not in _OUT:
        raise ValueError("fp8_grouped_mm: c must be bfloat16 or float16")
    if a.dim() != 2 or b.dim() != 3 or a.shape[1] != b.shape[2]:
        raise ValueError("fp8_grouped_mm: a must be [m, k] and b [groups, n, k]")
    m, k = a.shape
    groups, n = b.shape[:2]
    if n % 64 != 0 or k % 128 != 0 or n == 0 or k == 0 or not 1 <= groups <= MAX_GROUPS:
        raise ValueError("fp8_grouped_mm: n % 64, k % 128 must be 0 and groups 1 .. 1024")
    if (tuple(c.shape) != (m, n) or tuple(a_scale.shape) != (m, k // 128) or tuple(offsets.shape) != (groups + 1,)
            or tuple(b_scale.shape) != (groups, (n + 127) // 128, k // 128)):
        raise ValueError("fp8_grouped_mm: shape mismatch")
    st = _lib.lib().rf_fp8_grouped_gemm(a.data_ptr(), b.data_ptr(), a_scale.data_ptr(), b_scale.data_ptr(), offsets.data_ptr(),
                                        c.data_ptr(), _OUT[c.dtype], m, groups, n, k, _lib.current_stream())
    _lib.check(st, "rf_fp8_grouped_gemm")
    return c
