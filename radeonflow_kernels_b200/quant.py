"""Python boundary of the FP8 quantisation: operands for `gemm.fp8_mm` and `grouped.fp8_grouped_mm`.

Every block of 128 columns of a row (activations) or of 128 x 128 elements (weights) gets one fp32 scale:

    a = max(largest magnitude of the block, 2**-100),  scale = a / 448,  q = e4m3fn(x * (448 / a))

The value that q stands for is q * scale.  A NaN makes its whole block NaN, an infinity makes the block's scale infinite.
Inputs are CUDA tensors in fp16, bf16 or fp32; the work runs on the current stream of the current device, where the
tensors have to be.  The reference has no counterpart (its FP8 operands arrive quantised).
"""
import torch

from . import _lib

BLOCK = 128
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}       # RF_F16, RF_BF16, RF_F32


def _check_input(what, name, x):
    if not x.is_cuda:
        raise ValueError(f"{what}: {name} must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what}: {name} must be float16, bfloat16 or float32")
    if x.device.index != torch.cuda.current_device():
        raise ValueError(f"{what}: {name} must be on the current device")
    if max(x.shape, default=0) >= 2 ** 31:
        raise ValueError(f"{what}: {name} must have fewer than 2^31 rows and columns")


def _outputs(what, out, q_shape, scale_shape, device):
    if out is None:
        return (torch.empty(q_shape, dtype=torch.float8_e4m3fn, device=device),
                torch.empty(scale_shape, dtype=torch.float32, device=device))
    q, scale = out
    for name, t, dtype, shape in (("q", q, torch.float8_e4m3fn, q_shape), ("scale", scale, torch.float32, scale_shape)):
        if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{what}: out's {name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on x's device")
    return q, scale


def fp8_quantize(x, rows=None, out=None):
    """x [m, k] -> (q e4m3fn [m, k], scale fp32 [m, k/128]), the A operand of the FP8 products.

    Columns are contiguous, rows may lie any distance apart; k % 128 == 0.  With ``rows`` (int32 indices, taken modulo m as
    unsigned numbers) row i of the result is x[rows[i]]: the gather of `MoE` token rows costs no pass of its own.
    ``out``: (q, scale) to write to, not overlapping x.
    """
    if out is None:
        hot = (_lib._tensors or _lib.tensors()).quantize(x, rows)         # (the same checks and call in native code, where nothing is amiss)
        if hot is not None:
            return hot
    _check_input("fp8_quantize", "x", x)
    if x.dim() != 2 or x.shape[1] % BLOCK != 0 or x.shape[1] == 0:
        raise ValueError("fp8_quantize: x must be [m, k] with k a multiple of 128")
    if x.stride(1) != 1:
        raise ValueError("fp8_quantize: x's columns must be contiguous")
    n_src, k = x.shape
    m = n_src
    if rows is not None:
        if not (rows.dtype == torch.int32 and rows.dim() == 1 and rows.is_contiguous() and rows.device == x.device):
            raise ValueError("fp8_quantize: rows must be a contiguous int32 vector on x's device")
        m = rows.shape[0]
        if n_src == 0 and m > 0:
            raise ValueError("fp8_quantize: x has no rows to take")
    q, scale = _outputs("fp8_quantize", out, (m, k), (m, k // BLOCK), x.device)
    st = _lib.lib().rf_fp8_quantize(x.data_ptr(), _DTYPES[x.dtype], x.stride(0), None if rows is None else rows.data_ptr(),
                                    n_src, m, k, q.data_ptr(), scale.data_ptr(), _lib.current_stream())
    _lib.check(st, "rf_fp8_quantize")
    return q, scale


def fp8_swiglu_quantize(gate_up, out=None):
    """gate_up [m, 2f] -> (q e4m3fn [m, f], scale fp32 [m, f/128]) of SiLU(gate_up[:, :f]) * gate_up[:, f:], computed in fp32.

    Columns are contiguous, rows may lie any distance apart; f % 128 == 0.
    """
    if out is None:
        hot = (_lib._tensors or _lib.tensors()).swiglu_quantize(gate_up)
        if hot is not None:
            return hot
    _check_input("fp8_swiglu_quantize", "gate_up", gate_up)
    if gate_up.dim() != 2 or gate_up.shape[1] % (2 * BLOCK) != 0 or gate_up.shape[1] == 0:
        raise ValueError("fp8_swiglu_quantize: gate_up must be [m, 2f] with f a multiple of 128")
    if gate_up.stride(1) != 1:
        raise ValueError("fp8_swiglu_quantize: gate_up's columns must be contiguous")
    m, f = gate_up.shape[0], gate_up.shape[1] // 2
    q, scale = _outputs("fp8_swiglu_quantize", out, (m, f), (m, f // BLOCK), gate_up.device)
    st = _lib.lib().rf_fp8_swiglu_quantize(gate_up.data_ptr(), _DTYPES[gate_up.dtype], gate_up.stride(0), m, f, q.data_ptr(),
                                           scale.data_ptr(), _lib.current_stream())
    _lib.check(st, "rf_fp8_swiglu_quantize")
    return q, scale


def fp8_quantize_blocks(w, out=None):
    """w [n, k] or [e, n, k] -> (q e4m3fn like w, contiguous; scale fp32 [(e,) ceil(n/128), k/128]), the B operand.

    One of the last two axes is contiguous: a weight held as [k, n] goes in as its transposed view and is turned round on the
    way.  k % 128 == 0; the last block of n may be shorter than 128.
    """
    if out is None:
        hot = (_lib._tensors or _lib.tensors()).quantize_blocks(w)
        if hot is not None:
            return hot
    _check_input("fp8_quantize_blocks", "w", w)
    if w.dim() not in (2, 3) or w.shape[-1] % BLOCK != 0 or w.shape[-1] == 0:
        raise ValueError("fp8_quantize_blocks: w must be [n, k] or [e, n, k] with k a multiple of 128")
    if w.stride(-1) != 1 and w.stride(-2) != 1:
        raise ValueError("fp8_quantize_blocks: one of w's last two axes must be contiguous")
    n, k = w.shape[-2:]
    e = w.shape[0] if w.dim() == 3 else 1
    scale_shape = (*w.shape[:-2], (n + BLOCK - 1) // BLOCK, k // BLOCK)
    q, scale = _outputs("fp8_quantize_blocks", out, tuple(w.shape), scale_shape, w.device)
    st = _lib.lib().rf_fp8_quantize_blocks(w.data_ptr(), _DTYPES[w.dtype], e, n, k, w.stride(0) if w.dim() == 3 else 0,
                                           w.stride(-2), w.stride(-1), q.data_ptr(), scale.data_ptr(), _lib.current_stream())
    _lib.check(st, "rf_fp8_quantize_blocks")
    return q, scale
