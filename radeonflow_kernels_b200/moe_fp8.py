"""The MoE layer with block-scaled FP8 experts, for any number of tokens.

Router, top-k and sort are the fp16 layer's stages; then the token rows are gathered and quantised in one pass, the experts'
products run on FP8 tensor cores (`grouped.fp8_grouped_mm`), SwiGLU quantises on its way, and the layer's combine adds up.
`moe_few.FewTokenMoE` takes the same weights for a decode step of up to 32 tokens, in one kernel and with fp16 activations.
The reference has no counterpart (its MoE layer is fp16 throughout).
"""
import torch

from . import _lib
from .grouped import fp8_grouped_mm
from .moe import _check_fp16_cuda
from .quant import BLOCK, fp8_quantize, fp8_quantize_blocks, fp8_swiglu_quantize


def quantize_experts(weights, config):
    """The fp16 layer's weights dict -> the dict of FP8 experts that `Fp8MoE` and `FewTokenMoE` take.

    'experts.gate_up.weight' e4m3fn [E, 2f, d] (gate rows first) and 'experts.gate_up.scale' fp32 [E, 2f/128, d/128],
    'experts.down.weight' [E, d, f] and its scale, the same under 'shared_experts' without the leading axis (the shared
    expert is d_expert * n_shared_experts wide), and the fp16 'router.weight' itself.  d_hidden and d_expert: multiples of 128.
    """
    d, f, e = (int(config[k]) for k in ("d_hidden", "d_expert", "n_routed_experts"))
    fs = f * int(config["n_shared_experts"])
    if d % BLOCK or f % BLOCK:
        raise ValueError("moe: FP8 experts need d_hidden and d_expert in multiples of 128")
    device = weights["router.weight"].device

    def stack(n, rows, cols):
        return (torch.empty(n, rows, cols, dtype=torch.float8_e4m3fn, device=device),
                torch.empty(n, rows // BLOCK, cols // BLOCK, dtype=torch.float32, device=device))

    out = {"router.weight": weights["router.weight"]}
    for prefix, n, width in (("experts", e, f),) + ((("shared_experts", 1, fs),) if fs else ()):
        gu, down = stack(n, 2 * width, d), stack(n, d, width)
        for i in range(n):
            name = f"experts.{i}" if prefix == "experts" else prefix
            mats = [weights[f"{name}.{j}.weight"] for j in range(3)]
            for j, (m, shape) in enumerate(zip(mats, ((d, width), (d, width), (width, d)))):
                _check_fp16_cuda(f"{name}.{j}.weight", m)
                if tuple(m.shape) != shape:
                    raise ValueError(f"moe: {name}.{j}.weight must be {list(shape)}")
            for j in range(2):
                at, blocks = slice(j * width, (j + 1) * width), slice(j * width // BLOCK, (j + 1) * width // BLOCK)
                fp8_quantize_blocks(mats[j].t(), out=(gu[0][i, at], gu[1][i, blocks]))
            fp8_quantize_blocks(mats[2].t(), out=(down[0][i], down[1][i]))
        for what, (q, s) in (("gate_up", gu), ("down", down)):
            out[f"{prefix}.{what}.weight"], out[f"{prefix}.{what}.scale"] = (q, s) if prefix == "experts" else (q[0], s[0])
    return out


class Fp8MoE:
    """The layer with the weights of `quantize_experts`.  ``config`` as in `moe.moe_forward` (n_shared_experts may be 0);
    ``router_bias``: fp32 [E], added to the logits.  Buffers come from torch's allocator at every call; calls on different
    streams may overlap.
    """

    def __init__(self, weights, config, router_bias=None):
        self.d, self.f, self.e, self.k = (int(config[n]) for n in ("d_hidden", "d_expert", "n_routed_experts",
                                                                   "n_experts_per_token"))
        self.fs = self.f * int(config["n_shared_experts"])
        self.router, self.bias = weights["router.weight"], router_bias
        _check_fp16_cuda("router.weight", self.router)
        if tuple(self.router.shape) != (self.e, self.d):
            raise ValueError(f"moe: router.weight must be [{self.e}, {self.d}]")
        device = self.router.device
        if router_bias is not None and not (router_bias.dtype == torch.float32 and tuple(router_bias.shape) == (self.e,)
                                            and router_bias.is_contiguous() and router_bias.device == device):
            raise ValueError(f"moe: router_bias must be a contiguous float32 vector of {self.e} on the weights' device")
        if self.d % BLOCK or self.f % BLOCK:
            raise ValueError("moe: FP8 experts need d_hidden and d_expert in multiples of 128")
        self.gate_up = self._operand(weights, "experts.gate_up", self.e, 2 * self.f, self.d)
        self.down = self._operand(weights, "experts.down", self.e, self.d, self.f)
        if self.fs:
            self.shared_gate_up = self._operand(weights, "shared_experts.gate_up", 1, 2 * self.fs, self.d)
            self.shared_down = self._operand(weights, "shared_experts.down", 1, self.d, self.fs)

    def _operand(self, weights, name, e, n, k):
        q, s = weights[f"{name}.weight"], weights[f"{name}.scale"]
        lead = (e,) if name.startswith("experts") else ()
        for t, dtype, shape in ((q, torch.float8_e4m3fn, (*lead, n, k)), (s, torch.float32, (*lead, n // BLOCK, k // BLOCK))):
            if not (t.is_cuda and t.dtype == dtype and tuple(t.shape) == shape and t.is_contiguous() and t.device == self.router.device):
                raise ValueError(f"moe: {name} must be a contiguous {dtype} tensor {list(shape)} on the router weight's device")
        return q.view(e, n, k), s.view(e, n // BLOCK, k // BLOCK)

    def _experts(self, a, a_scale, gate_up, down, offsets):
        m = a.shape[0]
        gu = torch.empty(m, gate_up[0].shape[1], dtype=torch.float16, device=a.device)
        fp8_grouped_mm(a, gate_up[0], a_scale, gate_up[1], offsets, gu)
        h, h_scale = fp8_swiglu_quantize(gu)
        y = torch.empty(m, self.d, dtype=torch.float16, device=a.device)
        return fp8_grouped_mm(h, down[0], h_scale, down[1], offsets, y)

    def forward(self, x):
        """x fp16 [..., d_hidden] -> the layer's output, same shape, on the current stream.  Synchronises nothing."""
        _check_fp16_cuda("input", x)
        if x.shape[-1] != self.d or x.device != self.router.device:
            raise ValueError(f"moe: input must be [..., {self.d}] on the weights' device")
        if x.device.index != torch.cuda.current_device():
            raise ValueError("moe: the input must be on the current device")
        t, e, k = x.numel() // self.d, self.e, self.k
        if t == 0:
            return torch.empty_like(x)
        L, stream, dev = _lib.lib(), _lib.current_stream(), x.device
        ints = lambda *s: torch.empty(*s, dtype=torch.int32, device=dev)
        half = lambda *s: torch.empty(*s, dtype=torch.float16, device=dev)
        scores, index, weight, source = half(t, e), ints(t * k), half(t * k), ints(t * k)
        _lib.check(L.rf_moe_router_gemm(x.data_ptr(), self.router.data_ptr(), None if self.bias is None else self.bias.data_ptr(),
                                        t, e, self.d, scores.data_ptr(), stream), "rf_moe_router_gemm")
        _lib.check(L.rf_moe_topk(scores.data_ptr(), t, e, k, index.data_ptr(), weight.data_ptr(), source.data_ptr(), stream),
                   "rf_moe_topk")
        experts, rows, offsets, rev, row_weight = ints(t * k), ints(t * k), ints(e + 1), ints(t * k), half(t * k)
        scratch = torch.empty(L.rf_moe_permute_scratch_bytes(t * k, e), dtype=torch.uint8, device=dev)
        _lib.check(L.rf_moe_permute(index.data_ptr(), source.data_ptr(), weight.data_ptr(), t, e, k, experts.data_ptr(),
                                    rows.data_ptr(), offsets.data_ptr(), rev.data_ptr(), row_weight.data_ptr(),
                                    scratch.data_ptr(), stream), "rf_moe_permute")
        flat = x.view(t, self.d)
        y = self._experts(*fp8_quantize(flat, rows=rows), self.gate_up, self.down, offsets)      # (rows count modulo t)
        if self.fs:
            ends = ints(2)
            ends[:1].zero_()
            ends[1:].fill_(t)
            shared = self._experts(*fp8_quantize(flat), self.shared_gate_up, self.shared_down, ends)
        else:
            shared = torch.zeros(t, self.d, dtype=torch.float16, device=dev)
        out = torch.empty_like(x)
        _lib.check(L.rf_moe_combine(y.data_ptr(), shared.data_ptr(), rev.data_ptr(), row_weight.data_ptr(), t, k, self.d,
                                    out.data_ptr(), stream), "rf_moe_combine")
        return out
