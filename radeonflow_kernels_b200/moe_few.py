"""The MoE layer for a few tokens, a decode step, in one kernel.

``FewTokenMoE`` computes the layer of `moe.moe_forward` (router, softmax and top-k, SwiGLU experts, shared expert, weighted sum)
for 1 to 32 tokens.  The experts are the layer's fp16 weights or block-scaled FP8 ones (`moe_fp8.quantize_experts`); tokens
and results are fp16, products are summed in fp32.  It chooses experts by the layer's rule: fp16 logits, probabilities rounded
to fp16, equal ones by the lowest index.  Unlike the layer it rounds nothing between the logits and the result but the
vector between an expert's two products, to fp16.
"""
import ctypes
import threading
import weakref

import torch

from . import _lib
from .moe import _check_fp16_cuda

MAX_TOKENS = 32
BLOCK = 128
_SHARED = "shared_experts"


class _Workspace:
    """Zeroed device memory, freed with the last layer that uses it."""

    def __init__(self, size):
        self.size, ptr = size, ctypes.c_void_p()
        _lib.check(_lib.lib().rf_moe_few_workspace_alloc(size, ctypes.byref(ptr)), "rf_moe_few_workspace_alloc")
        self.ptr, self._free = ptr.value, _lib.lib().rf_moe_few_workspace_free

    def __del__(self):
        if getattr(self, "ptr", None):
            self._free(self.ptr)


class _CaptureWorkspace:
    """Zeroed device memory of the graph that `stream` is being captured into: it lives as long as the graph and its executables."""

    def __init__(self, stream, capture, size):
        self.capture, self.size, ptr = capture, size, ctypes.c_void_p()
        _lib.check(_lib.lib().rf_moe_few_workspace_alloc_captured(stream, size, ctypes.byref(ptr)),
                   "rf_moe_few_workspace_alloc_captured")
        self.ptr = ptr.value


# (device, stream) -> workspace.  The layers of a model run one after the other on a stream, so they share them.
_workspaces = weakref.WeakValueDictionary()
# (device, stream) -> workspace of the last capture on it; of no use when the capture has ended (its number never comes again)
_captured = {}
_lock = threading.Lock()        # over the maps of workspaces while one is looked for and made


def captured_workspace_bytes():
    """Device memory that captured graphs hold as workspaces of this module's layers.  What graphs that are gone have left is freed,
    as it is at the next capture or new workspace."""
    size = ctypes.c_size_t()
    _lib.check(_lib.lib().rf_moe_few_workspace_reap(ctypes.byref(size)), "rf_moe_few_workspace_reap")
    return size.value


class FewTokenMoE:
    """One layer's handle: what its kernel needs of the weights, which have to stay where they are.

    ``weights``: the layer's dict ('router.weight', 'experts.{i}.{0,1,2}.weight', 'shared_experts.{0,1,2}.weight', fp16), or the
    dict of FP8 experts ('router.weight' fp16; 'experts.gate_up.weight' e4m3fn [E, 2f, d], gate rows first,
    'experts.gate_up.scale' fp32 [E, 2f/128, d/128], 'experts.down.weight' [E, d, f], 'experts.down.scale' and the same under
    'shared_experts' without the leading axis).  ``config``: d_hidden, d_expert, n_routed_experts (a power of two, at most 256),
    n_experts_per_token (at most 8), n_shared_experts (0: no shared expert).  ``router_bias``: fp32 [E], added to the logits.

    Calls on different streams may overlap: each stream has a workspace of its own, which the layers called on it share, and so
    has each capture.  A captured graph uses the handle's tables: the handle has to outlive it.  Its workspace is the graph's own, outside
    torch's allocator, and goes with it.  32 tokens through 8 of 256 experts of 7168 x 2048 take 102 MB, one token 3.
    """

    def __init__(self, weights, config, router_bias=None):
        d, f, e = (int(config[k]) for k in ("d_hidden", "d_expert", "n_routed_experts"))
        n_shared = int(config["n_shared_experts"])
        self._handle = None
        self.fp8 = "experts.gate_up.weight" in weights
        self.config = _lib.RfMoeFewConfig(d, f, e, int(config["n_experts_per_token"]), n_shared, int(self.fp8))
        self.d_hidden, self._held, self._sizes = d, {}, {}
        router = weights["router.weight"]
        _check_fp16_cuda("router.weight", router)
        self.device = router.device
        self._check_device("the weights")
        if tuple(router.shape) != (e, d):
            raise ValueError(f"moe: router.weight must be [{e}, {d}]")
        if router_bias is not None and not (router_bias.dtype == torch.float32 and tuple(router_bias.shape) == (e,)
                                            and router_bias.is_contiguous() and router_bias.device == self.device):
            raise ValueError(f"moe: router_bias must be a contiguous float32 vector of {e} on the weights' device")
        take = self._fp8_matrices if self.fp8 else self._fp16_matrices
        matrices, scales = take(weights, d, f, e, n_shared)
        self._keep = (router, router_bias, matrices, scales)
        arrays = [(ctypes.c_void_p * len(m))(*m) for m in zip(*[[t.data_ptr() for t in row] for row in matrices])]
        scale_arrays = [(ctypes.c_void_p * len(m))(*m) for m in zip(*[[t.data_ptr() for t in row] for row in scales])] or [None] * 3
        handle = ctypes.c_void_p()
        st = _lib.lib().rf_moe_few_create(ctypes.byref(self.config), router.data_ptr(),
                                          None if router_bias is None else router_bias.data_ptr(), *arrays, *scale_arrays,
                                          ctypes.byref(handle))
        _lib.check(st, "rf_moe_few_create")
        self._handle, self._destroy = handle, _lib.lib().rf_moe_few_destroy

    def _check_device(self, what):
        if self.device.index != torch.cuda.current_device():
            raise ValueError(f"moe: {what} must be on the current device")

    def _fp16_matrices(self, weights, d, f, e, n_shared):
        rows = []
        for prefix, width in [(f"experts.{i}", f) for i in range(e)] + [(_SHARED, f * n_shared)] * (n_shared > 0):
            row = [weights[f"{prefix}.{j}.weight"] for j in range(3)]
            for j, (t, shape) in enumerate(zip(row, ((d, width), (d, width), (width, d)))):
                _check_fp16_cuda(f"{prefix}.{j}.weight", t)
                if tuple(t.shape) != shape or t.device != self.device:
                    raise ValueError(f"moe: {prefix}.{j}.weight must be {list(shape)} on the router weight's device")
            rows.append(row)
        return rows, []

    def _fp8_matrices(self, weights, d, f, e, n_shared):
        def stack(prefix, name, *shape):
            w, s = weights[f"{prefix}.{name}.weight"], weights[f"{prefix}.{name}.scale"]
            blocks = (*shape[:-2], (shape[-2] + BLOCK - 1) // BLOCK, shape[-1] // BLOCK)
            for t, dtype, want in ((w, torch.float8_e4m3fn, shape), (s, torch.float32, blocks)):
                if not (t.is_cuda and t.dtype == dtype and t.is_contiguous() and tuple(t.shape) == want and t.device == self.device):
                    raise ValueError(f"moe: {prefix}.{name} must be a contiguous {dtype} tensor {list(want)} on the router "
                                     "weight's device")
            return w, s

        if d % BLOCK or f % BLOCK:
            raise ValueError("moe: FP8 experts need d_hidden and d_expert in multiples of 128")
        gu, gus = stack("experts", "gate_up", e, 2 * f, d)
        dn, dns = stack("experts", "down", e, d, f)
        rows = [[gu[i, :f], gu[i, f:], dn[i]] for i in range(e)]
        scales = [[gus[i, :f // BLOCK], gus[i, f // BLOCK:], dns[i]] for i in range(e)]
        if n_shared > 0:
            fs = f * n_shared
            gu, gus = stack(_SHARED, "gate_up", 2 * fs, d)
            dn, dns = stack(_SHARED, "down", d, fs)
            rows.append([gu[:fs], gu[fs:], dn])
            scales.append([gus[:fs // BLOCK], gus[fs // BLOCK:], dns])
        return rows, scales

    def _workspace(self, n_tokens, stream):
        L = _lib.lib()
        size = self._sizes.get(n_tokens)
        if size is None:
            size = self._sizes[n_tokens] = L.rf_moe_few_workspace_bytes(ctypes.byref(self.config), n_tokens)
        capture = ctypes.c_ulonglong()          # (of this call: another thread's may come in between)
        _lib.check(L.rf_stream_capture_id(stream, ctypes.byref(capture)), "rf_stream_capture_id")
        key = (self.device.index, stream)
        if capture.value:
            with _lock:
                ws = _captured.get(key)
                if ws is None or ws.capture != capture.value or ws.size < size:
                    ws = _captured[key] = _CaptureWorkspace(stream, capture.value, size)
            return ws
        held = self._held.get(key)
        if held is not None and held[-1].size >= size:
            return held[-1]
        with _lock:             # threads may share a stream
            shared = _workspaces.get(key)
            if shared is None or shared.size < size:
                # (one that has become too small stays: earlier calls may still use it)
                shared = _workspaces[key] = _Workspace(1 << (size - 1).bit_length())
            held = self._held.get(key, ())
            if not held or held[-1] is not shared:
                self._held[key] = (*held, shared)       # never seen empty
        return shared

    def reset(self):
        """Forgets the workspaces of this process's layers.  Needed after `gemm.device_status()` has told of a lost wait: until then
        every call with a workspace that such a call left behind refuses to run and reports a lost wait again.  The other layers
        have to be reset too, and a graph whose replay lost a wait has to be captured again."""
        with _lock:
            _workspaces.clear()
            _captured.clear()
            self._held.clear()

    def forward(self, x, out=None):
        """x fp16 [..., d_hidden], 1 to 32 tokens -> out, same shape (given, it must not overlap x).  Enqueues one kernel on the
        current stream."""
        if not (x.is_cuda and x.dtype == torch.float16 and x.is_contiguous() and x.device == self.device):
            raise ValueError("moe: input must be a contiguous CUDA fp16 tensor on the weights' device (there is no CPU path)")
        self._check_device("the input")
        if x.shape[-1] != self.d_hidden:
            raise ValueError(f"moe: input must be [..., {self.d_hidden}]")
        n_tokens = x.numel() // self.d_hidden
        if n_tokens > MAX_TOKENS:
            raise ValueError(f"moe: at most {MAX_TOKENS} tokens (moe_forward and Fp8MoE take more)")
        if out is None:
            out = torch.empty_like(x)
        elif not (out.dtype == torch.float16 and out.shape == x.shape and out.is_contiguous() and out.device == x.device):
            raise ValueError("moe: out must be a contiguous fp16 tensor like the input")
        elif abs(out.data_ptr() - x.data_ptr()) < 2 * x.numel():
            raise ValueError("moe: out must not overlap the input, which is read until the kernel's end")
        if n_tokens == 0:
            return out
        stream = _lib.current_stream()
        ws = self._workspace(n_tokens, stream)
        st = _lib.lib().rf_moe_few_forward(self._handle, x.data_ptr(), n_tokens, out.data_ptr(), ws.ptr, ws.size, stream)
        _lib.check(st, "rf_moe_few_forward")
        return out

    def __del__(self):
        if getattr(self, "_handle", None):
            self._destroy(self._handle)
