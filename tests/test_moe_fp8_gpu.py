"""The layer with FP8 experts, put together from its operators, against the same steps in plain torch and against the layers
with fp16 activations.

The steps' own tolerances are tested with each operator.  Together: one fp16 step of a gate or up value (2^-11) can turn an
e4m3 rounding behind it over, 2^-3 of a single value of h; of random sign, in a share of about 2^-11 / 2^-4 of the values, it
moves the norm of the result by 2^-3 sqrt(2^-7) = 1.1e-2 at the very most.

Against unquantised activations: e4m3 has a step of 2^-3 at mantissa 1 <= m < 2, an error of step / sqrt(12) on the mean, and m^2
is 7/3 on the mean, so a quantised vector, and a sum over it, is off by q = 2^-3 / sqrt(12 * 7/3) = 2.4 % of its norm.  x's
error reaches gate and up.  d(silu(g) u) / (silu(g) u) = dg (1 + g (1 - sigmoid(g))) / g + du / u, where the bracket is at most
1.5 on the mean of normal g: sqrt(1.5^2 + 1) q = 4.3 %, with h's own 2.4 % behind it 4.9 %.  That is a mean; a result of few
terms scatters about it: ACT = twice that.  Quantised weights add q to each of gate, up and down: sqrt(2) * 4.3 % = 6.0 %, with
h's and the down weight's 2.4 % 6.9 %: ALL = twice that.
"""
import numpy as np
import pytest
import torch

from oracle import moe as o
from radeonflow_kernels_b200 import gemm, moe, moe_few, moe_fp8, quant

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACT, ALL = 0.098, 0.138


def make(t, d, f, e, k, ns, seed):
    x, w, cfg = o.generate_input(d, f, e, max(ns, 1), k, t, seed)
    cfg["n_shared_experts"] = ns
    w = {n: torch.from_numpy(v).to(DEV) for n, v in w.items() if ns or not n.startswith("shared")}
    # logits of small multiples of powers of two: exact in any order, so that every path chooses the same experts
    g = torch.Generator(device=DEV).manual_seed(seed)
    w["router.weight"] = (torch.randint(-1, 2, (e, d), generator=g, device=DEV) * 2.0 ** -5).half()
    x = (torch.randint(-8, 9, (1, t, d), generator=g, device=DEV) / 8).half()
    return x, w, cfg


def value(q, s):
    return (q.float().double().unflatten(-1, (-1, 128)) * s.double()[..., None]).flatten(-2)


def weight_value(q, s):
    return value(q, s.repeat_interleave(128, -2))


def plain(x, w8, cfg):
    t, d = x.shape
    k, e, ns = cfg["n_experts_per_token"], cfg["n_routed_experts"], cfg["n_shared_experts"]
    logits = (x.double() @ w8["router.weight"].double().t()).half()
    idx, p, _ = o.route(logits.cpu().numpy(), k)
    a = value(*quant.fp8_quantize(x))

    def expert(rows, gu, down):
        g, u = (rows @ gu.t()).half().double().chunk(2, 1)
        h = value(*quant.fp8_quantize((g / (1 + torch.exp(-g)) * u).float()))
        return (h @ down.t()).half().double()

    out = torch.zeros(t, d, dtype=torch.float64, device=DEV)
    gu, down = (weight_value(w8[f"experts.{n}.weight"], w8[f"experts.{n}.scale"]) for n in ("gate_up", "down"))
    for i in range(e):
        tt, kk = np.nonzero(idx == i)
        if len(tt):
            rows = torch.from_numpy(tt).to(DEV)
            out[rows] += torch.from_numpy(p[tt, kk].astype(np.float64)).to(DEV)[:, None] * expert(a[rows], gu[i], down[i])
    if ns:
        gu, down = (weight_value(w8[f"shared_experts.{n}.weight"], w8[f"shared_experts.{n}.scale"]) for n in ("gate_up", "down"))
        out += expert(a, gu, down)
    return out


@pytest.mark.parametrize("t,d,f,e,k,ns", [(1, 128, 128, 4, 2, 1), (37, 384, 256, 32, 4, 1), (300, 1024, 512, 8, 2, 2),
                                          (2000, 256, 384, 16, 8, 0)])
def test_the_steps_together(t, d, f, e, k, ns):
    x, w, cfg = make(t, d, f, e, k, ns, 3)
    w8 = moe_fp8.quantize_experts(w, cfg)
    layer = moe_fp8.Fp8MoE(w8, cfg)
    got = layer.forward(x)
    torch.cuda.synchronize()
    assert got.shape == x.shape and gemm.device_status() == 0
    want = plain(x[0], w8, cfg)
    assert float((got[0].double() - want).norm() / want.norm()) < 1.1e-2
    assert torch.equal(layer.forward(x), got)
    if t <= 32:
        few = moe_few.FewTokenMoE(w8, cfg).forward(x)
        assert float((got.double() - few.double()).norm() / few.double().norm()) < ACT
    if ns:
        full, _ = moe.moe_forward(x, w, cfg)
        assert float((got.double() - full.double()).norm() / full.double().norm()) < ALL


def test_prefill_and_decode_from_the_same_weights():
    """As a serving program has them: one set of FP8 weights, a prefill, then decode steps, some of them captured."""
    x, w, cfg = make(40, 512, 256, 16, 4, 1, 5)
    w8 = moe_fp8.quantize_experts(w, cfg)
    prefill, decode = moe_fp8.Fp8MoE(w8, cfg), moe_few.FewTokenMoE(w8, cfg)
    long = prefill.forward(x)
    steps = torch.cat([decode.forward(x[:, i:i + 5].contiguous()) for i in range(0, 40, 5)], 1)
    assert float((long.double() - steps.double()).norm() / steps.double().norm()) < ACT
    buf = x[:, :5].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decode.forward(buf)
        both = prefill.forward(buf)
    for i in range(0, 40, 5):
        buf.copy_(x[:, i:i + 5])
        graph.replay()
        assert torch.equal(out, steps[:, i:i + 5])
        assert float((both.double() - out.double()).norm() / out.double().norm()) < ACT
    assert gemm.device_status() == 0


def test_weights_with_a_bias():
    x, w, cfg = make(64, 256, 128, 8, 2, 1, 6)
    w8 = moe_fp8.quantize_experts(w, cfg)
    bias = torch.zeros(8, device=DEV)
    bias[5] = 8.0
    got, few = moe_fp8.Fp8MoE(w8, cfg, router_bias=bias).forward(x), moe_few.FewTokenMoE(w8, cfg, router_bias=bias)
    steps = torch.cat([few.forward(x[:, i:i + 32].contiguous()) for i in (0, 32)], 1)
    assert float((got.double() - steps.double()).norm() / steps.double().norm()) < ACT


def test_refusals():
    x, w, cfg = make(4, 256, 128, 4, 2, 1, 7)
    with pytest.raises(ValueError, match="multiples of 128"):
        moe_fp8.quantize_experts(w, {**cfg, "d_expert": 64})
    with pytest.raises(ValueError, match="shared_experts.0.weight"):
        moe_fp8.quantize_experts(w, {**cfg, "n_shared_experts": 2})
    w8 = moe_fp8.quantize_experts(w, cfg)
    with pytest.raises(ValueError, match="experts.down"):
        moe_fp8.Fp8MoE({**w8, "experts.down.scale": w8["experts.down.scale"].half()}, cfg)
    layer = moe_fp8.Fp8MoE(w8, cfg)
    with pytest.raises(ValueError, match="256"):
        layer.forward(x[..., :128].contiguous())
    with pytest.raises(ValueError, match="fp16"):
        layer.forward(x.float())
    assert layer.forward(x[:, :0]).shape == (1, 0, 256)
    few = moe_few.FewTokenMoE(w8, cfg)
    for bad, match in ((x.float(), "fp16"), (x[..., :128].contiguous(), "256"), (x.expand(9, 4, 256).contiguous(), "32 tokens"),
                       (x.transpose(1, 2).contiguous().transpose(1, 2), "contiguous"), (x.cpu(), "CUDA")):
        with pytest.raises(ValueError, match=match):
            few.forward(bad)
