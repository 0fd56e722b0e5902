"""The layer for a few tokens against a plain computation in 64 bits.

Routing is compared exactly: x and the router hold small multiples of powers of two, so that every sum of a logit is exact in
fp32, and `oracle.moe.route` reproduces softmax, rounding and ties bit for bit.

Tolerance of the result, with u = 2^-11 (fp16), s(K) = (K/16 + 40) 2^-23: an fp32 sum of K products, 16 to an MMA, cut off at
every step, and 40 more additions of partial sums:
    dg <= s(d) sum |x||Wg|, du likewise;  dh <= u |h| + 2^-24 + 1.1 dg |u| + |silu(g)| du + 2^-20 |h|     (1.1 >= |silu'|)
    dy <= sum dh |Wd| + s(f) sum |h||Wd|;  dout <= u |out| + 2^-25 + (1 + 2^-20) sum_i p_i dy_i
"""
import ctypes
import gc
import threading
import time

import numpy as np
import pytest
import torch

from oracle import moe as o
from radeonflow_kernels_b200 import _lib, gemm, moe, moe_few, quant

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -11


def make(t, d, f, e, k, ns, fp8, seed, router_scale=2.0 ** -5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ri = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device=DEV)
    cfg = {"d_hidden": d, "d_expert": f, "n_routed_experts": e, "n_experts_per_token": k, "n_shared_experts": ns}
    x = (ri(-8, 9, t, d) / 8).half()
    router = (ri(-1, 2, e, d) * router_scale).half()
    rn = lambda rows, cols, fan: torch.randn(rows, cols, generator=g, device=DEV).mul_(fan ** -0.5)
    sets = [(f"experts.{i}", f) for i in range(e)] + [("shared_experts", f * ns)] * (ns > 0)
    dense = {}         # prefix -> gate, up [d, width], down [width, d] in fp64, as the kernel's weights stand for
    w = {"router.weight": router}
    if not fp8:
        for prefix, width in sets:
            mats = [rn(d, width, d).half(), rn(d, width, d).half(), rn(width, d, max(width, 1)).half()]
            for j, m in enumerate(mats):
                w[f"{prefix}.{j}.weight"] = m
            dense[prefix] = [m.double() for m in mats]
        return x, w, cfg, dense

    def pack(prefix, q, s, name, lead):
        w[f"{prefix}.{name}.weight"], w[f"{prefix}.{name}.scale"] = (q, s) if lead else (q[0], s[0])
        return (q.float().double().unflatten(-1, (-1, 128)) * s.double().repeat_interleave(128, -2)[..., None]).flatten(-2)

    for prefix, n, width in (("experts", e, f),) + ((("shared_experts", 1, f * ns),) if ns else ()):
        gu = torch.stack([rn(2 * width, d, d) for _ in range(n)])
        dn = torch.stack([rn(d, width, width) for _ in range(n)])
        gu = pack(prefix, *quant.fp8_quantize_blocks(gu), "gate_up", n == e and prefix == "experts")
        dn = pack(prefix, *quant.fp8_quantize_blocks(dn), "down", n == e and prefix == "experts")
        for i in range(n):
            dense[f"experts.{i}" if prefix == "experts" else prefix] = [gu[i, :width].t(), gu[i, width:].t(), dn[i].t()]
    return x, w, cfg, dense


def reference(x, w, cfg, dense, bias=None):
    """fp64 result, and how far the kernel may be from it."""
    t, d = x.shape
    k = cfg["n_experts_per_token"]
    logits = x.double() @ w["router.weight"].double().t()
    logits = logits.float()                 # exact
    if bias is not None:
        logits = logits + bias
    idx, p, _ = o.route(logits.half().cpu().numpy(), k)
    s = lambda n: (n / 16 + 40) * 2.0 ** -23
    out, tol = torch.zeros(t, d, dtype=torch.float64, device=DEV), torch.zeros(t, d, dtype=torch.float64, device=DEV)

    def add(rows, weight, mats):
        gate, up, down = mats
        xs = x[rows].double()
        g, u = xs @ gate, xs @ up
        sig = 1 / (1 + torch.exp(-g))
        h = g * sig * u
        dg, du = s(d) * (xs.abs() @ gate.abs()), s(d) * (xs.abs() @ up.abs())
        dh = (U + 2.0 ** -20) * h.abs() + 2.0 ** -24 + 1.1 * dg * u.abs() + (g * sig).abs() * du
        dy = dh @ down.abs() + s(gate.shape[1]) * (h.abs() @ down.abs())
        out[rows] += weight[:, None] * (h @ down)
        tol[rows] += weight[:, None] * dy * (1 + 2.0 ** -20)

    for e in np.unique(idx):
        tt, kk = np.nonzero(idx == e)
        add(torch.from_numpy(tt).to(DEV), torch.from_numpy(p[tt, kk].astype(np.float64)).to(DEV), dense[f"experts.{e}"])
    if cfg["n_shared_experts"]:
        add(torch.arange(t, device=DEV), torch.ones(t, dtype=torch.float64, device=DEV), dense["shared_experts"])
    return out, tol + U * out.abs() + 2.0 ** -25, idx


def check(got, ref, tol):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float((err / tol).max()))


SHAPES = [
    # t, d, f, e, k, shared
    (1, 128, 128, 4, 1, 1), (1, 1024, 512, 8, 2, 1), (2, 256, 128, 256, 8, 0), (3, 384, 256, 32, 4, 2), (7, 640, 128, 16, 8, 1),
    (8, 512, 384, 64, 8, 1), (9, 256, 256, 1, 1, 1), (16, 1152, 128, 128, 4, 1), (17, 128, 640, 8, 8, 0), (31, 256, 256, 32, 3, 3),
    (32, 1024, 256, 256, 8, 1), (32, 2176, 1152, 4, 4, 1),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,d,f,e,k,ns", SHAPES)
def test_against_64_bits(t, d, f, e, k, ns, fp8):
    x, w, cfg, dense = make(t, d, f, e, k, ns, fp8, seed=t + d)
    ref, tol, _ = reference(x, w, cfg, dense)
    layer = moe_few.FewTokenMoE(w, cfg)
    full = torch.full((t + 2, d), 77.0, device=DEV, dtype=torch.float16)
    got = layer.forward(x, out=full[1:t + 1])
    torch.cuda.synchronize()
    assert gemm.device_status() == 0
    check(got, ref, tol)
    assert (full[0] == 77).all() and (full[-1] == 77).all()
    again = layer.forward(x)                # the workspace as the first call left it
    assert torch.equal(again, got)


@pytest.mark.parametrize("t,d,f,e,k,ns", [(1, 64, 64, 4, 2, 1), (5, 192, 64, 8, 3, 1), (20, 320, 192, 16, 2, 2)])
def test_widths_of_64(t, d, f, e, k, ns):
    """fp16 widths that end inside a tile of 128 columns."""
    x, w, cfg, dense = make(t, d, f, e, k, ns, False, seed=9)
    ref, tol, _ = reference(x, w, cfg, dense)
    check(moe_few.FewTokenMoE(w, cfg).forward(x), ref, tol)


@pytest.mark.parametrize("fp8", [False, True])
def test_every_number_of_tokens_on_one_workspace(fp8):
    x, w, cfg, dense = make(32, 256, 128, 16, 4, 1, fp8, seed=3)
    layer = moe_few.FewTokenMoE(w, cfg)
    ref, tol, _ = reference(x, w, cfg, dense)
    for t in [32, 1, 31, 2, *range(3, 31, 3), 32, 1]:
        check(layer.forward(x[:t]), ref[:t], tol[:t])
    assert layer.forward(x[:0]).shape == (0, 256) and gemm.device_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_bias_sends_all_tokens_to_the_same_experts(fp8):
    x, w, cfg, dense = make(32, 384, 256, 32, 4, 1, fp8, seed=4)
    bias = torch.zeros(32, device=DEV)
    bias[[3, 9, 30]] = 16.0
    ref, tol, idx = reference(x, w, cfg, dense, bias)
    assert (np.sort(idx, 1)[:, 1:] == [3, 9, 30]).sum() > 60
    check(moe_few.FewTokenMoE(w, cfg, router_bias=bias).forward(x), ref, tol)


def test_equal_logits_take_the_lowest_experts():
    x, w, cfg, dense = make(6, 256, 128, 64, 8, 1, False, seed=5)
    w["router.weight"].zero_()
    ref, tol, idx = reference(x, w, cfg, dense)
    assert (idx == np.arange(8)).all()
    check(moe_few.FewTokenMoE(w, cfg).forward(x), ref, tol)


@pytest.mark.parametrize("fp8", [False, True])
def test_nan_stays_in_its_token(fp8):
    x, w, cfg, dense = make(11, 256, 128, 16, 4, 1, fp8, seed=6)
    layer = moe_few.FewTokenMoE(w, cfg)
    want = layer.forward(x)
    for row, value in ((4, float("nan")), (10, float("inf"))):
        y = x.clone()
        y[row, 100] = value
        got = layer.forward(y)
        assert got[row].isnan().all()
        keep = [i for i in range(11) if i != row]
        assert torch.equal(got[keep], want[keep])
    assert gemm.device_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [8, 16, 24, 32])
def test_same_bits_every_time(t, fp8):
    """Weights that stay in L2, so that a stage of them is refilled as soon as it is given back: a warp that still read it when it
    gave it back would multiply some of the next one's (one call in twenty did)."""
    x, w, cfg, _ = make(t, 1024, 512, 32, 4, 1, fp8, seed=t)
    layer = moe_few.FewTokenMoE(w, cfg)
    runs = torch.stack([layer.forward(x) for _ in range(400)])
    assert not (runs != runs[0]).any()
    assert gemm.device_status() == 0


def test_beside_the_layer():
    """The same layer through moe_forward, whose intermediate roundings (fp16 gate, up, outputs of the experts) are more: the
    layer's own tolerance, 1e-2 absolute and relative.  Both choose on the logits that they compute themselves."""
    x, w, cfg = o.generate_input(1024, 512, 32, 1, 4, 24, 7)
    tx, tw = torch.from_numpy(x).to(DEV), {n: torch.from_numpy(v).to(DEV) for n, v in w.items()}
    want, _ = moe.moe_forward(tx, tw, cfg)
    got = moe_few.FewTokenMoE(tw, cfg).forward(tx)
    assert got.shape == tx.shape
    ok, nbad, mx = o.check(got.cpu().numpy(), want.cpu().numpy())
    assert ok, (nbad, mx)


@pytest.mark.parametrize("fp8", [False, True])
def test_large_layer(fp8):
    """The benchmark layer's widths; the weights of one shared and a few routed experts."""
    for t in (1, 12):
        x, w, cfg, dense = make(t, 7168, 2048, 8, 2, 1, fp8, seed=8, router_scale=2.0 ** -6)
        ref, tol, _ = reference(x, w, cfg, dense)
        check(moe_few.FewTokenMoE(w, cfg).forward(x), ref, tol)
        assert gemm.device_status() == 0


def test_streams_and_graphs_at_once():
    """Calls on several streams, and graphs captured from one handle, each with a workspace of its own."""
    x, w, cfg, _ = make(8, 1024, 512, 32, 4, 1, False, seed=10)
    layer = moe_few.FewTokenMoE(w, cfg)
    xs = [x, x.flip(0).contiguous(), (x * 0.5)]
    want = [layer.forward(v).clone() for v in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[] for _ in xs]
    for _ in range(5):
        for i, (v, st) in enumerate(zip(xs, streams)):
            with torch.cuda.stream(st):
                got[i].append(layer.forward(v))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(3) for g in got[i])
    graphs, outs = [], []
    for v in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = layer.forward(v)
            outs.append((a, layer.forward(a.clamp(-1, 1))))
        graphs.append(graph)
    second = [layer.forward(v.clamp(-1, 1)).clone() for v in want]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        got_eager = layer.forward(x)
    torch.cuda.synchronize()
    assert torch.equal(got_eager, want[0]) and gemm.device_status() == 0
    for i in range(3):
        assert torch.equal(outs[i][0], want[i]) and torch.equal(outs[i][1], second[i])


def test_a_marked_workspace_is_refused_until_reset():
    """A workspace that a lost wait left behind holds counts that belong to nothing."""
    x, w, cfg, dense = make(2, 128, 128, 4, 2, 1, False, seed=11)
    layer = moe_few.FewTokenMoE(w, cfg)
    want = layer.forward(x)
    torch.cuda.synchronize()
    assert gemm.device_status() == 0
    one, mark = ctypes.c_int(1), [held[-1].ptr + 256 for held in layer._held.values()]
    cudart = ctypes.CDLL("libcudart.so.12")
    for at in mark:
        assert cudart.cudaMemcpy(ctypes.c_void_p(at), ctypes.byref(one), ctypes.c_size_t(4), 1) == 0
    out = torch.full_like(x, 5.0)
    layer.forward(x, out=out)
    assert gemm.device_status() == 5 and (out == 5).all()
    layer.forward(x, out=out)
    assert gemm.device_status() == 5 and (out == 5).all()
    layer.reset()
    assert torch.equal(layer.forward(x, out=out), want) and gemm.device_status() == 0


def test_weights_are_read_at_every_call():
    x, w, cfg, dense = make(3, 256, 128, 8, 2, 1, False, seed=12)
    layer = moe_few.FewTokenMoE(w, cfg)
    layer.forward(x)
    for n in w:
        if n.endswith(".2.weight"):
            w[n].mul_(-2)
    dense = {n: [m[0], m[1], -2 * m[2]] for n, m in dense.items()}
    ref, tol, _ = reference(x, w, cfg, dense)
    check(layer.forward(x), ref, tol)


def test_out_that_overlaps_the_input_is_refused():
    x, w, cfg, _ = make(3, 256, 128, 8, 2, 1, False, seed=1)
    layer = moe_few.FewTokenMoE(w, cfg)
    both = torch.cat([x, x])
    for out in (both[:3], both[1:4], both[2:5]):
        with pytest.raises(ValueError, match="overlap"):
            layer.forward(both[:3], out=out)
    ws = layer._workspace(3, torch.cuda.current_stream().cuda_stream)
    assert _lib.lib().rf_moe_few_forward(layer._handle, both.data_ptr(), 3, both[2:].data_ptr(), ws.ptr, ws.size, 0) == 7
    assert torch.equal(layer.forward(both[:3], out=both[3:]), layer.forward(x))


def test_host_threads_at_once():
    """One layer, called from threads with a stream each."""
    x, w, cfg, _ = make(20, 512, 256, 16, 4, 1, False, seed=2)
    layer = moe_few.FewTokenMoE(w, cfg)
    inputs = [x[i:i + 5].contiguous() for i in range(0, 20, 5)]
    want = [layer.forward(v) for v in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                if not torch.equal(layer.forward(inputs[i]), want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    assert gemm.device_status() == 0


@pytest.mark.parametrize("fp8", [False, True])
def test_first_call_on_a_stream_of_its_own(fp8):
    """A layer is made and called at once on a stream that is ordered behind nothing, then freed: the next one's tables lie where
    its tables lay."""
    made = [make(4, 512, 256, 16, 4, 1, fp8, seed=20 + i) for i in range(2)]
    want = [reference(x, w, cfg, dense) for x, w, cfg, dense in made]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(40):
        x, w, cfg, _ = made[i % 2]
        layer = moe_few.FewTokenMoE(w, cfg)
        with torch.cuda.stream(side):
            got = layer.forward(x)
        side.synchronize()
        check(got, *want[i % 2][:2])
        del layer
    assert gemm.device_status() == 0


def settled(want):
    """Bytes that graphs hold, once CUDA has told of those that are gone (it does so on a thread of its own)."""
    for _ in range(200):
        gc.collect()
        if moe_few.captured_workspace_bytes() == want:
            return True
        time.sleep(0.02)
    return False


def capture(layer, x):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer.forward(x)
    return graph, out


def test_a_graphs_workspace_goes_with_it():
    x, w, cfg, _ = make(32, 1024, 512, 32, 4, 1, False, seed=13)
    layer, other = moe_few.FewTokenMoE(w, cfg), moe_few.FewTokenMoE(w, cfg)
    size = lambda t: _lib.lib().rf_moe_few_workspace_bytes(ctypes.byref(layer.config), t)
    want = {t: layer.forward(x[:t]).clone() for t in (1, 8, 32)}
    torch.cuda.synchronize()
    gc.collect()
    time.sleep(0.2)
    before = moe_few.captured_workspace_bytes()
    graphs = {t: capture(layer, x[:t]) for t in want}
    assert settled(before + sum(size(t) for t in want))
    both = torch.cuda.CUDAGraph()
    with torch.cuda.graph(both):            # two layers and two sizes in one graph: one workspace, and the larger one
        outs = layer.forward(x[:8]), other.forward(x[:8]), other.forward(x[:32]), layer.forward(x[:1])
    assert settled(before + sum(size(t) for t in want) + size(8) + size(32))
    both.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[o.shape[0]]) for o in outs)
    # one goes; the others stay whole while what it had is used again
    del graphs[8], both, outs
    assert settled(before + size(1) + size(32))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(layer.forward(x), want[32])
    for t, (graph, out) in graphs.items():
        for _ in range(5):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want[t])
    graphs[32][0].replay()                  # (gone while it runs)
    del graph, out, graphs
    assert settled(before) and gemm.device_status() == 0
    # captured over and over
    free = torch.cuda.mem_get_info()[0]
    for _ in range(30):
        graph, out = capture(layer, x)
        graph.replay()
        assert torch.equal(out, want[32])
        del graph, out
    assert settled(before) and torch.cuda.mem_get_info()[0] >= free - 4 * size(32) - (8 << 20)
    assert len(layer._held) == 2 and gemm.device_status() == 0


def test_a_capture_that_fails_leaves_nothing():
    x, w, cfg, _ = make(4, 256, 128, 8, 2, 1, False, seed=14)
    layer = moe_few.FewTokenMoE(w, cfg)
    want = layer.forward(x).clone()
    gc.collect()
    time.sleep(0.2)
    before = moe_few.captured_workspace_bytes()
    with pytest.raises(RuntimeError, match="given up"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.forward(x)
            raise RuntimeError("given up")
    del graph
    assert settled(before)
    graph, out = capture(layer, x)
    graph.replay()
    assert torch.equal(out, want) and torch.equal(layer.forward(x), want)


def test_workspaces_of_captures_only(rf_lib):
    got = ctypes.c_void_p()
    assert rf_lib.rf_moe_few_workspace_alloc_captured(torch.cuda.Stream().cuda_stream, 1000, ctypes.byref(got)) == 7 and not got


class Scattered(moe_few.FewTokenMoE):
    """The same weights, each matrix in memory of its own, the experts in descending order: no distance is even."""

    def _copies(self, rows):
        gap = 48
        buf = torch.empty(sum(t.numel() * t.element_size() + gap for row in rows for t in row) + 16, dtype=torch.uint8, device=DEV)
        at, out = 0, [None] * len(rows)
        for i in reversed(range(len(rows))):
            out[i] = []
            for t in rows[i]:
                n = t.numel() * t.element_size()
                out[i].append(buf[at:at + n].view(t.dtype).view(t.shape).copy_(t))
                at += n + gap
        return out

    def _fp16_matrices(self, *args):
        rows, scales = super()._fp16_matrices(*args)
        return self._copies(rows), scales

    def _fp8_matrices(self, *args):
        rows, scales = super()._fp8_matrices(*args)
        return self._copies(rows), scales


def stacked(w, cfg, interleaved):
    """The fp16 layer's dict as views of stacks."""
    e, w = cfg["n_routed_experts"], dict(w)
    mats = [torch.stack([w[f"experts.{i}.{j}.weight"] for i in range(e)]) for j in range(3)]
    if interleaved:                 # gate and up in one stack
        both = torch.stack(mats[:2], 1)
        mats[:2] = both[:, 0], both[:, 1]
    for i in range(e):
        for j in range(3):
            w[f"experts.{i}.{j}.weight"] = mats[j][i]
    return w


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,d,f,e,k,ns", [(1, 256, 128, 16, 4, 1), (8, 640, 256, 8, 2, 2), (13, 1152, 384, 32, 8, 1), (32, 512, 128, 4, 2, 0), (5, 384, 128, 1, 1, 1)])
def test_weights_may_lie_anywhere(t, d, f, e, k, ns, fp8):
    """Stacks (one tensor map each), and matrices anywhere (a table of them): the same bits."""
    x, w, cfg, dense = make(t, d, f, e, k, ns, fp8, seed=d + e)
    ref, tol, _ = reference(x, w, cfg, dense)
    layers = [moe_few.FewTokenMoE(w, cfg), Scattered(w, cfg)]
    if not fp8:
        layers += [moe_few.FewTokenMoE(stacked(w, cfg, interleaved), cfg) for interleaved in (False, True)]
    got = [layer.forward(x) for layer in layers]
    check(got[0], ref, tol)
    assert all(torch.equal(g, got[0]) for g in got)
    for _ in range(50):
        for layer in layers:
            assert torch.equal(layer.forward(x), got[0])
    assert gemm.device_status() == 0


def test_widths_of_64_in_stacks():
    for t, d, f, e, k, ns in ((1, 64, 64, 4, 2, 1), (20, 320, 192, 16, 2, 2)):
        x, w, cfg, dense = make(t, d, f, e, k, ns, False, seed=9)
        ref, tol, _ = reference(x, w, cfg, dense)
        got = moe_few.FewTokenMoE(stacked(w, cfg, False), cfg).forward(x)
        check(got, ref, tol)
        assert torch.equal(Scattered(w, cfg).forward(x), got)


@pytest.mark.parametrize("fp8", [False, True])
def test_scattered_layers_made_one_where_the_other_was(fp8):
    made = [make(4, 512, 256, 16, 4, 1, fp8, seed=30 + i) for i in range(2)]
    want = [reference(x, w, cfg, dense) for x, w, cfg, dense in made]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(40):
        x, w, cfg, _ = made[i % 2]
        layer = Scattered(w, cfg)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = layer.forward(x)
        side.synchronize()
        check(got, *want[i % 2][:2])
        del layer
    assert gemm.device_status() == 0
