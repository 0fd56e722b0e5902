"""FP8 quantisation against a plain computation in 64 bits.

Tolerances.  scale = a / 448 is one correctly rounded fp32 division: off by at most eps32 / 2 = 2^-24 relative.  q is
e4m3(x * r) with r = fl(448 / a): x * r is off by at most 2 * 2^-24 relative before the conversion, which rounds by half a
step: 2^-4 relative for normal values (|v| >= 2^-6), 2^-10 absolute below.  So |q - v| <= 2^-4 |v| (1 + 2^-22) + 2^-10.
SwiGLU: h in fp32 has an exponential (2 ulp), a sum, a division (2 ulp) and a product: 2^-21 relative is more than their sum.
"""
import numpy as np
import pytest
import torch

from radeonflow_kernels_b200 import _lib, gemm, quant
from tests.helpers import assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def blocks_of(x):                 # [..., k] -> [..., k/128, 128]
    return x.reshape(*x.shape[:-1], -1, 128)


def check(q, scale, x, a, slack=0.0):
    """q, scale (device) against x in blocks [..., 128] (float64 numpy) whose largest magnitudes are a."""
    a = np.maximum(a, 2.0 ** -100)
    s = scale.double().cpu().numpy()
    np.testing.assert_allclose(s, a / 448, rtol=2.0 ** -24 * 1.01 + slack)
    v = x * (448 / a)[..., None]
    got = blocks_of(q.float().double().cpu().numpy())
    bad = np.abs(got - v) > 2.0 ** -4 * np.abs(v) * (1 + 2.0 ** -22 + 2 * slack) + 2.0 ** -10
    assert not bad.any(), (int(bad.sum()), got[bad][:4], v[bad][:4])


def data(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, generator=g, device=DEV) * torch.exp(2 * torch.randn(shape[0], *[1] * (len(shape) - 1), generator=g, device=DEV))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 128), (3, 128), (1, 7168), (7, 384), (130, 1152), (2049, 2048)])
def test_rows(dtype, m, k):
    x = data((m, k), dtype, m + k)
    q, s = quant.fp8_quantize(x)
    assert q.shape == (m, k) and s.shape == (m, k // 128)
    xb = blocks_of(x.double().cpu().numpy())
    check(q, s, xb, np.abs(xb).max(-1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_strided_unaligned_and_no_write_outside(dtype):
    big = data((40, 1000), dtype, 5)
    x = big[3:24, 5:5 + 384]                       # rows 1000 elements apart, starting at odd addresses
    q = torch.full((30, 384), 1.0, device=DEV).to(torch.float8_e4m3fn)
    s = torch.full((30, 3), 7.0, device=DEV)
    quant.fp8_quantize(x, out=(q[4:25], s[4:25]))
    xb = blocks_of(x.double().cpu().numpy())
    check(q[4:25], s[4:25], xb, np.abs(xb).max(-1))
    assert (q.float()[:4] == 1).all() and (q.float()[25:] == 1).all() and (s[:4] == 7).all() and (s[25:] == 7).all()
    # a broadcast row
    q, s = quant.fp8_quantize(x[:1].expand(9, 384))
    assert (q.view(torch.uint8) == q.view(torch.uint8)[:1]).all() and (s == s[:1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_gather(dtype):
    x = data((50, 640), dtype, 6)
    rows = torch.randint(0, 50, (333,), device=DEV, dtype=torch.int32)
    rows[0], rows[1], rows[2] = 49, 49, 0
    q, s = quant.fp8_quantize(x, rows=rows + 50 * 3)              # indices count modulo the number of rows
    q1, s1 = quant.fp8_quantize(x[rows.long()].contiguous())
    assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)
    q, s = quant.fp8_quantize(x, rows=rows[:0])
    assert q.shape == (0, 640) and s.shape == (0, 5)
    # no index, whatever its value, reads outside x
    wild = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1], device=DEV, dtype=torch.int32)
    q, s = quant.fp8_quantize(x, rows=wild)
    i = [(v % 2 ** 32) % 50 for v in (-1, -2 ** 31, 2 ** 31 - 1)]
    q1, s1 = quant.fp8_quantize(x[i].contiguous())
    assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(dtype):
    x = torch.randn(6, 384, device=DEV).to(dtype)
    x[0] = 0
    x[1, :128] = 0
    x[2, 5] = float("nan")
    x[3, 130] = float("inf")
    x[4] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).smallest_normal / 4
    q, s = quant.fp8_quantize(x)
    f = q.float()
    assert (f[0] == 0).all() and (f[1, :128] == 0).all() and torch.isfinite(s[:2]).all()
    assert f[2, :128].isnan().all() and s[2, 0].isnan() and torch.isfinite(f[2, 128:]).all()
    assert s[3, 1].isinf() and f[3, 130].isnan() and (f[3, 128:130] == 0).all() and torch.isfinite(f[3, :128]).all()
    assert (f[4] == 448).all()
    xb = blocks_of(x[5:].double().cpu().numpy())
    check(q[5:], s[5:], xb, np.abs(xb).max(-1))
    # blocks take the same care of them
    w = x.repeat(1, 1)
    q, s = quant.fp8_quantize_blocks(w[2:3])
    assert q.float()[0, :128].isnan().all() and s[0, 0].isnan() and torch.isfinite(q.float()[0, 128:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,f", [(1, 128), (5, 384), (131, 2048), (1201, 640), (1024, 768)])
def test_swiglu(dtype, m, f):
    gu = data((m, 2 * f), dtype, m + f).clamp_(-60, 60)
    gu = torch.cat([gu, gu[:, :8]], 1)[:, :2 * f]               # rows 2f + 8 apart
    q, s = quant.fp8_swiglu_quantize(gu)
    x = gu.double().cpu().numpy()
    h = x[:, :f] / (1 + np.exp(-x[:, :f])) * x[:, f:]
    hb = blocks_of(h)
    check(q, s, hb, np.abs(hb).max(-1), slack=2.0 ** -21)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,pad", [(640, 0), (640, 3), (384, 8), (128, 0), (1024, 0)])
def test_long_calls_are_short_ones(dtype, k, pad):
    """Long calls reduce four blocks together: the same bits as calls of a few rows, which take one block at a time.  With blocks that
    run over the ends of rows, a rest of one to three blocks, special values in single blocks, and (pad 3) rows at odd addresses."""
    m = 40003 if k == 128 else 8191
    x = data((m, k + pad), dtype, k)[:, pad:]
    x[5, 129 % k], x[77, k - 1], x[m - 1, 0] = float("nan"), float("inf"), float("nan")
    x[100:103] = 0
    rows = torch.randint(0, m, (m + 2,), device=DEV, dtype=torch.int32)
    pieces = list(range(0, m, 500))

    def bits(*calls):
        return torch.cat([q.view(torch.uint8) for q, _ in calls]), torch.cat([s.view(torch.int32) for _, s in calls])

    for got, want in ((bits(quant.fp8_quantize(x)), bits(*(quant.fp8_quantize(x[i:i + 500]) for i in pieces))),
                      (bits(quant.fp8_quantize(x, rows=rows)),
                       bits(*(quant.fp8_quantize(x, rows=rows[i:i + 500]) for i in range(0, m + 2, 500))))):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if k % 256 == 0:
        x = x.clamp(-60, 60)
        got, want = bits(quant.fp8_swiglu_quantize(x)), bits(*(quant.fp8_swiglu_quantize(x[i:i + 500]) for i in pieces))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("e,n,k", [(1, 1, 128), (1, 127, 256), (1, 128, 128), (3, 576, 384), (2, 200, 1024), (5, 130, 128)])
def test_blocks(dtype, turned, e, n, k):
    w = data((e, k, n) if turned else (e, n, k), dtype, n + k)
    if turned:
        w = w.transpose(1, 2)
    q, s = quant.fp8_quantize_blocks(w)
    assert q.shape == (e, n, k) and q.is_contiguous() and s.shape == (e, (n + 127) // 128, k // 128)
    x = w.double().cpu().numpy()
    for i in range(e):
        for b in range((n + 127) // 128):
            xb = blocks_of(x[i, 128 * b:128 * b + 128])                       # [rows, k/128, 128]
            a = np.abs(xb).max((0, 2))
            check(q[i, 128 * b:128 * b + 128], s[i, b][None].expand(xb.shape[0], -1), xb, np.broadcast_to(a, xb.shape[:2]))
    one = quant.fp8_quantize_blocks(w[0])
    assert torch.equal(one[0].view(torch.uint8), q[0].view(torch.uint8)) and torch.equal(one[1], s[0])


def test_blocks_of_views():
    """Rows further apart than they are long, odd starts, experts in another order."""
    big = torch.randn(4, 150, 700, device=DEV)
    for w in (big[1:3, 7:140, 3:3 + 512], big[::2, :130, :384], big.flip(0)[:, 2:4, :128],
              torch.randn(3, 256, 77, device=DEV).transpose(1, 2)[:, 3:70], big[:, :128, 9:300].transpose(1, 2)):
        q, s = quant.fp8_quantize_blocks(w)
        q1, s1 = quant.fp8_quantize_blocks(w.contiguous())
        assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)


def test_offsets_beyond_32_bits():
    """The last rows of a matrix of more than 2^32 bytes (and elements)."""
    m, k = 4_300_000, 1024
    x = torch.zeros(m, k, device=DEV, dtype=torch.float16)
    x[-3:] = torch.randn(3, k, device=DEV, dtype=torch.float16)
    q, s = quant.fp8_quantize(x)
    q1, s1 = quant.fp8_quantize(x[-3:])
    assert torch.equal(q[-3:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-3:], s1)
    assert not q[:-3].view(torch.uint8).any()


def test_on_another_stream_and_in_a_graph():
    x = torch.randn(64, 512, device=DEV)
    want = quant.fp8_quantize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = quant.fp8_quantize(x)
    side.synchronize()
    assert torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = quant.fp8_quantize(x)
        twice = quant.fp8_swiglu_quantize(x)
    x.mul_(-3)
    graph.replay()
    want = quant.fp8_quantize(x), quant.fp8_swiglu_quantize(x)
    for a, b in ((got, want[0]), (twice, want[1])):
        assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])


def test_operands_of_the_gemm():
    """Quantised operands through the GEMM: each factor is off by at most 2^-4 relative plus 2^-10 of its block's 448 steps."""
    m, n, k = 70, 192, 512
    x, w = torch.randn(m, k, device=DEV, dtype=torch.bfloat16), torch.randn(k, n, device=DEV, dtype=torch.float16) * k ** -0.5
    a, a_s = quant.fp8_quantize(x)
    b, b_s = quant.fp8_quantize_blocks(w.t())
    c = gemm.fp8_mm(a, b, a_s, b_s, torch.empty(m, n, device=DEV, dtype=torch.bfloat16))
    da = (blocks_of(a.float().double().cpu().numpy()) * a_s.double().cpu().numpy()[..., None]).reshape(m, k)
    sb = b_s.double().cpu().numpy().repeat(128, 0)[:n]
    db = (blocks_of(b.float().double().cpu().numpy()) * sb[..., None]).reshape(n, k)
    ref = da @ db.T
    # bf16 rounding 2^-8 of the value; the fp32 sum over k blocks and the tensor cores' sums inside one: 2^-12 of the terms
    assert (np.abs(c.double().cpu().numpy() - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -12 * (np.abs(da) @ np.abs(db).T)).all()


def test_without_the_extension_the_same_bits(monkeypatch):
    x = torch.randn(33, 640, device=DEV).bfloat16()
    rows = torch.tensor([3, 3, 32, 0], device=DEV, dtype=torch.int32)
    w = torch.randn(3, 256, 200, device=DEV).half().transpose(1, 2)
    calls = (lambda: quant.fp8_quantize(x), lambda: quant.fp8_quantize(x[:, 128:384], rows=rows), lambda: quant.fp8_quantize_blocks(w),
             lambda: quant.fp8_quantize_blocks(w[1]), lambda: quant.fp8_swiglu_quantize(x[:, :512]), lambda: quant.fp8_quantize(x[:0]))
    assert _lib.tensors() is not _lib._NoTensors
    native = [f() for f in calls]
    monkeypatch.setattr(_lib, "_tensors", _lib._NoTensors)
    for f, (q, s) in zip(calls, native):
        q1, s1 = f()
        assert q.dtype == q1.dtype and q.shape == q1.shape and s.shape == s1.shape and q.is_contiguous()
        assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)


@pytest.mark.parametrize("native", [True, False])
def test_refusals_on_the_gpu(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_lib, "_tensors", _lib._NoTensors)
    x = torch.zeros(4, 256, device=DEV)
    for bad, match in ((x[:, :100], "multiple of 128"), (x[0], "multiple of 128"), (x.t(), "multiple of 128"), (x.double(), "float16"),
                       (x.cpu(), "CUDA"), (torch.zeros(256, 256, device=DEV)[:, ::2], "contiguous")):
        with pytest.raises(ValueError, match=match):
            quant.fp8_quantize(bad)
    for rows in (torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int32), torch.zeros(6, device=DEV, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="rows"):
            quant.fp8_quantize(x, rows=rows)
    with pytest.raises(ValueError, match="no rows"):
        quant.fp8_quantize(x[:0], rows=torch.zeros(3, device=DEV, dtype=torch.int32))
    with pytest.raises(ValueError, match="multiple of 128"):
        quant.fp8_swiglu_quantize(x[:, :128])
    with pytest.raises(ValueError, match="contiguous"):
        quant.fp8_quantize_blocks(torch.zeros(2, 256, 512, device=DEV)[:, ::2, ::2])


def formula_bits(x, amax):
    """Blocks [..., 128] of fp32 values and their largest magnitudes, numpy -> bytes and scale by the formula in fp32."""
    a = np.maximum(amax, np.float32(2.0 ** -100)).astype(np.float32)
    v = x * (np.float32(448) / a)[..., None]
    return torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), a / np.float32(448)


def near_ties(n, seed):
    """n blocks of fp32 whose elements, times 448 / a, fall on the middle between two e4m3 values or a unit or two beside it."""
    rng = np.random.default_rng(seed)
    a = (rng.uniform(1, 2, n) * 2.0 ** rng.integers(-90, 90, n)).astype(np.float32)
    e4m3 = torch.arange(0x08, 0x7E, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()        # normal values to 448
    middle = (e4m3[1:] + e4m3[:-1]) / 2
    x = (middle[rng.integers(0, len(middle), (n, 128))] / (np.float32(448) / a)[:, None]).astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-2, 3, x.shape, dtype=np.int32)).view(np.float32) * rng.choice([-1, 1], x.shape).astype(np.float32)
    x[np.arange(n), rng.integers(0, 128, n)] = a
    return x


@pytest.mark.parametrize("m,k", [(60, 128), (700, 384), (9000, 1024)])
def test_ties_go_where_the_formula_sends_them(m, k):
    """q is e4m3(x * (448 / a)) with both operations rounded to nearest in fp32, to the bit: short calls, long ones, gathered ones."""
    x = near_ties(m * k // 128, m).reshape(m, k // 128, 128)
    want, scale = formula_bits(x, np.abs(x).max(-1))
    t = torch.from_numpy(x.reshape(m, k)).to(DEV)
    rows = torch.randperm(m, device=DEV, dtype=torch.int32)
    for (q, s), order in ((quant.fp8_quantize(t), slice(None)), (quant.fp8_quantize(t, rows=rows), rows.cpu().numpy())):
        assert np.array_equal(q.view(torch.uint8).cpu().numpy(), want.reshape(m, k)[order])
        assert np.array_equal(s.cpu().numpy(), scale[order])


@pytest.mark.parametrize("turned", [False, True])
def test_ties_of_blocks(turned):
    n, k = 300, 512
    x = near_ties(n * k // 128, 3).reshape(n, k // 128, 128) if not turned else near_ties(n * k // 128, 4).reshape(n, k // 128, 128)
    x /= np.abs(x).max(-1, keepdims=True)                       # one magnitude for the block: ties of its largest are a few
    want, scale = [], []
    for b in range(0, n, 128):
        p = x[b:b + 128]
        a = np.abs(p).max((0, 2))
        q, s = formula_bits(p, np.broadcast_to(a, p.shape[:2]))
        want.append(q.reshape(-1, k))
        scale.append(s[0])
    t = torch.from_numpy(x.reshape(n, k)).to(DEV)
    q, s = quant.fp8_quantize_blocks(t.t().contiguous().t() if turned else t)
    assert np.array_equal(q.view(torch.uint8).cpu().numpy(), np.concatenate(want)) and np.array_equal(s.cpu().numpy(), np.stack(scale))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_type_to_the_bit(dtype):
    for m, k in ((3, 128), (700, 1152), (3000, 2048)):
        x = data((m, k), dtype, m)
        xb = blocks_of(x.float().cpu().numpy())
        want, scale = formula_bits(xb, np.abs(xb).max(-1))
        q, s = quant.fp8_quantize(x)
        assert np.array_equal(q.view(torch.uint8).cpu().numpy(), want.reshape(m, k)) and np.array_equal(s.cpu().numpy(), scale)


# SwiGLU far below zero.  Its fp32 arithmetic, as quant.cu has it: 2^t within 2^-22, the reciprocal within 2^-23, four roundings of
# 2^-24 on the way to SiLU, one for the product with up: 11 * 2^-24 < 2^-20.  Below -87: twice an exponential of (g / 2) within 2
# ulp = 2^-22 each, three products, and 1 / (1 + exp(-g)) = exp(g) (1 - 2^-125): 2^-21 + 3 * 2^-24 < 2^-20.  The magnitude of a
# block, and so its scale, is off by as much; x * r by two more roundings.
SWIGLU = 2.0 ** -20


def check_swiglu(gu, q, s):
    f = gu.shape[1] // 2
    x = gu.double()
    h = blocks_of(x[:, :f] / (1 + torch.exp(-x[:, :f])) * x[:, f:])
    a = h.abs().amax(-1).clamp(min=2.0 ** -100)
    assert_within(s, a / 448, (2.0 ** -24 * 1.01 + SWIGLU) * a / 448)
    v = h * (448 / a)[..., None]
    assert_within(blocks_of(q.float()), v, 2.0 ** -4 * v.abs() * (1 + 2.0 ** -22 + 2 * SWIGLU) + 2.0 ** -10)


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e36), (torch.bfloat16, 1e36), (torch.float32, 1.0), (torch.bfloat16, 1.0),
                                        (torch.float16, 6e4)])
@pytest.mark.parametrize("lo,hi", [(-60, -30), (-86.9, -80), (-95, -85), (-104, -87), (80, 95), (-1e-3, 1e-3)])
@pytest.mark.parametrize("m", [4, 1500])
def test_swiglu_of_far_gates(dtype, size, lo, hi, m):
    f = 256
    g = torch.Generator(device=DEV).manual_seed(m)
    gate = lo + (hi - lo) * torch.rand(m, f, generator=g, device=DEV)
    up = torch.randn(m, f, generator=g, device=DEV) * (size / 6 if hi < 0 or size == 6e4 else 1.0)
    gu = torch.cat([gate, up], 1).to(dtype)
    check_swiglu(gu, *quant.fp8_swiglu_quantize(gu))


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_at_the_ends(dtype):
    """SiLU(-inf) is -inf * 0, the largest negative gate gives zero, +inf infinity."""
    top = torch.finfo(dtype).max
    gu = torch.ones(5, 256, device=DEV, dtype=dtype)
    gu[0, 3], gu[1, 3], gu[2, :128], gu[3, 3], gu[4, 3] = -float("inf"), float("inf"), -top, float("nan"), -top
    q, s = quant.fp8_swiglu_quantize(gu)
    assert s[0, 0].isnan() and s[1, 0].isinf() and s[3, 0].isnan()
    assert (q[2].float() == 0).all() and s[2, 0] == 2.0 ** -100 / 448
    one = 1 / (1 + np.exp(-1.0))
    assert q[4, 3].float() == 0 and (q[4, 4:].float() == 448).all() and abs(float(s[4, 0]) * 448 / one - 1) < SWIGLU


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_gates_in_long_calls_are_those_of_short_ones(dtype):
    """A thread takes the long way for all of its gates when one needs it: what it does beside that is the same arithmetic."""
    m, f = 8191, 640
    gu = torch.randn(m, 2 * f, device=DEV).mul_(40).clamp_(-104, 104).to(dtype)
    q, s = quant.fp8_swiglu_quantize(gu)
    for i in (0, 500, 4000, m - 300):
        q1, s1 = quant.fp8_swiglu_quantize(gu[i:i + 300])
        assert torch.equal(q[i:i + 300].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[i:i + 300], s1)
    check_swiglu(gu, q, s)
