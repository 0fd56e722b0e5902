"""Performance cases of the operators around FP8 experts and of the layer for a few tokens.

Kinds of case:
  quantize   `quant.fp8_quantize`: rows to e4m3 with one scale per 1 x 128 block, optionally gathered on the way
  blocks     `quant.fp8_quantize_blocks`: weights to e4m3 with one scale per 128 x 128 block, from either memory order
  swiglu     `quant.fp8_swiglu_quantize`: SiLU(gate) * up of one matrix [gate | up], quantised like `quantize`
  grouped    `grouped.fp8_grouped_mm`: the block-scaled FP8 product, each group of rows by weights of its own
  few        `moe_few.FewTokenMoE`: a whole MoE layer for a few tokens, experts in fp16 or in block-scaled FP8

With `own` false every operator runs in its plain form: elementary torch operations in 32 bits, rounded once at the end.
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BLOCK = 128
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "fp8": 1}


def listed():
    return [
        # The activations of a decode batch in front of an FP8 projection: a few kilobytes, latency only.
        {"name": "quantize_24x7168_fp16", "kind": "quantize", "m": 24, "k": 7168, "dtype": "fp16", "rows": 0},
        # Prefill through top-4 experts: 8192 tokens gathered in expert order and quantised in the same pass.
        {"name": "quantize_gather_32768x7168_bf16", "kind": "quantize", "m": 8192, "k": 7168, "dtype": "bf16", "rows": 32768},
        # One projection's weights at load time, with a last block of half a block's rows.
        {"name": "blocks_576x7168_fp32", "kind": "blocks", "e": 1, "n": 576, "k": 7168, "dtype": "fp32", "t": False},
        # A layer's fp16 down projections, [in, out] as the MoE layer holds them, turned into FP8 operands.
        {"name": "blocks_t_32x7168x2048_fp16", "kind": "blocks", "e": 32, "n": 7168, "k": 2048, "dtype": "fp16", "t": True},
        # Between the experts' two products in a small decode batch, an odd number of rows.
        {"name": "swiglu_37x2048_bf16", "kind": "swiglu", "m": 37, "f": 2048, "dtype": "bf16"},
        # The same in prefill.
        {"name": "swiglu_32768x2048_fp16", "kind": "swiglu", "m": 32768, "f": 2048, "dtype": "fp16"},
        # Decode of 128 sequences, top-4 of 32 experts: the weight stream, a dozen rows per expert.
        {"name": "grouped_512_32x7168x2048", "kind": "grouped", "m": 512, "e": 32, "n": 7168, "k": 2048, "skew": 0.0,
         "tail": 0, "out": "fp16"},
        # A short prefill on a small model with popular and unused experts, rows behind the last group, odd widths.
        {"name": "grouped_1777_64x1472x1024_skew", "kind": "grouped", "m": 1777, "e": 64, "n": 1472, "k": 1024, "skew": 1.0,
         "tail": 23, "out": "bf16"},
        # Gate and up projections of 8192 tokens through top-4 of 32 experts.
        {"name": "grouped_32768_32x4096x7168", "kind": "grouped", "m": 32768, "e": 32, "n": 4096, "k": 7168, "skew": 0.0,
         "tail": 0, "out": "bf16"},
        # One token through a small model: nothing but latency.
        {"name": "few_1_1024x512_e64k8_fp16", "kind": "few", "t": 1, "d": 1024, "f": 512, "e": 64, "k": 8, "w": "fp16"},
        # One sequence in decode, the benchmark layer's experts in fp16.
        {"name": "few_1_7168x2048_e32k4_fp16", "kind": "few", "t": 1, "d": 7168, "f": 2048, "e": 32, "k": 4, "w": "fp16"},
        # A dozen sequences in decode, 256 experts in FP8.
        {"name": "few_13_7168x2048_e256k8_fp8", "kind": "few", "t": 13, "d": 7168, "f": 2048, "e": 256, "k": 8, "w": "fp8"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 32768 rows of 128 to 7168 columns, weights of 1 to 64 experts, layers of 1 to 32 tokens."""
    kind = rng.choice(["quantize", "blocks", "swiglu", "grouped", "grouped", "few", "few"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    if kind == "quantize":
        m, k = _log_int(rng, 1, 8192), BLOCK * _log_int(rng, 1, 56)
        return {"kind": kind, "m": m, "k": k, "dtype": dtype, "rows": rng.choice([0, 0, m * rng.choice([1, 2, 4])])}
    if kind == "blocks":
        return {"kind": kind, "e": _log_int(rng, 1, 16), "n": _log_int(rng, 1, 7168), "k": BLOCK * _log_int(rng, 1, 16),
                "dtype": dtype, "t": rng.random() < 0.5}
    if kind == "swiglu":
        return {"kind": kind, "m": _log_int(rng, 1, 16384), "f": BLOCK * _log_int(rng, 1, 16), "dtype": dtype}
    if kind == "grouped":
        m = _log_int(rng, 1, 8192)
        return {"kind": kind, "m": m, "e": rng.choice([1, 3, 8, 32, 64]), "n": 64 * _log_int(rng, 1, 64),
                "k": BLOCK * _log_int(rng, 1, 16), "skew": rng.choice([0.0, 0.5, 1.0]), "tail": rng.choice([0, 0, 1, 77]),
                "out": rng.choice(["bf16", "fp16"])}
    d, f = rng.choice([(7168, 2048), (4096, 1536), (1024, 512), (1280, 384)])
    e = rng.choice([4, 8, 32, 64]) if d == 7168 else rng.choice([4, 8, 32, 64, 128, 256])
    return {"kind": kind, "t": _log_int(rng, 1, 12 if d == 7168 else 32), "d": d, "f": f, "e": e,
            "k": rng.choice([2, 4, 8]) if e >= 8 else rng.choice([2, 4]), "w": rng.choice(["fp16", "fp8"])}


# ------------------------------------------------------------------------------------------------ inputs --
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _activations(m, k, dtype, g):
    """Rows of unit variance with a magnitude of their own, a few channels far larger than the others, as hidden states are."""
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=g, device=DEV))
    x *= 1.0 + 20.0 * (torch.rand(1, k, generator=g, device=DEV) < 0.002)
    return x.to(DTYPES[dtype])


def _fp8_operand(e, n, k, fan, g):
    """Weights N(0, 1/fan) in e4m3 with 128 x 128 scales: q [e, n, k], scale [e, ceil(n/128), k/128]; expert by expert, as a
    checkpoint is loaded."""
    kb, nb = k // BLOCK, -(-n // BLOCK)
    q = torch.empty(e, n, k, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(e, nb, kb, device=DEV)
    for i in range(e):
        w = torch.zeros(nb * BLOCK, k, device=DEV)
        w[:n] = torch.randn(n, k, generator=g, device=DEV) * fan ** -0.5
        w = w.view(nb, BLOCK, kb, BLOCK)
        scale[i] = w.abs().amax((1, 3)) / E4M3_MAX
        q[i] = (w / scale[i][:, None, :, None]).view(nb * BLOCK, k)[:n].to(torch.float8_e4m3fn)
    return q, scale


def _prepare_grouped(case, seed, g):
    m, e, n, k = (case[q] for q in "menk")
    kb = k // BLOCK
    rng = np.random.default_rng(seed)
    p = (1.0 + np.arange(e)) ** -case["skew"]
    counts = rng.multinomial(m, rng.permutation(p / p.sum()))
    x = torch.randn(m + case["tail"], kb, BLOCK, generator=g, device=DEV)
    a_scale = x.abs().amax(-1) / E4M3_MAX
    a = (x / a_scale[..., None]).view(-1, k).to(torch.float8_e4m3fn)
    b, b_scale = _fp8_operand(e, n, k, k, g)
    c = torch.randn(m + case["tail"], n, generator=g, device=DEV).to(DTYPES[case["out"]])
    offsets = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).to(DEV)
    return {"a": a, "b": b, "a_scale": a_scale, "b_scale": b_scale, "offsets": offsets, "c": c, "total": m,
            "largest": int(counts.max())}


def _prepare_few(case, g):
    t, d, f, e = (case[q] for q in "tdfe")

    def randn(*shape, fan):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16).mul_(fan ** -0.5)

    config = {"d_hidden": d, "d_expert": f, "n_routed_experts": e, "n_shared_experts": 1, "n_experts_per_token": case["k"],
              "batch_size": t, "seq_len": 1}
    s = {"x": torch.randn(t, 1, d, generator=g, device=DEV, dtype=torch.float16), "config": config,
         "router": randn(e, d, fan=d)}
    if case["w"] == "fp16":
        # the shared expert is the last of each stack; the layer's dict holds views of the stacks
        s["gate"], s["up"], s["down"] = randn(e + 1, d, f, fan=f), randn(e + 1, d, f, fan=f), randn(e + 1, f, d, fan=d)
        w = {"router.weight": s["router"]}
        for i in range(e + 1):
            prefix = f"experts.{i}" if i < e else "shared_experts"
            w.update({f"{prefix}.0.weight": s["gate"][i], f"{prefix}.1.weight": s["up"][i], f"{prefix}.2.weight": s["down"][i]})
    else:
        s["gate_up"], s["gate_up_scale"] = _fp8_operand(e + 1, 2 * f, d, f, g)
        s["down"], s["down_scale"] = _fp8_operand(e + 1, d, f, d, g)
        w = {"router.weight": s["router"],
             "experts.gate_up.weight": s["gate_up"][:e], "experts.gate_up.scale": s["gate_up_scale"][:e],
             "experts.down.weight": s["down"][:e], "experts.down.scale": s["down_scale"][:e],
             "shared_experts.gate_up.weight": s["gate_up"][e], "shared_experts.gate_up.scale": s["gate_up_scale"][e],
             "shared_experts.down.weight": s["down"][e], "shared_experts.down.scale": s["down_scale"][e]}
    if own:
        from radeonflow_kernels_b200 import moe_few
        s["layer"] = moe_few.FewTokenMoE(w, config)       # the handle that a serving program keeps per layer
    return s


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "quantize":
        s = {"x": _activations(case["m"], case["k"], case["dtype"], g), "rows": None}
        if case["rows"]:
            s["rows"] = torch.randint(0, case["m"], (case["rows"],), generator=g, device=DEV, dtype=torch.int32)
    elif kind == "blocks":
        e, n, k = case["e"], case["n"], case["k"]
        w = torch.randn(e, *((k, n) if case["t"] else (n, k)), generator=g, device=DEV, dtype=DTYPES[case["dtype"]])
        s = {"w": (w * k ** -0.5).transpose(1, 2) if case["t"] else w * k ** -0.5}
    elif kind == "swiglu":
        s = {"gate_up": torch.randn(case["m"], 2 * case["f"], generator=g, device=DEV).mul_(1.5).to(DTYPES[case["dtype"]])}
    elif kind == "grouped":
        s = _prepare_grouped(case, seed, g)
    else:
        s = _prepare_few(case, g)
    return dict(s, kind=kind, w8=case.get("w") == "fp8")


# ------------------------------------------------------------------------------------------- plain forms --
def _quantize(x):
    """x [m, k] fp32 -> (e4m3 [m, k], scale [m, k/128])."""
    x = x.view(x.shape[0], -1, BLOCK)
    amax = x.abs().amax(-1, keepdim=True).clamp(min=AMAX_FLOOR)
    return (x * (E4M3_MAX / amax)).view(x.shape[0], -1).to(torch.float8_e4m3fn), (amax / E4M3_MAX).squeeze(-1)


def _quantize_blocks(w):
    e, n, k = w.shape
    nb = -(-n // BLOCK)
    x = torch.zeros(e, nb * BLOCK, k, device=w.device)
    x[:, :n] = w.float()
    x = x.view(e, nb, BLOCK, k // BLOCK, BLOCK)
    amax = x.abs().amax((2, 4), keepdim=True).clamp(min=AMAX_FLOOR)
    q = (x * (E4M3_MAX / amax)).view(e, nb * BLOCK, k)[:, :n].to(torch.float8_e4m3fn)
    return q.contiguous(), (amax / E4M3_MAX).view(e, nb, k // BLOCK)


def _swiglu_quantize(gate_up):
    gate, up = gate_up.float().chunk(2, 1)
    return _quantize(gate / (1.0 + torch.exp(-gate)) * up)


def _dequantize(q, scale):
    """e4m3 [e, n, k] with 128 x 128 scales -> fp32."""
    e, n, k = q.shape
    s = scale.repeat_interleave(BLOCK, 1)[:, :n]
    return (q.float().view(e, n, -1, BLOCK) * s[..., None]).view(e, n, k)


def _grouped(s):
    k, starts, counts = s["a"].shape[1], s["offsets"][:-1], s["offsets"][1:] - s["offsets"][:-1]
    x = (s["a"].float().view(-1, k // BLOCK, BLOCK) * s["a_scale"][..., None]).view(-1, k)
    slots = torch.arange(s["largest"], device=x.device)
    slots = torch.minimum(slots, (counts[:, None] - 1).clamp(min=0))
    y = torch.bmm(x[(starts[:, None] + slots).clamp(max=x.shape[0] - 1)], _dequantize(s["b"], s["b_scale"]).transpose(1, 2))
    rows = torch.arange(s["total"], device=x.device)
    group = (rows[:, None] >= s["offsets"][1:]).sum(1)
    s["c"][:s["total"]] = y[group, rows - starts[group]].to(s["c"].dtype)
    return s["c"]


def _few(s):
    x, e, top = s["x"].flatten(0, 1).float(), s["router"].shape[0], s["config"]["n_experts_per_token"]
    logits = (x @ s["router"].float().t()).half().float()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = (p / p.sum(1, keepdim=True)).half()
    p, idx = torch.sort(p, dim=1, descending=True, stable=True)
    w = torch.nn.functional.pad(p[:, :top].float(), (0, 1), value=1.0)             # the shared expert's weight is one
    idx = torch.nn.functional.pad(idx[:, :top], (0, 1), value=e)
    pairs, xs = idx.flatten(), x.repeat_interleave(top + 1, 0)[:, None]
    if s["w8"]:
        gate, up = torch.bmm(xs, _dequantize(s["gate_up"][pairs], s["gate_up_scale"][pairs]).transpose(1, 2)).chunk(2, 2)
    else:
        gate, up = torch.bmm(xs, s["gate"][pairs].float()), torch.bmm(xs, s["up"][pairs].float())
    h = gate / (1.0 + torch.exp(-gate)) * up
    if s["w8"]:
        y = torch.bmm(h, _dequantize(s["down"][pairs], s["down_scale"][pairs]).transpose(1, 2))
    else:
        y = torch.bmm(h, s["down"][pairs].float())
    return (w[..., None] * y.view(x.shape[0], top + 1, -1)).sum(1).half().view(s["x"].shape)


# ------------------------------------------------------------------------------------------------ one pass --
@functools.lru_cache(maxsize=1)
def _framework():
    from radeonflow_kernels_b200 import grouped, quant
    return grouped, quant


def run(state):
    kind = state["kind"]
    if own:
        grouped, quant = _framework()
        if kind == "quantize":
            return quant.fp8_quantize(state["x"], rows=state["rows"])
        if kind == "blocks":
            return quant.fp8_quantize_blocks(state["w"])
        if kind == "swiglu":
            return quant.fp8_swiglu_quantize(state["gate_up"])
        if kind == "grouped":
            return grouped.fp8_grouped_mm(state["a"], state["b"], state["a_scale"], state["b_scale"], state["offsets"],
                                          state["c"])
        return state["layer"].forward(state["x"])
    if kind == "quantize":
        x = state["x"] if state["rows"] is None else state["x"][state["rows"].long()]
        return _quantize(x.float())
    if kind == "blocks":
        return _quantize_blocks(state["w"])
    if kind == "swiglu":
        return _swiglu_quantize(state["gate_up"])
    return _grouped(state) if kind == "grouped" else _few(state)


def work(case):
    kind = case["kind"]
    if kind == "quantize":
        m, k, rows = case["m"], case["k"], case["rows"] or case["m"]
        # (a gather reads each row that it takes once)
        return {"bytes": min(m, rows) * k * BYTES[case["dtype"]] + rows * (k + 4 * k // BLOCK) + 4 * case["rows"],
                "flops": 3.0 * rows * k}
    if kind == "blocks":
        e, n, k = case["e"], case["n"], case["k"]
        return {"bytes": e * (n * k * (BYTES[case["dtype"]] + 1) + 4 * -(-n // BLOCK) * (k // BLOCK)), "flops": 3.0 * e * n * k}
    if kind == "swiglu":
        m, f = case["m"], case["f"]
        return {"bytes": m * (2 * f * BYTES[case["dtype"]] + f + 4 * f // BLOCK), "flops": 8.0 * m * f}
    if kind == "grouped":
        m, e, n, k = (case[q] for q in "menk")
        kb, hit = k // BLOCK, min(e, m)
        return {"bytes": m * (k + 4 * kb) + hit * (n * k + 4 * -(-n // BLOCK) * kb) + 2 * m * n + 4 * (e + 1),
                "flops": 2.0 * m * n * k}
    t, d, f, e, k = (case[q] for q in "tdfek")
    hit = e * (1.0 - (1.0 - k / e) ** t) + 1            # experts hit by t tokens that choose evenly, and the shared one
    return {"bytes": 3.0 * d * f * BYTES[case["w"]] * hit + 2 * e * d + 4 * t * d, "flops": 2.0 * t * (3 * d * f * (k + 1) + e * d)}


# ----------------------------------------------------------------------------------------------- in 64 bits --
def exact(case, seed):
    """What `run` gives, computed in fp64 row block by row block and expert by expert."""
    s = prepare(case, seed)
    kind = case["kind"]

    def blocks(v):            # the last axis in pieces of 128
        return v.unflatten(-1, (-1, BLOCK))

    def with_scale(v, floor=AMAX_FLOOR):
        top = torch.linalg.vector_norm(blocks(v), ord=math.inf, dim=-1).clamp_(min=floor)
        return (blocks(v) / (top / E4M3_MAX)[..., None]).flatten(-2), top / E4M3_MAX

    if kind == "quantize":
        x = s["x"].double()
        return with_scale(x if s["rows"] is None else torch.index_select(x, 0, s["rows"]))
    if kind == "swiglu":
        f = case["f"]
        v = s["gate_up"].double()
        return with_scale(torch.sigmoid(v[:, :f]) * v[:, :f] * v[:, f:])
    if kind == "blocks":
        qs, scales = [], []
        for w in s["w"]:
            w = w.double()
            tops = torch.stack([torch.linalg.vector_norm(blocks(p), ord=math.inf, dim=(0, 2)) for p in w.split(BLOCK)])
            tops.clamp_(min=AMAX_FLOOR)
            qs.append(torch.cat([(blocks(p) * (E4M3_MAX / top)[None, :, None]).flatten(1) for p, top in zip(w.split(BLOCK), tops)]))
            scales.append(tops / E4M3_MAX)
        return torch.stack(qs), torch.stack(scales)

    def weight(q, scale):      # one expert's [n, k]
        n = q.shape[0]
        return (blocks(q.double()) * scale.double()[torch.arange(n, device=DEV) // BLOCK][..., None]).flatten(1)

    if kind == "grouped":
        if 2.0 * case["m"] * case["n"] * case["k"] > 3e14:
            return None
        out = s["c"].double()
        a = (blocks(s["a"].double()) * s["a_scale"].double()[..., None]).flatten(1)
        bounds = s["offsets"].tolist()
        for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            if hi > lo:
                out[lo:hi] = a[lo:hi] @ weight(s["b"][i], s["b_scale"][i]).t()
        return out

    d, f, e, top = case["d"], case["f"], case["e"], case["k"]
    x = s["x"].view(-1, d).double()
    # the layer chooses by probabilities rounded to fp16, of logits rounded to fp16; equal ones by the lowest index
    prob = torch.softmax((x @ s["router"].double().t()).half().double(), 1).half().double()
    out = torch.zeros(x.shape[0], d, dtype=torch.float64, device=DEV)
    share = torch.zeros(x.shape[0], e + 1, dtype=torch.float64, device=DEV)
    share[:, e] = 1.0
    for row, p in enumerate(prob.tolist()):
        for i in sorted(range(e), key=lambda j: (-p[j], j))[:top]:
            share[row, i] = p[i]
    for i in range(e + 1):
        if i < e and not bool(share[:, i].any()):
            continue
        if case["w"] == "fp8":
            gate, up = (x @ weight(s["gate_up"][i], s["gate_up_scale"][i]).t()).split(f, 1)
            down = weight(s["down"][i], s["down_scale"][i]).t()
        else:
            gate, up, down = x @ s["gate"][i].double(), x @ s["up"][i].double(), s["down"][i].double()
        out += share[:, i:i + 1] * ((torch.sigmoid(gate) * gate * up) @ down)
    return out.view(s["x"].shape)
