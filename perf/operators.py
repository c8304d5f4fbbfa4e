"""The sequence operators of annc_b200, as cases that can be timed and compared: what a ranking model runs
that scores candidates against a user's history, beside the embedding bags and the fp32 / BF16 layers.

A case is a dict of plain values; `kind` names the operator and the rest its sizes:

  gemm_i8   device.gemm_i8: product of 8-bit integers with a scale per token and per output channel, bias and
            activation in the epilogue
  linear_i8 device.quantize_rows + device.gemm_i8: a layer on floating-point activations, quantised per token
  rotary    device.Rotary.run: rotary positions on the queries and keys of a batch of tokens
  attention device.PrefixAttention.run: tokens that share one long prefix of keys and values, each sequence with
            a few keys of its own behind it

`own` false computes them from elementary torch operations, true by the framework.  Inputs are drawn on the GPU
from the seed alone; the lengths of ragged batches follow from the case.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_ACT = {"none": 0, "relu": 1, "sigmoid": 2}  # annc_b200.ACT_*
_T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one sample through the widest layer of the large recsys model: latency, the weight is all there is to read
        dict(name="i8_m1", kind="gemm_i8", m=1, n=1024, k=8192, out="f32", bias=True, act="relu"),
        # a serving batch through a square-ish layer (the prepacked-weight layer of the benchmark)
        dict(name="i8_m200", kind="gemm_i8", m=200, n=4096, k=2048, out="f32", bias=True, act="none"),
        # extents that are multiples of nothing, sigmoid scores
        dict(name="i8_odd", kind="gemm_i8", m=1999, n=1003, k=1001, out="bf16", bias=True, act="sigmoid"),
        # the wide layer at the recsys batch
        dict(name="i8_m16384", kind="gemm_i8", m=16384, n=1024, k=8192, out="bf16", bias=True, act="relu"),
        # the layer a compiled graph calls, on a small serving batch of fp32 activations
        dict(name="linear_m16", kind="linear_i8", m=16, n=1024, k=1024, x="f32", out="f32", bias=True, act="relu"),
        # a throughput batch of bf16 activations
        dict(name="linear_m8192", kind="linear_i8", m=8192, n=4096, k=2048, x="bf16", out="bf16", bias=False,
             act="none"),
        # the new tokens of one decoding step
        dict(name="rotary_t16", kind="rotary", tokens=16, heads=16, kv_heads=4, dim=128, rot=128, dtype="bf16",
             layout="half", scaling="none", far=4000),
        # a history that is read in: half of every head turned, positions beyond what the model was trained on
        dict(name="rotary_t8191", kind="rotary", tokens=8191, heads=32, kv_heads=8, dim=128, rot=64, dtype="bf16",
             layout="interleaved", scaling="yarn", far=131072),
        # one candidate against a short history
        dict(name="attn_b1", kind="attention", seqs=1, max_q=1, heads=8, kv_heads=8, dim=64, prefix=1000, max_own=4,
             dtype="bf16", lse=False),
        # a decoding step of a batch behind a long prompt: keys and values are what there is to read
        dict(name="attn_b64", kind="attention", seqs=64, max_q=1, heads=32, kv_heads=8, dim=128, prefix=32768,
             max_own=200, dtype="bf16", lse=False),
        # candidates of one to eight tokens each
        dict(name="attn_ragged", kind="attention", seqs=500, max_q=8, heads=8, kv_heads=8, dim=64, prefix=2047,
             max_own=16, dtype="f16", lse=True),
        # a throughput batch of candidates against a long history
        dict(name="attn_b2048", kind="attention", seqs=2048, max_q=1, heads=16, kv_heads=2, dim=128, prefix=8192,
             max_own=33, dtype="bf16", lse=False),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["gemm_i8", "gemm_i8", "linear_i8", "linear_i8", "rotary", "attention", "attention", "attention"])
    if kind in ("gemm_i8", "linear_i8"):
        n, k = _log(rng, 16, 8192), _log(rng, 16, 8192)
        if rng.random() < 0.7:  # layer widths are multiples of 16, batches are not
            n, k = (n + 15) // 16 * 16, (k + 15) // 16 * 16
        m = _log(rng, 1, max(1, min(16384, 130_000_000_000 // (n * k), 45_000_000 // (n + k))))
        c = dict(kind=kind, m=m, n=n, k=k, out=rng.choice(["f32", "bf16", "f16"]), bias=rng.random() < 0.7,
                 act=rng.choice(["none", "relu", "sigmoid"]))
        if kind == "linear_i8":
            c["x"] = rng.choice(["f32", "bf16", "f16"])
        return c
    if kind == "rotary":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 8])
        return dict(kind=kind, tokens=_log(rng, 1, max(1, min(65536, 20_000_000 // (dim * (heads + kv))))), heads=heads,
                    kv_heads=kv, dim=dim, rot=rng.choice([dim, dim, dim // 2]), dtype=rng.choice(["f32", "bf16", "f16"]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    far=_log(rng, 100, 1_000_000))
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8])
    max_q = rng.choice([1, 1, 1, rng.randint(2, 16)])
    prefix = _log(rng, 1, 32768)
    # score elements, and the own keys that the plain form spreads out, within the listed cases' reach
    rows = min(8192, 240_000_000 // (heads * prefix))
    max_own = rng.choice([0, _log(rng, 1, 256)])
    rows = min(rows, 120_000_000 // (max(1, max_own) * kv * dim))
    return dict(kind=kind, seqs=_log(rng, 1, max(1, 2 * rows // (max_q + 1))), max_q=max_q, heads=heads, kv_heads=kv,
                dim=dim, prefix=prefix, max_own=max_own, dtype=rng.choice(["bf16", "f16"]), lse=rng.random() < 0.3)


# ---------------------------------------------------------------- inputs

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def _pitched_i8(rows: int, cols: int):
    """int8 [rows, cols] whose rows start on 16 bytes, as a program lays weights and activations out."""
    return torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :cols]


def _random_i8(g, rows: int, cols: int):
    out = _pitched_i8(rows, cols)
    out.copy_((torch.randn((rows, cols), device="cuda", generator=g) * 36).round_().clamp_(-127, 127))
    return out


def _lengths(case):
    """Tokens and own keys of every sequence: from one token to max_q, from no key to max_own, at least the
    sequence's own tokens where it has keys at all."""
    i = np.arange(case["seqs"], dtype=np.int64)
    nq = 1 + (i * 13 + 5) % case["max_q"]
    if case["max_own"] == 0:
        return nq, np.zeros_like(nq)
    return nq, np.maximum((i * 37 + 11) % (case["max_own"] + 1), nq if case["max_q"] > 1 else 0)


def _linear_state(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    s = dict(w=_random_i8(g, n, k), w_scale=torch.rand(n, device="cuda", generator=g) * 1e-3 + 2e-4,
             bias=_normal(g, n, scale=0.1) if case["bias"] else None,
             c=torch.empty((m, n), dtype=_T[case["out"]], device="cuda"))
    if case["kind"] == "gemm_i8":
        s.update(a=_random_i8(g, m, k), a_scale=torch.rand(m, device="cuda", generator=g) * 0.03 + 0.01)
    else:
        # activations behind a layer: tokens of different size
        x = _normal(g, m, k) * (torch.rand((m, 1), device="cuda", generator=g) * 2 + 0.1)
        s.update(x=x.to(_T[case["x"]]), a=_pitched_i8(m, k), a_scale=torch.empty(m, device="cuda"))
    return s


def _rotary_state(case, g):
    t, dt = case["tokens"], _T[case["dtype"]]
    q = _normal(g, t, case["heads"], case["dim"], dtype=dt)
    k = _normal(g, t, case["kv_heads"], case["dim"], dtype=dt)
    pos = torch.randint(0, case["far"], (t,), device="cuda", generator=g)
    return dict(q=q, k=k, pos=pos, out_q=torch.empty_like(q), out_k=torch.empty_like(k))


def _attention_state(case, g):
    nq, no = _lengths(case)
    dt, kv, dim = _T[case["dtype"]], case["kv_heads"], case["dim"]
    tokens, rows = int(nq.sum()), int(no.sum())
    up = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)
    return dict(q=_normal(g, tokens, case["heads"], dim, dtype=dt), kp=_normal(g, case["prefix"], kv, dim, dtype=dt),
                vp=_normal(g, case["prefix"], kv, dim, dtype=dt),
                ko=_normal(g, max(rows, 1), kv, dim, dtype=dt), vo=_normal(g, max(rows, 1), kv, dim, dtype=dt),
                own_begin=up(np.cumsum(no) - no, torch.int64), own_len=up(no, torch.int32),
                q_begin=up(np.concatenate([[0], np.cumsum(nq)]), torch.int32),
                out=torch.empty((tokens, case["heads"], dim), dtype=dt, device="cuda"),
                lse=torch.empty((tokens, case["heads"]), device="cuda") if case["lse"] else None)


_ROTARY = dict(base=10000.0, factor=8.0, original=4096)


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = (_linear_state if kind in ("gemm_i8", "linear_i8") else _rotary_state if kind == "rotary" else _attention_state)(case, g)
    s["case"] = case
    if own:  # the plans that a user's program makes once
        from annc_b200 import device as dev
        if kind == "rotary":
            s["plan"] = dev.Rotary(case["rot"], base=_ROTARY["base"], layout=case["layout"], scaling=case["scaling"],
                                   factor=_ROTARY["factor"], original_len=_ROTARY["original"])
        elif kind == "attention":
            s["plan"] = dev.PrefixAttention(case["heads"], case["kv_heads"], case["dim"], s["q"].shape[0],
                                            dtype=s["q"].dtype)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    kind = c["kind"]
    if own:
        return _own(s, c, kind)
    if kind == "gemm_i8":
        return _plain_product(s, c, s["a"], s["a_scale"])
    if kind == "linear_i8":
        # the quotients are taken in 64 bits: the scale is the nearest one in 32, values lie next to borders of steps
        x = s["x"].double()
        scale = (x.abs().amax(1) / 127.0).clamp_min(2.0 ** -126).float()
        q = torch.round(x / scale.double()[:, None]).clamp_(-127, 127)
        return [_plain_product(s, c, q, scale), scale]
    if kind == "rotary":
        return _plain_rotary(s, c)
    return _plain_attention(s, c)


def _own(s, c, kind):
    from annc_b200 import device as dev
    if kind in ("gemm_i8", "linear_i8"):
        if kind == "linear_i8":
            dev.quantize_rows(s["x"], s["a"], s["a_scale"])
        dev.gemm_i8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["c"], bias=s["bias"], activation=_ACT[c["act"]])
        return s["c"] if kind == "gemm_i8" else [s["c"], s["a_scale"]]
    if kind == "rotary":
        s["plan"].run(s["pos"], s["q"], s["out_q"], s["k"], s["out_k"])
        return [s["out_q"], s["out_k"]]
    s["plan"].run(s["q"], s["kp"], s["vp"], s["out"], k_own=s["ko"], v_own=s["vo"], own_begin=s["own_begin"],
                  own_len=s["own_len"], q_begin=s["q_begin"] if c["max_q"] > 1 else None, lse=s["lse"])
    return [s["out"], s["lse"]] if c["lse"] else s["out"]


def _plain_product(s, c, a, a_scale):
    y = torch.matmul(a.float(), s["w"].float().t()) * a_scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "relu":
        y = y.clamp_min(0)
    elif c["act"] == "sigmoid":
        y = 1 / (1 + torch.exp(-y))
    return y.to(s["c"].dtype)


def _plain_frequencies(c):
    """Angle per position of every pair, and what queries and keys are scaled by."""
    rot, base, f, orig = c["rot"], _ROTARY["base"], _ROTARY["factor"], _ROTARY["original"]
    if c["scaling"] == "ntk" and rot > 2:
        base = base * f ** (rot / (rot - 2))
    inv = base ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    if c["scaling"] == "linear":
        return inv / f, 1.0
    if c["scaling"] != "yarn":
        return inv, 1.0
    # pairs that turn often within the trained length keep their speed, slow ones are stretched, a ramp between
    turns = lambda n: rot * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(turns(32.0)), 0), min(math.ceil(turns(1.0)), rot - 1)
    ramp = ((torch.arange(rot // 2, device="cuda", dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
    return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0


def _plain_rotary(s, c):
    inv, size = _plain_frequencies(c)
    angle = s["pos"].double()[:, None] * inv  # 64 bits: far positions
    cos, sin = (torch.cos(angle) * size).float()[:, None], (torch.sin(angle) * size).float()[:, None]
    rot, both = c["rot"], []
    for x in (s["q"], s["k"]):
        y = x.float()
        if c["layout"] == "half":
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        both.append(torch.cat([turned, y[..., rot:]], -1).to(x.dtype))
    return both


def _plain_attention(s, c):
    kv, dim = c["kv_heads"], c["dim"]
    q = s["q"].float()
    tokens, group = q.shape[0], c["heads"] // kv
    q = q.view(tokens, kv, group, dim).permute(1, 0, 2, 3).reshape(kv, tokens * group, dim) * dim ** -0.5
    scores = torch.matmul(q, s["kp"].float().permute(1, 2, 0))
    if c["max_own"]:
        # own keys, spread out to one list a token; token i of n sees all but the last n - 1 - i of its sequence
        t = torch.arange(tokens, device="cuda")
        seq = torch.searchsorted(s["q_begin"].long(), t, right=True) - 1
        seen = s["own_len"][seq] - (s["q_begin"][seq + 1] - 1 - t)
        j = torch.arange(max(c["max_own"], c["max_q"]), device="cuda")
        there = j < seen[:, None]
        at = torch.where(there, s["own_begin"][seq][:, None] + j, 0)
        ko, vo = s["ko"].float()[at], s["vo"].float()[at]  # [tokens, keys, kv, dim]
        own_scores = torch.einsum("htgd,tjhd->htgj", q.view(kv, tokens, group, dim), ko)
        own_scores = own_scores.masked_fill(~there[None, :, None], -math.inf).reshape(kv, tokens * group, -1)
        top = torch.maximum(scores.amax(-1), own_scores.amax(-1))[..., None]
    else:
        top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    total = p.sum(-1)
    out = torch.matmul(p, s["vp"].float().permute(1, 0, 2))
    if c["max_own"]:
        p = torch.exp(own_scores - top)
        total = total + p.sum(-1)
        out = out + torch.einsum("htgj,tjhd->htgd", p.view(kv, tokens, group, -1), vo).reshape(out.shape)
    back = lambda x: x.view(kv, tokens, group, -1).permute(1, 0, 2, 3).reshape(tokens, c["heads"], -1)
    out = back(out / total[..., None]).to(s["q"].dtype)
    return [out, back(top[..., 0] + torch.log(total))[..., 0].contiguous()] if c["lse"] else out


# ---------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if kind in ("gemm_i8", "linear_i8"):
        m, n, k = case["m"], case["n"], case["k"]
        x = m * k * size[case["x"]] if kind == "linear_i8" else m * k
        return {"bytes": x + n * k + 4 * (m + n * (2 if case["bias"] else 1)) + m * n * size[case["out"]],
                "flops": 2.0 * m * n * k}
    if kind == "rotary":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * size[case["dtype"]] * values + 8 * case["tokens"],
                "flops": 3.0 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]}
    nq, no = _lengths(case)
    seen = float(sum(np.maximum(no - i, 0)[nq > i].sum() for i in range(int(nq.max()))))  # own keys of all tokens
    tokens, e = int(nq.sum()), 2
    return {"bytes": e * case["dim"] * (2 * tokens * case["heads"] + 2 * case["kv_heads"] * (case["prefix"] + int(no.sum()))),
            "flops": 4.0 * case["heads"] * case["dim"] * (tokens * case["prefix"] + seen)}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("gemm_i8", "linear_i8"):
        if kind == "linear_i8":
            top = s["x"].double().abs().max(dim=1).values
            scale = torch.maximum(top / 127, torch.full_like(top, 2.0 ** -126)).float()  # held in 32 bits
            a, sa = torch.round(s["x"].double() / scale.double().unsqueeze(1)), scale.double()
        else:
            a, sa = s["a"].double(), s["a_scale"].double()
        y = (a @ s["w"].double().T) * torch.outer(sa, s["w_scale"].double())
        if case["bias"]:
            y += s["bias"].double()
        y = {"none": lambda v: v, "relu": torch.relu, "sigmoid": torch.sigmoid}[case["act"]](y)
        return y if kind == "gemm_i8" else [y, sa]
    if kind == "rotary":
        rot, outs = case["rot"], []
        theta = np.array([_exact_frequency(case, j) for j in range(rot // 2)])
        turn = torch.polar(torch.full((case["tokens"], rot // 2), 1.0 if case["scaling"] != "yarn" else
                                      0.1 * math.log(_ROTARY["factor"]) + 1.0, dtype=torch.float64, device="cuda"),
                           torch.outer(s["pos"].double(), torch.from_numpy(theta).cuda()))
        for x in (s["q"], s["k"]):
            y = x.double().clone()
            first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if case["layout"] == "half" else \
                (slice(0, rot, 2), slice(1, rot, 2))
            z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn.unsqueeze(1)
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return outs
    # attention, one head at a time
    nq, no = _lengths(case)
    tokens, kv, heads = int(nq.sum()), case["kv_heads"], case["heads"]
    seq = torch.from_numpy(np.repeat(np.arange(case["seqs"]), nq)).cuda()
    rank = torch.from_numpy(np.concatenate([np.arange(n) for n in nq])).cuda()  # token's place in its sequence
    last = torch.from_numpy(no).cuda()[seq] - (torch.from_numpy(nq).cuda()[seq] - 1 - rank)
    width = int(last.max().clamp_min(0))
    j = torch.arange(width, device="cuda")
    hidden = j >= last[:, None]
    rows = (s["own_begin"][seq][:, None] + j).masked_fill(hidden, 0)
    out = torch.empty((tokens, heads, case["dim"]), dtype=torch.float64, device="cuda")
    lse = torch.empty((tokens, heads), dtype=torch.float64, device="cuda")
    for h in range(heads):
        g = h // (heads // kv)
        q = s["q"][:, h].double() / math.sqrt(case["dim"])
        z = q @ s["kp"][:, g].double().T
        if width:
            own_z = (q[:, None] * s["ko"][:, g].double()[rows]).sum(-1).masked_fill(hidden, -math.inf)
            z = torch.cat([z, own_z], 1)
        lse[:, h] = torch.logsumexp(z, 1)
        w = torch.softmax(z, 1)
        out[:, h] = w[:, :case["prefix"]] @ s["vp"][:, g].double()
        if width:
            out[:, h] += (w[:, case["prefix"]:, None] * s["vo"][:, g].double()[rows]).sum(1)
    return [out, lse] if case["lse"] else out


def _exact_frequency(case, j):
    rot, base, f, orig = case["rot"], _ROTARY["base"], _ROTARY["factor"], _ROTARY["original"]
    w = base ** (-2.0 * j / rot)
    if case["scaling"] == "linear":
        return w / f
    if case["scaling"] == "ntk":
        return (base * f ** (rot / (rot - 2.0))) ** (-2.0 * j / rot)
    if case["scaling"] == "yarn":
        at = lambda turns: rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        slow = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
        return w * (slow / f + 1.0 - slow)
    return w
