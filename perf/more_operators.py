"""The operators of this package with which other tokens read an image's, as they are measured: the rotation of heads by
their positions, attention of queries to keys and values of another length, and the end of a block with the norms on
both sides of it.

Every case runs in two forms. `own = False`: plain torch arithmetic in 32 bits (angles in 64), rounded once at the end.
`own = True`: this package's kernels through `foidfinder_b200.ops`.

- rotation: of every head the columns [start, start + r) are r / 2 pairs (y0, y1), neighbours ("pairs") or a half apart
  ("halves"), and become scale * (y0 cos t - y1 sin t, y0 sin t + y1 cos t) with t = position * frequency; the head's
  other columns stay. Several positions per row (axes of an image's grid) take equal shares of the pairs, in order.
- cross attention: out = softmax(scale q k^T over the keys that take part) v for every sequence and head; query head h
  reads key head h // (heads / kv_heads); a query without keys gives zeros.
- block end: out = alpha x + c * act(gate) * post(y) and normed = pre(out), where post and pre are RMS norms, LayerNorms
  or nothing, and pre sees `out` before it is rounded.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6


# ---------------------------------------------------------------- cases
def listed():
    return [
        # The queries of one new token at a far position: latency counts.
        dict(name="rotate one token", op="rope", dtype="fp16", rows=1, heads=16, dim=64, rotary=64, start=0, pairing="halves", axes=1, far=131072, scaling="linear"),
        # Queries and keys of a batch of 64 images of 448 pixels, by row and column of the patch.
        dict(name="rotate axial bs64", op="rope", dtype="fp16", rows=65600, heads=32, dim=64, rotary=64, start=0, pairing="pairs", axes=2, far=32, scaling=None),
        # Half of every head rotated for a context beyond the one trained on, an odd number of rows.
        dict(name="rotate part of the head, long context", op="rope", dtype="bf16", rows=32001, heads=8, dim=128, rotary=64, start=64, pairing="halves", axes=1, far=131072, scaling="yarn"),
        # One decoder token after its cross attention, behind a tanh gate.
        dict(name="block end one token", op="end", dtype="fp16", branch="fp16", rows=1, cols=1024, post=None, pre="layer", gate="scalar", act="tanh", scale=False, alpha=1.0, per=1),
        # A batch of 8 in a 32-bit residual stream, per-channel scale, LayerNorm before the next block (EVA02-B's width).
        dict(name="block end fp32 stream bs8", op="end", dtype="fp32", branch="bf16", rows=8200, cols=768, post="layer", pre="layer", gate=None, act=None, scale=True, alpha=1.0, per=1025),
        # Hidden rows of 2730 columns with a sigmoid gate for every element.
        dict(name="block end hidden rows, gated by element", op="end", dtype="bf16", branch="bf16", rows=16400, cols=2730, post="rms", pre=None, gate="element", act="sigmoid", scale=False, alpha=1.0, per=1),
        # A batch of 64, RMS norms on both sides, a gate per image and channel and a residual scale.
        dict(name="block end bs64", op="end", dtype="bf16", branch="bf16", rows=65600, cols=1024, post="rms", pre="rms", gate="sample", act=None, scale=True, alpha=0.875, per=1025),
        # One decoder token reads one image's tokens: latency counts.
        dict(name="one token reads one image", op="cross", dtype="fp16", sequences=1, queries=1, keys=1025, heads=16, kv_heads=16, dim=64, layout="even", mask=False, lengths=0),
        # 32 learned queries read each of 64 images.
        dict(name="32 queries read 64 images", op="cross", dtype="fp16", sequences=64, queries=32, keys=1025, heads=16, kv_heads=16, dim=64, layout="even", mask=False, lengths=0),
        # One token per sequence reads the frames of a long recording, shared key heads, padded to the longest.
        dict(name="one token reads 4 long recordings", op="cross", dtype="bf16", sequences=4, queries=1, keys=32800, heads=16, kv_heads=4, dim=128, layout="padded", mask=False, lengths=5),
        # Captions of any length over images of any size with letterbox borders masked, packed one behind the other.
        dict(name="ragged captions over ragged images", op="cross", dtype="bf16", sequences=24, queries=200, keys=1300, heads=16, kv_heads=4, dim=128, layout="ragged", mask=True, lengths=11),
        # Every second patch of a 1008-pixel image as a query over all of another's 5184.
        dict(name="2592 queries read 5184 patches", op="cross", dtype="fp16", sequences=4, queries=2592, keys=5184, heads=16, kv_heads=16, dim=64, layout="even", mask=False, lengths=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "end", "cross", "cross"])
    if op == "rope":
        dim = rng.choice([32, 64, 80, 128, 256])
        part = rng.random() < 0.5
        axes = rng.choice([1, 1, 2])
        rotary = max(4, int(dim * rng.choice([0.25, 0.5, 0.75])) // 4 * 4) if part else dim
        heads = rng.choice([1, 2, 5, 8, 16, 32])
        rows = min(_log(rng, 1, 65600), 65600 * 32 * 64 // (heads * dim))
        return dict(op=op, dtype=rng.choice(["fp16", "bf16", "fp32"]), rows=rows, heads=heads, dim=dim, rotary=rotary, start=rng.choice([0, dim - rotary]),
                    pairing=rng.choice(["pairs", "halves"]), axes=axes, far=32 if axes == 2 else _log(rng, 64, 1 << 20),
                    scaling=None if axes == 2 else rng.choice([None, "linear", "ntk", "yarn"]))
    if op == "end":
        dtype = rng.choice(["fp16", "bf16", "fp32"])
        cols = _log(rng, 17, 8192)
        rows = min(_log(rng, 1, 65600), 65600 * 1024 // cols)
        post = rng.choice([None, "rms", "layer"])
        gate = rng.choice([None, "scalar", "sample", "element"])
        return dict(op=op, dtype=dtype, branch=rng.choice(["fp32", "bf16", "fp16"]) if dtype == "fp32" else dtype, rows=rows, cols=cols, post=post,
                    pre=rng.choice([None, "rms", "layer"]), gate=gate, act=rng.choice([None, "sigmoid", "tanh"]) if gate else None, scale=rng.random() < 0.5,
                    alpha=rng.choice([1.0, 1.0, 0.875]), per=rng.choice([1, 197, 1025]))
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = min(kv_heads * rng.choice([1, 1, 2, 4, 8]), 32 // kv_heads * kv_heads)
    sequences, queries, keys = _log(rng, 1, 64), _log(rng, 1, 2592), _log(rng, 1, 32800)
    if rng.random() < 0.3:
        queries = rng.choice([1, 1, 2, 4])
    while sequences * queries * keys * heads * dim > 4 * 2592 * 5184 * 16 * 64 or sequences * keys * kv_heads * dim > 4 * 32800 * 4 * 128:
        if sequences > 1:
            sequences = max(1, sequences // 2)
        elif keys > queries:
            keys = keys * 2 // 3
        else:
            queries = queries * 2 // 3
    return dict(op=op, dtype=rng.choice(["fp16", "bf16"]), sequences=sequences, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim,
                layout=rng.choice(["even", "ragged", "padded"]), mask=rng.random() < 0.3, lengths=rng.randint(1, 1000))


def _lengths(case):
    """Queries and keys of every sequence, from the case alone."""
    n, q, k = case["sequences"], case["queries"], case["keys"]
    rng = random.Random(case["lengths"])
    qs, ks = [q] * n, [k] * n
    if case["layout"] == "ragged":
        qs = [rng.randint(1, 2 * q - 1) for _ in range(n)]
        ks = [0 if n > 2 and rng.random() < 0.1 else rng.randint(1, 2 * k - 1) for _ in range(n)]
    elif case["layout"] == "padded":
        ks = [rng.randint((k + 1) // 2, k) for _ in range(n)]
    return qs, ks


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _raw(case, seed):
    """The inputs of a case from the seed alone (both forms and the 64-bit definition start from these)."""
    g = _gen(seed)
    dt = TYPES[case["dtype"]]
    r = {}
    if case["op"] == "rope":
        r["x"] = (torch.randn(case["rows"], case["heads"] * case["dim"], generator=g, device="cuda") * 1.5).to(dt)
        size = (case["rows"],) if case["axes"] == 1 else (case["rows"], case["axes"])
        r["positions"] = torch.randint(0, case["far"], size, generator=g, device="cuda", dtype=torch.int32)
    elif case["op"] == "end":
        rows, cols = case["rows"], case["cols"]
        bt = TYPES[case["branch"]]
        r["x"] = (torch.randn(rows, cols, generator=g, device="cuda") * 2).to(dt)
        r["y"] = (torch.randn(rows, cols, generator=g, device="cuda") * 0.7 + 0.1).to(bt)
        for side in ("post", "pre"):
            if case[side]:
                r[side + "_weight"] = 1 + 0.1 * torch.randn(cols, generator=g, device="cuda")
            if case[side] == "layer":
                r[side + "_bias"] = 0.1 * torch.randn(cols, generator=g, device="cuda")
        if case["gate"] == "scalar":
            r["gate"] = torch.randn(1, 1, generator=g, device="cuda")
        elif case["gate"] == "sample":
            r["gate"] = torch.randn(-(-rows // case["per"]), cols, generator=g, device="cuda")
        elif case["gate"] == "element":
            r["gate"] = torch.randn(rows, cols, generator=g, device="cuda").to(bt)
        if case["scale"]:
            r["scale"] = 0.1 + 0.02 * torch.randn(cols, generator=g, device="cuda")
    else:
        qs, ks = _lengths(case)
        hd, kd = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        pitch = sum(ks) if case["layout"] != "padded" else case["sequences"] * case["keys"]
        r["q"] = torch.randn(sum(qs), hd, generator=g, device="cuda").to(dt)
        r["kv"] = torch.randn(pitch, 2 * kd, generator=g, device="cuda").to(dt)  # keys | values, as their projection leaves them
        if case["mask"]:
            r["mask"] = torch.rand(pitch, generator=g, device="cuda") > 0.25
            if case["sequences"] > 1:
                r["mask"][: ks[0]] = False  # the first image has nothing to read
    return r


def prepare(case, seed):
    s = _raw(case, seed)
    s["case"] = case
    if case["op"] == "rope":
        if own:
            from foidfinder_b200 import ops

            s["frequencies"], s["scale"] = ops.rope_frequencies(case["rotary"] // case["axes"], scaling=case["scaling"], factor=8.0, trained=4096)
            s["frequencies"] = s["frequencies"].repeat(case["axes"]).cuda()
            s["out"] = torch.empty_like(s["x"])
        else:
            s["frequencies"], s["scale"] = _plain_frequencies(case)
    elif case["op"] == "end":
        if own:
            s["out"] = torch.empty_like(s["x"])
            s["normed"] = torch.empty_like(s["y"]) if case["pre"] else None
    else:
        qs, ks = _lengths(case)
        kd = case["kv_heads"] * case["dim"]
        s["k"], s["v"] = s["kv"][:, :kd], s["kv"][:, kd:]
        s["lengths"] = qs, ks
        if own:
            ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")
            s["out"] = torch.empty_like(s["q"])
            s["pieces"] = dict(sequences=case["sequences"])
            if case["layout"] == "ragged":
                s["pieces"] |= dict(q_start=ints([sum(qs[:i]) for i in range(len(qs) + 1)]), k_start=ints([sum(ks[:i]) for i in range(len(ks) + 1)]))
            elif case["layout"] == "padded":
                s["pieces"] |= dict(k_len=ints(ks))
    return s


# ---------------------------------------------------------------- plain form
def _plain_frequencies(case):
    """(frequencies [rotary / 2], factor of the rotated values) for a context trained on 4096 tokens, 8 times as long."""
    r, base, factor, trained = case["rotary"] // case["axes"], 10000.0, 8.0, 4096
    scale = 1.0
    if case["scaling"] == "ntk":
        base = base * factor ** (r / (r - 2)) if r > 2 else base
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "yarn":
        turn = lambda n: r * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), r - 1)
        ramp = ((torch.arange(r // 2, device="cuda").double() - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        scale = 0.1 * math.log(factor) + 1
    return f.repeat(case["axes"]), scale


def _plain_rope(s, case):
    rows, heads, dim, r, start = case["rows"], case["heads"], case["dim"], case["rotary"], case["start"]
    p = s["positions"].double().reshape(rows, case["axes"]).repeat_interleave(r // 2 // case["axes"], 1)
    angle = p * s["frequencies"]
    c, sn = (angle.cos() * s["scale"]).float()[:, None], (angle.sin() * s["scale"]).float()[:, None]
    x = s["x"].float().reshape(rows, heads, dim)
    y = x[..., start : start + r]
    if case["pairing"] == "pairs":
        y0, y1 = y[..., 0::2], y[..., 1::2]
        y = torch.stack([y0 * c - y1 * sn, y0 * sn + y1 * c], -1).flatten(-2)
    else:
        y0, y1 = y[..., : r // 2], y[..., r // 2 :]
        y = torch.cat([y0 * c - y1 * sn, y0 * sn + y1 * c], -1)
    return torch.cat([x[..., :start], y, x[..., start + r :]], -1).reshape(rows, -1).to(s["x"].dtype)


def _plain_norm(x, kind, w, b):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    return y if b is None else y + b


def _plain_end(s, case):
    y = s["y"].float()
    if case["post"]:
        y = _plain_norm(y, case["post"], s["post_weight"], s.get("post_bias"))
    if case["gate"]:
        gate = s["gate"].float()
        if case["act"] == "sigmoid":
            gate = 1 / (1 + torch.exp(-gate))
        elif case["act"] == "tanh":
            gate = torch.tanh(gate)
        if case["gate"] == "sample":
            gate = gate[torch.arange(case["rows"], device=gate.device) // case["per"]]
        y = y * gate
    if case["scale"]:
        y = y * s["scale"]
    out = case["alpha"] * s["x"].float() + y
    outs = [out.to(s["x"].dtype)]
    if case["pre"]:
        outs.append(_plain_norm(out, case["pre"], s["pre_weight"], s.get("pre_bias")).to(s["y"].dtype))
    return outs


def _plain_cross(s, case):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    qs, ks = s["lengths"]
    outs, qa, ka = [], 0, 0
    for nq, nk in zip(qs, ks):
        q = s["q"][qa : qa + nq].float().reshape(nq, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
        k = s["k"][ka : ka + nk].float().reshape(nk, kv_heads, dim).permute(1, 2, 0)
        v = s["v"][ka : ka + nk].float().reshape(nk, kv_heads, dim).transpose(0, 1)
        if nk == 0:
            o = torch.zeros_like(q)
        else:
            t = torch.matmul(q, k) * dim**-0.5
            if case["mask"]:
                t = t.masked_fill(~s["mask"][ka : ka + nk], -torch.inf)
            top = t.amax(-1, keepdim=True)
            p = torch.exp(t - torch.where(top == -torch.inf, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
        outs.append(o.reshape(kv_heads, -1, nq, dim).permute(2, 0, 1, 3).reshape(nq, heads * dim).to(s["q"].dtype))
        qa += nq
        ka += nk if case["layout"] != "padded" else case["keys"]
    return torch.cat(outs)


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "rope":
            return [_plain_rope(s, case)]
        return _plain_end(s, case) if case["op"] == "end" else [_plain_cross(s, case)]
    from foidfinder_b200 import ops

    if case["op"] == "rope":
        ops.rope(s["x"], s["out"], s["positions"], s["frequencies"], heads=case["heads"], head_dim=case["dim"], start=case["start"], pairing=case["pairing"],
                 scale=s["scale"])
    elif case["op"] == "end":
        gate_rows = {"scalar": case["rows"], "sample": case["per"]}.get(case["gate"], 1)
        ops.norm_residual(s["x"], s["y"], s["out"], alpha=case["alpha"], post=case["post"], post_weight=s.get("post_weight"), post_bias=s.get("post_bias"),
                          gate=s.get("gate"), gate_act=case["act"], gate_rows=gate_rows, scale=s.get("scale"), normed=s["normed"], pre=case["pre"],
                          pre_weight=s.get("pre_weight"), pre_bias=s.get("pre_bias"), eps=EPS)
        if case["pre"]:
            return [s["out"], s["normed"]]
    else:
        ops.cross_attention(s["q"], s["k"], s["v"], s["out"], heads=case["heads"], kv_heads=case["kv_heads"], head_dim=case["dim"], mask=s.get("mask"), **s["pieces"])
    return [s["out"]]


# ---------------------------------------------------------------- what a pass cannot do without
def _size(name):
    return 4 if name == "fp32" else 2


def work(case):
    if case["op"] == "rope":  # values read and written once, positions and frequencies read once
        n = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * _size(case["dtype"]) + 4 * case["rows"] * case["axes"] + 4 * case["rotary"], "flops": 3 * case["rows"] * case["heads"] * case["rotary"]}
    if case["op"] == "end":  # x and y read, out and normed written; gate and weights read once
        n = case["rows"] * case["cols"]
        bytes_ = n * (2 * _size(case["dtype"]) + (2 if case["pre"] else 1) * _size(case["branch"]))
        bytes_ += {"element": n * _size(case["branch"]), "sample": 4 * -(-case["rows"] // case["per"]) * case["cols"], "scalar": 4}.get(case["gate"], 0)
        bytes_ += 4 * case["cols"] * sum({"rms": 1, "layer": 2}.get(case[side], 0) for side in ("post", "pre")) + (4 * case["cols"] if case["scale"] else 0)
        return {"bytes": bytes_, "flops": n * (2 + 4 * bool(case["post"]) + 4 * bool(case["pre"]) + bool(case["gate"]) + case["scale"])}
    qs, ks = _lengths(case)  # queries, keys and values read once, results written once
    bytes_ = 2 * case["dim"] * (2 * sum(qs) * case["heads"] + 2 * sum(ks) * case["kv_heads"]) + (sum(ks) if case["mask"] else 0)
    return {"bytes": bytes_, "flops": 4 * case["heads"] * case["dim"] * sum(a * b for a, b in zip(qs, ks))}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_frequency(j, r, scaling):
    """Frequency of pair j of r / 2 in radians per position, and the factor of the rotated values."""
    theta, longer = math.exp(-2 * j / r * math.log(10000)), 8
    if scaling == "linear":
        return theta / longer, 1.0
    if scaling == "ntk":  # the slowest pair turns `longer` times as slowly, the fastest as before
        return theta * longer ** (-2 * j / (r - 2)) if r > 2 else theta, 1.0
    if scaling == "yarn":  # pairs that turn more than 32 times in the trained context stay, those that turn less than once slow down
        first, last = (math.log(4096 / (2 * math.pi * n)) / math.log(10000) * r / 2 for n in (32, 1))
        first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
        share = min(max((j - first) / (last - first if last > first else 0.001), 0), 1)
        return theta * ((1 - share) + share / longer), 1 + math.log(longer) / 10
    return theta, 1.0


def _exact_rope(r, case):
    rows, dim, a, n = case["rows"], case["dim"], case["start"], case["rotary"]
    x = r["x"].double().reshape(rows, case["heads"], dim)
    each = n // 2 // case["axes"]
    pos = r["positions"].double().reshape(rows, -1)
    turns = torch.tensor([_exact_frequency(j, 2 * each, case["scaling"])[0] for j in range(each)], dtype=torch.float64, device="cuda")
    factor = _exact_frequency(0, 2 * each, case["scaling"])[1]
    w = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"), torch.einsum("ta,j->taj", pos, turns).reshape(rows, 1, n // 2))
    y = x[..., a : a + n]
    y = y.reshape(rows, -1, n // 2, 2) if case["pairing"] == "pairs" else y.reshape(rows, -1, 2, n // 2).transpose(2, 3)
    y = torch.view_as_real(torch.view_as_complex(y.contiguous()) * w)
    x[..., a : a + n] = (y if case["pairing"] == "pairs" else y.transpose(2, 3)).reshape(rows, -1, n)
    return x.reshape(rows, -1)


def _exact_norm(x, kind, w, b):
    mean = x.sum(-1, keepdim=True) / x.shape[-1] if kind == "layer" else 0.0
    y = (x - mean) / ((x - mean).square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w.double()
    return y if b is None else y + b.double()


def exact(case, seed):
    r = _raw(case, seed)
    if case["op"] == "rope":
        return [_exact_rope(r, case)]
    if case["op"] == "end":
        y = r["y"].double()
        if case["post"]:
            y = _exact_norm(y, case["post"], r["post_weight"], r.get("post_bias"))
        if case["gate"]:
            gate = r["gate"].double()
            gate = {"sigmoid": torch.sigmoid, "tanh": torch.tanh, None: lambda t: t}[case["act"]](gate)
            y = y * (gate.repeat_interleave(case["per"], 0)[: case["rows"]] if case["gate"] == "sample" else gate)
        y = y * (r["scale"].double() if case["scale"] else 1.0) + r["x"].double() * case["alpha"]
        return [y] + ([_exact_norm(y, case["pre"], r["pre_weight"], r.get("pre_bias"))] if case["pre"] else [])
    heads, dim, group = case["heads"], case["dim"], case["heads"] // case["kv_heads"]
    qs, ks = _lengths(case)
    out = torch.zeros(sum(qs), heads, dim, dtype=torch.float64, device="cuda")
    q_at = k_at = 0
    for nq, nk in zip(qs, ks):
        keep = torch.arange(k_at, k_at + nk, device="cuda")
        if case["mask"]:
            keep = keep[r["mask"][k_at : k_at + nk]]
        if nq and keep.numel():
            kv = r["kv"][keep].double().reshape(keep.numel(), 2, case["kv_heads"], dim)
            for h in range(heads):
                q = r["q"][q_at : q_at + nq, h * dim : (h + 1) * dim].double()
                out[q_at : q_at + nq, h] = torch.softmax(q @ kv[:, 0, h // group].t() / math.sqrt(dim), -1) @ kv[:, 1, h // group]
        q_at += nq
        k_at += case["keys"] if case["layout"] == "padded" else nk
    return [out.reshape(sum(qs), heads * dim)]
