"""The 4-bit operators of this package as they are measured: block-scaled 4-bit quantisation, the linear layer
on 4-bit operands with its fused epilogues, and the per-head normalisation of queries and keys with the rotary
position rotation.

Every case runs in two forms. `own = False`: plain torch arithmetic in 32 bits, rounded once at the end.
`own = True`: this package's kernels through `foidfinder_b200.ops` and `foidfinder_b200.fp4`.

The 4-bit formats. A code is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}; ties go to the code with an even mantissa bit.
- "nv": blocks of 16 columns share an unsigned 8-bit scale S (4 exponent, 3 mantissa bits) and every row has a
  32-bit scale s: s = the smallest power of two (2^-110 at least) with amax(row) <= 2688 s, S = round(amax(block) / (6 s)),
  code = round(x / (S s)), saturating at +-6.
- "mx": blocks of 32 columns share a power of two 2^E, E = floor(log2(amax(block))) - 2, code = round(x / 2^E),
  saturating at +-6.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
NV_TOP = 2688.0  # 6 (the largest code) x 448 (the largest block scale)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One 448-pixel image's tokens (EVA02-L), quantised ahead of a product: latency counts.
        dict(name="quantise one image", op="quantise", fmt="nv", dtype="fp16", rows=1025, cols=1024),
        # A batch of 64's SwiGLU hidden rows, whose 2730 columns end inside a block and whose rows start unaligned.
        dict(name="quantise hidden rows bs64", op="quantise", fmt="mx", dtype="bf16", rows=65600, cols=2730),
        # A 32-bit checkpoint's gate|up weight when it is loaded.
        dict(name="quantise fp32 weight", op="quantise", fmt="nv", dtype="fp32", rows=5460, cols=1024),
        # The tag head on the (already normalised) class token of one image: one row, a wide odd output in 32 bits.
        dict(name="tag head one row", op="linear", epi="bias", fmt="nv", dtype="fp16", out="fp32", m=1, k=1024, n=30877, norm=False),
        # The attention projection of one image, added to the residual stream.
        dict(name="proj one image", op="linear", epi="residual", fmt="nv", dtype="fp16", out="fp16", m=1025, k=1024, n=1024, norm=False),
        # EVA02-B: pre-norm, query/key/value projection with per-head normalisation and rotation, batch of 8.
        dict(name="qkv EVA02-B bs8", op="linear", epi="qkv", fmt="nv", dtype="fp16", out="fp16", m=8200, k=768, n=2304, norm=True, tokens=1025),
        # EVA02-B: pre-norm and SwiGLU up-projection, batch of 8 (hidden 2048).
        dict(name="gate/up EVA02-B bs8", op="linear", epi="swiglu", fmt="mx", dtype="fp16", out="fp16", m=8200, k=768, n=2048, norm=True),
        # PixAI: GELU up-projection of one image's 5184 patches, hidden 4736, bfloat16.
        dict(name="fc1 PixAI one image", op="linear", epi="gelu", fmt="mx", dtype="bf16", out="bf16", m=5184, k=1024, n=4736, norm=True),
        # EVA02-L: pre-norm and SwiGLU up-projection, batch of 64 (hidden 2730): the largest product.
        dict(name="gate/up EVA02-L bs64", op="linear", epi="swiglu", fmt="nv", dtype="fp16", out="fp16", m=65600, k=1024, n=2730, norm=True),
        # EVA02-L: hidden norm and down-projection (odd depth 2730) added to the residual stream, batch of 64.
        dict(name="down EVA02-L bs64", op="linear", epi="residual", fmt="nv", dtype="bf16", out="bf16", m=65600, k=2730, n=1024, norm=True),
        # Queries and keys of one image behind an existing projection.
        dict(name="qk norm one image", op="qknorm", norm="rms", pairing="pairs", dtype="fp16", rows=1025, qheads=16, kheads=16, dim=64, tokens=1025),
        # Queries and keys of a batch of 64, layer-normalised.
        dict(name="qk norm bs64", op="qknorm", norm="layer", pairing="pairs", dtype="fp16", rows=65600, qheads=16, kheads=16, dim=64, tokens=1025),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantise", "linear", "linear", "qknorm"])
    if op == "quantise":
        return dict(op=op, fmt=rng.choice(["nv", "mx"]), dtype=rng.choice(["fp16", "bf16", "fp32"]), rows=_log(rng, 1, 32000), cols=_log(rng, 17, 4864))
    if op == "linear":
        epi = rng.choice(["bias", "residual", "swiglu", "gelu", "qkv"])
        dtype = rng.choice(["fp16", "bf16"])
        case = dict(op=op, epi=epi, fmt=rng.choice(["nv", "mx"]), dtype=dtype, out=dtype, m=_log(rng, 1, 32000), k=_log(rng, 128, 4864),
                    n=_log(rng, 64, 4864), norm=rng.random() < 0.5)
        if epi == "qkv":
            case |= dict(n=192 * rng.randint(1, 16), tokens=rng.choice([1, 197, 576, 1025, 5184]))
        elif epi == "swiglu":
            case |= dict(n=_log(rng, 64, 2730))
        elif epi == "bias" and rng.random() < 0.4:
            case |= dict(out="fp32", m=_log(rng, 1, 64), n=_log(rng, 1000, 98782), norm=False)
        case["m"] = min(case["m"], 65600 * 1024 * 5460 // (case["k"] * case["n"] * (2 if epi == "swiglu" else 1)))  # at most the largest listed product
        return case
    kheads = rng.choice([1, 2, 4, 8, 12, 16])
    dim = rng.choice([32, 64, 128])
    return dict(op=op, norm=rng.choice(["rms", "layer"]), pairing=rng.choice(["pairs", "halves"]), dtype=rng.choice(["fp16", "bf16"]), rows=_log(rng, 1, 32000),
                qheads=kheads * rng.choice([1, 1, 2]), kheads=kheads, dim=dim, tokens=rng.choice([1, 197, 576, 1025, 5184]))


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, cols, dtype, g):
    """N(0, 1) with 1% of the values 20 times as large, as transformer activations have them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return torch.where(torch.rand(rows, cols, generator=g, device="cuda") < 0.01, 20 * x, x).to(dtype)


def _pitched(rows, cols, dtype, by=8):
    """An output whose rows start 16 bytes apart or more, as the engine's buffers do: the view of its first `cols` columns."""
    return torch.empty(rows, -(-cols // by) * by, device="cuda", dtype=dtype)[:, :cols]


def _angles(tokens, half, dtype):
    """Axial rotation angles of a square grid of tokens (row 0 is the class token where the rest is a square), [tokens, half]."""
    grid = math.isqrt(tokens)
    cls = 0 if grid * grid == tokens else 1
    grid = max(1, math.isqrt(tokens - cls)) if tokens > cls else 1
    i = torch.arange(tokens, device="cuda") - cls
    on = (i >= 0).to(dtype)
    y, x = (torch.div(i.clamp_min(0), grid, rounding_mode="floor") % 128).to(dtype), (i.clamp_min(0) % grid).to(dtype)
    nb = half // 2
    bands = torch.exp(torch.arange(nb, device="cuda").to(dtype) * (-math.log(10000.0) / nb))
    return torch.cat([(y * on)[:, None] * bands, (x * on)[:, None] * bands], 1)


def _raw(case, seed):
    """The inputs of a case from the seed alone (both forms and the 64-bit definition start from these)."""
    g = _gen(seed)
    dt = TYPES[case["dtype"]]
    r = {}
    if case["op"] == "quantise":
        r["x"] = _activations(case["rows"], case["cols"], dt, g)
        if case["dtype"] == "fp32":
            r["x"] = r["x"] * 0.02
    elif case["op"] == "linear":
        m, k, n, epi = case["m"], case["k"], case["n"], case["epi"]
        nw = 2 * n if epi == "swiglu" else n
        x = _pitched(m, k, dt)
        x.copy_(_activations(m, k, dt, g))
        r["x"] = x
        r["w"] = torch.randn(nw, k, generator=g, device="cuda") * 0.02
        r["bias"] = torch.randn(nw, generator=g, device="cuda") * 0.02
        if case["norm"]:
            r["gamma"] = 1 + 0.02 * torch.randn(k, generator=g, device="cuda")
            r["beta"] = 0.02 * torch.randn(k, generator=g, device="cuda")
        if epi == "residual":
            r["residual"] = _pitched(m, n, TYPES[case["out"]])
            r["residual"].copy_(torch.randn(m, n, generator=g, device="cuda"))
        if epi == "qkv":
            r["qw"] = 1 + 0.1 * torch.randn(64, generator=g, device="cuda")
            r["kw"] = 1 + 0.1 * torch.randn(64, generator=g, device="cuda")
            a = _angles(case["tokens"], 32, torch.float64)
            r["cos"], r["sin"] = a.cos().float().t().contiguous(), a.sin().float().t().contiguous()
    else:
        d, heads = case["dim"], case["qheads"] + case["kheads"]
        # columns q | k | v, as the projection leaves them
        r["x"] = (torch.randn(case["rows"], (heads + case["kheads"]) * d, generator=g, device="cuda") * 1.5).to(dt)
        for name in ("qw", "kw"):
            r[name] = 1 + 0.1 * torch.randn(d, generator=g, device="cuda")
        if case["norm"] == "layer":
            for name in ("qb", "kb"):
                r[name] = 0.1 * torch.randn(d, generator=g, device="cuda")
        a = _angles(case["tokens"], d // 2, torch.float64)
        r["cos"], r["sin"] = a.cos().float().t().contiguous(), a.sin().float().t().contiguous()  # [dim / 2, tokens]
    return r


def prepare(case, seed):
    s = _raw(case, seed)
    s["case"] = case
    if case["op"] == "linear":
        w, bias = s.pop("w"), s.pop("bias")
        if own:
            from foidfinder_b200 import fp4

            qkv = {}
            if case["epi"] == "qkv":
                qkv = dict(rope=(s["cos"], s["sin"]), q_weight=s["qw"], k_weight=s["kw"], norm="rms", qk_eps=1e-6)
            s["layer"] = fp4.Fp4Linear(w, bias, fmt=case["fmt"], epilogue=case["epi"], gamma=s.get("gamma"), beta=s.get("beta"), eps=1e-6, **qkv)
            s["out"] = _pitched(case["m"], case["n"], TYPES[case["out"]]) if case["out"] != "fp32" else torch.empty(case["m"], case["n"], device="cuda")
        else:
            s["w"], s["bias"] = _plain_values(w, case["fmt"]), bias  # the values that the 4-bit weight stands for
    elif own:
        from foidfinder_b200 import fp4

        if case["op"] == "quantise":
            s["q"] = fp4.Fp4Tensor.empty(case["rows"], case["cols"], case["fmt"], device="cuda")
            s["out"] = torch.empty_like(s["x"])
        else:
            s["out"] = torch.empty(case["rows"], (case["qheads"] + case["kheads"]) * case["dim"], device="cuda", dtype=s["x"].dtype)
    return s


# ---------------------------------------------------------------- plain form
def _plain_values(x, fmt):
    """The 32-bit values that the 4-bit codes and scales of x stand for."""
    rows, cols = x.shape
    size = 16 if fmt == "nv" else 32
    v = torch.nn.functional.pad(x.float(), (0, -cols % size)).view(rows, -1, size)
    top = v.abs().amax(2, keepdim=True)
    if fmt == "nv":
        m, e = torch.frexp(top.amax(1, keepdim=True))  # m in [0.5, 1); NV_TOP = 0.65625 x 2^12
        e = torch.where(m > NV_TOP / 4096, e - 11, e - 12).clamp_min(-110)
        six = torch.full_like(top, 6.0)
        scale = torch.ldexp((torch.ldexp(top, -e) / six).to(torch.float8_e4m3fn).float(), e)
    else:
        _, e = torch.frexp(top)
        scale = torch.ldexp(torch.ones_like(top), torch.where(top > 0, (e - 3).clamp_min(-127), torch.full_like(e, -127)))
    y = torch.where(scale > 0, v / scale, torch.zeros_like(v))
    a = y.abs()
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float()) + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float()
    return (torch.where(y < 0, -q, q) * scale).view(rows, -1)[:, :cols]


def _plain_layer_norm(x, w, b, eps):
    d = x - x.mean(-1, keepdim=True)
    y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + eps) * w
    return y if b is None else y + b


def _plain_heads(x, w, b, norm, cos, sin, pairing):
    """x [rows, heads, dim] normalised over dim and rotated; cos, sin [rows, dim / 2]."""
    if norm == "rms":
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    else:
        y = _plain_layer_norm(x, w, b, 1e-6)
    c, s = cos[:, None], sin[:, None]
    if pairing == "pairs":
        y0, y1 = y[..., 0::2], y[..., 1::2]
        return torch.stack([y0 * c - y1 * s, y0 * s + y1 * c], -1).flatten(-2)
    h = x.shape[-1] // 2
    y0, y1 = y[..., :h], y[..., h:]
    return torch.cat([y0 * c - y1 * s, y0 * s + y1 * c], -1)


def _plain_qk(x, q_cols, k_cols, dim, case_norm, s, tokens, pairing):
    rows = x.shape[0]
    at = torch.arange(rows, device=x.device) % tokens
    cos, sin = s["cos"].t()[at], s["sin"].t()[at]
    q = _plain_heads(x[:, :q_cols].reshape(rows, -1, dim), s["qw"], s.get("qb"), case_norm, cos, sin, pairing)
    k = _plain_heads(x[:, q_cols : q_cols + k_cols].reshape(rows, -1, dim), s["kw"], s.get("kb"), case_norm, cos, sin, pairing)
    return torch.cat([q.reshape(rows, -1), k.reshape(rows, -1)], 1)


def _plain_linear(s, case):
    x = s["x"].float()
    if case["norm"]:
        x = _plain_layer_norm(x, s["gamma"], s["beta"], 1e-6)
    y = _plain_values(x, case["fmt"]) @ s["w"].t() + s["bias"]
    n = case["n"]
    if case["epi"] == "residual":
        y = y + s["residual"].float()
    elif case["epi"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    elif case["epi"] == "swiglu":
        y = y[:, :n] / (1 + torch.exp(-y[:, :n])) * y[:, n:]
    elif case["epi"] == "qkv":
        y = torch.cat([_plain_qk(y, n // 3, n // 3, 64, "rms", s, case["tokens"], "pairs"), y[:, 2 * n // 3 :]], 1)
    return y.to(TYPES[case["out"]])


def run(s):
    case = s["case"]
    if not own:
        if case["op"] == "quantise":
            return [_plain_values(s["x"], case["fmt"]).to(s["x"].dtype)]
        if case["op"] == "linear":
            return [_plain_linear(s, case)]
        d = case["dim"]
        return [_plain_qk(s["x"].float(), case["qheads"] * d, case["kheads"] * d, d, case["norm"], s, case["tokens"], case["pairing"]).to(s["x"].dtype)]
    from foidfinder_b200 import fp4, ops

    if case["op"] == "quantise":
        fp4.quantize(s["x"], out=s["q"])
        fp4.dequantize(s["q"], out=s["out"])
    elif case["op"] == "linear":
        s["layer"](s["x"], out=s["out"], residual=s.get("residual"))
    else:
        ops.qk_norm_rope(s["x"], s["out"], q_heads=case["qheads"], k_heads=case["kheads"], head_dim=case["dim"], norm=case["norm"], q_weight=s["qw"],
                         k_weight=s["kw"], q_bias=s.get("qb"), k_bias=s.get("kb"), eps=1e-6, rope_cos=s["cos"], rope_sin=s["sin"], pairing=case["pairing"])
    return [s["out"]]


# ---------------------------------------------------------------- what a pass cannot do without
def _size(name):
    return 4 if name == "fp32" else 2


def _packed(rows, cols, fmt):
    return rows * cols / 2 + rows * -(-cols // (16 if fmt == "nv" else 32)) + (4 * rows if fmt == "nv" else 0)


def work(case):
    if case["op"] == "quantise":  # codes and scales written and read once, values read and written once
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * _size(case["dtype"]) + 2 * _packed(case["rows"], case["cols"], case["fmt"]), "flops": 4 * n}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        nw = 2 * n if case["epi"] == "swiglu" else n
        out = m * n * _size(case["out"])
        return {"bytes": m * k * _size(case["dtype"]) + _packed(nw, k, case["fmt"]) + 4 * nw + out * (2 if case["epi"] == "residual" else 1), "flops": 2 * m * nw * k}
    n = case["rows"] * (case["qheads"] + case["kheads"]) * case["dim"]
    return {"bytes": 2 * n * _size(case["dtype"]) + 4 * case["tokens"] * case["dim"], "flops": 10 * n}


# ---------------------------------------------------------------- the definition in 64 bits
def _floor_power(x):
    """The largest power of two that is not above x > 0 (64-bit), from its exponent field."""
    return (x.view(torch.int64) & (0x7FF << 52)).view(torch.float64)


def _exact_scales(x, fmt):
    """Scale of every column of x (64-bit), [rows, cols]."""
    size = 16 if fmt == "nv" else 32
    rows, cols = x.shape
    nb = -(-cols // size)
    a = torch.zeros(rows, nb * size, dtype=torch.float64, device=x.device)
    a[:, :cols] = x.abs()
    top = a.reshape(rows, nb, size).max(-1).values
    if fmt == "mx":
        scale = _floor_power(top.clamp_min(2.0**-125)) / 4
    else:
        most = (top.max(-1, keepdim=True).values / 2688).clamp_min(2.0**-110)
        s = _floor_power(most)
        s = torch.where(most > s, 2 * s, s)
        t = top / (6 * s)
        step = _floor_power(t.clamp_min(2.0**-6)) / 8
        scale = (torch.round(t / step) * step).clamp_max(448) * s
    return scale.repeat_interleave(size, 1)[:, :cols]


def _exact_values(x, fmt):
    scale = _exact_scales(x, fmt)
    y = x / torch.where(scale > 0, scale, torch.inf)
    step = _floor_power(y.abs().clamp(1.0, 4.0)) / 2
    return (torch.round(y / step) * step).clamp(-6, 6) * scale


def _exact_norm(x, w, b, layer):
    if layer:
        x = x - x.sum(-1, keepdim=True) / x.shape[-1]
    y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
    return y if b is None else y + b.double()


def _exact_rotate(y, angle, pairing):
    """y [rows, heads, dim] as complex numbers, turned by angle [rows, dim / 2]."""
    rows, heads, d = y.shape
    z = y.reshape(rows, heads, d // 2, 2) if pairing == "pairs" else y.reshape(rows, heads, 2, d // 2).transpose(2, 3)
    t = torch.view_as_real(torch.view_as_complex(z.contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None])
    return (t if pairing == "pairs" else t.transpose(2, 3)).reshape(rows, heads * d)


def exact(case, seed):
    r = _raw(case, seed)
    x = r["x"].double()
    if case["op"] == "quantise":
        return [_exact_values(x, case["fmt"])]
    if case["op"] == "linear":
        if case["norm"]:
            x = _exact_norm(x, r["gamma"], r["beta"], True)
        y = _exact_values(x, case["fmt"]) @ _exact_values(r["w"].double(), case["fmt"]).t()
        y += r["bias"].double()
        n = case["n"]
        if case["epi"] == "residual":
            y += r["residual"].double()
        elif case["epi"] == "gelu":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y**3))
        elif case["epi"] == "swiglu":
            y = y[:, :n] * torch.sigmoid(y[:, :n]) * y[:, n:]
        elif case["epi"] == "qkv":
            angle = _angles(case["tokens"], 32, torch.float64).repeat(-(-case["m"] // case["tokens"]), 1)[: case["m"]]
            parts = [_exact_rotate(_exact_norm(p.reshape(case["m"], -1, 64), w, None, False), angle, "pairs") for p, w in zip(y.split(n // 3, 1), (r["qw"], r["kw"]))]
            y = torch.cat(parts + [y[:, 2 * n // 3 :]], 1)
        return [y]
    d, layer = case["dim"], case["norm"] == "layer"
    angle = _angles(case["tokens"], d // 2, torch.float64).repeat(-(-case["rows"] // case["tokens"]), 1)[: case["rows"]]
    q, k, _ = x.split([case["qheads"] * d, case["kheads"] * d, case["kheads"] * d], 1)
    parts = [_exact_rotate(_exact_norm(p.reshape(case["rows"], -1, d), w, b, layer), angle, case["pairing"]) for p, w, b in ((q, r["qw"], r.get("qb")), (k, r["kw"], r.get("kb")))]
    return [torch.cat(parts, 1)]
