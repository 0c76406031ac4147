"""Rotation by positions, the end of a block and cross attention on the GPU, against the 64-bit oracle (oracle/cross.py).

Tolerances, from the arithmetic:
- rotation: the part of a turn is rounded to 2^-26 of one, 2 pi 2^-26 < 2^-23 radians, sine and cosine are within 2^-23 of
  theirs, a product and the sum round by 2^-24 each: at most 2^-21 of the partners' magnitudes. In 64 bits an angle is off by
  a few 2^-53 of itself.
- block end: oracle/cross.py bounds the error of the f32 statistics and products.
- attention: scores are sums of up to 128 products in f32, off by at most 2^-20 of the sum of their magnitudes (half that,
  if every step were truncated), which changes a weight by that factor; exponentials are within 2^-21. Weights are rounded to 16 bits for
  their product with V: half a unit of each, so of the sum of p |v|. Weights in fp16 have a factor of 2^7 at least for the
  largest, so a step below fp16's smallest normal is at most 2^-25 / 2^7 of the largest weight, for every key.
- every output is rounded once: half a unit in the last place.
"""

from __future__ import annotations

import math

import pytest
import torch

from foidfinder_b200 import ops
from oracle import cross as O

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TINY = {F16: 2.0**-25, BF16: 2.0**-134, F32: 2.0**-150}


def _half_ulp(t):
    return torch.finfo(t).eps / 2


def _close(got, want, err, dtype):
    tol = err + (want.abs() + err) * _half_ulp(dtype) + TINY[dtype]
    bad = (got.double().cpu() - want).abs() > tol
    worst = ((got.double().cpu() - want).abs() / tol).max().item() if want.numel() else 0
    assert not bad.any() and not got.isnan().any(), f"{int(bad.sum())} of {bad.numel()} off, worst {worst:.2f} of the tolerance"


def _randn(*shape, seed=0, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


# ---------------------------------------------------------------- rotation
def _rope(x, positions, f, *, heads, dim, start=0, pairing="pairs", scale=1.0, out=None):
    want, size, top = O.rope(x, positions, f, heads=heads, head_dim=dim, start=start, pairing=pairing, scale=scale)
    d = x.cuda()
    o = torch.empty_like(d) if out is None else out
    ops.rope(d, o, positions.cuda(), f.cuda(), heads=heads, head_dim=dim, start=start, pairing=pairing, scale=scale)
    _close(o, want, size * (2.0**-21 + 4 * top * 2.0**-53), x.dtype)
    return o


@pytest.mark.parametrize("pairing", ["pairs", "halves"])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize(("rows", "heads", "dim", "rotary", "start"), [
    (1, 1, 2, 2, 0), (1, 16, 64, 64, 0), (5, 3, 80, 20, 60), (300, 32, 64, 64, 0), (131, 5, 80, 60, 20), (77, 2, 256, 64, 0), (40, 7, 34, 14, 9),
    (2001, 1, 32, 32, 0), (1, 128, 128, 64, 64), (3, 700, 16, 8, 4), (9, 1, 1024, 1024, 0), (8, 2, 13, 10, 3)])
def test_rope(cuda_device, rows, heads, dim, rotary, start, dtype, pairing):
    x = _randn(rows, heads * dim, seed=1, dtype=dtype, scale=2)
    positions = torch.randint(-5, 1 << 17, (rows,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    f, s = ops.rope_frequencies(rotary, scaling="yarn", factor=4.0, trained=2048)
    _rope(x, positions, f, heads=heads, dim=dim, start=start, pairing=pairing, scale=s)


@pytest.mark.parametrize("axes", [2, 3])
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64])
def test_rope_axes_and_types(cuda_device, axes, ptype):
    x = _randn(197, 4 * 96, seed=3, dtype=F16)
    positions = torch.randint(0, 72, (197, axes), generator=torch.Generator().manual_seed(4), dtype=ptype)
    f = ops.rope_frequencies(96 // axes)[0].repeat(axes)
    _rope(x, positions, f, heads=4, dim=96)
    _rope(x, positions, f.float(), heads=4, dim=96, pairing="halves")


@pytest.mark.parametrize("far", [1 << 20, 1 << 30, 1 << 40])
def test_rope_far_positions(cuda_device, far):
    x = _randn(64, 2 * 64, seed=5, dtype=F32)
    positions = far - torch.arange(64, dtype=torch.int64) * 977
    _rope(x, positions, ops.rope_frequencies(64)[0], heads=2, dim=64)


@pytest.mark.parametrize("pairing", ["pairs", "halves"])
@pytest.mark.parametrize(("dim", "rotary", "start"), [(64, 64, 0), (128, 32, 96), (30, 10, 5)])
def test_rope_in_place_in_a_packed_projection(cuda_device, dim, rotary, start, pairing):
    """Rotated in place within wider rows (q | k | v): nothing else changes."""
    x = _randn(133, 6 * dim + 8, seed=6, dtype=BF16)
    positions = torch.arange(133, dtype=torch.int32)
    f = ops.rope_frequencies(rotary)[0]
    want, size, _ = O.rope(x[:, : 4 * dim].contiguous(), positions, f, heads=4, head_dim=dim, start=start, pairing=pairing, scale=1.0)
    d = x.cuda()
    ops.rope(d, d, positions.cuda(), f.cuda(), heads=4, head_dim=dim, start=start, pairing=pairing)
    _close(d[:, : 4 * dim], want, size * 2.0**-21, BF16)
    assert torch.equal(d[:, 4 * dim :].cpu(), x[:, 4 * dim :])
    untouched = torch.ones(4, dim, dtype=torch.bool)
    untouched[:, start : start + rotary] = False
    assert torch.equal(d[:, : 4 * dim][:, untouched.reshape(-1).cuda()].cpu(), x[:, : 4 * dim][:, untouched.reshape(-1)])


def test_rope_strides_and_alignment(cuda_device):
    f = ops.rope_frequencies(64)[0]
    positions = torch.arange(50, dtype=torch.int32) * 31
    wide = _randn(50, 2 * 64 + 9, seed=7, dtype=F16)
    for offset in range(9):  # every alignment of the rows
        x = wide[:, offset : offset + 128]
        want, size, _ = O.rope(x, positions, f, heads=2, head_dim=64, start=0, pairing="pairs", scale=1.0)
        d, o = wide.cuda(), torch.full((50, 200), 7.0, dtype=F16, device="cuda")
        ops.rope(d[:, offset : offset + 128], o[:, 3 : 3 + 128], positions.cuda(), f.cuda(), heads=2, head_dim=64)
        _close(o[:, 3 : 3 + 128], want, size * 2.0**-21, F16)
        assert (o[:, :3] == 7).all() and (o[:, 131:] == 7).all()


def test_rope_no_rows_or_heads(cuda_device):
    f = ops.rope_frequencies(8)[0].cuda()
    x = torch.empty(0, 32, dtype=F16, device="cuda")
    ops.rope(x, x, torch.empty(0, dtype=torch.int32, device="cuda"), f, heads=4, head_dim=8)
    y = torch.ones(3, 32, dtype=F16, device="cuda")
    ops.rope(y, y, torch.arange(3, device="cuda"), f, heads=0, head_dim=8)
    assert (y == 1).all()


def test_rope_non_finite_values_stay_in_their_pair(cuda_device):
    x = _randn(4, 64, seed=8, dtype=F32)
    x[1, 6], x[2, 9] = math.inf, math.nan
    d = x.cuda()
    o = torch.empty_like(d)
    ops.rope(d, o, torch.arange(1, 5, device="cuda"), ops.rope_frequencies(64)[0].cuda(), heads=1, head_dim=64)
    finite = o.isfinite().cpu()
    assert not finite[1, 6:8].any() and not finite[2, 8:10].any()
    assert finite.sum() == 4 * 64 - 4


# ---------------------------------------------------------------- block end
def _end_inputs(rows, cols, xt, yt, *, gate=None, seed=0, scale=True):
    x, y = _randn(rows, cols, seed=seed, dtype=xt, scale=2), _randn(rows, cols, seed=seed + 1, scale=0.7).add(0.1).to(yt)
    kw = dict(post_weight=1 + _randn(cols, seed=seed + 2, scale=0.1), pre_weight=1 + _randn(cols, seed=seed + 3, scale=0.1),
              post_bias=_randn(cols, seed=seed + 4, scale=0.1), pre_bias=_randn(cols, seed=seed + 5, scale=0.1))
    if gate is not None:
        per, gcols, gt = gate
        kw |= dict(gate=_randn(-(-rows // per) if rows else 1, cols if gcols else 1, seed=seed + 6, dtype=gt), gate_rows=per)
    if scale:
        kw["scale"] = 0.1 + _randn(cols, seed=seed + 7, scale=0.02)
    return x, y, kw


def _end(x, y, kw, *, out=None, normed=None, dx=None, dy=None):
    want, err, n, n_err = O.block_end(x, y, **kw)
    dx, dy = x.cuda() if dx is None else dx, y.cuda() if dy is None else dy
    out = torch.empty_like(dx) if out is None else out
    if kw.get("pre") and normed is None:
        normed = torch.empty_like(dy)
    ops.norm_residual(dx, dy, out, normed=normed, **{k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()})
    _close(out, want, err, x.dtype)
    if normed is not None:
        _close(normed, n, n_err, y.dtype)
    return out, normed


TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)]


@pytest.mark.parametrize(("xt", "yt"), TYPES)
@pytest.mark.parametrize(("rows", "cols"), [(1, 1), (1, 1024), (3, 7), (5, 257), (130, 768), (4, 2730), (2, 4097), (3, 8192), (2, 16384), (2500, 40), (2400, 1024),
                                            (2400, 515), (9601, 40), (3001, 250), (1201, 770), (901, 1000), (701, 2056)])
def test_block_end(cuda_device, rows, cols, xt, yt):
    x, y, kw = _end_inputs(rows, cols, xt, yt, gate=(3, True, F32))
    _end(x, y, kw | dict(post="rms", pre="layer", gate_act="tanh", alpha=0.875))


@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("pre", [None, "rms", "layer"])
@pytest.mark.parametrize("act", [None, "sigmoid", "tanh"])
def test_block_end_norms_and_gates(cuda_device, post, pre, act):
    for cols in (1024, 518):
        x, y, kw = _end_inputs(67, cols, BF16, BF16, gate=(1, True, BF16), scale=False)
        _end(x, y, kw | dict(post=post, pre=pre, gate_act=act))


@pytest.mark.parametrize("gate", [(67, False, F32), (5, True, F32), (1, True, F32), (67, False, F16), (7, True, F16), (1, False, F16), (1 << 40, True, F32)])
@pytest.mark.parametrize("cols", [512, 301])
def test_block_end_gate_layouts(cuda_device, gate, cols):
    x, y, kw = _end_inputs(67, cols, F16, F16, gate=gate)
    _end(x, y, kw | dict(post="layer", pre="rms", gate_act="sigmoid"))


def test_block_end_without_weights(cuda_device):
    x, y, _ = _end_inputs(33, 400, F32, F32)
    _end(x, y, dict(post="layer", pre="rms"))
    _end(x, y, dict())
    _end(x, y, dict(post="rms", pre="layer", eps=1e-3, pre_eps=1e-5))


@pytest.mark.parametrize(("xt", "yt"), TYPES)
@pytest.mark.parametrize("cols", [256, 250])
def test_block_end_rows_off_a_chunk(cuda_device, xt, yt, cols):
    """Every alignment of the rows, the same in all matrices or different ones; nothing beside the rows is written."""
    x, y, kw = _end_inputs(21, cols, xt, yt, gate=(1, True, yt))
    kw |= dict(post="layer", pre="rms", gate_act="sigmoid")
    for pitch in (264, 267, 270):
        for offset in range(0, 8):
            for other in (offset, (offset + 3) % 8):
                dx, out = (torch.full((21, pitch + 8), 9.0, dtype=xt, device="cuda") for _ in range(2))
                dy, normed = (torch.full((21, pitch + 8), 9.0, dtype=yt, device="cuda") for _ in range(2))
                at, there = slice(offset, offset + cols), slice(other, other + cols)
                dx[:, at], dy[:, at] = x.cuda(), y.cuda()
                _end(x, y, kw, dx=dx[:, at], dy=dy[:, at], out=out[:, there], normed=normed[:, at])
                for t, s in ((out, there), (normed, at)):
                    beside = torch.ones(pitch + 8, dtype=torch.bool, device="cuda")
                    beside[s] = False
                    assert (t[:, beside] == 9).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize(("rows", "cols", "plain"), [(21, 258, True), (700, 518, True), (900, 770, True), (130, 2050, False), (400, 2730, True), (9, 6002, False),
                                                     (3, 16370, False), (3, 16384, False)])
def test_block_end_rows_equally_off_16_bytes(cuda_device, rows, cols, plain, dtype):
    """Rows of every matrix, the gate's among them, begin equally far off 16 bytes, each row differently; with few parameters and
    many; nothing beside the rows is written, and what is there (NaN) does not count."""
    x, y, kw = _end_inputs(rows, cols, dtype, dtype, gate=(1, True, dtype), scale=not plain)
    kw |= dict(post="layer", gate_act="sigmoid") | (dict(post_weight=None, post_bias=None, pre_weight=None, pre_bias=None) if plain else dict(pre="rms"))
    want, err, n, n_err = O.block_end(x, y, **kw)
    for pitch, offset in ((cols + 8, 2), (cols + 10, 6), (cols + 12, 1), (cols + 14, 0)):
        at = slice(offset, offset + cols)
        dx, dy, gate = (torch.full((rows, pitch), math.nan, dtype=dtype, device="cuda") for _ in range(3))
        out, normed = (torch.full((rows, pitch), 9.0, dtype=dtype, device="cuda") for _ in range(2))
        dx[:, at], dy[:, at], gate[:, at] = x.cuda(), y.cuda(), kw["gate"].cuda()
        on_device = {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()} | dict(gate=gate[:, at])
        ops.norm_residual(dx[:, at], dy[:, at], out[:, at], normed=None if plain else normed[:, at], **on_device)
        _close(out[:, at], want, err, dtype)
        if not plain:
            _close(normed[:, at], n, n_err, dtype)
        beside = torch.ones(pitch, dtype=torch.bool, device="cuda")
        beside[at] = False
        assert (out[:, beside] == 9).all() and (normed[:, beside] == 9).all()


@pytest.mark.parametrize("cols", [1024, 99, 5000])
def test_block_end_in_place(cuda_device, cols):
    x, y, kw = _end_inputs(300, cols, BF16, BF16)
    dx, dy = x.cuda(), y.cuda()
    _end(x, y, kw | dict(post="rms", pre="rms"), dx=dx, dy=dy, out=dx, normed=dy)


def test_block_end_no_rows_or_columns(cuda_device):
    for rows, cols in ((0, 64), (3, 0)):
        x, y, kw = _end_inputs(rows, cols, F16, F16)
        _end(x, y, kw | dict(post="rms", pre="layer"))


def test_block_end_rows_are_apart(cuda_device):
    """A row with NaN or infinity, or of one value, leaves the others alone; a constant row's LayerNorm is its bias."""
    x, y, kw = _end_inputs(40, 300, F32, F32, scale=False)
    y[3, 5], x[7, 0] = math.nan, math.inf
    y[11] = 2.5
    dx, dy, out, normed = x.cuda(), y.cuda(), torch.empty(40, 300, device="cuda"), torch.empty(40, 300, device="cuda")
    ops.norm_residual(dx, dy, out, normed=normed, post="layer", pre="rms", **{k: v.cuda() for k, v in kw.items()})
    keep = [i for i in range(40) if i not in (3, 7)]
    want, err, n, n_err = O.block_end(x[keep], y[keep], post="layer", pre="rms", **kw)
    _close(out[keep], want, err, F32)
    _close(normed[keep], n, n_err, F32)
    assert normed[3].isnan().all() and not out[7].isfinite().all()
    assert torch.equal(out[11].cpu(), x[11] + kw["post_bias"])


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("cols", [512, 301])
@pytest.mark.parametrize(("xt", "yt"), [(F16, F16), (F32, F32)])
def test_block_end_gates_of_any_size(cuda_device, act, cols, xt, yt):
    """Gates far from zero on both sides and next to it; a NaN is one."""
    x, y, kw = _end_inputs(40, cols, xt, yt, gate=(1, True, yt), scale=False)
    sizes = torch.tensor([0.0, 1e-4, -3e-3, 0.1, -0.34, 0.36, 2.0, -6.0, 11.0, -20.0, 60.0, -90.0, 300.0, -2e4, math.inf, -math.inf])
    kw["gate"] = sizes[torch.arange(40 * cols) % 16].reshape(40, cols).to(yt)
    out, _ = _end(x, y, kw | dict(gate_act=act))
    gate = kw["gate"].cuda()
    gate[5, 7] = math.nan
    ops.norm_residual(x.cuda(), y.cuda(), out, gate=gate, gate_act=act)
    assert out[5, 7].isnan() and out.isnan().sum() == 1


def test_block_end_large_mean(cuda_device):
    """LayerNorm of values far from zero: the variance comes from centred values."""
    x, y, kw = _end_inputs(9, 1000, F32, F32)
    _end(x, y + 4096.0, kw | dict(post="layer", pre="layer"))


# ---------------------------------------------------------------- cross attention
def _pieces(nq, nk, mask=None, k_at=None):
    """Rows of every sequence from lengths; keys that the mask leaves out are dropped."""
    out, qa, ka = [], 0, 0
    for i, (a, b) in enumerate(zip(nq, nk)):
        s = ka if k_at is None else k_at[i]
        keys = torch.arange(s, s + b)
        out.append((torch.arange(qa, qa + a), keys if mask is None else keys[mask[s : s + b]]))
        qa, ka = qa + a, ka + b
    return out


def _starts(n, at=0):
    return torch.tensor([at] + n).cumsum(0).int()


def _check_attention(out, q, k, v, *, heads, kv_heads, dim, pieces, scale=None, finite=None):
    scale = dim**-0.5 if scale is None else scale
    want, size, dot, longest = O.attention(q, k, v, heads=heads, kv_heads=kv_heads, head_dim=dim, pieces=pieces, scale=scale)
    vmax = max([v[ki].abs().max().item() for _, ki in pieces if len(ki)], default=0.0)
    err = size * (_half_ulp(q.dtype) + 2 * 2.0**-20 * dot + 2.0**-20) + longest * 2.0**-32 * vmax
    rows = torch.cat([qi for qi, _ in pieces]) if pieces else torch.arange(0)
    _close(out[rows.cuda()], want[rows], err[rows], q.dtype)


def _attend(q, k, v, **kw):
    out = torch.full((q.shape[0], q.shape[1]), 9.0, dtype=q.dtype, device="cuda")
    ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), out, **{n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()})
    return out


def _qkv(tq, tk, heads, kv_heads, dim, dtype, seed=0):
    return _randn(tq, heads * dim, seed=seed, dtype=dtype), _randn(tk, kv_heads * dim, seed=seed + 1, dtype=dtype), _randn(tk, kv_heads * dim, seed=seed + 2, dtype=dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize(("sequences", "nq", "nk", "heads", "kv_heads", "dim"), [
    (1, 1, 1, 1, 1, 16), (1, 1, 1025, 16, 16, 64), (1, 1, 5000, 2, 1, 128), (3, 1, 63, 4, 4, 64), (2, 1, 64, 4, 2, 32), (2, 2, 65, 4, 1, 96),
    (1, 5, 129, 6, 2, 80), (4, 17, 127, 2, 2, 64), (2, 33, 128, 3, 3, 48), (2, 64, 1000, 2, 2, 128), (2, 7, 300, 16, 2, 64), (1, 65, 200, 2, 2, 64),
    (3, 128, 256, 2, 1, 64), (2, 129, 257, 4, 4, 128), (1, 256, 128, 2, 2, 112), (2, 300, 1025, 4, 2, 64), (1, 1025, 700, 2, 2, 64), (1, 513, 1, 2, 2, 64),
    (5, 257, 130, 3, 1, 128), (1, 200, 3000, 1, 1, 32), (40, 90, 40, 8, 8, 64), (70, 260, 150, 4, 2, 64), (200, 3, 70, 4, 2, 128)])
def test_attention(cuda_device, no_device_error, sequences, nq, nk, heads, kv_heads, dim, dtype):
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, kv_heads, dim, dtype)
    out = _attend(q, k, v, heads=heads, kv_heads=kv_heads, head_dim=dim, sequences=sequences)
    _check_attention(out, q, k, v, heads=heads, kv_heads=kv_heads, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences))


RAGGED = {
    "short": ([1, 3, 2, 7, 1], [10, 0, 64, 200, 1]),
    "long": ([300, 1, 0, 129, 700], [100, 1000, 50, 0, 257]),
    "few read much": ([1, 1, 1], [5000, 1, 2049]),
    "uneven": ([1, 1, 1, 1, 1000], [64, 65, 63, 1, 190]),
    "uneven the other way": ([900, 500, 400] + [1] * 12, [100] * 15),
    "nothing": ([0, 0, 5], [7, 0, 0]),
    "short on average": ([2, 1, 3] + [1] * 20, [900, 0, 130] + [3] * 20),
    "queries of one tile and of two": ([128, 129, 1, 256, 257, 384, 100], [128, 129, 300, 64, 257, 700, 1000]),
    "many": ([i % 5 for i in range(150)], [(7 * i) % 90 for i in range(150)]),
    "many long": ([(37 * i) % 300 for i in range(40)], [(53 * i) % 400 for i in range(40)]),
}


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize(("heads", "kv_heads", "dim", "dtype"), [(4, 4, 64, F16), (6, 2, 128, BF16), (2, 1, 80, F16)])
@pytest.mark.parametrize("name", RAGGED)
def test_attention_ragged(cuda_device, no_device_error, name, heads, kv_heads, dim, dtype, masked):
    """Sequences packed with rows before, behind and between nothing; what takes no part is NaN or infinite, and rows
    outside the sequences keep what they held."""
    nq, nk = RAGGED[name]
    before, behind = 3, 130
    q, k, v = _qkv(sum(nq) + before + behind, sum(nk) + before + behind, heads, kv_heads, dim, dtype)
    mask = None
    if masked:
        g = torch.Generator().manual_seed(9)
        mask = torch.rand(k.shape[0], generator=g) < 0.6
        mask[before : before + nk[0]] = False  # the first sequence has nothing left
        at = before + sum(nk[:-1])
        mask[at : at + 300] = mask[at : at + 300].clone().fill_(False)  # a stretch of whole tiles
    ks = _starts(nk, before)
    pieces = [(qi + before, ki) for qi, ki in _pieces(nq, nk, mask, [int(s) for s in ks[:-1]])]
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for _, ki in pieces:
        used[ki] = True
    k[~used], v[~used] = math.nan, math.inf
    v[~used, ::2] = math.nan
    out = _attend(q, k, v, heads=heads, kv_heads=kv_heads, head_dim=dim, q_start=_starts(nq, before), k_start=ks, mask=mask)
    _check_attention(out, q, torch.where(used[:, None], k, 0), torch.where(used[:, None], v, 0), heads=heads, kv_heads=kv_heads, dim=dim, pieces=pieces)
    assert (out[:before] == 9).all() and (out[before + sum(nq) :] == 9).all()
    for qi, ki in pieces:
        if len(ki) == 0 and len(qi):
            assert (out[qi.cuda()] == 0).all()


@pytest.mark.parametrize(("sequences", "dim"), [(320, 64), (321, 64), (320, 80), (321, 80)])
def test_attention_of_many_sequences_of_many_queries(cuda_device, no_device_error, sequences, dim):
    """As many sequences as are put in order by their lengths, and one more; equal lengths and none among them."""
    nq, nk = [(37 * i) % 390 for i in range(sequences)], [(53 * i) % 100 // 8 * 8 for i in range(sequences)]
    q, k, v = _qkv(sum(nq), sum(nk), 2, 2, dim, F16)
    out = _attend(q, k, v, heads=2, kv_heads=2, head_dim=dim, q_start=_starts(nq, 0), k_start=_starts(nk, 0))
    _check_attention(out, q, k, v, heads=2, kv_heads=2, dim=dim, pieces=_pieces(nq, nk))


@pytest.mark.parametrize("nq", [1, 20, 150])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_padded(cuda_device, no_device_error, nq, dtype):
    """Equal pieces of which the first k_len keys take part, lengths out of range included; mixed with q_start."""
    lens = [1, 0, 77, 200, 128, 999, -5]
    kept = [min(max(n, 0), 200) for n in lens]
    q, k, v = _qkv(7 * nq, 7 * 200, 4, 2, 64, dtype)
    k_at = [200 * i for i in range(7)]
    pieces = _pieces([nq] * 7, kept, None, k_at)
    used = torch.zeros(1400, dtype=torch.bool)
    for _, ki in pieces:
        used[ki] = True
    k[~used], v[~used] = math.inf, math.nan
    kw = dict(heads=4, kv_heads=2, head_dim=64, k_len=torch.tensor(lens).int())
    want = (q, torch.where(used[:, None], k, 0), torch.where(used[:, None], v, 0))
    for more in (dict(), dict(sequences=7), dict(q_start=_starts([nq] * 7))):
        out = _attend(q, k, v, **kw, **more)
        _check_attention(out, *want, heads=4, kv_heads=2, dim=64, pieces=pieces)


@pytest.mark.parametrize("nq", [1, 150])
def test_attention_starts_beyond_the_rows(cuda_device, no_device_error, nq):
    """Starts past the rows that there are (or before the first) are taken back to them."""
    q, k, v = _qkv(2 * nq, 300, 2, 2, 64, F16)
    out = _attend(q, k, v, heads=2, head_dim=64, q_start=torch.tensor([-4, nq, 5 * nq + 9]).int(), k_start=torch.tensor([-100, 100, 1 << 30]).int())
    _check_attention(out, q, k, v, heads=2, kv_heads=2, dim=64, pieces=_pieces([nq, nq], [100, 200]))


@pytest.mark.parametrize(("sequences", "nq", "nk", "dim"), [(150, 300, 130, 128), (150, 100, 400, 128), (160, 130, 200, 64), (300, 40, 300, 64), (9, 3000, 70, 64), (160, 1, 100, 32)])
def test_attention_of_many_items_in_a_row(cuda_device, no_device_error, sequences, nq, nk, dim):
    """More items than SMs, one behind the other in the CTAs' pipelines."""
    q, k, v = _qkv(sequences * nq, sequences * nk, 2, 1, dim, BF16)
    out = _attend(q, k, v, heads=2, kv_heads=1, head_dim=dim, sequences=sequences)
    _check_attention(out, q, k, v, heads=2, kv_heads=1, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences))


def test_attention_with_offsets_beyond_32_bits(cuda_device, no_device_error):
    """Keys and values whose rows lie more than 2^32 bytes and 2^31 elements from the first."""
    rows, pitch = 700_000, 4096
    big = torch.empty(rows, pitch, dtype=F16, device="cuda")
    for nq in (1, 300):
        q, k, v = _qkv(nq, 500, 2, 2, 64, F16, seed=nq)
        at = rows - 500
        big[at:, :128], big[at:, 2048:2176] = k.cuda(), v.cuda()
        starts = torch.tensor([at, rows]).int().cuda()
        out = torch.empty(nq, 128, dtype=F16, device="cuda")
        ops.cross_attention(q.cuda(), big[:, :128], big[:, 2048:2176], out, heads=2, head_dim=64, k_start=starts, q_start=torch.tensor([0, nq]).int().cuda())
        _check_attention(out, q, k, v, heads=2, kv_heads=2, dim=64, pieces=_pieces([nq], [500]))


@pytest.mark.parametrize("nq", [2, 140])
def test_attention_views(cuda_device, no_device_error, nq):
    """Keys and values as halves of a packed projection, queries and results in wider rows."""
    heads, dim = 4, 64
    q, kv = _randn(nq, 3 * heads * dim, seed=1, dtype=F16), _randn(333, 2 * heads * dim + 16, seed=2, dtype=F16)
    cols = heads * dim
    out = torch.full((nq, cols + 24), 9.0, dtype=F16, device="cuda")
    dq, dkv = q.cuda(), kv.cuda()
    ops.cross_attention(dq[:, cols : 2 * cols], dkv[:, 8 : 8 + cols], dkv[:, 16 + cols :], out[:, 8 : 8 + cols], heads=heads, head_dim=dim)
    _check_attention(out[:, 8 : 8 + cols], q[:, cols : 2 * cols], kv[:, 8 : 8 + cols], kv[:, 16 + cols :], heads=heads, kv_heads=heads, dim=dim, pieces=_pieces([nq], [333]))
    assert (out[:, :8] == 9).all() and (out[:, 8 + cols :] == 9).all()


@pytest.mark.parametrize("nq", [1, 40, 130])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_large_and_small_scores(cuda_device, no_device_error, nq, dtype):
    """A maximum that grows from tile to tile, a key that takes all the weight, and weights that are nearly equal."""
    q, k, v = _qkv(nq, 1000, 2, 2, 64, dtype)
    k = (k.float() * torch.linspace(0.01, 4, 1000)[:, None]).to(dtype)
    _check_attention(_attend(q, k, v, heads=2, head_dim=64), q, k, v, heads=2, kv_heads=2, dim=64, pieces=_pieces([nq], [1000]))
    for scale in (1e-6, 1.0):
        out = _attend(q, k, v, heads=2, head_dim=64, scale=scale)
        _check_attention(out, q, k, v, heads=2, kv_heads=2, dim=64, pieces=_pieces([nq], [1000]), scale=scale)
    k[500] = 60 * q[0, :128].sign()
    _check_attention(_attend(q, k, v, heads=2, head_dim=64), q, k, v, heads=2, kv_heads=2, dim=64, pieces=_pieces([nq], [1000]))


@pytest.mark.parametrize("nq", [1, 130])
def test_attention_of_non_finite_keys_and_queries(cuda_device, no_device_error, nq):
    """A NaN in one sequence's key, or in a query, stays with what reads it."""
    q, k, v = _qkv(2 * nq, 2 * 100, 2, 2, 64, F16)
    want = q.clone(), k.clone(), v.clone()
    k[150, 3] = math.nan  # sequence 1, head 0
    q[0, 64] = math.nan  # sequence 0, query 0, head 1
    out = _attend(q, k, v, heads=2, head_dim=64, sequences=2)
    assert out[nq:, :64].isnan().all() and out[0, 64:].isnan().all()
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[nq:, :64] = True
    bad[0, 64:] = True
    good, size, dot, _ = O.attention(*want, heads=2, kv_heads=2, head_dim=64, pieces=_pieces([nq] * 2, [100] * 2), scale=0.125)
    fixed = torch.where(bad.cpu(), good, out.double().cpu())
    _close(fixed, good, size * (2.0**-11 + 2 * 2.0**-20 * dot + 2.0**-20) + 100 * 2.0**-32 * 5, F16)


@pytest.mark.parametrize("nq", [1, 200])
def test_attention_without_keys_or_queries(cuda_device, nq):
    q, k, v = _qkv(nq, 0, 2, 2, 64, F16)
    assert (_attend(q, k, v, heads=2, head_dim=64) == 0).all()
    out = _attend(q[:0], *_qkv(0, 50, 2, 2, 64, F16)[1:], heads=2, head_dim=64)
    assert out.shape == (0, 128)


@pytest.mark.parametrize(("nq", "nk"), [(1, 3000), (30, 1025), (300, 600)])
def test_attention_same_bits_every_time_and_on_other_streams(cuda_device, no_device_error, nq, nk):
    heads, dim = 4, 64
    sets = [tuple(t.cuda() for t in _qkv(nq, nk, heads, heads, dim, BF16, seed=10 * i)) for i in range(4)]
    outs = [torch.empty_like(s[0]) for s in sets]
    for s, o in zip(sets, outs):
        ops.cross_attention(*s, o, heads=heads, head_dim=dim)
    torch.cuda.synchronize()
    again = [torch.empty_like(o) for o in outs]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for st, s, o in zip(streams, sets, again):
            with torch.cuda.stream(st):
                ops.cross_attention(*s, o, heads=heads, head_dim=dim)
    torch.cuda.synchronize()
    for a, b in zip(outs, again):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- together
def _reading_block(s, image, tokens, out, work):
    """q rotated, cross attention to the image's tokens, block end; into `out` and work["normed"]."""
    heads, dim = s["heads"], s["dim"]
    ops.rope(tokens, work["q"], s["positions"], s["frequencies"], heads=heads, head_dim=dim, pairing="halves", scale=s["scale"])
    kv = heads * dim
    ops.rope(image[:, :kv], work["k"], s["patches"], s["axial"], heads=heads, head_dim=dim)
    ops.cross_attention(work["q"], work["k"], image[:, kv:], work["o"], heads=heads, head_dim=dim, q_start=s["q_start"], k_start=s["k_start"], mask=s["mask"])
    ops.norm_residual(tokens, work["o"], out, post="rms", post_weight=s["w"], gate=s["gate"], gate_act="tanh", gate_rows=1 << 20, normed=work["normed"],
                      pre="layer", pre_weight=s["w"], pre_bias=s["b"])


def _reading_state(nq, nk, seed):
    heads, dim = 4, 64
    T, K = sum(nq), sum(nk)
    f, scale = ops.rope_frequencies(dim, scaling="yarn", factor=8.0, trained=4096)
    g = torch.Generator().manual_seed(seed)
    return dict(heads=heads, dim=dim, positions=torch.randint(0, 30000, (T,), generator=g), frequencies=f, scale=scale,
                patches=torch.randint(0, 32, (K, 2), generator=g, dtype=torch.int32), axial=ops.rope_frequencies(dim // 2)[0].repeat(2), q_start=_starts(nq), k_start=_starts(nk),
                mask=torch.rand(K, generator=g) < 0.8, w=1 + _randn(256, seed=seed, scale=0.1), b=_randn(256, seed=seed + 1, scale=0.1), gate=_randn(1, 1, seed=seed))


def _reading_oracle(s, image, tokens, nq, nk):
    r = lambda x, p, f, **kw: O.rope(x, p, f, heads=4, head_dim=64, start=0, **kw)[0].to(F16)
    q, k = r(tokens, s["positions"], s["frequencies"], pairing="halves", scale=s["scale"]), r(image[:, :256], s["patches"], s["axial"], pairing="pairs", scale=1.0)
    o = O.attention(q, k, image[:, 256:], heads=4, kv_heads=4, head_dim=64, pieces=_pieces(nq, nk, s["mask"]), scale=0.125)[0].to(F16)
    return O.block_end(tokens, o, post="rms", post_weight=s["w"], gate=s["gate"], gate_act="tanh", gate_rows=1 << 20, pre="layer", pre_weight=s["w"], pre_bias=s["b"])[::2]


@pytest.mark.parametrize("nq", [[1, 1, 1], [3, 200, 150]])
def test_tokens_read_an_image(cuda_device, no_device_error, nq):
    """The operators one behind the other, eager, captured into a graph, and replayed on new inputs while an eager run
    of the same shape goes on beside it. Between the operators values are rounded to fp16, in the oracle too, and may
    fall to the next fp16 number there: 2^-10 of the values (about 4 at most) and of their norms (about 5)."""
    nk = [70, 0, 400]
    s = _reading_state(nq, nk, 3)
    d = {k: v.cuda() if torch.is_tensor(v) else v for k, v in s.items()}
    sets = [(_randn(sum(nk), 512, seed=20 + i, dtype=F16), _randn(sum(nq), 256, seed=30 + i, dtype=F16)) for i in range(3)]
    make = lambda: {n: torch.empty(sum(nk) if n == "k" else sum(nq), 256, dtype=F16, device="cuda") for n in ("q", "k", "o", "normed")}

    def check(i, out, work):
        want, n = _reading_oracle(s, *sets[i], nq, nk)
        assert (out.double().cpu() - want).abs().max() < 5 * 2.0**-9
        assert (work["normed"].double().cpu() - n).abs().max() < 5 * 2.0**-8

    image, tokens, out, work = sets[0][0].cuda(), sets[0][1].cuda(), torch.empty(sum(nq), 256, dtype=F16, device="cuda"), make()
    _reading_block(d, image, tokens, out, work)
    check(0, out, work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _reading_block(d, image, tokens, out, work)
    image.copy_(sets[1][0])
    tokens.copy_(sets[1][1])
    graph.replay()
    other, other_work = torch.empty_like(out), make()
    image2, tokens2 = sets[2][0].cuda(), sets[2][1].cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _reading_block(d, image2, tokens2, other, other_work)
    graph.replay()
    torch.cuda.synchronize()
    check(1, out, work)
    check(2, other, other_work)


# ---------------------------------------------------------------- refusals and ways into the calls
def _every_call():
    """The three calls on one set of tensors, as functions of what to replace."""
    d = "cuda"
    x = torch.zeros(4, 128, dtype=F16, device=d)
    pos, f, w = torch.zeros(4, dtype=torch.int32, device=d), torch.zeros(32, dtype=torch.float64, device=d), torch.ones(128, device=d)
    k = torch.zeros(6, 128, dtype=F16, device=d)
    rope = dict(x=x, out=torch.zeros_like(x), positions=pos, frequencies=f, heads=2, head_dim=64)
    end = dict(x=x, y=torch.zeros_like(x), out=torch.zeros_like(x), post="rms", post_weight=w, normed=torch.zeros_like(x), pre="layer", pre_weight=w, pre_bias=w,
               gate=torch.zeros(4, 1, device=d), gate_act="tanh")
    cross = dict(q=x, k=k, v=k, out=torch.zeros_like(x), heads=2, head_dim=64, q_start=torch.tensor([0, 1, 4]).int().cuda(), k_start=torch.tensor([0, 3, 6]).int().cuda(),
                 k_len=torch.tensor([3, 3]).int().cuda(), mask=torch.ones(6, dtype=torch.bool, device=d))
    return (ops.rope, rope), (ops.norm_residual, end), (ops.cross_attention, cross)


@pytest.mark.parametrize("short", [True, False])
def test_refusals(cuda_device, monkeypatch, short):
    """What a call does not take raises before any launch, through the extension module and without it."""
    if not short:
        monkeypatch.setattr(ops, "_calls", lambda: ops._NoCalls)
    (rope, r), (end, e), (cross, c) = _every_call()
    x, d = r["x"], "cuda"
    for fn, kw in ((rope, r), (end, e), (cross, c)):
        fn(**kw)
    strided = torch.zeros(4, 256, dtype=F16, device=d)[:, ::2]
    for change in (dict(x=x.cpu()), dict(out=x.bfloat16()), dict(out=x[:3]), dict(x=x[:, :100]), dict(x=strided), dict(positions=r["positions"][:3]),
                   dict(positions=r["positions"].float()), dict(positions=r["positions"].cpu()), dict(frequencies=r["frequencies"].half()), dict(frequencies=r["frequencies"][None]),
                   dict(frequencies=r["frequencies"].repeat(2)), dict(frequencies=r["frequencies"][:0]), dict(pairing="both"), dict(start=1), dict(start=-2), dict(head_dim=0),
                   dict(heads=-1), dict(heads=3), dict(positions=torch.zeros(4, 3, dtype=torch.int32, device=d)), dict(positions=torch.zeros(4, 0, dtype=torch.int32, device=d)),
                   dict(x=x.int(), out=x.int())):
        with pytest.raises(RuntimeError):
            rope(**(r | change))
    for change in (dict(x=x.cpu()), dict(y=x.bfloat16()), dict(y=x.float()), dict(out=x.float()), dict(out=x[:3]), dict(normed=None), dict(pre=None), dict(post="other"), dict(pre="other"),
                   dict(post_weight=e["post_weight"][:5]), dict(pre_bias=e["pre_bias"].half()), dict(gate=torch.zeros(3, 1, device=d)), dict(gate=torch.zeros(4, 2, device=d)),
                   dict(gate=x.bfloat16()), dict(gate_act="relu"), dict(gate_rows=0), dict(scale=e["post_weight"].cpu()), dict(y=strided), dict(normed=e["out"]), dict(out=e["y"])):
        with pytest.raises(RuntimeError):
            end(**(e | change))
    for change in (dict(q=x.cpu()), dict(q=x.float()), dict(k=c["k"].bfloat16()), dict(v=c["v"][:5]), dict(out=x[:3]), dict(heads=3), dict(kv_heads=1), dict(heads=0), dict(head_dim=32),
                   dict(head_dim=24, heads=2), dict(q_start=c["q_start"].long()), dict(q_start=c["q_start"].cpu()), dict(k_start=c["k_start"][:2]), dict(k_len=c["q_start"]),
                   dict(mask=c["mask"][:5]), dict(mask=c["mask"].float()), dict(sequences=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(out=x),
                   dict(sequences=4, q_start=None, k_start=None, k_len=None), dict(q=torch.zeros(4, 132, dtype=F16, device=d)[:, :128]), dict(v=strided[:4].repeat(2, 1)[:6, :64])):
        with pytest.raises(RuntimeError):
            cross(**(c | change))


def test_the_short_and_the_long_way_into_these_calls_agree(cuda_device, no_device_error, monkeypatch):
    x, y, kw = _end_inputs(67, 256, F16, F16, gate=(67, False, F32))
    kw = {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()} | dict(post="rms", pre="layer", gate_act="tanh")
    q, k, v = (t.cuda() for t in _qkv(40, 3000, 4, 2, 64, F16))
    f, pos = ops.rope_frequencies(32)[0].cuda(), torch.arange(67, device="cuda")

    def everything():
        o = [torch.full_like(t, 3.0) for t in (x.cuda(), x.cuda(), x.cuda(), q)]
        ops.rope(x.cuda(), o[0], pos, f, heads=4, head_dim=64, start=32, pairing="halves", scale=1.25)
        ops.norm_residual(x.cuda(), y.cuda(), o[1], normed=o[2], **kw)
        ops.cross_attention(q, k, v, o[3], heads=4, kv_heads=2, head_dim=64, sequences=10)
        return o

    def taken(real):
        def call(*args):
            r = real(*args)
            assert r == 0
            return r
        return call

    short = ops._calls()
    with monkeypatch.context() as m:
        for name in ("rope", "norm_residual", "cross_attention"):
            m.setattr(short, name, taken(getattr(short, name)))
        a = everything()
    monkeypatch.setattr(ops, "_calls", lambda: ops._NoCalls)
    for u, w in zip(a, everything()):
        assert torch.equal(u, w)


def test_rows_beyond_32_bits(cuda_device):
    """Rows that start more than 2^32 columns behind the first: rotation and block end."""
    pitch, rows = (1 << 30) + 8, 6
    x = _randn(rows, 256, seed=3, dtype=F16)
    whole = torch.empty(rows * pitch, dtype=F16, device="cuda")
    far = whole.as_strided((rows, 256), (pitch, 1))
    far.copy_(x)
    positions, f = torch.arange(rows, dtype=torch.int32) * 100, ops.rope_frequencies(64)[0]
    want, size, _ = O.rope(x, positions, f, heads=4, head_dim=64, start=0, pairing="halves", scale=1.0)
    ops.rope(far, far, positions.cuda(), f.cuda(), heads=4, head_dim=64, pairing="halves")
    _close(far, want, size * 2.0**-21, F16)
    _, y, kw = _end_inputs(rows, 256, F16, F16)
    far.copy_(x)
    _end(x, y, kw | dict(post="rms"), dx=far, out=far)
    del far, whole
    torch.cuda.empty_cache()


def test_microbench_cross(cuda_device, no_device_error, capsys):
    from foidfinder_b200 import microbench

    microbench.bench_cross(1, 1, 3)
    assert len(capsys.readouterr().out.splitlines()) == 4
