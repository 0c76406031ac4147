"""Cross attention of many queries on the GPU, at sizes that the choice of kernel sends to the tensor-core kernels, with the
kernel that ran asserted, against the 64-bit oracle. Tolerances are those of test_gpu_cross.py; what differs is derived
at the test."""

from __future__ import annotations

import math

import pytest
import torch

from foidfinder_b200 import ops
from oracle import cross as O
from test_gpu_cross import BF16, F16, _attend, _check_attention, _pieces, _qkv, _randn, _starts

pytestmark = pytest.mark.gpu

NARROW, WIDE = "cross_tc64_kernel", "cross_tc_kernel"


def _kernel(dim):
    return NARROW if dim <= 64 else WIDE


@pytest.fixture(scope="module")
def kernels_of(cuda_device):
    """f -> (f(), names of the cross attention kernels that it launched, or None where the profiler sees no kernels at all)."""

    def run(f):
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            r = f()
            torch.cuda.synchronize()
        return r, {e.key for e in prof.key_averages()}

    x = torch.ones(8, device=cuda_device)
    sees = any("elementwise" in n for n in run(lambda: x + 1)[1])

    def named(f):
        r, names = run(f)
        return r, {n for n in names if "cross_" in n} if sees else None

    return named


def _ran(names, kernel):
    """This kernel alone (whole names: one is the beginning of another's)."""
    assert names is None or (len(names) == 1 and kernel + "<" in next(iter(names))), names


def _ran_first(names, kernel):
    """This kernel, perhaps with another that joins its parts."""
    assert names is None or any(kernel + "<" in n for n in names), names


def _levels(tiles, tile, steps):
    """A score for every key: within each tile of keys a step up (nats) from one 32 keys to the next, each tile above the last."""
    out, level = [], 0.0
    for _ in range(tiles):
        for i in range(tile // 32):
            level += steps[i % len(steps)]
            out += [level] * 32
    return torch.tensor(out)


# Nats between one stretch of 32 keys and the next. Growth beyond 8 powers of two (5.5 nats) is what moves the maximum.
STEPS = {
    "every stretch": [6.0, 6.5, 7.0, 6.0],
    "twice per tile": [0.5, 6.0, 0.25, 8.0],
    "the last of a tile": [0.0, 0.25, 0.5, 9.0],
    "hundreds": [90.0, 0.0, 200.0, 50.0],
    "and down again": [12.0, -30.0, 45.0, -20.0],
}


@pytest.mark.parametrize("silent", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize(("dim", "sequences", "nq"), [(64, 16, 300), (64, 36, 100), (128, 16, 300), (128, 16, 100), (80, 12, 200)])
@pytest.mark.parametrize("steps", STEPS)
def test_maxima_that_grow(no_device_error, kernels_of, steps, dim, sequences, nq, dtype, silent):
    """Scores that jump between the stretches of a tile, twice per tile, and from tile to tile, for items of one query tile
    and of two; with `silent` the values of each tile's highest keys are zero, so that the result is what smaller weights
    leave. The first two columns of q are 1 and 1/8, and k's there hold the level in two parts."""
    heads, nk = 8, 290
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, dtype, seed=5)
    k = k / 8  # the random part of a score is small beside a step
    level = _levels(3, 128, STEPS[steps])[:nk].repeat(sequences)
    whole = level.round()
    for h in range(heads):
        q[:, h * dim], q[:, h * dim + 1] = 1.0, 0.125
        k[:, h * dim], k[:, h * dim + 1] = whole.to(dtype), ((level - whole) * 8).to(dtype)
    if silent:
        v[torch.arange(sequences * nk) % nk % 128 >= 96] = 0
        v[torch.arange(sequences * nk) % nk >= 256] = 0
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences, scale=1.0))
    _ran(names, _kernel(dim))
    _check_attention(out, q, k, v, heads=heads, kv_heads=heads, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences), scale=1.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_are_rounded_once(no_device_error, kernels_of, dim, dtype):
    """Three keys take part, in three stretches of 32: one that sets the maximum, one near it, whose value alone is not zero, and
    one far above both. The result is the second key's weight: rounded to 16 bits when it is stored, and once more in the
    output, and not when the third key scales it down."""
    sequences, heads, nq, nk = 16, 8, 300, 128
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, dtype, seed=11)
    q[:], k[:], v[:] = 0, 0, 0
    for h in range(heads):
        q[:, h * dim] = 1.0
        q[:, h * dim + 1 : h * dim + 3] = torch.rand(sequences * nq, 2, generator=torch.Generator().manual_seed(h)).to(dtype)
        for b in range(sequences):
            k[b * nk + 32, h * dim + 1] = 2.0  # between 0 and 2
            k[b * nk + 64, h * dim], k[b * nk + 64, h * dim + 2] = 8.0, 2.0  # between 8 and 10: at least 8 powers of two above
    v[32::nk] = 1 + torch.rand(sequences, heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype)
    mask = torch.zeros(sequences * nk, dtype=torch.bool)
    for i in (0, 32, 64):
        mask[i::nk] = True
    at = [nk * i for i in range(sequences)]
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences, scale=1.0, mask=mask))
    _ran(names, _kernel(dim))
    _check_attention(out, q, k, v, heads=heads, kv_heads=heads, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences, mask, at), scale=1.0)


# What reaches each kernel: sequences, queries and keys of each, heads of how many columns.
EACH_KERNEL = {"cross_few_kernel": [(3, 1, 300, 64), (2, 1, 1100, 128), (2, 20, 150, 80), (5, 4, 40, 16)], NARROW: [(16, 300, 290, 64), (48, 100, 290, 48)],
               WIDE: [(16, 300, 290, 128), (16, 100, 290, 80)]}
EACH_KERNEL = [pytest.param(name, *shape, id="-".join(map(str, (name, *shape)))) for name, shapes in EACH_KERNEL.items() for shape in shapes]


@pytest.mark.parametrize("order", ["rising", "falling", "mixed", "late"])
@pytest.mark.parametrize(("dtype", "q0", "k0", "apart"), [
    pytest.param(dtype, q0, k0, apart, id=f"{str(dtype)[6:]}-{math.copysign(math.log2(abs(q0 * k0)), q0 * k0):.0f}")
    for dtype, q0, k0, apart in (
        (F16, 2.0**6, 2.0**10, 1.0), (F16, 2.0**14, 2.0**10, 1.0), (F16, 2.0**14, -(2.0**10), 1.0), (F16, 2.0**14, -(2.0**14), 16.0), (F16, 2.0**15, 2.0**14, 16.0),
        (BF16, 2.0**20, 2.0**20, 2.0**13), (BF16, 2.0**40, -(2.0**50), 2.0**43), (BF16, -(2.0**60), 2.0**60, 2.0**53))])
@pytest.mark.parametrize(("kernel", "sequences", "nq", "nk", "dim"), EACH_KERNEL)
def test_scores_far_from_zero(no_device_error, kernels_of, kernel, sequences, nq, nk, dim, dtype, q0, k0, apart, order):
    """Scores of up to 2^120, whose fractions 32 bits do not hold, exact multiples of q0 apart (64 at least, so the second best has no
    weight): the result is the mean of the best key's values and those of its doubles. Their weights are equal: one
    rounding to 16 bits, and the sum's in 32; then the output's."""
    heads = 8
    n = torch.arange(nk) % 100
    late = torch.arange(nk) > nk - 10
    level = {"rising": n, "falling": 99 - n, "mixed": 37 * n % 100, "late": n * late}[order].double()
    keys = k0 + apart * level
    if order == "late" and k0 > 0:
        keys = torch.where(late, keys, 0.0)
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, dtype, seed=3)
    q[:], k[:] = 0, 0
    q[:, ::dim] = q0
    k[:, ::dim] = keys.to(dtype).repeat(sequences)[:, None]
    assert torch.equal(k[:nk, 0].double(), keys)
    top = (q0 * keys == (q0 * keys).max()).nonzero()[:, 0]
    best = v.reshape(sequences, nk, heads * dim)[:, top].double()
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences, scale=1.0))
    _ran_first(names, kernel)
    want, size = best.mean(1)[:, None], best.abs().mean(1)[:, None]
    half = torch.finfo(dtype).eps / 2
    off = (out.double().cpu().reshape(sequences, nq, -1) - want).abs()
    assert (off <= size * (half + 2.0**-20) + want.abs() * half * (1 + half) + 2.0**-25).all(), off.max()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize(("kernel", "sequences", "nq", "nk", "dim"), EACH_KERNEL)
def test_scores_far_from_zero_and_near_each_other(no_device_error, kernels_of, kernel, sequences, nq, nk, dim, dtype):
    """Scores from 2^21 to 2^22 (exact, in steps of 2^14) times scale 2^-14: the best has most of the weight, its neighbours e^-1,
    e^-2 and so on. And the same ones 2^24 times as large, where the best has all. Exponents are exact but for scale *
    log2(e), within 2^-23 of itself: times at most 128 * 1.45, and times ln 2 in a weight, that is 2^-15."""
    heads = 8
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, dtype, seed=7)
    level = 37 * torch.arange(nk) % 100 + 128
    q[:], k[:] = 0, 0
    q[:, ::dim] = 2.0**7
    k[:, ::dim] = (2.0**7 * level).to(dtype).repeat(sequences)[:, None]
    at = [slice(i * nk, (i + 1) * nk) for i in range(sequences)]
    pieces = [(slice(i * nq, (i + 1) * nq), s) for i, s in enumerate(at)]
    half = torch.finfo(dtype).eps / 2
    for scale in (2.0**-14, 2.0**10):
        (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences, scale=scale))
        _ran_first(names, kernel)
        want, size, _, _ = O.attention(q, k, v, heads=heads, kv_heads=heads, head_dim=dim, pieces=pieces, scale=scale)
        off = (out.double().cpu() - want).abs()
        assert (off <= size * (half + 2 * 2.0**-15 + 2.0**-20) + want.abs() * half * (1 + half) + nk * 2.0**-32 * 5 + 2.0**-25).all(), off.max()


@pytest.mark.parametrize("size", [3e38, 1e30, 1e-25])
@pytest.mark.parametrize(("kernel", "sequences", "nq", "nk", "dim"), EACH_KERNEL)
def test_values_of_any_size(no_device_error, kernels_of, kernel, sequences, nq, nk, dim, size):
    """bf16 values next to the type's largest, and far below 1: sums of weights times values stay numbers of 32 bits. (Scores near each
    other, so that all weights count. The smallest products are off by f32's smallest normal number at most, 2^-126, where
    1e-25 times a weight of 2^-28 is 2^-111: within the 2^-9 of a weight's rounding, which few come near.)"""
    heads = 8
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, BF16, seed=13)
    q = q / 16
    v = (v.float().clamp(-1, 1) * size).to(BF16)
    v[::nk] = size
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences))
    _ran_first(names, kernel)
    assert out.isfinite().all()
    pieces = [(slice(i * nq, (i + 1) * nq), slice(i * nk, (i + 1) * nk)) for i in range(sequences)]
    want, magnitude, dot, _ = O.attention(q, k, v, heads=heads, kv_heads=heads, head_dim=dim, pieces=pieces, scale=dim**-0.5)
    off, half = (out.double().cpu() - want).abs(), 2.0**-9
    assert (off <= magnitude * (half + 2 * 2.0**-20 * dot + 2.0**-20) + want.abs() * half * (1 + half)).all(), (off / magnitude).max()


def _check(out, q, k, v, *, heads, kv_heads=None, dim, pieces):
    _check_attention(out, q, k, v, heads=heads, kv_heads=kv_heads or heads, dim=dim, pieces=pieces)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim", range(16, 129, 16))
@pytest.mark.parametrize(("sequences", "nq", "nk", "heads", "kv_heads"), [(37, 500, 130, 2, 2), (37, 250, 130, 4, 1), (74, 128, 65, 2, 2), (2, 700, 1500, 48, 16), (37, 250, 1, 4, 4)])
def test_every_head_size(no_device_error, kernels_of, sequences, nq, nk, heads, kv_heads, dim, dtype):
    """Items of one query tile and of two, last tiles of one query and of few, keys that end within a step, and longer than the
    ring of loads."""
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, kv_heads, dim, dtype)
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, kv_heads=kv_heads, head_dim=dim, sequences=sequences))
    _ran(names, _kernel(dim))
    _check(out, q, k, v, heads=heads, kv_heads=kv_heads, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences))


@pytest.mark.parametrize(("dim", "heads"), [(64, 32), (128, 16)])
def test_more_items_than_are_looked_up_ahead(no_device_error, kernels_of, dim, heads):
    """More than 16 items for each of 148 CTAs."""
    sequences, nq, nk = 151, 128, 200
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, F16)
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences))
    _ran(names, _kernel(dim))
    _check(out, q, k, v, heads=heads, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nk", [1, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 192, 193, 255, 257, 511, 513, 1000])
@pytest.mark.parametrize("nq", [100, 128, 129, 256, 257])
def test_every_end_of_a_tile(no_device_error, kernels_of, nq, nk, dim):
    sequences, heads = 37, 4 if nq <= 256 else 2  # 148 items
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, 2, dim, BF16)
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, kv_heads=2, head_dim=dim, sequences=sequences))
    _ran(names, _kernel(dim))
    _check(out, q, k, v, heads=heads, kv_heads=2, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize(("sequences", "heads", "kv_heads", "dim"), [(40, 16, 16, 64), (40, 16, 4, 128), (40, 12, 2, 48), (330, 4, 2, 64), (700, 4, 1, 80)])
def test_packed(no_device_error, kernels_of, sequences, heads, kv_heads, dim, dtype, masked):
    """Sequences of any lengths, none among them, packed with rows before and behind; a mask that leaves some of them nothing. What
    takes no part is NaN or infinite, and rows outside the sequences stay. (Items are many and short: the CTAs walk them, up to 33 each.)"""
    nq, nk = [(137 * i) % 390 for i in range(sequences)], [(253 * i) % 700 * (i % 9 != 4) for i in range(sequences)]
    if sequences > 300:
        nk = [n // 8 for n in nk]
    before, behind = 5, 200
    q, k, v = _qkv(sum(nq) + before + behind, sum(nk) + before + behind, heads, kv_heads, dim, dtype)
    ks = _starts(nk, before)
    mask = None
    if masked:
        mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(4)) < 0.6
        for b in range(0, sequences, 7):
            mask[ks[b] : ks[b + 1]] = False
        at = int(ks[sequences // 2])
        mask[at : at + 500] = False  # whole tiles
    pieces = [(qi + before, ki) for qi, ki in _pieces(nq, nk, mask, [int(s) for s in ks[:-1]])]
    used = torch.zeros(k.shape[0], dtype=torch.bool)
    for _, ki in pieces:
        used[ki] = True
    k[~used], v[~used] = math.nan, math.inf
    v[~used, ::2] = math.nan
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, kv_heads=kv_heads, head_dim=dim, q_start=_starts(nq, before), k_start=ks, mask=mask))
    _ran(names, _kernel(dim))
    _check(out, q, torch.where(used[:, None], k, 0), torch.where(used[:, None], v, 0), heads=heads, kv_heads=kv_heads, dim=dim, pieces=pieces)
    assert (out[:before] == 9).all() and (out[before + sum(nq) :] == 9).all()
    for qi, ki in pieces:
        if len(ki) == 0 and len(qi):
            assert (out[qi.cuda()] == 0).all()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("sequences", [20, 320, 321, 400])
@pytest.mark.parametrize("dim", [64, 80])
def test_packed_in_any_order(no_device_error, kernels_of, dim, sequences, masked):
    """Enough keys (450 on average) that every item has a CTA of its own: the longest first, up to 320 sequences; equal lengths and
    none among them."""
    heads = 16 if sequences == 20 else 2
    nq, nk = [(37 * i) % 390 for i in range(sequences)], [(53 * i) % 113 * 8 for i in range(sequences)]
    q, k, v = _qkv(sum(nq), sum(nk), heads, 2, dim, F16)
    mask = torch.rand(sum(nk), generator=torch.Generator().manual_seed(5)) < 0.7 if masked else None
    at = [int(n) for n in _starts(nk)[:-1]]
    call = lambda: _attend(q, k, v, heads=heads, kv_heads=2, head_dim=dim, q_start=_starts(nq, 0), k_start=_starts(nk, 0), mask=mask)
    (out, names) = kernels_of(call)
    _ran(names, _kernel(dim))
    _check(out, q, k, v, heads=heads, kv_heads=2, dim=dim, pieces=_pieces(nq, nk, mask, at))


@pytest.mark.parametrize(("sequences", "nk"), [(30, 400), (50, 200)])
@pytest.mark.parametrize("nq", [100, 300])
@pytest.mark.parametrize("dim", [64, 96])
def test_padded(no_device_error, kernels_of, dim, nq, sequences, nk):
    """Equal pieces of which the first k_len keys take part, lengths out of range included, with and without q_start and a mask; a
    CTA per item, and CTAs that walk them."""
    heads = 16
    lens = [(97 * i) % nk for i in range(sequences)]
    lens[3], lens[4], lens[5] = 999, -7, 0
    kept = [min(max(n, 0), nk) for n in lens]
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, 4, dim, F16)
    at = [nk * i for i in range(sequences)]
    for mask in (None, torch.rand(sequences * nk, generator=torch.Generator().manual_seed(8)) < 0.8):
        pieces = _pieces([nq] * sequences, kept, mask, at)
        used = torch.zeros(sequences * nk, dtype=torch.bool)
        for _, ki in pieces:
            used[ki] = True
        dirty = torch.where(used[:, None], k, math.inf), torch.where(used[:, None], v, math.nan)
        clean = torch.where(used[:, None], k, 0), torch.where(used[:, None], v, 0)
        for more in (dict(sequences=sequences), dict(q_start=_starts([nq] * sequences))):
            kw = dict(heads=heads, kv_heads=4, head_dim=dim, k_len=torch.tensor(lens).int(), mask=mask, **more)
            (out, names) = kernels_of(lambda: _attend(q, *dirty, **kw))
            _ran(names, _kernel(dim))
            _check(out, q, *clean, heads=heads, kv_heads=4, dim=dim, pieces=pieces)


@pytest.mark.parametrize("dim", [64, 128])
def test_starts_beyond_the_rows(no_device_error, kernels_of, dim):
    """Starts past the rows that there are, or before the first, are taken back to them."""
    nq, heads = 300, 160
    q, k, v = _qkv(2 * nq, 300, heads, 8, dim, F16)
    starts = dict(q_start=torch.tensor([-4, nq, 5 * nq + 9]).int(), k_start=torch.tensor([-100, 100, 1 << 30]).int())
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, kv_heads=8, head_dim=dim, **starts))
    _ran(names, _kernel(dim))
    _check(out, q, k, v, heads=heads, kv_heads=8, dim=dim, pieces=_pieces([nq, nq], [100, 200]))


@pytest.mark.parametrize("dim", [64, 112])
def test_views(no_device_error, kernels_of, dim):
    """Keys and values as halves of a packed projection, queries and results in wider rows, each 16 bytes further in."""
    sequences, heads, nq, nk = 20, 16, 140, 333
    cols = heads * dim
    q, kv = _randn(sequences * nq, 3 * cols, seed=1, dtype=F16), _randn(sequences * nk, 2 * cols + 16, seed=2, dtype=F16)
    out = torch.full((sequences * nq, cols + 24), 9.0, dtype=F16, device="cuda")
    dq, dkv = q.cuda(), kv.cuda()
    call = lambda: ops.cross_attention(dq[:, cols : 2 * cols], dkv[:, 8 : 8 + cols], dkv[:, 16 + cols :], out[:, 8 : 8 + cols], heads=heads, head_dim=dim, sequences=sequences)
    _, names = kernels_of(call)
    _ran(names, _kernel(dim))
    _check(out[:, 8 : 8 + cols], q[:, cols : 2 * cols], kv[:, 8 : 8 + cols], kv[:, 16 + cols :], heads=heads, dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences))
    assert (out[:, :8] == 9).all() and (out[:, 8 + cols :] == 9).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_offsets_beyond_32_bits(no_device_error, kernels_of, dim):
    """Rows of every matrix that lie more than 2^32 bytes and 2^31 elements from the first."""
    rows, pitch, heads, nq, nk = 300_000, 8192, 16, 600, 700
    big = torch.empty(rows, pitch, dtype=F16, device="cuda")
    assert big.nbytes > 1 << 32 and big.numel() > 1 << 31
    cols = heads * dim
    q, k, v = _qkv(4 * nq, 4 * nk, heads, heads, dim, F16)
    q_at, k_at = rows - 4 * nq, rows - 4 * nk
    parts = [big[:, i * 2048 : i * 2048 + cols] for i in range(4)]
    for part, t in zip(parts, (q, k, v)):
        part[rows - t.shape[0] :] = t.cuda()
    parts[3][:] = 9
    starts = dict(q_start=_starts([nq] * 4, q_at).cuda(), k_start=_starts([nk] * 4, k_at).cuda())
    _, names = kernels_of(lambda: ops.cross_attention(*parts, heads=heads, head_dim=dim, **starts))
    _ran(names, _kernel(dim))
    _check(parts[3][q_at:], q, k, v, heads=heads, dim=dim, pieces=_pieces([nq] * 4, [nk] * 4))
    assert (parts[3][:q_at] == 9).all()
    del big, parts
    torch.cuda.empty_cache()


@pytest.mark.parametrize("nq", [100, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_non_finite_keys_and_queries(no_device_error, kernels_of, dim, nq):
    """A NaN or an infinite score stays with what reads it. (A score of -inf counts nothing; the sequence with it is not compared.)"""
    sequences, heads, nk = 16, 8, 400
    q, k, v = _qkv(sequences * nq, sequences * nk, heads, heads, dim, F16)
    want = q.clone(), k.clone(), v.clone()
    k[nk + 150, 3] = math.nan  # sequence 1, head 0
    k[2 * nk + 390, 1 * dim + 5] = math.inf  # sequence 2, head 1: a score of either infinity
    v[3 * nk + 7, 2 * dim + 1] = math.nan  # sequence 3, head 2, column 1
    q[nq - 1, dim] = math.nan  # sequence 0, last query, head 1
    (out, names) = kernels_of(lambda: _attend(q, k, v, heads=heads, head_dim=dim, sequences=sequences))
    _ran(names, _kernel(dim))
    bad = torch.zeros(sequences * nq, heads * dim, dtype=torch.bool)
    bad[nq : 2 * nq, :dim] = True
    bad[3 * nq : 4 * nq, 2 * dim + 1] = True
    bad[nq - 1, dim : 2 * dim] = True
    rows = torch.arange(2 * nq, 3 * nq)
    plus = rows[q[rows, dim + 5] > 0]  # its score is +inf: no difference to it is a number
    bad[plus, dim : 2 * dim] = True
    got = out.cpu()
    assert got[bad].isnan().all()
    good, size, dot, _ = O.attention(*want, heads=heads, kv_heads=heads, head_dim=dim, pieces=_pieces([nq] * sequences, [nk] * sequences), scale=dim**-0.5)
    rest = ~bad & (torch.arange(sequences * nq)[:, None] // nq != 2)
    tol = size * (2.0**-11 + 2 * 2.0**-20 * 60 + 2.0**-20) + nk * 2.0**-32 * 5 + good.abs() * 2.0**-11 * 1.001 + 2.0**-25
    assert ((got.double() - good).abs() <= tol)[rest].all()
    assert got[~bad].isfinite().all()


@pytest.mark.parametrize("dim", [64, 128])
def test_same_bits_every_time_on_other_streams_and_in_a_graph(no_device_error, kernels_of, dim):
    """Equal pieces and packed ones: the same bits again, several calls at once on streams of their own, and as a graph that is
    replayed on other inputs beside eager calls."""
    heads, sequences = 16, 10
    nq, nk = [260, 100, 0, 513, 128, 300, 77, 256, 30, 400], [300, 700, 64, 0, 900, 129, 500, 64, 200, 1000]
    even = [_qkv(10 * 300, 10 * 600, heads, 4, dim, BF16, seed=10 * i) for i in range(2)]
    packed = [_qkv(sum(nq), sum(nk), heads, 4, dim, BF16, seed=100 + 10 * i) for i in range(2)]
    starts = dict(q_start=_starts(nq).cuda(), k_start=_starts(nk).cuda())
    calls = [(tuple(t.cuda() for t in s), kw) for some, kw in ((even, dict(sequences=sequences)), (packed, starts)) for s in some]
    run = lambda c, o: ops.cross_attention(*c[0], o, heads=heads, kv_heads=4, head_dim=dim, **c[1])
    outs = [torch.zeros_like(c[0][0]) for c in calls]
    _, names = kernels_of(lambda: [run(c, o) for c, o in zip(calls, outs)])
    _ran(names, _kernel(dim))
    _check(outs[1], *even[1], heads=heads, kv_heads=4, dim=dim, pieces=_pieces([300] * 10, [600] * 10))
    _check(outs[3], *packed[1], heads=heads, kv_heads=4, dim=dim, pieces=_pieces(nq, nk))
    again, streams = [torch.zeros_like(o) for o in outs], [torch.cuda.Stream() for _ in outs]
    for _ in range(3):
        for st, c, o in zip(streams, calls, again):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                run(c, o)
    torch.cuda.synchronize()
    for a, b in zip(outs, again):
        assert torch.equal(a, b)
    for first in (0, 2):
        c, static = calls[first], tuple(t.clone() for t in calls[first][0])
        o, beside = torch.zeros_like(outs[first]), torch.zeros_like(outs[first])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run((static, c[1]), o)
        graph.replay()
        assert torch.equal(o, outs[first])
        for t, n in zip(static, calls[first + 1][0]):
            t.copy_(n)
        side = streams[0]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(c, beside)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, outs[first + 1]) and torch.equal(beside, outs[first])
