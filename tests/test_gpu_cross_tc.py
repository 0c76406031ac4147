"""Cross attention of many queries on the GPU, at sizes that the choice of kernel sends to the tensor-core kernels, with the
kernel that ran asserted, against the 64-bit oracle. Tolerances are those of test_gpu_cross.py; what differs is derived
at the test."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import cross as O
from test_gpu_cross import BF16, F16, _attend, _check_attention, _pieces, _qkv

pytestmark = pytest.mark.gpu

NARROW, WIDE = "cross_tc64_kernel", "cross_tc_kernel"


def _kernel(dim):
    return NARROW if dim <= 64 else WIDE


@pytest.fixture(scope="module")
def kernels_of(cuda_device):
    """f -> (f(), names of the cross attention kernels that it launched)."""

    def run(f):
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
            r = f()
            torch.cuda.synchronize()
        names = {e.key for e in prof.key_averages() if "cross_" in e.key}
        assert names, "the profiler has seen no kernel"
        return r, names

    return run


def _ran(names, *kernels):
    """Exactly these kernels (whole names: one is the beginning of another's)."""
    assert len(names) == len(kernels) and all(any(k + "<" in n for n in names) for k in kernels), names


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
    assert any(kernel + "<" in n for n in names), names
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
        assert any(kernel + "<" in n for n in names), names
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
    assert any(kernel + "<" in n for n in names), names
    assert out.isfinite().all()
    pieces = [(slice(i * nq, (i + 1) * nq), slice(i * nk, (i + 1) * nk)) for i in range(sequences)]
    want, magnitude, dot, _ = O.attention(q, k, v, heads=heads, kv_heads=heads, head_dim=dim, pieces=pieces, scale=dim**-0.5)
    off, half = (out.double().cpu() - want).abs(), 2.0**-9
    assert (off <= magnitude * (half + 2 * 2.0**-20 * dot + 2.0**-20) + want.abs() * half * (1 + half)).all(), (off / magnitude).max()
