"""Cross attention of many queries on the GPU, at sizes that the choice of kernel sends to the tensor-core kernels, with the
kernel that ran asserted, against the 64-bit oracle. Tolerances are those of test_gpu_cross.py; what differs is derived
at the test."""

from __future__ import annotations

import pytest
import torch

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
