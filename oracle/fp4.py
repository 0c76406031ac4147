"""Oracle of the block-scaled 4-bit operators in 64 bits (CPU, torch) — test infrastructure only. The formats and
formulas are those of include/foidfinder_b200.h (ff_quantize_fp4, ff_gemm_fp4, ff_qk_norm_rope); the reference has
no counterpart.
"""

from __future__ import annotations

import math

import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BLOCK = {"nv": 16, "mx": 32}


def nearest(y: torch.Tensor, grid: torch.Tensor) -> torch.Tensor:
    """Index of the value of the ascending `grid` nearest to y >= 0; ties to the even index (the even mantissa)."""
    hi = torch.searchsorted(grid, y.contiguous()).clamp(1, len(grid) - 1)
    lo = hi - 1
    dl, dh = y - grid[lo], grid[hi] - y
    up = (dh < dl) | ((dh == dl) & (hi % 2 == 0))
    return torch.where(up, hi, lo)


def e4m3_grid() -> torch.Tensor:
    """The non-negative e4m3 values by byte, 0 .. 448 (byte 126)."""
    v = [m * 2.0**-9 for m in range(8)]
    v += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64)


def quantize(x: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """x [T, C] -> codes uint8 [T, C] (sign in bit 3), scale bytes [T, ceil(C / block)], row scale [T] f64."""
    x = x.double()
    T, C = x.shape
    B = BLOCK[fmt]
    nb = -(-C // B)
    v = torch.zeros(T, nb * B, dtype=torch.float64)
    v[:, :C] = x
    v = v.view(T, nb, B)
    finite = torch.isfinite(v)
    top = torch.where(finite, v.abs(), torch.zeros_like(v)).amax(2)
    row = torch.ones(T, dtype=torch.float64)
    if fmt == "nv":
        bad = ~finite.all(2).all(1)
        for r in range(T):
            m = top[r].max().item()
            e = -110
            if m > 0:
                e = max(e, math.frexp(m)[1] - 13)
                while m > 2688 * 2.0**e:
                    e += 1
            row[r] = 2.0**e
        bytes_ = nearest((top / (6 * row[:, None])).clamp_max(448), e4m3_grid())
        scale = e4m3_grid()[bytes_] * row[:, None]
        bytes_[bad] = 0
        scale[bad] = 0
        row[bad] = math.nan
    else:
        bad = ~finite.all(2)
        e = torch.zeros_like(top, dtype=torch.int64)
        nz = top > 0
        e[nz] = torch.frexp(top[nz])[1].long() - 3
        e[~nz] = -127
        e = e.clamp_min(-127)
        bytes_ = e + 127
        scale = 2.0 ** e.double()
        bytes_[bad] = 255
        scale[bad] = 0
    y = torch.where((scale > 0)[..., None], v / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None], torch.zeros_like(v))
    y = torch.where(torch.isfinite(y), y, torch.zeros_like(y))
    codes = nearest(y.abs().clamp_max(6), VALUES)
    codes = torch.where(y < 0, codes + 8, codes).view(T, -1)[:, :C]
    return codes.to(torch.uint8), bytes_.to(torch.uint8), row


def values(codes: torch.Tensor, bytes_: torch.Tensor, row: torch.Tensor, fmt: str) -> torch.Tensor:
    """The 64-bit values of an operand."""
    v = VALUES[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    s = e4m3_grid()[bytes_.long()] if fmt == "nv" else torch.where(bytes_ == 255, math.nan, 2.0 ** (bytes_.double() - 127))
    return v * s.repeat_interleave(BLOCK[fmt], 1)[:, : codes.shape[1]] * row[:, None]


def unpack_codes(packed: torch.Tensor, T: int, C: int) -> torch.Tensor:
    p = packed.cpu().view(T, -1)
    return torch.stack([p & 15, p >> 4], 2).view(T, -1)[:, :C]


def scale_index(T: int, C: int, fmt: str) -> torch.Tensor:
    """Byte of every (row, block) of the padded columns in the scale buffer, [T, blocks]."""
    blocks = -(-C // 256) * 256 // BLOCK[fmt]
    r, b = torch.arange(T)[:, None], torch.arange(blocks)[None]
    tile = blocks // 4 * 512
    return (r // 128) * tile + (b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4


def layer_norm(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor | None, eps: float) -> torch.Tensor:
    x = x.double()
    d = x - x.mean(-1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + eps) * w.double()
    return y if b is None else y + b.double()


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    x = x.double()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def rotate(y: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pairing: str) -> torch.Tensor:
    """y [T, heads, D] by cos/sin [T, D / 2]."""
    c, s = cos.double()[:, None], sin.double()[:, None]
    if pairing == "pairs":
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    h = y.shape[-1] // 2
    a, b = y[..., :h], y[..., h:]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def heads(x, n, D, w, b, norm, eps, cos, sin, pairing) -> torch.Tensor:
    """n heads of D columns of x, normalised and rotated; cos/sin angle-major [D / 2, tokens], position row % tokens."""
    T = x.shape[0]
    y = x.double().reshape(T, n, D)
    y = rms_norm(y, w, eps) if norm == "rms" else layer_norm(y, w, b, eps)
    at = torch.arange(T) % cos.shape[1]
    return rotate(y, cos.t()[at], sin.t()[at], pairing).reshape(T, n * D)


def gelu_tanh(y: torch.Tensor) -> torch.Tensor:
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))


def silu_mul(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    return g * torch.sigmoid(g) * u
