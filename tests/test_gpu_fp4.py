"""Block-scaled 4-bit quantisation, the 4-bit product with its epilogues and the query/key head norms with rotation,
against the 64-bit oracle (oracle/fp4.py).

Tolerances. Quantisation without a norm is exact. After a LayerNorm the f32 statistics move a value by up to about
2^-20 of itself, which moves a code or a block scale only next to a rounding boundary: at most 1 in 1000 codes may
differ. Products are compared on the same codes: the tensor cores add in f32, one rounding (or truncation) of at most
2^-22 of the sum of magnitudes per 64-column step, plus the output type's own rounding (half a unit in the last place)
and, for the epilogues with transcendental functions, their relative error of 2^-18.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import fp4 as O

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-130, torch.float32: 2.0**-130}
FMT = {"nv": 0, "mx": 1}


def _x(rows, cols, dtype, seed, outliers=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if outliers:
        x = torch.where(torch.rand(rows, cols, generator=g) < 0.01, 20 * x, x)
    return x.to(dtype)


def _read(q):
    """(codes [T, C], scale bytes of the padded columns [T, blocks], row scale) of an Fp4Tensor."""
    codes = O.unpack_codes(q.codes, q.rows, q.cols)
    s = q.scales.cpu()[O.scale_index(q.rows, q.cols, q.fmt)]
    row = q.row_scale.cpu().double() if q.fmt == "nv" else torch.ones(q.rows, dtype=torch.float64)
    return codes, s, row


def _check_exact(q, x):
    codes, s, row = _read(q)
    ec, es, er = O.quantize(x, q.fmt)
    same = (codes == ec) | ((codes & 7) + (ec & 7) == 0)  # +0 and -0 are one value
    assert same.all(), f"{(~same).sum()} codes differ"
    assert torch.equal(s[:, : es.shape[1]], es)
    assert s[:, es.shape[1] :].count_nonzero() == 0, "padded block scales must be zero"
    torch.testing.assert_close(row, er, rtol=0, atol=0, equal_nan=True)
    packed = q.codes.cpu().view(q.rows, -1)
    if packed.shape[1] * 2 > q.cols:  # padding columns
        tail = torch.stack([packed & 15, packed >> 4], 2).view(q.rows, -1)[:, q.cols :]
        assert tail.count_nonzero() == 0


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("rows", "cols"), [(1, 1), (1, 16), (3, 17), (129, 32), (33, 255), (257, 256), (5, 512), (130, 1024), (64, 1100),
                                            (9, 2730), (4, 4864), (3, 6200), (2, 12289), (2, 20000)])
def test_quantize_is_exact(cuda_device, no_device_error, fmt, dtype, rows, cols):
    from foidfinder_b200 import fp4

    x = _x(rows, cols, dtype, rows * 7 + cols)
    q = fp4.quantize(x.to(cuda_device), fmt)
    _check_exact(q, x)
    v = O.values(*O.quantize(x, fmt), fmt)
    for out in (torch.float16, torch.bfloat16, torch.float32):
        got = fp4.dequantize(q, out).cpu()
        ref = v.float().to(out)  # code * scale is exact in f32
        assert torch.equal(got, ref)


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5, 8])
def test_quantize_and_dequantize_any_alignment(cuda_device, no_device_error, fmt, dtype, shift):
    """Rows that start anywhere inside a 16-byte granule, with NaN around them that must not be read as data."""
    from foidfinder_b200 import fp4

    rows, cols = 37, 333
    x = _x(rows, cols, dtype, 3)
    big = torch.full((rows, cols + 20), math.nan, dtype=dtype, device=cuda_device)
    view = big[:, shift : shift + cols]
    view.copy_(x)
    flat = torch.full((rows * cols + 32,), math.nan, dtype=dtype, device=cuda_device)
    dense = flat[shift : shift + rows * cols].view(rows, cols)
    dense.copy_(x)
    for t in (view, dense):
        _check_exact(fp4.quantize(t, fmt), x)
    q = fp4.quantize(x.to(cuda_device), fmt)
    ref = O.values(*O.quantize(x, fmt), fmt).float().to(dtype)
    for buf, t in ((big, view), (flat, dense)):
        before = torch.isnan(buf).sum().item()
        fp4.dequantize(q, out=t)
        assert torch.equal(t.cpu(), ref)
        assert torch.isnan(buf).sum().item() == before  # nothing outside the rows was written


@pytest.mark.parametrize(("low", "high"), [(-20, 20), (-120, 118)])
def test_quotients_next_to_ties(cuda_device, no_device_error, low, high):
    """f32 values that are e2m1 ties times their block's scale, or up to two units in the last place off them."""
    from foidfinder_b200 import fp4

    g = torch.Generator().manual_seed(high)
    rows, cols = 256, 256
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64)
    x[:, 0] = 2688 * torch.rand(rows, generator=g, dtype=torch.float64).clamp_min(0.51)
    first = x.view(rows, -1, 16)[:, :, 0]  # each block's largest value fixes its scale
    first[:, 1:] = 2688 * torch.rand(rows, cols // 16 - 1, generator=g, dtype=torch.float64) ** 4
    x = (x * 2.0 ** torch.randint(low, high, (rows, 1), generator=g)).float()
    _, s, row = O.quantize(x, "nv")
    scale = s.view(torch.float8_e4m3fn).double() * row.double()[:, None]
    tie = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    v = (tie[torch.randint(0, 7, (rows, cols // 16, 15), generator=g)] * scale[:, :, None]).float()
    v = (v.view(torch.int32) + torch.randint(-2, 3, v.shape, generator=g).int()).view(torch.float32).where(v > 0, 0.0)
    blocks = x.view(rows, -1, 16)
    v = v.where(v <= blocks[:, :, :1].abs(), 0.0)
    blocks[:, :, 1:] = v.where(torch.rand(v.shape, generator=g) < 0.5, -v)
    _check_exact(fp4.quantize(x.to(cuda_device), "nv"), x)


@pytest.mark.parametrize("fmt", ["nv", "mx"])
def test_quantize_special_values(cuda_device, no_device_error, fmt):
    from foidfinder_b200 import fp4

    x = _x(140, 96, torch.float32, 5)
    x[0] = 0
    x[1, :32] = 0
    x[2] = -0.0
    x[3] *= 1e-30
    x[4] *= 1e36
    x[5] = 2688.0
    x[6, 0], x[6, 1:] = 2690.0, 1.0
    x[7, 5] = math.inf
    x[8, 40] = math.nan
    x[9, 95] = -math.inf
    x[10] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]).repeat(12)  # ties
    x[11] = 1e-42  # below the smallest normal number
    x[12] = torch.finfo(torch.float32).max
    q = fp4.quantize(x.to(cuda_device), fmt)
    _check_exact(q, x)
    v = fp4.dequantize(q, torch.float32).cpu()
    if fmt == "nv":
        assert torch.isnan(v[[7, 8, 9]]).all()
    else:
        assert torch.isnan(v[7, :32]).all() and torch.isfinite(v[7, 32:]).all()
        assert torch.isnan(v[8, 32:64]).all() and torch.isnan(v[9, 64:]).all()
    assert torch.isfinite(v[[0, 1, 2, 3, 4, 5, 6, 10, 11]]).all()
    # the largest f32 value may round up to a block scale times 6 beyond f32: whatever the codes stand for, in f32
    assert torch.equal(v[12], O.values(*O.quantize(x, fmt), fmt)[12].float())


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize(("rows", "cols"), [(1, 768), (130, 1024), (17, 2730), (5, 13000), (3, 33)])
def test_layernorm_quantize(cuda_device, no_device_error, fmt, dtype, rows, cols):
    from foidfinder_b200 import fp4

    x = _x(rows, cols, dtype, cols)
    g = torch.Generator().manual_seed(9)
    gamma, beta = 1 + 0.1 * torch.randn(cols, generator=g), 0.1 * torch.randn(cols, generator=g)
    q = fp4.quantize(x.to(cuda_device), fmt, gamma=gamma.to(cuda_device), beta=beta.to(cuda_device), eps=1e-5)
    codes, s, row = _read(q)
    ec, es, er = O.quantize(O.layer_norm(x, gamma, beta, 1e-5), fmt)
    assert torch.equal(row, er)
    nb = es.shape[1]
    assert (s[:, :nb].int() - es.int()).abs().max() <= 1 and (s[:, :nb] != es).float().mean() <= 1e-3
    assert s[:, nb:].count_nonzero() == 0
    assert (codes != ec).float().mean() <= 1e-3


def _operand(rows, cols, fmt, seed, device, std=1.0, dtype=torch.float32):
    from foidfinder_b200 import fp4

    x = (_x(rows, cols, torch.float32, seed) * std).to(dtype)
    q = fp4.quantize(x.to(device), fmt)
    return q, O.values(*O.quantize(x, fmt), fmt)


def _product(av, wv, bias):
    """Exact product, and the error bound of its f32 accumulation."""
    y = av @ wv.t()
    steps = -(-av.shape[1] // 64) + 8
    tol = steps * 2.0**-22 * (av.abs() @ wv.abs().t())
    if bias is not None:
        y = y + bias.double()
        tol = tol + 2.0**-23 * (y.abs() + bias.double().abs())
    return y, tol


def _close(got, ref, tol, dtype):
    got = got.cpu().double()
    limit = tol + HALF_ULP[dtype] * (ref.abs() + tol) + TINY[dtype]
    bad = ~((got - ref).abs() <= limit)
    assert not bad.any(), f"{bad.sum()} of {bad.numel()} values off, worst {((got - ref).abs() / limit).max():.3g} x the bound"


GEMM_SHAPES = [(1, 1, 1), (1, 7, 32), (2, 129, 64), (3, 64, 65), (127, 128, 256), (128, 128, 512), (129, 100, 300), (200, 257, 768),
               (300, 520, 1100), (257, 333, 2730), (515, 384, 1600)]


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize(("cols", "dtype"), [(96, torch.float32), (200, torch.float16), (1301, torch.bfloat16), (2736, torch.float16)])
def test_rows_do_not_depend_on_each_other(cuda_device, no_device_error, cols, dtype, norm, fmt):
    """More rows than the GPU holds at once (each warp goes on to further rows), against the same rows a few at a time:
    equal to the last bit, and so are their values."""
    from foidfinder_b200 import fp4

    rows = 12345
    x = _x(rows, cols, dtype, cols).to(cuda_device)
    kw = dict(gamma=torch.linspace(0.5, 2, cols, device=cuda_device), beta=torch.linspace(-1, 1, cols, device=cuda_device)) if norm else {}
    q = fp4.quantize(x, fmt, **kw)
    codes, scales, row = _read(q)
    v = {t: fp4.dequantize(q, t) for t in (torch.float16, torch.float32)}
    for first in (0, 127, 5921, rows - 301):
        part = slice(first, first + 301)
        p = fp4.quantize(x[part].clone(), fmt, **kw)
        pc, ps, pr = _read(p)
        assert torch.equal(pc, codes[part]) and torch.equal(ps, scales[part]) and torch.equal(pr, row[part])
        for t, a in v.items():
            assert torch.equal(fp4.dequantize(p, t), a[part])


@pytest.mark.parametrize("fmt", ["nv", "mx"])
def test_the_short_and_the_long_way_into_a_call_agree(cuda_device, no_device_error, monkeypatch, fmt):
    """The extension module takes plain calls (it must be there); what it leaves to Python gives the same."""
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    assert ops._calls() is not ops._NoCalls
    x = _x(70, 200, torch.float16, 1).to(d)
    g = torch.linspace(0.5, 1.5, 200, device=d)
    t, hw = torch.linspace(0, 1, 16 * 7, device=d).view(16, 7), torch.ones(32, device=d)
    layer = fp4.Fp4Linear(_x(200, 200, torch.float32, 2).to(d), g, fmt=fmt, epilogue="residual", gamma=g, beta=g)

    def everything():
        q = fp4.quantize(x, fmt, gamma=g, beta=g)
        h = torch.zeros(70, 200, device=d, dtype=torch.float16)
        ops.qk_norm_rope(x, h, q_heads=4, k_heads=2, head_dim=32, norm="layer", q_weight=hw, k_weight=hw, k_bias=hw, rope_cos=t, rope_sin=t, pairing="halves")
        return [*_read(q), fp4.dequantize(q, torch.float32), layer(x, residual=x), h]

    def taken(*args):
        r = real(*args)
        assert r == 0
        return r

    short = ops._calls()
    for name in ("quantize", "dequantize", "linear", "qk_norm_rope"):
        real = getattr(short, name)
        with monkeypatch.context() as m:
            m.setattr(short, name, taken)
            a = everything()
    monkeypatch.setattr(ops, "_calls", lambda: ops._NoCalls)
    for u, v in zip(a, everything()):
        assert torch.equal(u, v)


def test_what_the_short_way_leaves(cuda_device, monkeypatch):
    from foidfinder_b200 import fp4, ops

    c = ops._calls()
    d = cuda_device
    x = torch.zeros(4, 64, dtype=torch.float16, device=d)
    q = fp4.Fp4Tensor.empty(4, 64, "nv")
    args = [x, q.codes, q.scales, q.row_scale, 0, None, None, 1e-6]
    assert c.quantize(*args) == 0
    for i, bad in ((0, x.cpu()), (0, x.t()), (0, x[0]), (0, x.int()), (0, x.cpu().numpy()), (1, q.codes[:8]), (1, q.codes.float()), (2, None), (3, None),
                   (3, q.row_scale.half()), (4, "nv"), (4, 1 << 40), (5, x), (7, 1)):
        assert c.quantize(*args[:i], bad, *args[i + 1 :]) is None, (i, bad)
    assert c.quantize(*args[:-1]) is None
    with pytest.raises(RuntimeError, match="unknown format"):  # the library's own check
        ops.quantize_fp4(x, q.codes, q.scales, q.row_scale, 7)


def test_calls_of_no_rows(cuda_device, no_device_error):
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    x = torch.empty(0, 64, dtype=torch.float16, device=d)
    q = fp4.quantize(x)
    assert fp4.dequantize(q).shape == (0, 64)
    for epilogue in ("bias", "residual"):
        layer = fp4.Fp4Linear(torch.ones(64, 64, device=d), epilogue=epilogue)
        assert layer(x, residual=x if epilogue == "residual" else None).shape == (0, 64)
    t, w = torch.ones(16, 5, device=d), torch.ones(32, device=d)
    ops.qk_norm_rope(x, x.clone(), q_heads=1, k_heads=1, head_dim=32, norm="rms", q_weight=w, k_weight=w, rope_cos=t, rope_sin=t)


def test_more_rows_than_an_index_holds_are_refused(cuda_device):
    from foidfinder_b200 import ops

    x = torch.zeros(1, 1, dtype=torch.float16, device=cuda_device).expand((1 << 30) + 1, 1)
    c = torch.zeros(16, dtype=torch.uint8, device=cuda_device)
    with pytest.raises(RuntimeError, match="2\\^30 rows"):
        ops.quantize_fp4(x, c, c, None, ops.FP4_MX)


@pytest.mark.parametrize("tile", [128, 512])
@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize(("M", "N", "K"), GEMM_SHAPES)
def test_gemm_bias_f32(cuda_device, no_device_error, M, N, K, fmt, tile):
    from foidfinder_b200 import ops

    A, av = _operand(M, K, fmt, 1, cuda_device)
    W, wv = _operand(N, K, fmt, 2, cuda_device, 0.02)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(4)) * 0.1
    out = torch.full((M, N), math.nan, device=cuda_device)
    ops.gemm_fp4(A.codes, A.scales, A.row_scale, W.codes, W.scales, W.row_scale, out, ops.EPI_BIAS, FMT[fmt], N=N, K=K,
                 bias=bias.to(cuda_device), tile=tile)
    y, tol = _product(av, wv, bias)
    _close(out, y, tol, torch.float32)


@pytest.mark.parametrize("tile", [128, 512])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("epi", ["bias", "nobias", "gelu", "residual", "inplace"])
@pytest.mark.parametrize(("M", "N", "K", "fmt"), [(1, 9, 48, "nv"), (130, 200, 320, "mx"), (300, 328, 1024, "nv"), (515, 270, 1500, "mx")])
def test_gemm_16bit_epilogues(cuda_device, no_device_error, M, N, K, fmt, epi, dtype, tile):
    from foidfinder_b200 import ops

    A, av = _operand(M, K, fmt, 1, cuda_device)
    W, wv = _operand(N, K, fmt, 2, cuda_device, 0.05)
    g = torch.Generator().manual_seed(4)
    bias = None if epi == "nobias" else torch.randn(N, generator=g) * 0.1
    pitch = (N + 7) // 8 * 8 + 8
    buf = torch.full((M, pitch), 77.0, device=cuda_device, dtype=dtype)
    out = buf[:, :N]
    y, tol = _product(av, wv, bias)
    kind, residual = ops.EPI_BIAS, None
    if epi == "gelu":
        kind = ops.EPI_GELU
        tol = 1.13 * tol + 2.0**-18 * y.abs()  # |gelu'| <= 1.13
        y = O.gelu_tanh(y)
    elif epi in ("residual", "inplace"):
        kind = ops.EPI_RESIDUAL
        r = torch.randn(M, N, generator=g).to(dtype)
        residual = out if epi == "inplace" else torch.zeros(M, pitch + 16, device=cuda_device, dtype=dtype)[:, :N]
        residual.copy_(r)
        y = y + r.double()
        tol = tol + 2.0**-23 * (y.abs() + r.double().abs())
    ops.gemm_fp4(A.codes, A.scales, A.row_scale, W.codes, W.scales, W.row_scale, out, kind, FMT[fmt], N=N, K=K,
                 bias=None if bias is None else bias.to(cuda_device), residual=residual, tile=tile)
    _close(out, y, tol, dtype)
    assert (buf[:, N:] == 77.0).all(), "columns past N were written"


@pytest.mark.parametrize("tile", [128, 512])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("M", "H", "K", "fmt"), [(1, 64, 64, "nv"), (129, 100, 256, "mx"), (300, 330, 768, "nv"), (260, 704, 512, "mx")])
def test_gemm_swiglu(cuda_device, no_device_error, M, H, K, fmt, dtype, tile):
    from foidfinder_b200 import fp4, ops

    A, av = _operand(M, K, fmt, 1, cuda_device)
    g = torch.Generator().manual_seed(4)
    w = torch.randn(2 * H, K, generator=g) * 0.1
    bias = torch.randn(2 * H, generator=g) * 0.1
    wv = O.values(*O.quantize(w, fmt), fmt)
    layer = fp4.Fp4Linear(w.to(cuda_device), bias.to(cuda_device), fmt=fmt, epilogue="swiglu")
    W = layer.weight
    out = torch.full((M, (H + 7) // 8 * 8), 77.0, device=cuda_device, dtype=dtype)
    ops.gemm_fp4(A.codes, A.scales, A.row_scale, W.codes, W.scales, W.row_scale, out[:, :H], ops.EPI_SWIGLU, FMT[fmt], N=layer.rows, K=K,
                 bias=layer.bias, tile=tile)
    y, tol = _product(av, wv, bias)
    gt, up, tg, tu = y[:, :H], y[:, H:], tol[:, :H], tol[:, H:]
    ref = O.silu_mul(gt, up)
    silu = O.silu_mul(gt, torch.ones_like(gt))
    _close(out[:, :H], ref, 1.1 * tg * (up.abs() + tu) + silu.abs() * tu + 2.0**-18 * ref.abs(), dtype)
    assert (out[:, H:] == 77.0).all()


def _tables(tokens, half, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(half, tokens, generator=g) * 6.28
    return a.cos().contiguous(), a.sin().contiguous()


@pytest.mark.parametrize("tile", [0, 128])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize(("M", "qh", "kh", "vh", "K", "tokens", "fmt", "dtype"), [
    (1, 1, 1, 1, 64, 1, "nv", torch.float16),
    (131, 4, 2, 2, 256, 50, "mx", torch.bfloat16),
    (300, 3, 3, 3, 768, 197, "nv", torch.float16),
])
def test_gemm_qkv_norm_rope(cuda_device, no_device_error, M, qh, kh, vh, K, tokens, fmt, dtype, norm, tile):
    from foidfinder_b200 import ops

    d = cuda_device
    N = 64 * (qh + kh + vh)
    A, av = _operand(M, K, fmt, 1, d)
    W, wv = _operand(N, K, fmt, 2, d, 0.05)
    g = torch.Generator().manual_seed(4)
    bias = torch.randn(N, generator=g) * 0.1
    qw, kw = 1 + 0.1 * torch.randn(64, generator=g), 1 + 0.1 * torch.randn(64, generator=g)
    qb, kb = (0.1 * torch.randn(64, generator=g), 0.1 * torch.randn(64, generator=g)) if norm == "layer" else (None, None)
    cos, sin = _tables(tokens, 32)
    dev = lambda t: None if t is None else t.to(d)  # noqa: E731
    out = torch.full((M, N), math.nan, device=d, dtype=dtype)
    ops.gemm_fp4(A.codes, A.scales, A.row_scale, W.codes, W.scales, W.row_scale, out, ops.EPI_QKV_NORM_ROPE, FMT[fmt], N=N, K=K, bias=bias.to(d),
                 tile=tile, norm=norm, q_heads=qh, k_heads=kh, q_weight=dev(qw), k_weight=dev(kw), q_bias=dev(qb), k_bias=dev(kb), qk_eps=1e-6,
                 rope_cos=dev(cos), rope_sin=dev(sin))
    y, tol = _product(av, wv, bias)
    q = O.heads(y[:, : 64 * qh], qh, 64, qw, qb, norm, 1e-6, cos, sin, "pairs")
    k = O.heads(y[:, 64 * qh : 64 * (qh + kh)], kh, 64, kw, kb, norm, 1e-6, cos, sin, "pairs")
    ref = torch.cat([q, k, y[:, 64 * (qh + kh) :]], 1)
    # The norm divides the product's error by the head's rms and spreads it over the head; f32 arithmetic of the norm
    # and rotation adds 2^-19 of values of order 1.
    qk = 64 * (qh + kh)
    h = y[:, :qk].reshape(M, -1, 64)
    if norm == "layer":
        h = h - h.mean(-1, keepdim=True)
    rms = h.square().mean(-1, keepdim=True).sqrt()
    spread = tol[:, :qk].reshape(M, -1, 64).amax(-1, keepdim=True) / rms * (2 + 2 * (h / rms).abs().amax(-1, keepdim=True))
    lim = torch.cat([(1.5 * 1.5 * spread + 2.0**-19 * (1 + (h / rms).abs().amax(-1, keepdim=True))).expand(-1, -1, 64).reshape(M, qk), tol[:, qk:]], 1)
    _close(out, ref, lim, dtype)


@pytest.mark.parametrize("rows", [1, 5, 130])
def test_nan_rows_stay_in_their_rows(cuda_device, no_device_error, rows):
    """A row with a NaN input is NaN in the output; the other rows are as without it, whatever the padding rows hold."""
    from foidfinder_b200 import fp4

    x = _x(rows, 300, torch.float16, 2).to(cuda_device)
    w = _x(96, 300, torch.float32, 3).to(cuda_device)
    for fmt in ("nv", "mx"):
        layer = fp4.Fp4Linear(w, fmt=fmt)
        good = layer(x)
        y = x.clone()
        y[rows // 2, 7] = math.nan
        got = layer(y)
        keep = torch.arange(rows, device=cuda_device) != rows // 2
        assert torch.isnan(got[rows // 2]).all()
        assert torch.equal(got[keep], good[keep])


@pytest.mark.parametrize("fmt", ["nv", "mx"])
def test_linear_is_quantize_then_gemm(cuda_device, no_device_error, fmt):
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    M, K, N = 300, 700, 264
    x = _x(M, K, torch.bfloat16, 2).to(d)
    g = torch.Generator().manual_seed(4)
    gamma, beta, bias = (torch.randn(n, generator=g).to(d) for n in (K, K, N))
    layer = fp4.Fp4Linear(_x(N, K, torch.float32, 3).to(d), bias, fmt=fmt, gamma=gamma, beta=beta)
    q = fp4.quantize(x, fmt, gamma=gamma, beta=beta)
    W = layer.weight
    out = torch.empty(M, N, device=d, dtype=torch.bfloat16)
    ops.gemm_fp4(q.codes, q.scales, q.row_scale, W.codes, W.scales, W.row_scale, out, ops.EPI_BIAS, FMT[fmt], N=N, K=K, bias=bias)
    assert torch.equal(layer(x), out)
    assert torch.equal(layer(x), layer(x))


def test_linear_on_another_stream(cuda_device, no_device_error):
    """Each call's workspace belongs to the stream it runs on: two streams at once give the single-stream results."""
    from foidfinder_b200 import fp4

    d = cuda_device
    layer = fp4.Fp4Linear(_x(512, 1024, torch.float32, 3).to(d))
    xs = [_x(2000, 1024, torch.float16, s).to(d) for s in (1, 2)]
    ref = [layer(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    outs = [[torch.empty(2000, 512, device=d, dtype=torch.float16) for _ in range(8)] for _ in xs]
    for i in range(8):
        for s, st in enumerate(streams):
            with torch.cuda.stream(st):
                layer(xs[s], out=outs[s][i])
    torch.cuda.synchronize()
    for s in range(2):
        for o in outs[s]:
            assert torch.equal(o, ref[s])


def test_linear_in_a_cuda_graph(cuda_device, no_device_error):
    from foidfinder_b200 import fp4

    d = cuda_device
    layer = fp4.Fp4Linear(_x(384, 768, torch.float32, 3).to(d), epilogue="gelu", fmt="mx")
    x = _x(700, 768, torch.float16, 1).to(d)
    out = torch.empty(700, 384, device=d, dtype=torch.float16)
    layer(x, out=out)  # loads the kernels
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        layer(x, out=out)
    x.copy_(_x(700, 768, torch.float16, 9))
    g.replay()
    torch.cuda.synchronize()
    got = out.clone()
    layer(x, out=out)
    assert torch.equal(got, out)
    del g


@pytest.mark.parametrize("pairing", ["pairs", "halves"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("rows", "qh", "kh", "dim", "tokens"), [(1, 1, 1, 32, 1), (3, 16, 16, 64, 2), (130, 5, 2, 64, 50), (77, 8, 1, 128, 197),
                                                                (33, 3, 3, 256, 9), (20, 7, 0, 32, 20)])
def test_qk_norm_rope(cuda_device, no_device_error, rows, qh, kh, dim, tokens, dtype, norm, pairing):
    from foidfinder_b200 import ops

    d = cuda_device
    cols = (qh + kh) * dim
    x = (_x(rows, cols + 16, torch.float32, rows, outliers=False) * 1.5).to(dtype)
    g = torch.Generator().manual_seed(4)
    qw, kw = 1 + 0.1 * torch.randn(dim, generator=g), 1 + 0.1 * torch.randn(dim, generator=g)
    qb, kb = (0.1 * torch.randn(dim, generator=g), 0.1 * torch.randn(dim, generator=g)) if norm == "layer" else (None, None)
    cos, sin = _tables(tokens, dim // 2)
    dev = lambda t: None if t is None else t.to(d)  # noqa: E731
    args = dict(q_heads=qh, k_heads=kh, head_dim=dim, norm=norm, q_weight=dev(qw), k_weight=dev(kw), q_bias=dev(qb), k_bias=dev(kb), eps=1e-6,
                rope_cos=dev(cos), rope_sin=dev(sin), pairing=pairing)
    out = torch.full((rows, cols + 8), 77.0, device=d, dtype=dtype)
    xd = x.to(d)
    ops.qk_norm_rope(xd, out, **args)
    q = O.heads(x[:, : qh * dim], qh, dim, qw, qb, norm, 1e-6, cos, sin, pairing)
    k = O.heads(x[:, qh * dim : cols], kh, dim, kw, kb, norm, 1e-6, cos, sin, pairing)
    ref = torch.cat([q, k], 1)
    # f32 arithmetic on values of order |n| <= 10: 2^-20 of the rotated pair's magnitude, then one rounding
    _close(out[:, :cols], ref, 2.0**-20 * torch.full_like(ref, 10.0), dtype)
    assert (out[:, cols:] == 77.0).all()
    ops.qk_norm_rope(xd, xd, **args)
    assert torch.equal(xd[:, :cols], out[:, :cols]) and torch.equal(xd[:, cols:].cpu(), x[:, cols:])


def test_qk_norm_of_zero_and_huge_heads(cuda_device, no_device_error):
    from foidfinder_b200 import ops

    d = cuda_device
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    x[1] = 1e18  # squares stay below the f32 maximum
    x[2, :64] = math.nan
    cos, sin = torch.ones(32, 4), torch.zeros(32, 4)
    w = torch.ones(64, device=d)
    out = torch.empty(4, 128, device=d, dtype=torch.bfloat16)
    ops.qk_norm_rope(x.to(d), out, q_heads=1, k_heads=1, head_dim=64, norm="rms", q_weight=w, k_weight=w, rope_cos=cos.to(d), rope_sin=sin.to(d))
    got = out.cpu().float()
    assert (got[0] == 0).all() and (got[1] == 1).all() and (got[3] == 0).all()
    assert torch.isnan(got[2, :64]).all() and (got[2, 64:] == 0).all()


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize("arch", ["eva02", "pixai"])
def test_fp4_block(cuda_device, no_device_error, arch, fmt):
    """Every linear layer of the block against 64 bits on the inputs that the block gave it, and the block's output as a
    whole. After a LayerNorm 1 in 1000 codes may be off by a step (a quarter of the value): sqrt(1e-3) / 4 = 0.8%, with
    the storage rounding 2% is left for each layer. Across layers a stored fp16 value that rounds the other way moves
    codes too, but the residual stream carries most of the output: 2% for the block."""
    from foidfinder_b200 import fp4
    from foidfinder_b200.config import EVA02_B, PIXAI_1008
    from foidfinder_b200.weights import random_raw

    d = cuda_device
    cfg = EVA02_B.with_(depth=1, image_size=56) if arch == "eva02" else PIXAI_1008.with_(depth=1, image_size=112, window=0, dim=256, heads=4, mlp_hidden=600)
    T, D, H = cfg.tokens, cfg.dim, cfg.heads
    g = torch.Generator().manual_seed(1)
    if arch == "eva02":
        raw = {k: v for k, v in random_raw(cfg, seed=2).items() if k.startswith("blocks.0.")}
    else:
        raw = {}
        for name, (n, k) in {"qkv": (3 * D, D), "proj": (D, D), "fc1": (cfg.mlp_hidden, D), "fc2": (D, cfg.mlp_hidden)}.items():
            raw[f"blocks.0.{name}.weight"] = torch.randn(n, k, generator=g) * 0.05
            raw[f"blocks.0.{name}.bias"] = torch.randn(n, generator=g) * 0.02
        for name in ("norm1", "norm2"):
            raw[f"blocks.0.{name}.weight"] = 1 + 0.02 * torch.randn(D, generator=g)
            raw[f"blocks.0.{name}.bias"] = 0.02 * torch.randn(D, generator=g)
    qw, kw = 1 + 0.1 * torch.randn(64, generator=g), 1 + 0.1 * torch.randn(64, generator=g)
    cos, sin = _tables(T, 32, 7)
    block = fp4.Fp4Block(raw, "blocks.0.", cfg, q_weight=qw.to(d), k_weight=kw.to(d), rope=(cos.to(d), sin.to(d)), fmt=fmt)
    x = (torch.randn(2 * T, D, generator=g) * 1.5).half()
    xd = x.to(d)
    got = block(xd)
    assert torch.equal(xd.cpu(), x)
    w = {k[len("blocks.0.") :]: v.double() for k, v in raw.items()}
    val = lambda t: O.values(*O.quantize(t, fmt), fmt)  # noqa: E731
    lin = lambda t, n: val(t) @ val(w[n + ".weight"].float()).t() + w[n + ".bias"]  # noqa: E731
    ln = lambda t, n: O.layer_norm(t, w[n + ".weight"], w[n + ".bias"], cfg.ln_eps)  # noqa: E731
    f16 = lambda t: t.half().double()  # noqa: E731
    def heads_of(y):
        q = O.heads(y[:, :D], H, 64, qw, None, "rms", cfg.ln_eps, cos, sin, "pairs")
        k = O.heads(y[:, D : 2 * D], H, 64, kw, None, "rms", cfg.ln_eps, cos, sin, "pairs")
        return torch.cat([q, k, y[:, 2 * D :]], 1)

    def close(name, got, ref):
        rel = ((got.cpu().double() - ref).norm() / ref.norm()).item()
        assert rel <= 2e-2, f"{name}: relative error {rel:.3g}"

    act = (lambda u: O.silu_mul(u[:, : cfg.mlp_hidden], u[:, cfg.mlp_hidden :])) if arch == "eva02" else O.gelu_tanh
    hidden = (lambda t: ln(t, "mlp_norm")) if arch == "eva02" else (lambda t: t)
    # layer by layer
    qkv = block.qkv(xd)
    close("qkv", qkv, heads_of(lin(ln(x, "norm1"), "qkv")))
    from foidfinder_b200 import ops

    o = torch.empty_like(xd)
    ops.attention(qkv, o, T, H, scale=0.125)
    x1 = block.proj(o, residual=xd)
    close("proj", x1 - xd, lin(o.cpu(), "proj"))
    h = block.fc1(x1)
    close("fc1", h, act(lin(ln(x1.cpu(), "norm2"), "fc1")))
    x2 = block.fc2(h, residual=x1)
    close("fc2", x2 - x1, lin(hidden(h.cpu()), "fc2"))
    assert torch.equal(got, x2)
    # as a whole
    q, k, v = (f16(t).view(2, T, H, 64).transpose(1, 2) for t in heads_of(lin(ln(x, "norm1"), "qkv")).split(D, 1))
    o = f16((torch.softmax(q @ k.transpose(-1, -2) / 8, -1) @ v).transpose(1, 2).reshape(2 * T, D))
    x1 = f16(x.double() + lin(o, "proj"))
    ref = x1 + lin(hidden(f16(act(lin(ln(x1, "norm2"), "fc1")))), "fc2")
    close("block", got, ref)


def test_swiglu_into_no_columns_writes_nothing(cuda_device, no_device_error):
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    layer = fp4.Fp4Linear(torch.ones(128, 64, device=d), epilogue="swiglu")
    x = torch.ones(4, 64, dtype=torch.float16, device=d)
    q, W = fp4.quantize(x), layer.weight
    buf = torch.full((4, 64), 77.0, dtype=torch.float16, device=d)
    with pytest.raises(RuntimeError, match="out is"):
        ops.gemm_fp4(q.codes, q.scales, q.row_scale, W.codes, W.scales, W.row_scale, buf[:, :0], ops.EPI_SWIGLU, 0, N=128, K=64)
    with pytest.raises(RuntimeError, match="out is"):
        ops.linear_fp4(x, W.codes, W.scales, W.row_scale, buf[:, :0], ops.EPI_SWIGLU, 0, N=128)
    assert (buf == 77.0).all()


@pytest.mark.parametrize("fmt", ["nv", "mx"])
def test_an_rms_norm_has_no_bias(cuda_device, no_device_error, fmt):
    """Biases given with an RMS head norm change nothing, neither in the product's epilogue nor by itself."""
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    g = torch.Generator().manual_seed(3)
    w, b = (1 + 0.1 * torch.randn(64, generator=g)).to(d), torch.full((64,), 3.0, device=d)
    cos, sin = (t.to(d) for t in _tables(7, 32))
    weight, x = _x(3 * 64, 128, torch.float32, 2).to(d), _x(40, 128, torch.float16, 5).to(d)
    kw = dict(fmt=fmt, epilogue="qkv", rope=(cos, sin), norm="rms", q_weight=w, k_weight=w)
    assert torch.equal(fp4.Fp4Linear(weight, q_bias=b, k_bias=b, **kw)(x), fp4.Fp4Linear(weight, **kw)(x))
    args = dict(q_heads=1, k_heads=1, head_dim=64, norm="rms", q_weight=w, k_weight=w, rope_cos=cos, rope_sin=sin)
    with_bias, without = torch.empty_like(x), torch.empty_like(x)
    ops.qk_norm_rope(x, with_bias, q_bias=b, k_bias=b, **args)
    ops.qk_norm_rope(x, without, **args)
    assert torch.equal(with_bias, without)


def _biases_only(values, epilogue, device):
    """A layer whose products are zero: its epilogue gets the biases, exactly."""
    from foidfinder_b200 import fp4

    v = torch.tensor(values)
    return fp4.Fp4Linear(torch.zeros(len(v), 64, device=device), v.to(device), epilogue=epilogue)


def _check_whole_range(got, ref, tol, dtype):
    """Within `tol` and the type's rounding where the type holds the value, its rounding (an infinity) where it does not."""
    top = torch.finfo(dtype).max
    inside = ref.abs() <= top
    _close(torch.where(inside, got.cpu().double(), 0), torch.where(inside, ref, 0), torch.where(inside, tol, 0), dtype)
    assert torch.equal(got.cpu()[~inside].float(), torch.copysign(torch.full_like(ref[~inside], math.inf), ref[~inside]).float())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_swiglu_over_the_whole_range_of_gates(cuda_device, no_device_error, dtype):
    """silu goes to zero below; f32 gates and ups of any size. 2^t with |t| <= 62 in f32 is within 62 * 2^-23 (2^-17) of
    itself, the remaining operations within 2^-21: 2^-16 of the result, and 2^-56 of the up where the gate is cut off."""
    gates = [-3e38, -1e20, -1e6, -200.0, -88.0, -60.0, -43.5, -43.0, -42.9, -30.0, -10.0, -1.0, -1e-20, 0.0, 1e-20, 0.5, 20.0, 43.5, 100.0, 1e6, 1e20]
    ups = [1.0, -2.5, 1e-20, 1e6, -1e20, 1e30, 3e37]
    g, u = torch.tensor(gates).repeat_interleave(len(ups)), torch.tensor(ups).repeat(len(gates))
    x = torch.ones(3, 64, dtype=dtype, device=cuda_device)
    got = _biases_only(torch.cat([g, u]).tolist(), "swiglu", cuda_device)(x)
    ref = (g.double() * torch.sigmoid(g.double()) * u.double())[None].expand(3, -1)
    edge = 2.0**-14 * torch.finfo(dtype).max
    clear = (ref.abs() - torch.finfo(dtype).max).abs() > edge  # not next to the largest value, where rounding decides
    assert clear.all()
    _check_whole_range(got, ref, 2.0**-16 * ref.abs() + 2.0**-56 * u.double().abs(), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gelu_over_the_whole_range(cuda_device, no_device_error, dtype):
    """The bounds are those of SwiGLU; where the argument is cut off the result is off by 7.6 * 2^-62 < 2^-59."""
    v = torch.tensor([-3e38, -1e20, -1e10, -1e5, -100.0, -10.0, -8.0, -7.7, -7.5, -5.0, -1.0, -1e-20, 0.0, 1e-20, 1.0, 7.7, 100.0, 1e4, 1e10, 1e20, 1e38])
    x = torch.ones(3, 64, dtype=dtype, device=cuda_device)
    got = _biases_only(v.tolist(), "gelu", cuda_device)(x)
    y = v.double()
    ref = (y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))[None].expand(3, -1)
    _check_whole_range(got, ref, 2.0**-16 * ref.abs() + 2.0**-59, dtype)


@pytest.mark.parametrize("epilogue", ["swiglu", "gelu"])
def test_a_nan_column_stays_in_its_column(cuda_device, no_device_error, epilogue):
    v = [0.5 + 0.01 * i for i in range(64)]
    x = torch.ones(3, 64, dtype=torch.float16, device=cuda_device)
    good = _biases_only(v, epilogue, cuda_device)(x)
    for at in (0, 7, 31):
        got = _biases_only(v[:at] + [math.nan] + v[at + 1 :], epilogue, cuda_device)(x)
        keep = torch.arange(good.shape[1], device=cuda_device) != at
        assert torch.isnan(got[:, at]).all() and torch.equal(got[:, keep], good[:, keep])


def _layers(device, fmt="nv"):
    from foidfinder_b200 import fp4

    g = torch.Generator().manual_seed(3)
    p = lambda n: (1 + 0.1 * torch.randn(n, generator=g)).to(device)  # noqa: E731
    rope = tuple(t.to(device) for t in _tables(7, 32))
    w = lambda n: _x(n, 128, torch.float32, n).to(device)  # noqa: E731
    return [fp4.Fp4Linear(w(96), p(96), fmt=fmt, gamma=p(128), beta=p(128)), fp4.Fp4Linear(w(80), p(80), fmt=fmt, epilogue="swiglu"),
            fp4.Fp4Linear(w(192), fmt=fmt, epilogue="qkv", norm="layer", rope=rope, q_weight=p(64), k_weight=p(64), q_bias=p(64), k_bias=p(64))]


@pytest.mark.parametrize("fmt", ["nv", "mx"])
def test_layers_can_be_copied_and_stored(cuda_device, no_device_error, fmt):
    """A copy has tensors of its own: what the first layer's memory holds afterwards does not matter."""
    import copy
    import pickle

    x = _x(33, 128, torch.float16, 1).to(cuda_device)
    for layer in _layers(cuda_device, fmt):
        ref = layer(x)
        copies = [copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))]
        for t in (layer.weight.codes, layer.weight.scales, layer.weight.row_scale, layer.bias, layer.gamma, layer.beta, *layer._heads.values()):
            if isinstance(t, torch.Tensor):
                t.zero_()
        for c in copies:
            assert torch.equal(c(x), ref)


def test_replaced_parameters_count(cuda_device, no_device_error):
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    x = _x(33, 128, torch.float16, 1).to(d)
    layer = _layers(d)[0]
    before = [layer.weight, layer.bias, layer.gamma, layer.beta]  # kept alive
    w = _x(96, 128, torch.float32, 5).to(d)
    bias, gamma, beta = (torch.linspace(a, 2, n, device=d) for a, n in ((0, 96), (1, 128), (-1, 128)))
    layer.weight, layer.bias, layer.gamma, layer.beta = fp4.quantize(w, "mx"), bias, gamma, beta
    ref = fp4.Fp4Linear(w, bias, fmt="mx", gamma=gamma, beta=beta)(x)
    assert torch.equal(layer(x), ref) and layer.fmt == "mx" and layer.bias is bias
    with pytest.MonkeyPatch.context() as m:  # and the long way
        m.setattr(ops, "_calls", lambda: ops._NoCalls)
        assert torch.equal(layer(x), ref)
    bias.data = torch.zeros(96, device=d)
    assert torch.equal(layer(x), fp4.Fp4Linear(w, fmt="mx", gamma=gamma, beta=beta)(x))
    layer.bias = None
    assert torch.equal(layer(x), fp4.Fp4Linear(w, fmt="mx", gamma=gamma, beta=beta)(x))
    with pytest.raises(RuntimeError, match="bias"):
        layer.bias = torch.zeros(95, device=d)
    layer.gamma = torch.ones(127, device=d)
    with pytest.raises(RuntimeError, match="gamma"):
        layer(x)
    layer.gamma, layer.weight = gamma, fp4.quantize(w[:95])
    with pytest.raises(RuntimeError, match="the weight is"):
        layer(x)
    del before


def test_f32_values_come_back_in_f32(cuda_device, no_device_error):
    """Without `out` a layer gives x's type: f32 values beyond fp16 stay finite where the epilogue can write f32."""
    from foidfinder_b200 import fp4

    d = cuda_device
    x, w = torch.full((3, 64), 960.0, device=d), torch.full((16, 64), 96.0, device=d)  # 6 x 320 / 2 and 6 x 256 / 16: exact in "nv"
    y = fp4.Fp4Linear(w)(x)
    assert y.dtype is torch.float32 and (y == 64 * 960.0 * 96.0).all()
    assert fp4.Fp4Linear(w)(x.half()).dtype is torch.float16 and fp4.Fp4Linear(w)(x.bfloat16()).dtype is torch.bfloat16
    assert fp4.Fp4Linear(w, epilogue="gelu")(x).dtype is torch.float16


def test_a_single_row_may_have_any_stride(cuda_device, no_device_error):
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    x, w = _x(1, 100, torch.float16, 1).to(d), _x(45, 100, torch.float32, 2).to(d)
    r = _x(1, 45, torch.float16, 3).to(d)
    for epilogue, residual in (("bias", None), ("residual", r)):
        layer = fp4.Fp4Linear(w, epilogue=epilogue)
        wide = None if residual is None else torch.cat([r, r], 1)[:, :48].contiguous()[:, :45]
        ref = layer(x, residual=wide)
        buf = torch.full((60,), 77.0, dtype=torch.float16, device=d)
        assert torch.equal(layer(x, out=buf[:45].view(1, 45), residual=residual), ref)
        assert (buf[45:] == 77.0).all()
    t, hw = torch.linspace(0, 1, 16 * 3, device=d).view(16, 3), torch.ones(32, device=d)
    args = dict(q_heads=1, k_heads=1, head_dim=32, norm="rms", q_weight=hw, k_weight=hw, rope_cos=t, rope_sin=t)
    ref = torch.empty(1, 64, dtype=torch.float16, device=d)
    ops.qk_norm_rope(x[:, :96], ref, **args)  # x: 100 elements from row to row
    narrow = x[:, :96].contiguous()
    ops.qk_norm_rope(narrow, narrow[:, :64], **args)
    assert torch.equal(narrow[:, :64], ref) and torch.equal(narrow[:, 64:], x[:, 64:96])


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize(("cols", "dtype"), [(8193, torch.float32), (9500, torch.float16), (9500, torch.float32), (11000, torch.bfloat16), (12288, torch.float16)])
def test_rows_that_fit_registers_stay_there(cuda_device, no_device_error, cols, dtype, fmt):
    """Up to 12288 columns a CTA's lanes hold the row (two or three pieces each); wider rows are read again for each step."""
    from foidfinder_b200 import fp4

    x = _x(5, cols, dtype, cols)
    xd = x.to(cuda_device)
    if dtype is torch.float32:
        _check_exact(fp4.quantize(xd, fmt), x)
    g = torch.Generator().manual_seed(9)
    gamma, beta = 1 + 0.1 * torch.randn(cols, generator=g), 0.1 * torch.randn(cols, generator=g)
    kw = dict(gamma=gamma.to(cuda_device), beta=beta.to(cuda_device), eps=1e-5)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        q = fp4.quantize(xd, fmt, **kw)
        torch.cuda.synchronize()
    names = [e.key for e in prof.key_averages() if "quantize_fp4" in e.key]
    assert not any("wide" in n for n in names), names  # none where the profiler is not available
    codes, s, row = _read(q)
    ec, es, er = O.quantize(O.layer_norm(x, gamma, beta, 1e-5), fmt)
    nb = es.shape[1]
    assert torch.equal(row, er)
    assert (s[:, :nb].int() - es.int()).abs().max() <= 1 and (s[:, :nb] != es).float().mean() <= 1e-3
    assert s[:, nb:].count_nonzero() == 0 and (codes != ec).float().mean() <= 1e-3


TIES = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]


def _ulps(v, n, dtype):
    """The n-th neighbours (above for n > 0) of the positive values v of type dtype."""
    bits = {torch.float32: torch.int32}.get(dtype, torch.int16)
    return (v.to(dtype).view(bits) + n).view(dtype)


@pytest.mark.parametrize(("dtype", "exponents"), [(torch.float32, (-100, -40, -3, 0, 1, 60, 115)), (torch.float16, (-4, 0, 3)), (torch.bfloat16, (-100, -7, 0, 100))])
def test_every_tie_of_every_block_scale(cuda_device, no_device_error, dtype, exponents):
    """All 7 ties times all 126 block scales, and the values next to them on either side, of either sign."""
    from foidfinder_b200 import fp4

    scales = O.e4m3_grid()[1:]
    v = torch.tensor(TIES, dtype=torch.float64)[None] * scales[:, None]  # [126, 7], exact in every type
    assert torch.equal(v.to(dtype).double(), v)
    v = torch.stack([_ulps(v, n, dtype) for n in (-1, 0, 1)], 2).reshape(126, 21).double()
    blocks = torch.zeros(126, 2, 16, dtype=torch.float64)
    blocks[:, :, 0] = 6 * scales[:, None]  # the block's largest value: its scale comes out exactly
    blocks[:, 0, 1:] = v[:, :15]
    blocks[:, 1, 1:7] = v[:, 15:]
    blocks[:, 1, 7:] = v[:, :9]
    sign = torch.where(torch.rand(126, 2, 16, generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0)
    rows = torch.zeros(17, 16, 16, dtype=torch.float64)
    rows[:, 0, 0] = 2688  # the row's largest value: row scale 1
    flat = (blocks * sign).reshape(252, 16)
    rows[:, 1:] = torch.cat([flat, flat[:3]]).view(17, 15, 16)
    x = torch.cat([rows.view(17, 256) * 2.0**e for e in exponents])
    low = x.to(dtype)
    if dtype is not torch.float16:  # fp16 runs out of exponents for the smallest ties: those are rounded, all others exact
        assert torch.equal(low.double(), x)
    _check_exact(fp4.quantize(low.to(cuda_device), "nv"), low)


@pytest.mark.parametrize("exponent", [-100, -20, 0, 90])
def test_block_maxima_next_to_the_ties_of_scales(cuda_device, no_device_error, exponent):
    """f32 block maxima that are 6 times a midpoint between two block scales, all 126 of them, or next to it."""
    from foidfinder_b200 import fp4

    grid = O.e4m3_grid()
    mid = 6 * (grid[:-1] + grid[1:]) / 2
    top = torch.stack([_ulps(mid, n, torch.float32) for n in (-1, 0, 1)], 1).double().reshape(-1)  # 378
    blocks = torch.rand(378, 16, generator=torch.Generator().manual_seed(2), dtype=torch.float64) * top[:, None] * 0.99
    blocks[:, 5] = -top
    rows = torch.zeros(27, 15, 16, dtype=torch.float64)
    rows[:, 0, 0] = 2688
    rows[:, 1:] = blocks.view(27, 14, 16)
    x = (rows.view(27, 240) * 2.0**exponent).float()
    _check_exact(fp4.quantize(x.to(cuda_device), "nv"), x)


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize(("tile", "epi", "N", "K", "dtype"), [
    (128, "bias", 4203, 320, torch.float32), (512, "bias", 4203, 320, torch.float32),
    (128, "bias", 4203, 320, torch.float16), (512, "bias", 4203, 1300, torch.bfloat16),
    (128, "gelu", 4200, 70, torch.bfloat16), (512, "gelu", 4200, 320, torch.float16),
    (128, "residual", 4203, 1300, torch.float16), (512, "residual", 4203, 320, torch.bfloat16),
    (128, "swiglu", 4202, 320, torch.bfloat16), (512, "swiglu", 4202, 320, torch.float16), (512, "swiglu", 4202, 1300, torch.bfloat16),
    (128, "qkv rms", 4224, 320, torch.float16), (128, "qkv layer", 4224, 1300, torch.bfloat16),
])
def test_products_of_many_tiles(cuda_device, no_device_error, tile, epi, N, K, dtype, fmt):
    """9 tiles or more for every CTA pair and 17 for every CTA of 148: both accumulators, the columns that they share, and
    every ring of buffers are used again and again, with partial last tiles both ways. Equal to the last bit to the same
    rows multiplied 250 at a time, where no CTA has a second tile (those are compared with the oracle above)."""
    from foidfinder_b200 import fp4, ops

    d = cuda_device
    M, part = 10000, 250
    g = torch.Generator().manual_seed(7)
    x, w = _x(M, K, torch.float16, 1).to(d), (torch.randn(N, K, generator=g) * 0.05).to(d)
    bias = (torch.randn(N, generator=g) * 0.1).to(d)
    kind = {"bias": ops.EPI_BIAS, "gelu": ops.EPI_GELU, "residual": ops.EPI_RESIDUAL, "swiglu": ops.EPI_SWIGLU}.get(epi, ops.EPI_QKV_NORM_ROPE)
    cols, kw = N, {}
    if epi == "swiglu":
        layer = fp4.Fp4Linear(w, bias, fmt=fmt, epilogue="swiglu")
        W, bias, cols = layer.weight, layer.bias, N // 2
    else:
        W = fp4.quantize(w, fmt)
    period = part
    if epi.startswith("qkv"):
        hw = [(1 + 0.1 * torch.randn(64, generator=g)).to(d) for _ in range(4)]
        cos, sin = (t.to(d) for t in _tables(period, 32))  # positions start again with every part
        kw = dict(norm=epi[4:], q_heads=30, k_heads=18, q_weight=hw[0], k_weight=hw[1], rope_cos=cos, rope_sin=sin)
        kw |= dict(q_bias=hw[2], k_bias=hw[3]) if epi == "qkv layer" else {}
    residual = torch.randn(M, cols, generator=g).to(dtype).to(d) if epi == "residual" else None

    def product(rows, out):
        q = fp4.quantize(x[rows], fmt)
        if residual is not None:
            out.copy_(residual[rows])  # in place
        ops.gemm_fp4(q.codes, q.scales, q.row_scale, W.codes, W.scales, W.row_scale, out, kind, FMT[fmt], N=W.rows, K=K, bias=bias,
                     residual=None if residual is None else out, tile=tile, **kw)

    pitch = (cols + 7) // 8 * 8 + 8
    buf = torch.full((M + 8, pitch), 77.0, dtype=dtype, device=d)
    ref = torch.full((M, pitch), 77.0, dtype=dtype, device=d)[:, :cols]
    for first in range(0, M, part):
        product(slice(first, first + part), ref[first : first + part])
    for _ in range(3):
        buf.fill_(77.0)
        product(slice(0, M), buf[:M, :cols])
        assert torch.equal(buf[:M, :cols], ref)
    assert (buf[M:] == 77.0).all() and (buf[:, cols:] == 77.0).all()


@pytest.mark.parametrize("pairing", ["pairs", "halves"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize(("rows", "qh", "kh", "dim", "tokens", "dtype"), [
    (50, 64, 16, 128, 7, torch.bfloat16),  # few rows: a warp for every chunk of heads
    (5, 9, 7, 256, 3, torch.float16),  # the same, chunks that are not full
    (3000, 20, 12, 128, 1025, torch.float16),  # four warps take turns with a row's five chunks
    (7500, 9, 5, 128, 1025, torch.bfloat16),  # a warp per row, several rows per warp, three chunks of both kinds
    (15000, 3, 2, 32, 577, torch.float16),  # the same, one chunk of each kind
])
def test_qk_norm_rope_of_many_heads_and_rows(cuda_device, no_device_error, rows, qh, kh, dim, tokens, dtype, norm, pairing):
    from foidfinder_b200 import ops

    d = cuda_device
    cols = (qh + kh) * dim
    x = (_x(rows, cols + 8, torch.float32, rows, outliers=False) * 1.5).to(dtype)
    g = torch.Generator().manual_seed(4)
    qw, kw = 1 + 0.1 * torch.randn(dim, generator=g), 1 + 0.1 * torch.randn(dim, generator=g)
    qb, kb = (0.1 * torch.randn(dim, generator=g), 0.1 * torch.randn(dim, generator=g)) if norm == "layer" else (None, None)
    cos, sin = _tables(tokens, dim // 2)
    dev = lambda t: None if t is None else t.to(d)  # noqa: E731
    args = dict(q_heads=qh, k_heads=kh, head_dim=dim, norm=norm, q_weight=dev(qw), k_weight=dev(kw), q_bias=dev(qb), k_bias=dev(kb), eps=1e-6,
                rope_cos=dev(cos), rope_sin=dev(sin), pairing=pairing)
    out = torch.full((rows, cols + 16), 77.0, device=d, dtype=dtype)
    xd = x.to(d)
    ops.qk_norm_rope(xd, out, **args)
    ref = torch.cat([O.heads(x[:, : qh * dim], qh, dim, qw, qb, norm, 1e-6, cos, sin, pairing),
                     O.heads(x[:, qh * dim : cols], kh, dim, kw, kb, norm, 1e-6, cos, sin, pairing)], 1)
    _close(out[:, :cols], ref, 2.0**-20 * torch.full_like(ref, 10.0), dtype)  # as in test_qk_norm_rope
    assert (out[:, cols:] == 77.0).all()
    ops.qk_norm_rope(xd, xd, **args)
    assert torch.equal(xd[:, :cols], out[:, :cols]) and torch.equal(xd[:, cols:].cpu(), x[:, cols:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [511, 512, 513, 1024, 1025, 1537, 2048, 2049, 3071, 3073, 4096, 4097, 5120, 5121])
def test_quantize_at_the_widths_where_variants_change(cuda_device, no_device_error, cols, dtype):
    from foidfinder_b200 import fp4

    x = _x(9, cols, dtype, cols)
    _check_exact(fp4.quantize(x.to(cuda_device), "nv"), x)
    wide = torch.full((9, (cols + 15) // 8 * 8), math.nan, dtype=dtype, device=cuda_device)[:, :cols]  # rows on 16-byte boundaries
    wide.copy_(x)
    _check_exact(fp4.quantize(wide, "nv"), x)


_FIRST_CALLS = """
import sys, torch
from foidfinder_b200 import fp4, ops
d = "cuda"
x, w = torch.randn(8, 64, device=d).half(), torch.randn(128, 64, device=d)
out, v, h = torch.empty(8, 128, device=d).half(), torch.empty(8, 64, device=d).half(), torch.empty(8, 64, device=d).half()
t, hw = torch.ones(16, 3, device=d), torch.ones(32, device=d)
q, weight = fp4.Fp4Tensor.empty(8, 64, "nv"), fp4.Fp4Tensor.empty(128, 64, "nv")
def calls():
    fp4.quantize(w, out=weight)
    fp4.quantize(x, out=q)
    fp4.dequantize(q, out=v)
    ops.linear_fp4(x, weight.codes, weight.scales, weight.row_scale, out, ops.EPI_BIAS, 0, N=128)
    ops.qk_norm_rope(x, h, q_heads=1, k_heads=1, head_dim=32, norm="rms", q_weight=hw, k_weight=hw, rope_cos=t, rope_sin=t)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (out, v, h)]
calls()
assert all(torch.equal(a, b) for a, b in zip(got, (out, v, h))) and ops.device_error(0) == 0
"""


def test_the_first_calls_of_a_process_can_be_captured(cuda_device):
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", _FIRST_CALLS], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
