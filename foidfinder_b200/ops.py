"""Per-kernel entry points on torch CUDA tensors, mirroring the reference's `torch.ops.foidfinder` ops
(foidfinder/backends/cuda/csrc/kernels.cu:267-281): outputs are caller-allocated and written in place,
shape/dtype violations raise, and every launch goes on the current CUDA stream. Each call goes through
the C ABI of `libfoidfinder_b200.so`; torch is only the memory and stream plumbing.
"""

from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import (
    EPI_BIAS, EPI_GELU, EPI_LOGITS, EPI_QKV_NORM_ROPE, EPI_QKV_ROPE, EPI_RESIDUAL, EPI_S32, EPI_STEM, EPI_SWIGLU, FP4_MX,
    FP4_NV, TILE_PAIR256, check, lib,
)

__all__ = [
    "EPI_QKV_ROPE", "EPI_RESIDUAL", "EPI_SWIGLU", "EPI_BIAS", "EPI_S32", "EPI_STEM", "EPI_LOGITS", "EPI_GELU", "TILE_PAIR256",
    "gemm_s8", "gemm_f16", "rot_q8", "rot_q8_1024", "rot_q8_h128", "attention", "patchify", "fill_cls",
    "layernorm", "topk", "tree_pool", "resize_pad", "patchify_windowed", "layernorm_pos", "pool_query_attention",
    "FP4_NV", "FP4_MX", "EPI_QKV_NORM_ROPE", "quantize_fp4", "dequantize_fp4", "gemm_fp4", "linear_fp4", "qk_norm_rope",
]


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda(*ts: torch.Tensor | None) -> None:
    for t in ts:
        if t is not None:
            _need(t.is_cuda and t.is_contiguous(), "expected contiguous CUDA tensors")


def gemm_s8(
    A: torch.Tensor,
    W: torch.Tensor,
    row_scale: torch.Tensor | None,
    col_scale: torch.Tensor | None,
    bias: torch.Tensor | None,
    out: torch.Tensor,
    epi: int,
    tile_n: int = 0,
    rope_cos: torch.Tensor | None = None,
    rope_sin: torch.Tensor | None = None,
    rope_cols: int = 0,
    tokens: int = 1,
) -> None:
    """A [M, K] int8 x W [N, K] int8 -> epilogue into out (see include/foidfinder_b200.h). RoPE tables
    for EPI_QKV_ROPE are angle-major [32, tokens]."""
    _cuda(A, W, row_scale, col_scale, bias, out, rope_cos, rope_sin)
    _need(A.dtype == torch.int8 and W.dtype == torch.int8, "gemm_s8: A and W must be int8")
    M, K = A.shape
    N = W.shape[0]
    _need(W.shape[1] == K, "gemm_s8: K mismatch")
    if epi == EPI_S32:
        _need(out.dtype == torch.int32 and tuple(out.shape) == (M, N), "gemm_s8: S32 out must be int32 [M, N]")
    else:
        cols = N // 2 if epi == EPI_SWIGLU else N
        _need(out.dtype == torch.float16 and tuple(out.shape) == (M, cols), f"gemm_s8: out must be fp16 [{M}, {cols}]")
        _need(row_scale.numel() == M and col_scale.numel() == N and bias.numel() == N, "gemm_s8: scale/bias sizes")
    with torch.cuda.device(A.device):
        check(
            lib().ff_gemm_s8(
                _ptr(A), _ptr(W), _ptr(row_scale), _ptr(col_scale), _ptr(bias), _ptr(out), M, N, K, epi,
                _ptr(rope_cos), _ptr(rope_sin), rope_cols, tokens, tile_n, _stream(A),
            ),
            "gemm_s8",
        )


def gemm_f16(
    A: torch.Tensor,
    W: torch.Tensor,
    out: torch.Tensor,
    epi: int,
    bias: torch.Tensor | None = None,
    n_valid: int | None = None,
    pos_bias: torch.Tensor | None = None,
    patches: int = 0,
    tokens: int = 0,
    tile_n: int = 0,
) -> None:
    """fp16 A [M, K] x W [N, K] with f32 accumulation: EPI_STEM into the token rows of x, EPI_LOGITS into f32."""
    _cuda(A, W, out, bias, pos_bias)
    _need(A.dtype == torch.float16 and W.dtype == torch.float16, "gemm_f16: A and W must be fp16")
    M, K = A.shape
    N = W.shape[0]
    ldo = out.shape[-1]
    nv = n_valid if n_valid is not None else min(N, ldo)
    with torch.cuda.device(A.device):
        check(
            lib().ff_gemm_f16(
                _ptr(A), _ptr(W), _ptr(bias), _ptr(out), M, N, K, epi, ldo, nv, _ptr(pos_bias), patches, tokens,
                tile_n, _stream(A),
            ),
            "gemm_f16",
        )


def rot_q8(
    x: torch.Tensor,
    gamma: torch.Tensor | None,
    beta: torch.Tensor | None,
    out: torch.Tensor,
    row_scale: torch.Tensor,
    *,
    block: int,
    eps: float = 1e-6,
    valid_cols: int | None = None,
) -> None:
    """x [T, C] fp16 -> (LayerNorm) -> block Hadamard -> int8 codes out [T, C] + row_scale [T]."""
    _cuda(x, gamma, beta, out, row_scale)
    _need(x.dtype == torch.float16 and out.dtype == torch.int8 and out.shape == x.shape, "rot_q8: dtypes/shapes")
    T, Ccols = x.shape
    with torch.cuda.device(x.device):
        check(
            lib().ff_rot_q8(
                _ptr(x), _ptr(gamma), _ptr(beta), eps, T, Ccols, valid_cols or Ccols, block, _ptr(out),
                _ptr(row_scale), _stream(x),
            ),
            "rot_q8",
        )


def rot_q8_1024(x, gamma, beta, out, row_scale) -> None:
    """Reference signature (kernels.cu:220): LayerNorm eps 1e-5 if gamma is given, H1024, int8."""
    rot_q8(x, gamma, beta, out, row_scale, block=1024, eps=1e-5)


def rot_q8_h128(x, out, row_scale) -> None:
    """Reference signature (kernels.cu:238): block-H128 rotation and int8, no norm."""
    rot_q8(x, None, None, out, row_scale, block=128)


def attention(
    qkv: torch.Tensor,
    out: torch.Tensor,
    seq_len: int,
    heads: int | None = None,
    rope: tuple[torch.Tensor, torch.Tensor] | None = None,
    scale: float = 1.0,
) -> None:
    """qkv [S * seq_len, 3 * heads * 64] fp16 -> out [S * seq_len, heads * 64] fp16 (non-causal). `rope` must be
    None: q and k arrive rotated, as in the reference (its QKV GEMM epilogue rotates them; here EPI_QKV_ROPE)."""
    _cuda(qkv, out)
    _need(qkv.dtype == torch.float16 and out.dtype == torch.float16, "attention: fp16 tensors expected")
    heads = heads or qkv.shape[1] // 192
    _need(qkv.shape[1] == 3 * heads * 64 and out.shape[1] == heads * 64, "attention: column sizes")
    _need(qkv.shape[0] % seq_len == 0 and out.shape[0] == qkv.shape[0], "attention: row sizes")
    cos, sin = rope if rope is not None else (None, None)
    _cuda(cos, sin)
    with torch.cuda.device(qkv.device):
        check(
            lib().ff_attention(
                _ptr(qkv), _ptr(out), qkv.shape[0] // seq_len, seq_len, heads, _ptr(cos), _ptr(sin), scale,
                _stream(qkv),
            ),
            "attention",
        )


def patchify(images: torch.Tensor, patch: int, mean, std, out: torch.Tensor) -> None:
    _cuda(images, out)
    _need(images.dtype == torch.uint8 and images.dim() == 4, "patchify: uint8 [B, S, S, 3] expected")
    B, S = images.shape[:2]
    m = (C.c_float * 3)(*map(float, mean))
    s = (C.c_float * 3)(*map(float, std))
    with torch.cuda.device(images.device):
        check(lib().ff_patchify(_ptr(images), B, S, patch, m, s, _ptr(out), out.shape[1], _stream(images)), "patchify")


def fill_cls(cls_row: torch.Tensor, x: torch.Tensor, B: int, tokens: int) -> None:
    _cuda(cls_row, x)
    with torch.cuda.device(x.device):
        check(lib().ff_fill_cls(_ptr(cls_row), _ptr(x), B, tokens, x.shape[-1], _stream(x)), "fill_cls")


def layernorm(x: torch.Tensor, row_stride: int, rows: int, cols: int, gamma, beta, eps: float, out: torch.Tensor) -> None:
    _cuda(x, gamma, beta, out)
    with torch.cuda.device(x.device):
        check(
            lib().ff_layernorm(_ptr(x), row_stride, _ptr(gamma), _ptr(beta), eps, rows, cols, _ptr(out), _stream(x)),
            "layernorm",
        )


def topk(logits: torch.Tensor, k: int, idx: torch.Tensor, val: torch.Tensor | None = None) -> None:
    _cuda(logits, idx, val)
    B, n = logits.shape
    with torch.cuda.device(logits.device):
        check(lib().ff_topk(_ptr(logits), B, n, k, _ptr(idx), _ptr(val), _stream(logits)), "topk")


def device_error(device: int = 0, clear: bool = True) -> int:
    """Error code left by a kernel whose bounded wait ran out (0 = none); synchronises the device."""
    return _lib.device_error(device, clear)


def tree_pool(cfg, weights: dict[str, torch.Tensor], x: torch.Tensor, leaf_out: torch.Tensor) -> None:
    """Haruka tree attention pool head: x [B * tokens, dim] fp16 (backbone output before its final
    LayerNorm) -> leaf_out [B, leaf_queries * leaf_dim] fp16. `weights` in the engine format
    (`weights.convert`), on x's device."""
    from .engine import _POOL_KEYS, c_config

    _cuda(x, leaf_out)
    _need(cfg.head == "tree", "tree_pool: config has no tree head")
    _need(x.dtype == torch.float16 and leaf_out.dtype == torch.float16, "tree_pool: fp16 tensors expected")
    B = x.shape[0] // cfg.tokens
    _need(x.shape == (B * cfg.tokens, cfg.dim) and leaf_out.shape == (B, cfg.head_in), "tree_pool: bad shapes")
    c = c_config(cfg)
    mw = _lib.ModelWeights()
    for field, key in {"norm_w": "norm.weight", "norm_b": "norm.bias"}.items():
        setattr(mw, field, weights[key].data_ptr())
    for field, key in _POOL_KEYS.items():
        setattr(mw, field, weights[key].data_ptr())
    nbytes = int(lib().ff_tree_pool_workspace_bytes(C.byref(c), B))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        check(lib().ff_tree_pool(C.byref(c), C.byref(mw), _ptr(x), B, _ptr(ws), nbytes, _ptr(leaf_out), _stream(x)),
              "tree_pool")
        torch.cuda.current_stream(x.device).synchronize()  # keeps the workspace alive until the pool has run


def resize_pad(image: torch.Tensor, new_h: int, new_w: int, size: int, out: torch.Tensor, *, bicubic: bool = True,
               fill: int = 255) -> None:
    """uint8 [h, w, 3] CUDA image -> out uint8 [size, size, 3]: Pillow-exact resize (bicubic or bilinear) to
    (new_h, new_w), centred on a `fill` canvas."""
    _cuda(image, out)
    _need(image.dtype == torch.uint8 and image.dim() == 3 and image.shape[2] == 3, "resize_pad: uint8 [h, w, 3]")
    _need(out.dtype == torch.uint8 and tuple(out.shape) == (size, size, 3), "resize_pad: out must be [size, size, 3]")
    h, w = image.shape[:2]
    flt = _lib.RESAMPLE_BICUBIC if bicubic else _lib.RESAMPLE_BILINEAR
    nbytes = int(lib().ff_resize_pad_workspace_bytes(h, w, new_h, new_w, flt))
    _need(nbytes > 0, "resize_pad: bad geometry")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=image.device)
    with torch.cuda.device(image.device):
        check(lib().ff_resize_pad(_ptr(image), h, w, new_h, new_w, size, flt, fill, _ptr(out), _ptr(ws), nbytes,
                                  _stream(image)), "resize_pad")
        torch.cuda.current_stream(image.device).synchronize()  # the workspace is freed on return


def letterbox_aa_f16(image: torch.Tensor, new_h: int, new_w: int, size: int, out: torch.Tensor) -> None:
    """uint8 [h, w, 3] CUDA image -> out fp16 [size, size, 3] normalised pixels: PixAI's float letterbox
    (foidfinder/backends/cuda/preprocess.py:16-32): /255, antialiased bilinear resize to (new_h, new_w) in
    f32, x * 2 - 1, centred on a canvas of -1."""
    _cuda(image, out)
    _need(image.dtype == torch.uint8 and image.dim() == 3 and image.shape[2] == 3, "letterbox_aa_f16: uint8 [h, w, 3]")
    _need(out.dtype == torch.float16 and tuple(out.shape[-3:]) == (size, size, 3) and out.is_contiguous(),
          "letterbox_aa_f16: out must be contiguous fp16 [size, size, 3]")
    image = image.contiguous()
    h, w = image.shape[:2]
    with torch.cuda.device(image.device):
        check(lib().ff_letterbox_aa_f16(_ptr(image), h, w, new_h, new_w, size, _ptr(out), _stream(image)),
              "letterbox_aa_f16")


def patchify_windowed(images: torch.Tensor, patch: int, mean, std, window: int, out: torch.Tensor) -> None:
    """uint8 [B, S, S, 3] -> fp16 patch rows [B * (S/patch)^2, k_pad] in window order (window x window tiles)."""
    _cuda(images, out)
    B, S = images.shape[:2]
    m = (C.c_float * 3)(*map(float, mean))
    s = (C.c_float * 3)(*map(float, std))
    with torch.cuda.device(images.device):
        check(lib().ff_patchify_windowed(_ptr(images), B, S, patch, m, s, _ptr(out), out.shape[1], window,
                                         _stream(images)), "patchify_windowed")


def layernorm_pos(x: torch.Tensor, gamma, beta, eps: float, pos: torch.Tensor, out: torch.Tensor) -> None:
    """LayerNorm of fp16 rows to fp16, then + pos[row % pos.shape[0]] in fp16."""
    _cuda(x, gamma, beta, pos, out)
    rows, cols = x.shape
    with torch.cuda.device(x.device):
        check(lib().ff_layernorm_pos(_ptr(x), cols, _ptr(gamma), _ptr(beta), eps, rows, cols, _ptr(pos), pos.shape[0],
                                     _ptr(out), _stream(x)), "layernorm_pos")


def pool_query_attention(q: torch.Tensor, kv: torch.Tensor, B: int, tokens: int, out: torch.Tensor) -> None:
    """q [heads * 64] f32 (scaled), kv [B * tokens, 2 * dim] fp16 -> out [B, dim] fp16."""
    _cuda(q, kv, out)
    heads = q.numel() // 64
    with torch.cuda.device(kv.device):
        check(lib().ff_pool_query_attention(_ptr(q), _ptr(kv), B, tokens, heads, _ptr(out), _stream(kv)),
              "pool_query_attention")


def int8_mma_peak(device: int = 0, iters: int = 200_000) -> float:
    """Measured dense int8 tensor-core throughput of `device` in TOPS (back-to-back tcgen05 MMAs on
    resident operands, one CTA per SM; about 50 ms)."""
    ms, ops = C.c_float(), C.c_double()
    with torch.cuda.device(device):
        check(lib().ff_int8_mma_peak(iters, C.byref(ms), C.byref(ops), torch.cuda.current_stream(device).cuda_stream),
              "int8_mma_peak")
    return ops.value / (ms.value * 1e-3) / 1e12


# ---------------------------------------------------------------- block-scaled 4-bit operands
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_NORMS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
_PAIRINGS = {"pairs": _lib.ROPE_PAIRS, "halves": _lib.ROPE_HALVES}


def _rows_2d(t: torch.Tensor, what: str) -> int:
    """Row stride of a 2-D tensor whose columns are contiguous."""
    _need(t.is_cuda and t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1), f"{what}: expected a 2-D CUDA tensor with contiguous columns")
    return max(t.stride(0), t.shape[1]) if t.shape[0] <= 1 else t.stride(0)


def _params(n: int, device: torch.device, what: str, **ts: torch.Tensor | None) -> None:
    for name, t in ts.items():
        if t is not None:
            _need(t.device == device and t.is_contiguous() and t.dtype == torch.float32 and t.numel() == n, f"{what}: {name} must be {n} contiguous f32 values on {device}")


def fp4_sizes(rows: int, cols: int, fmt: int) -> tuple[int, int]:
    """Bytes of the code and scale buffers of a [rows, cols] operand."""
    return int(lib().ff_fp4_code_bytes(rows, cols)), int(lib().ff_fp4_scale_bytes(rows, cols, fmt))


def _fp4_operand(codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor | None, rows: int, cols: int, fmt: int, what: str) -> None:
    _cuda(codes, scales, row_scale)
    nc, ns = fp4_sizes(rows, cols, fmt)
    _need(codes.dtype == torch.uint8 and codes.numel() >= nc, f"{what}: codes must be uint8, {nc} bytes for [{rows}, {cols}]")
    _need(scales.dtype == torch.uint8 and scales.numel() >= ns, f"{what}: scales must be uint8, {ns} bytes for [{rows}, {cols}]")
    _need(scales.device == codes.device, f"{what}: codes and scales are on different devices")
    if fmt == FP4_NV:
        _params(rows, codes.device, what, row_scale=row_scale)
        _need(row_scale is not None, f"{what}: FP4_NV needs row_scale")


def quantize_fp4(
    x: torch.Tensor,
    codes: torch.Tensor,
    scales: torch.Tensor,
    row_scale: torch.Tensor | None,
    fmt: int,
    *,
    gamma: torch.Tensor | None = None,
    beta: torch.Tensor | None = None,
    eps: float = 1e-6,
) -> None:
    """x [T, C] fp16, bf16 or f32 (columns contiguous, any row stride) -> (LayerNorm) -> 4-bit codes and block scales
    (`fp4_sizes` bytes) and, for FP4_NV, row_scale [T] f32."""
    ldx = _rows_2d(x, "quantize_fp4")
    _need(x.dtype in _DTYPES, "quantize_fp4: x must be fp16, bf16 or f32")
    T, cols = x.shape
    _fp4_operand(codes, scales, row_scale, T, cols, fmt, "quantize_fp4")
    _need(codes.device == x.device, "quantize_fp4: x and codes are on different devices")
    _params(cols, x.device, "quantize_fp4", gamma=gamma, beta=beta)
    with torch.cuda.device(x.device):
        check(
            lib().ff_quantize_fp4(
                _ptr(x), _DTYPES[x.dtype], ldx, _ptr(gamma), _ptr(beta), eps, T, cols, fmt, _ptr(codes), _ptr(scales),
                _ptr(row_scale), _stream(x),
            ),
            "quantize_fp4",
        )


def dequantize_fp4(codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor | None, out: torch.Tensor, fmt: int) -> None:
    """The values of a 4-bit operand into out [T, C] (fp16, bf16 or f32; columns contiguous, any row stride)."""
    ldo = _rows_2d(out, "dequantize_fp4")
    _need(out.dtype in _DTYPES, "dequantize_fp4: out must be fp16, bf16 or f32")
    T, cols = out.shape
    _fp4_operand(codes, scales, row_scale, T, cols, fmt, "dequantize_fp4")
    _need(codes.device == out.device, "dequantize_fp4: codes and out are on different devices")
    with torch.cuda.device(out.device):
        check(
            lib().ff_dequantize_fp4(
                _ptr(codes), _ptr(scales), _ptr(row_scale), T, cols, fmt, _ptr(out), _DTYPES[out.dtype], ldo, _stream(out)
            ),
            "dequantize_fp4",
        )


def fp4_epilogue(
    epi: int,
    N: int,
    device: torch.device,
    *,
    bias: torch.Tensor | None = None,
    norm: str = "rms",
    q_heads: int = 0,
    k_heads: int = 0,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    q_bias: torch.Tensor | None = None,
    k_bias: torch.Tensor | None = None,
    qk_eps: float = 1e-6,
    rope_cos: torch.Tensor | None = None,
    rope_sin: torch.Tensor | None = None,
) -> _lib.Fp4Epilogue:
    """The part of a gemm_fp4 epilogue that does not change from call to call (the tensors must outlive it)."""
    e = _lib.Fp4Epilogue(kind=epi)
    _params(N, device, "fp4_epilogue", bias=bias)
    e.bias = _ptr(bias)
    if epi == EPI_QKV_NORM_ROPE:
        _need(norm in _NORMS, "fp4_epilogue: norm must be 'rms' or 'layer'")
        _params(64, device, "fp4_epilogue", q_weight=q_weight, k_weight=k_weight, q_bias=q_bias, k_bias=k_bias)
        _need(rope_cos is not None and rope_sin is not None and rope_cos.dim() == 2 and rope_cos.shape[0] == 32 and rope_sin.shape == rope_cos.shape,
              "fp4_epilogue: rotation tables must be [32, tokens]")
        _params(rope_cos.numel(), device, "fp4_epilogue", rope_cos=rope_cos, rope_sin=rope_sin)
        e.norm, e.q_heads, e.k_heads, e.tokens, e.qk_eps = _NORMS[norm], q_heads, k_heads, rope_cos.shape[1], qk_eps
        e.q_w, e.k_w, e.q_b, e.k_b = _ptr(q_weight), _ptr(k_weight), _ptr(q_bias), _ptr(k_bias)
        e.rope_cos, e.rope_sin = _ptr(rope_cos), _ptr(rope_sin)
    return e


def _bind_out(e: _lib.Fp4Epilogue, M: int, N: int, out: torch.Tensor, residual: torch.Tensor | None, device: torch.device, what: str) -> None:
    ldo = _rows_2d(out, what)
    cols = out.shape[1]
    _need(out.device == device and out.dtype in _DTYPES, f"{what}: out must be fp16, bf16 or f32 on {device}")
    _need(out.shape[0] == M and (cols <= N // 2 if e.kind == EPI_SWIGLU else cols == N), f"{what}: out has shape {tuple(out.shape)} for M={M} N={N}")
    e.out_dtype, e.out, e.ldo, e.out_cols = _DTYPES[out.dtype], _ptr(out), ldo, cols
    e.residual = None
    if e.kind == EPI_RESIDUAL:
        _need(residual is not None, f"{what}: EPI_RESIDUAL needs the residual")
        e.ldr = _rows_2d(residual, what)
        _need(residual.shape == out.shape and residual.dtype == out.dtype and residual.device == device, f"{what}: the residual must be like out")
        e.residual = _ptr(residual)


def gemm_fp4(
    A: torch.Tensor,
    A_scales: torch.Tensor,
    row_scale: torch.Tensor | None,
    W: torch.Tensor,
    W_scales: torch.Tensor,
    col_scale: torch.Tensor | None,
    out: torch.Tensor,
    epilogue: int | _lib.Fp4Epilogue,
    fmt: int,
    *,
    N: int,
    K: int,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    tile: int = 0,
    **heads,
) -> None:
    """4-bit A [M, K] x W [N, K] (operands of `quantize_fp4`) -> epilogue into out (see include/foidfinder_b200.h).
    `epilogue` is an EPI_* number, with `bias` and the head arguments of `fp4_epilogue`, or a prepared
    `fp4_epilogue`."""
    M = out.shape[0]
    _fp4_operand(A, A_scales, row_scale, M, K, fmt, "gemm_fp4")
    _fp4_operand(W, W_scales, col_scale, N, K, fmt, "gemm_fp4")
    _need(W.device == A.device, "gemm_fp4: A and W are on different devices")
    e = fp4_epilogue(epilogue, N, A.device, bias=bias, **heads) if isinstance(epilogue, int) else epilogue
    _bind_out(e, M, N, out, residual, A.device, "gemm_fp4")
    with torch.cuda.device(A.device):
        check(
            lib().ff_gemm_fp4(
                _ptr(A), _ptr(A_scales), _ptr(row_scale), _ptr(W), _ptr(W_scales), _ptr(col_scale), fmt, M, N, K,
                C.byref(e), tile, _stream(A),
            ),
            "gemm_fp4",
        )


def linear_fp4(
    x: torch.Tensor,
    W: torch.Tensor,
    W_scales: torch.Tensor,
    col_scale: torch.Tensor | None,
    out: torch.Tensor,
    epilogue: int | _lib.Fp4Epilogue,
    fmt: int,
    *,
    N: int,
    gamma: torch.Tensor | None = None,
    beta: torch.Tensor | None = None,
    eps: float = 1e-6,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    **heads,
) -> None:
    """quantize_fp4 of x [M, K] (with the LayerNorm, if gamma is given) and gemm_fp4 in one call; the codes of x live
    in a workspace from torch's allocator on the current stream."""
    ldx = _rows_2d(x, "linear_fp4")
    M, K = x.shape
    _need(x.dtype in _DTYPES, "linear_fp4: x must be fp16, bf16 or f32")
    _fp4_operand(W, W_scales, col_scale, N, K, fmt, "linear_fp4")
    _need(W.device == x.device, "linear_fp4: x and W are on different devices")
    _params(K, x.device, "linear_fp4", gamma=gamma, beta=beta)
    e = fp4_epilogue(epilogue, N, x.device, bias=bias, **heads) if isinstance(epilogue, int) else epilogue
    _bind_out(e, M, N, out, residual, x.device, "linear_fp4")
    with torch.cuda.device(x.device):
        nbytes = lib().ff_linear_fp4_workspace_bytes(M, K, fmt)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        check(
            lib().ff_linear_fp4(
                _ptr(x), _DTYPES[x.dtype], ldx, _ptr(gamma), _ptr(beta), eps, _ptr(W), _ptr(W_scales), _ptr(col_scale),
                fmt, M, N, K, C.byref(e), _ptr(ws), nbytes, _stream(x),
            ),
            "linear_fp4",
        )


def qk_norm_rope(
    x: torch.Tensor,
    out: torch.Tensor,
    *,
    q_heads: int,
    k_heads: int,
    head_dim: int,
    norm: str,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    rope_cos: torch.Tensor,
    rope_sin: torch.Tensor,
    q_bias: torch.Tensor | None = None,
    k_bias: torch.Tensor | None = None,
    eps: float = 1e-6,
    pairing: str = "pairs",
) -> None:
    """x [T, >= (q_heads + k_heads) * head_dim] fp16 or bf16, q heads then k heads -> every head normalised ("rms" or
    "layer") and rotated by position row % tokens, into the first columns of out (x itself: in place). Tables are
    angle-major [head_dim / 2, tokens] f32; `pairing` "pairs" rotates (2i, 2i + 1), "halves" (i, i + head_dim / 2)."""
    ldx, ldo = _rows_2d(x, "qk_norm_rope"), _rows_2d(out, "qk_norm_rope")
    cols = (q_heads + k_heads) * head_dim
    _need(x.dtype in (torch.float16, torch.bfloat16) and out.dtype == x.dtype, "qk_norm_rope: x and out must be fp16 or bf16, alike")
    _need(x.shape[1] >= cols and out.shape[1] >= cols and out.shape[0] == x.shape[0] and out.device == x.device, "qk_norm_rope: shapes")
    _need(norm in _NORMS and pairing in _PAIRINGS, "qk_norm_rope: norm is 'rms' or 'layer', pairing 'pairs' or 'halves'")
    _params(head_dim, x.device, "qk_norm_rope", q_weight=q_weight, k_weight=k_weight, q_bias=q_bias, k_bias=k_bias)
    _need(rope_cos.dim() == 2 and rope_cos.shape[0] == head_dim // 2 and rope_sin.shape == rope_cos.shape, "qk_norm_rope: rotation tables must be [head_dim / 2, tokens]")
    _params(rope_cos.numel(), x.device, "qk_norm_rope", rope_cos=rope_cos, rope_sin=rope_sin)
    with torch.cuda.device(x.device):
        check(
            lib().ff_qk_norm_rope(
                _ptr(x), _DTYPES[x.dtype], ldx, _ptr(out), ldo, x.shape[0], q_heads, k_heads, head_dim, _NORMS[norm],
                _ptr(q_weight), _ptr(q_bias), _ptr(k_weight), _ptr(k_bias), eps, _ptr(rope_cos), _ptr(rope_sin),
                rope_cos.shape[1], _PAIRINGS[pairing], _stream(x),
            ),
            "qk_norm_rope",
        )
