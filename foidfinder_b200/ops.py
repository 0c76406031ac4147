"""Per-kernel entry points on torch CUDA tensors, mirroring the reference's `torch.ops.foidfinder` ops
(foidfinder/backends/cuda/csrc/kernels.cu:267-281): outputs are caller-allocated and written in place,
shape/dtype violations raise, and every launch goes on the current CUDA stream. Each call goes through
the C ABI of `libfoidfinder_b200.so`; torch is only the memory and stream plumbing. Calls made once per layer
take a short way to it (csrc/calls.cpp) where their arguments are plain.
"""

from __future__ import annotations

import ctypes as C
import math
import warnings
from functools import cache

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
    "rope", "rope_frequencies", "norm_residual", "cross_attention",
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
# These calls are made once per layer, some for a single row, so their checks read each tensor attribute once and
# build no message that is not needed.
_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_NORMS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
_PAIRINGS = {"pairs": _lib.ROPE_PAIRS, "halves": _lib.ROPE_HALVES}
# torch.cuda's own functions without their device guards and lazy initialisation (a CUDA tensor is at hand), which cost
# more than what they call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_alloc = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_alloc", None) or (lambda n, s: torch.cuda.caching_allocator_alloc(n, stream=s))
_free = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_delete", None) or torch.cuda.caching_allocator_delete


class _NoCalls:
    """In the place of the extension module where it has not been built: every call goes the long way."""

    quantize = dequantize = linear = qk_norm_rope = rope = norm_residual = cross_attention = staticmethod(lambda *args: None)


@cache
def _calls():
    """The extension module of csrc/calls.cpp, bound to the kernels' library."""
    try:
        from . import _calls as module
    except ImportError:
        return _NoCalls
    built_for = getattr(module, "built_for", "?")
    if built_for != torch.__version__:  # it reads torch's C++ objects
        warnings.warn(f"foidfinder_b200._calls was built for torch {built_for}, not {torch.__version__}; build it with `python -m foidfinder_b200.build`")
        return _NoCalls
    h = lib()
    names = ("ff_quantize_fp4", "ff_dequantize_fp4", "ff_linear_fp4_workspace_bytes", "ff_linear_fp4", "ff_qk_norm_rope", "ff_rope",
             "ff_norm_residual", "ff_cross_attention_workspace_bytes", "ff_cross_attention")
    module.bind(*(C.cast(getattr(h, name), C.c_void_p).value for name in names))
    return module


def _launch(what: str, fn, device: int, *args) -> None:
    """fn(*args, stream) on the current stream of CUDA device `device`."""
    if device == _current_device():
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        check(rc, what)


def _matrix(t: torch.Tensor, what: str) -> tuple[int, int, int, int]:
    """(rows, columns, row stride, device index) of a 2-D CUDA tensor whose columns are contiguous."""
    device = t.get_device()
    if device < 0 or t.dim() != 2:
        raise RuntimeError(f"{what}: expected a 2-D CUDA tensor, got {t.dim()}-D on {t.device}")
    rows, cols = t.shape
    ld, step = t.stride()
    if rows > 1 << 30:
        raise RuntimeError(f"{what}: at most 2^30 rows, got {rows}")
    if step != 1 and cols > 1:
        raise RuntimeError(f"{what}: expected contiguous columns, got strides {t.stride()}")
    return rows, cols, ld if rows > 1 else max(ld, cols), device


def _vector(t: torch.Tensor | None, n: int, device: int, what: str) -> int | None:
    """Address of an optional f32 parameter of n values."""
    if t is None:
        return None
    if t.get_device() != device or t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous():
        raise RuntimeError(f"{what}: expected {n} contiguous f32 values on cuda:{device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def fp4_sizes(rows: int, cols: int, fmt: int) -> tuple[int, int]:
    """Bytes of the code and scale buffers of a [rows, cols] operand."""
    return rows * ((cols + 31) // 32 * 16), (rows + 127) // 128 * ((cols + 255) // 256 * (2048 if fmt == FP4_NV else 1024))


def _operand(codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor | None, rows: int, cols: int, fmt: int, device: int,
             what: str) -> tuple[int, int, int | None]:
    """Addresses of a 4-bit operand's buffers."""
    nc, ns = fp4_sizes(rows, cols, fmt)
    for t, n in ((codes, nc), (scales, ns)):
        if t.get_device() != device or t.dtype is not torch.uint8 or t.numel() < n or not t.is_contiguous():
            raise RuntimeError(f"{what}: codes and scales of [{rows}, {cols}] must be contiguous uint8 of {nc} and {ns} bytes on cuda:{device}")
    if fmt != FP4_NV:
        return codes.data_ptr(), scales.data_ptr(), None
    if row_scale is None:
        raise RuntimeError(f"{what}: FP4_NV needs row_scale")
    return codes.data_ptr(), scales.data_ptr(), _vector(row_scale, rows, device, what)


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
    rc = _calls().quantize(x, codes, scales, row_scale, fmt, gamma, beta, eps)
    if rc is not None:
        return check(rc, "quantize_fp4") if rc else None
    T, cols, ldx, device = _matrix(x, "quantize_fp4")
    dtype = _DTYPES.get(x.dtype)
    _need(dtype is not None, "quantize_fp4: x must be fp16, bf16 or f32")
    c, s, r = _operand(codes, scales, row_scale, T, cols, fmt, device, "quantize_fp4")
    g, b = _vector(gamma, cols, device, "quantize_fp4: gamma"), _vector(beta, cols, device, "quantize_fp4: beta")
    _launch("quantize_fp4", lib().ff_quantize_fp4, device, x.data_ptr(), dtype, ldx, g, b, eps, T, cols, fmt, c, s, r)


def dequantize_fp4(codes: torch.Tensor, scales: torch.Tensor, row_scale: torch.Tensor | None, out: torch.Tensor, fmt: int) -> None:
    """The values of a 4-bit operand into out [T, C] (fp16, bf16 or f32; columns contiguous, any row stride)."""
    rc = _calls().dequantize(codes, scales, row_scale, out, fmt)
    if rc is not None:
        return check(rc, "dequantize_fp4") if rc else None
    T, cols, ldo, device = _matrix(out, "dequantize_fp4")
    dtype = _DTYPES.get(out.dtype)
    _need(dtype is not None, "dequantize_fp4: out must be fp16, bf16 or f32")
    c, s, r = _operand(codes, scales, row_scale, T, cols, fmt, device, "dequantize_fp4")
    _launch("dequantize_fp4", lib().ff_dequantize_fp4, device, c, s, r, T, cols, fmt, out.data_ptr(), dtype, ldo)


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
    """The part of a gemm_fp4 epilogue that does not change from call to call. It holds its tensors (`tensors`), and every
    call reads their addresses anew."""
    e = _lib.Fp4Epilogue(kind=epi)
    heads = (None,) * 6
    if epi == EPI_QKV_NORM_ROPE:
        _need(norm in _NORMS, "fp4_epilogue: norm must be 'rms' or 'layer'")
        _need(q_weight is not None and k_weight is not None, "fp4_epilogue: q and k norm weights are required")
        heads = (q_weight, q_bias, k_weight, k_bias, rope_cos, rope_sin)
        e.norm, e.q_heads, e.k_heads, e.qk_eps = _NORMS[norm], q_heads, k_heads, qk_eps
    e.tensors = (bias, *heads)
    _address(e, N, device.index if device.index is not None else torch.cuda.current_device(), "fp4_epilogue")
    return e


def _address(e: _lib.Fp4Epilogue, N: int, device: int, what: str) -> None:
    """The addresses of an epilogue's tensors into its fields. (One that was filled in by hand has no tensors.)"""
    tensors = getattr(e, "tensors", None)
    if tensors is None:
        return
    bias, q_weight, q_bias, k_weight, k_bias, cos, sin = tensors
    e.bias = _vector(bias, N, device, f"{what}: bias")
    if e.kind == EPI_QKV_NORM_ROPE:
        e.q_w, e.k_w = _vector(q_weight, 64, device, f"{what}: q_weight"), _vector(k_weight, 64, device, f"{what}: k_weight")
        e.q_b, e.k_b = _vector(q_bias, 64, device, f"{what}: q_bias"), _vector(k_bias, 64, device, f"{what}: k_bias")
        e.rope_cos, e.rope_sin, e.tokens = _tables(cos, sin, 32, device, what)


def _tables(cos: torch.Tensor | None, sin: torch.Tensor | None, half: int, device: int, what: str) -> tuple[int, int, int]:
    """Addresses of the angle-major rotation tables [half, tokens] and the number of tokens."""
    if cos is None or sin is None or cos.dim() != 2 or cos.shape[0] != half or cos.shape != sin.shape:
        raise RuntimeError(f"{what}: rotation tables must be two [{half}, tokens] tensors")
    n = cos.numel()
    return _vector(cos, n, device, what), _vector(sin, n, device, what), cos.shape[1]


def _bind(e: _lib.Fp4Epilogue, M: int, N: int, out: torch.Tensor, residual: torch.Tensor | None, device: int, what: str) -> None:
    """The tensors of one call, and its own, into an epilogue."""
    _address(e, N, device, what)
    rows, cols, e.ldo, d = _matrix(out, what)
    dtype = _DTYPES.get(out.dtype)
    if d != device or dtype is None or rows != M or (not 0 < cols <= N // 2 if e.kind == EPI_SWIGLU else cols != N):  # the library takes 0 for N / 2
        raise RuntimeError(f"{what}: out is {out.dtype} {list(out.shape)} on {out.device} for M={M} N={N} on cuda:{device}")
    e.out_dtype, e.out, e.out_cols = dtype, out.data_ptr(), cols
    if e.kind == EPI_RESIDUAL:
        _need(residual is not None, "EPI_RESIDUAL needs the residual")
        rows, rcols, e.ldr, d = _matrix(residual, what)
        if d != device or residual.dtype is not out.dtype or rows != M or rcols != cols:
            raise RuntimeError(f"{what}: the residual ({residual.dtype} {list(residual.shape)} on {residual.device}) must be like out")
        e.residual = residual.data_ptr()


def _copy(epilogue: _lib.Fp4Epilogue) -> _lib.Fp4Epilogue:
    e = _lib.Fp4Epilogue.from_buffer_copy(epilogue)
    e.tensors = getattr(epilogue, "tensors", None)
    return e


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
    M, device = out.shape[0], out.get_device()
    a = _operand(A, A_scales, row_scale, M, K, fmt, device, "gemm_fp4")
    w = _operand(W, W_scales, col_scale, N, K, fmt, device, "gemm_fp4")
    if isinstance(epilogue, int):
        e = fp4_epilogue(epilogue, N, out.device, bias=bias, **heads)
    else:
        e = _copy(epilogue)
    _bind(e, M, N, out, residual, device, "gemm_fp4")
    _launch("gemm_fp4", lib().ff_gemm_fp4, device, *a, *w, fmt, M, N, K, C.byref(e), tile)


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
    e = fp4_epilogue(epilogue, N, x.device, bias=bias, **heads) if isinstance(epilogue, int) else epilogue
    _linear(x, (W, W_scales, col_scale), fmt, N, x.shape[-1], gamma, beta, eps, e, out, residual)


def _linear(x, W, fmt, N, K, gamma, beta, eps, epilogue, out, residual) -> None:
    """linear_fp4 with the weight's tensors (codes, scales, row scale) and a prepared epilogue."""
    rc = _calls().linear(x, W, fmt, N, K, gamma, beta, eps, epilogue, out, residual)
    if rc is not None:
        return check(rc, "linear_fp4") if rc else None
    M, cols, ldx, device = _matrix(x, "linear_fp4")
    if device != _current_device():
        with torch.cuda.device(device):
            return _linear(x, W, fmt, N, K, gamma, beta, eps, epilogue, out, residual)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None or cols != K:
        raise RuntimeError(f"linear_fp4: x must be fp16, bf16 or f32 [M, {K}], got {x.dtype} {list(x.shape)}")
    w = _operand(*W, N, K, fmt, device, "linear_fp4")
    g, b = _vector(gamma, K, device, "linear_fp4: gamma"), _vector(beta, K, device, "linear_fp4: beta")
    e = _copy(epilogue)
    _bind(e, M, N, out, residual, device, "linear_fp4")
    nbytes = _linear_workspace(M, K, fmt)
    if M == 0:
        return
    stream = _raw_stream(device)
    ws = _alloc(nbytes, stream)  # torch's stream-ordered cache: free for the stream's next use as soon as the call has returned
    try:
        rc = lib().ff_linear_fp4(x.data_ptr(), dtype, ldx, g, b, eps, *w, fmt, M, N, K, C.byref(e), ws, nbytes, stream)
    finally:
        _free(ws)
    if rc:
        check(rc, "linear_fp4")


def _linear_workspace(M: int, K: int, fmt: int) -> int:
    """ff_linear_fp4_workspace_bytes: codes, scales and row scales, each rounded up to 256 bytes."""
    codes, scales = fp4_sizes(M, K, fmt)
    return (codes + 255 & ~255) + (scales + 255 & ~255) + (4 * M + 255 & ~255)


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
    n, p = _NORMS.get(norm), _PAIRINGS.get(pairing)
    rc = _calls().qk_norm_rope(x, out, q_heads, k_heads, head_dim, n, q_weight, q_bias, k_weight, k_bias, eps, rope_cos, rope_sin, p)
    if rc is not None:
        return check(rc, "qk_norm_rope") if rc else None
    rows, xcols, ldx, device = _matrix(x, "qk_norm_rope")
    orows, ocols, ldo, odevice = _matrix(out, "qk_norm_rope")
    cols, dtype = (q_heads + k_heads) * head_dim, x.dtype
    if dtype is torch.float32 or dtype not in _DTYPES or out.dtype is not dtype:
        raise RuntimeError(f"qk_norm_rope: x and out must be fp16 or bf16, alike, got {dtype} and {out.dtype}")
    if xcols < cols or ocols < cols or orows != rows or odevice != device:
        raise RuntimeError(f"qk_norm_rope: x {list(x.shape)} and out {list(out.shape)} must hold {cols} columns of the same rows on one device")
    _need(n is not None and p is not None, "qk_norm_rope: norm is 'rms' or 'layer', pairing 'pairs' or 'halves'")
    what = "qk_norm_rope"
    qw, qb = _vector(q_weight, head_dim, device, what), _vector(q_bias, head_dim, device, what)
    kw, kb = _vector(k_weight, head_dim, device, what), _vector(k_bias, head_dim, device, what)
    cos, sin, tokens = _tables(rope_cos, rope_sin, head_dim // 2, device, what)
    _launch(what, lib().ff_qk_norm_rope, device, x.data_ptr(), _DTYPES[dtype], ldx, out.data_ptr(), ldo, rows, q_heads, k_heads, head_dim, n,
            qw, qb, kw, kb, eps, cos, sin, tokens, p)


# ---------------------------------------------------------------- tokens that read an image's
_KINDS = {None: _lib.NORM_NONE, **_NORMS}
_GATES = {None: _lib.GATE_PLAIN, "sigmoid": _lib.GATE_SIGMOID, "tanh": _lib.GATE_TANH}


def rope_frequencies(
    rotary: int,
    base: float = 10000.0,
    *,
    scaling: str | None = None,
    factor: float = 1.0,
    trained: int = 0,
    fast: float = 32.0,
    slow: float = 1.0,
) -> tuple[torch.Tensor, float]:
    """Frequencies [rotary / 2] (f64, radians per position; base^(-2 i / rotary)) and the scale for `rope`. `scaling` stretches
    them for contexts `factor` times as long: "linear" divides all of them, "ntk" raises the base so that the slowest is
    divided and the fastest stays, "yarn" leaves pairs that turn more than `fast` times within the `trained` context, divides
    those that turn less than `slow` times, blends between, and scales by 0.1 ln(factor) + 1."""
    _need(rotary >= 2 and rotary % 2 == 0, f"rope_frequencies: {rotary} columns are no pairs")
    _need(base > 1 and factor >= 1, "rope_frequencies: base must be above 1 and factor at least 1")
    _need(scaling in (None, "linear", "ntk", "yarn"), f"rope_frequencies: unknown scaling {scaling!r}")
    scale = 1.0
    if scaling == "ntk" and rotary > 2:
        base *= factor ** (rotary / (rotary - 2))
    f = base ** (torch.arange(0, rotary, 2, dtype=torch.float64) / -rotary)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        _need(trained > 0 and fast > slow > 0, "rope_frequencies: yarn needs the trained context's length and fast > slow > 0")
        # the pair (a fraction of one) that turns n times within the trained context
        pair = lambda n: rotary * math.log(trained / (2 * math.pi * n)) / (2 * math.log(base))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rotary - 1)
        ramp = ((torch.arange(rotary // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        ramp[f * trained < 2 * math.pi * slow] = 1  # the first pair too, where even that turns less than `slow` times
        f = f * (1 - ramp) + f / factor * ramp
        scale = 0.1 * math.log(factor) + 1
    return f, scale


def rope(
    x: torch.Tensor,
    out: torch.Tensor,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    *,
    heads: int,
    head_dim: int,
    start: int = 0,
    pairing: str = "pairs",
    scale: float = 1.0,
) -> None:
    """x [T, >= heads * head_dim] fp16, bf16 or f32 -> every head's columns [start, start + 2 * frequencies.numel()) rotated by
    positions[row] * frequencies (radians; the angles in 64 bits), times `scale`, its other columns as they are, into the
    first columns of out (x itself: in place). `positions` [T] or [T, axes] int32 or int64 (axes take equal shares of the
    pairs, in order), `frequencies` f64 or f32 (`rope_frequencies`); `pairing` "pairs" rotates (2i, 2i + 1) of them, "halves" (i, i + r / 2)."""
    what = "rope"
    rc = _calls().rope(x, out, positions, frequencies, heads, head_dim, start, _PAIRINGS.get(pairing), scale)
    if rc is not None:
        return check(rc, what) if rc else None
    rows, xcols, ldx, device = _matrix(x, what)
    orows, ocols, ldo, odevice = _matrix(out, what)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None or out.dtype is not x.dtype:
        raise RuntimeError(f"rope: x and out must be fp16, bf16 or f32, alike, got {x.dtype} and {out.dtype}")
    cols = heads * head_dim
    if heads < 0 or head_dim < 1 or xcols < cols or ocols < cols or orows != rows or odevice != device:
        raise RuntimeError(f"rope: x {list(x.shape)} and out {list(out.shape)} must hold {cols} columns of the same rows on one device")
    _need(pairing in _PAIRINGS, "rope: pairing is 'pairs' or 'halves'")
    axes = 1 if positions.dim() == 1 else positions.shape[1] if positions.dim() == 2 else 0
    if positions.get_device() != device or positions.dtype not in (torch.int32, torch.int64) or axes < 1 or positions.shape[0] != rows or not positions.is_contiguous():
        raise RuntimeError(f"rope: positions must be contiguous int32 or int64 [{rows}] or [{rows}, axes] on cuda:{device}, got {positions.dtype} {list(positions.shape)} on {positions.device}")
    if frequencies.get_device() != device or frequencies.dtype not in (torch.float32, torch.float64) or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise RuntimeError(f"rope: frequencies must be a contiguous f64 or f32 vector on cuda:{device}, got {frequencies.dtype} {list(frequencies.shape)} on {frequencies.device}")
    _launch(what, lib().ff_rope, device, x.data_ptr(), dtype, ldx, out.data_ptr(), ldo, rows, heads, head_dim, start, 2 * frequencies.numel(),
            _PAIRINGS[pairing], positions.data_ptr(), positions.element_size(), axes, frequencies.data_ptr(), frequencies.element_size(), scale)


def norm_residual(
    x: torch.Tensor,
    y: torch.Tensor,
    out: torch.Tensor,
    *,
    alpha: float = 1.0,
    post: str | None = None,
    post_weight: torch.Tensor | None = None,
    post_bias: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    gate_act: str | None = None,
    gate_rows: int = 1,
    scale: torch.Tensor | None = None,
    normed: torch.Tensor | None = None,
    pre: str | None = None,
    pre_weight: torch.Tensor | None = None,
    pre_bias: torch.Tensor | None = None,
    eps: float = 1e-6,
    pre_eps: float | None = None,
) -> None:
    """The end of a block and the norm before the next one: out = alpha * x + scale * act(gate) * post(y), normed = pre(out) (of
    out before it is rounded). x and out [T, C] are the residual stream (out may be x), y the block's result; normed, y's
    type, may be y. `post` and `pre`: None, "rms" or "layer" with weights and biases [C] (f32, or None). `gate` [G, C] or [G, 1],
    f32 or y's type, after `gate_act` None, "sigmoid" or "tanh"; row t reads gate row t // gate_rows. `scale` [C] f32. Types: fp16,
    bf16 or f32 alike, or x and out in f32 with a 16-bit y; C is at most 16384. Rows that start 16 bytes apart are the fastest."""
    what = "norm_residual"
    rc = _calls().norm_residual(x, y, out, normed, alpha, _KINDS.get(post), post_weight, post_bias, gate, _GATES.get(gate_act), gate_rows, scale, _KINDS.get(pre),
                                pre_weight, pre_bias, eps, eps if pre_eps is None else pre_eps)
    if rc is not None:
        return check(rc, what) if rc else None
    rows, cols, ldx, device = _matrix(x, what)
    n = _lib.NormResidualArgs(rows=rows, cols=cols, alpha=alpha, ldx=ldx, x=x.data_ptr(), post_eps=eps, pre_eps=eps if pre_eps is None else pre_eps)
    for name, ld, t, like in (("y", "ldy", y, y), ("out", "ldo", out, x), ("normed", "ldn", normed, y)):
        if t is None:
            continue
        trows, tcols, tld, tdevice = _matrix(t, f"norm_residual: {name}")
        if (trows, tcols, tdevice) != (rows, cols, device) or t.dtype is not like.dtype:
            raise RuntimeError(f"norm_residual: {name} is {t.dtype} {list(t.shape)} on {t.device} beside x [{rows}, {cols}] on cuda:{device} and {like.dtype}")
        setattr(n, name, t.data_ptr())
        setattr(n, ld, tld)
    if x.dtype not in _DTYPES or y.dtype not in _DTYPES or (x.dtype is not y.dtype and x.dtype is not torch.float32):
        raise RuntimeError(f"norm_residual: x and y must be fp16, bf16 or f32 alike, or x f32, got {x.dtype} and {y.dtype}")
    n.x_type, n.y_type = _DTYPES[x.dtype], _DTYPES[y.dtype]
    if post not in (None, *_NORMS) or pre not in (None, *_NORMS) or (pre is None) != (normed is None):
        raise RuntimeError("norm_residual: post and pre are None, 'rms' or 'layer', and pre comes with normed")
    if post is not None:
        n.post, n.post_w, n.post_b = _NORMS[post], _vector(post_weight, cols, device, what), _vector(post_bias, cols, device, what)
    if pre is not None:
        n.pre, n.pre_w, n.pre_b = _NORMS[pre], _vector(pre_weight, cols, device, what), _vector(pre_bias, cols, device, what)
    n.scale = _vector(scale, cols, device, what)
    if gate is not None:
        grows, gcols, n.ldg, gdevice = _matrix(gate, "norm_residual: gate")
        if gdevice != device or gcols not in (1, cols) or (gate.dtype is not torch.float32 and gate.dtype is not y.dtype) or gate_act not in _GATES:
            raise RuntimeError(f"norm_residual: the gate must be f32 or {y.dtype} [G, {cols}] or [G, 1] on cuda:{device} behind None, 'sigmoid' or 'tanh', got {gate.dtype} {list(gate.shape)} on {gate.device} and {gate_act!r}")
        if gate_rows < 1 or grows * gate_rows < rows:
            raise RuntimeError(f"norm_residual: {grows} gate rows for {gate_rows} rows each are too few for {rows}")
        n.gate, n.gate_type, n.gate_cols, n.gate_act = gate.data_ptr(), _DTYPES[gate.dtype], gcols, _GATES[gate_act]
        n.gate_rows = min(gate_rows, max(rows, 1))
    _launch(what, lib().ff_norm_residual, device, C.byref(n))


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    *,
    heads: int,
    head_dim: int,
    kv_heads: int | None = None,
    sequences: int | None = None,
    q_start: torch.Tensor | None = None,
    k_start: torch.Tensor | None = None,
    k_len: torch.Tensor | None = None,
    mask: torch.Tensor | None = None,
    scale: float | None = None,
) -> None:
    """out = softmax(scale * q k^T) v for every sequence and head, with queries and keys of different lengths: q and out [Tq, heads *
    head_dim], k and v [Tk, kv_heads * head_dim], fp16 or bf16 (views with contiguous columns and 16-byte rows, such as the
    halves of a packed projection). Query head h reads key head h // (heads // kv_heads).

    Sequences are equal pieces of the rows (`sequences` of them), or sequence b has rows q_start[b] to q_start[b + 1] and
    k_start[b] to k_start[b + 1] (ascending int32 [sequences + 1] on the device, one or both); of its keys the first k_len[b]
    (int32 [sequences]) take part. `mask` [Tk] bool leaves out keys where it is False. What is left out counts nothing, whatever
    it holds. A query without keys gives zeros; rows of out outside the sequences stay as they were. `scale` is head_dim**-0.5 unless given."""
    what = "cross_attention"
    kv_heads = heads if kv_heads is None else kv_heads
    for t, more in ((q_start, 1), (k_start, 1), (k_len, 0)):
        if sequences is None and t is not None:
            sequences = t.numel() - more
    sequences = 1 if sequences is None else sequences
    scale = head_dim**-0.5 if scale is None and head_dim > 0 else scale
    rc = _calls().cross_attention(q, k, v, out, heads, kv_heads, head_dim, sequences, q_start, k_start, k_len, mask, scale)
    if rc is not None:
        return check(rc, what) if rc else None
    tq, qcols, ldq, device = _matrix(q, what)
    tk, kcols, ldk, kdevice = _matrix(k, what)
    shape_v, shape_o = _matrix(v, what), _matrix(out, what)
    dtype = q.dtype
    if dtype is torch.float32 or dtype not in _DTYPES or k.dtype is not dtype or v.dtype is not dtype or out.dtype is not dtype:
        raise RuntimeError(f"cross_attention: q, k, v and out must be fp16 or bf16, alike, got {q.dtype}, {k.dtype}, {v.dtype} and {out.dtype}")
    if qcols != heads * head_dim or kcols != kv_heads * head_dim or shape_v[:2] != (tk, kcols) or shape_o[:2] != (tq, qcols):
        raise RuntimeError(f"cross_attention: q {list(q.shape)}, k {list(k.shape)}, v {list(v.shape)}, out {list(out.shape)} for {heads} and {kv_heads} heads of {head_dim}")
    if kdevice != device or shape_v[3] != device or shape_o[3] != device:
        raise RuntimeError("cross_attention: q, k, v and out must be on one device")
    for name, t, n in (("q_start", q_start, sequences + 1), ("k_start", k_start, sequences + 1), ("k_len", k_len, sequences)):
        if t is not None and (t.get_device() != device or t.dtype is not torch.int32 or t.numel() != n or not t.is_contiguous()):
            raise RuntimeError(f"cross_attention: {name} must be {n} contiguous int32 values on cuda:{device}, got {t.dtype} {list(t.shape)} on {t.device}")
    if mask is not None and (mask.get_device() != device or mask.dtype not in (torch.bool, torch.uint8) or mask.numel() != tk or not mask.is_contiguous()):
        raise RuntimeError(f"cross_attention: mask must be {tk} contiguous bool values on cuda:{device}, got {mask.dtype} {list(mask.shape)} on {mask.device}")
    if sequences < 0 or heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise RuntimeError(f"cross_attention: {sequences} sequences, {heads} query heads over {kv_heads} key heads")
    if device != _current_device():
        with torch.cuda.device(device):
            return cross_attention(q, k, v, out, heads=heads, head_dim=head_dim, kv_heads=kv_heads, sequences=sequences, q_start=q_start,
                                   k_start=k_start, k_len=k_len, mask=mask, scale=scale)
    nbytes = lib().ff_cross_attention_workspace_bytes(tq, tk, sequences, heads, kv_heads, head_dim)
    stream = _raw_stream(device)
    ws = _alloc(nbytes, stream) if nbytes else None  # torch's stream-ordered cache: free for the stream's next use on return
    try:
        rc = lib().ff_cross_attention(q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), shape_v[2], out.data_ptr(), shape_o[2], _DTYPES[dtype],
                                      tq, tk, sequences, _ptr(q_start), _ptr(k_start), _ptr(k_len), _ptr(mask), heads, kv_heads, head_dim,
                                      scale, ws, nbytes, stream)
    finally:
        if ws is not None:
            _free(ws)
    if rc:
        check(rc, what)
