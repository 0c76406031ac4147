"""Block-scaled 4-bit linear layers: weights quantised once, activations quantised per call, products on the 4-bit
tensor cores (`ops.quantize_fp4`, `ops.gemm_fp4`, `ops.linear_fp4`).

`Fp4Linear` keeps a packed weight with its epilogue; `Fp4Block` runs a pre-norm transformer block (EVA02 layout,
with per-head query and key norms) on them. Formats: "nv" (16-column blocks, 8-bit scales, a scale per row) and
"mx" (32-column blocks, power-of-two scales).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, ops
from .config import ModelConfig

FORMATS = {"nv": _lib.FP4_NV, "mx": _lib.FP4_MX}
EPILOGUES = {
    "bias": _lib.EPI_BIAS,
    "gelu": _lib.EPI_GELU,
    "swiglu": _lib.EPI_SWIGLU,
    "residual": _lib.EPI_RESIDUAL,
    "qkv": _lib.EPI_QKV_NORM_ROPE,
}


@dataclass
class Fp4Tensor:
    """A 4-bit operand [rows, cols]: codes, block scales in the tensor cores' order and (nv) a scale per row."""

    codes: torch.Tensor
    scales: torch.Tensor
    row_scale: torch.Tensor | None
    rows: int
    cols: int
    fmt: str

    @classmethod
    def empty(cls, rows: int, cols: int, fmt: str, device: torch.device | str = "cuda") -> Fp4Tensor:
        if fmt not in FORMATS:
            raise RuntimeError(f"fp4: unknown format {fmt!r} (nv or mx)")
        nc, ns = ops.fp4_sizes(rows, cols, FORMATS[fmt])
        return cls(
            torch.empty(nc, dtype=torch.uint8, device=device),
            torch.empty(ns, dtype=torch.uint8, device=device),
            torch.empty(rows, dtype=torch.float32, device=device) if fmt == "nv" else None,
            rows,
            cols,
            fmt,
        )


def quantize(x: torch.Tensor, fmt: str = "nv", *, gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None, eps: float = 1e-6,
             out: Fp4Tensor | None = None) -> Fp4Tensor:
    """x [rows, cols] (fp16, bf16 or f32) -> (LayerNorm) -> 4-bit; into `out` (whose format counts) when it is given."""
    if out is None:
        out = Fp4Tensor.empty(x.shape[0], x.shape[1], fmt, x.device)
    if (out.rows, out.cols) != tuple(x.shape):
        raise RuntimeError(f"fp4.quantize: out is [{out.rows}, {out.cols}], x {list(x.shape)}")
    ops.quantize_fp4(x, out.codes, out.scales, out.row_scale, FORMATS[out.fmt], gamma=gamma, beta=beta, eps=eps)
    return out


def dequantize(q: Fp4Tensor, dtype: torch.dtype = torch.float16, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values that q stands for, rounded to dtype."""
    if out is None:
        out = torch.empty(q.rows, q.cols, dtype=dtype, device=q.codes.device)
    if tuple(out.shape) != (q.rows, q.cols):
        raise RuntimeError(f"fp4.dequantize: out is {list(out.shape)}, q [{q.rows}, {q.cols}]")
    ops.dequantize_fp4(q.codes, q.scales, q.row_scale, out, FORMATS[q.fmt])
    return out


def _f32(t: torch.Tensor | None, device: torch.device) -> torch.Tensor | None:
    return None if t is None else t.detach().to(device=device, dtype=torch.float32).contiguous()


class Fp4Linear:
    """y = epilogue(x @ W^T + bias) with W [N, K] held in 4 bits and x quantised on the way in, after a LayerNorm over
    K when gamma and beta are given.

    epilogue: "bias"; "gelu"; "swiglu" (weight rows are the H gates, then the H ups; y [M, H]); "residual" (y +
    residual); "qkv" (N = 3 * heads * 64, or q_heads + 2 * k_heads of them; q and k heads normalised by `norm`
    "rms" or "layer" with q_weight/k_weight [64] (and, for "layer", biases) and rotated by the `rope` tables (cos, sin), each
    [32, tokens]).

    `weight`, `bias`, `gamma` and `beta` are read at every call and may be replaced by others of their shape and kind."""

    def __init__(
        self,
        weight: torch.Tensor,
        bias: torch.Tensor | None = None,
        *,
        fmt: str = "nv",
        epilogue: str = "bias",
        gamma: torch.Tensor | None = None,
        beta: torch.Tensor | None = None,
        eps: float = 1e-6,
        rope: tuple[torch.Tensor, torch.Tensor] | None = None,
        norm: str = "rms",
        q_weight: torch.Tensor | None = None,
        k_weight: torch.Tensor | None = None,
        q_bias: torch.Tensor | None = None,
        k_bias: torch.Tensor | None = None,
        q_heads: int | None = None,
        qk_eps: float = 1e-6,
    ) -> None:
        if fmt not in FORMATS or epilogue not in EPILOGUES:
            raise RuntimeError(f"Fp4Linear: unknown format {fmt!r} or epilogue {epilogue!r}")
        if not weight.is_cuda or weight.dim() != 2:
            raise RuntimeError("Fp4Linear: weight must be a 2-D CUDA tensor")
        if (gamma is None) != (beta is None):
            raise RuntimeError("Fp4Linear: give both gamma and beta or neither")
        d = weight.device
        w = weight.detach()
        bias = _f32(bias, d)
        self.out_features = w.shape[0]
        if epilogue == "swiglu":
            if w.shape[0] % 2:
                raise RuntimeError("Fp4Linear: swiglu needs an even number of weight rows")
            h = self.out_features = w.shape[0] // 2
            w = _interleave(w, h)
            bias = None if bias is None else _interleave(bias, h)
        self.in_features, self.rows, self.eps = w.shape[1], w.shape[0], eps
        self.weight = quantize(w if w.stride(1) == 1 or w.shape[1] == 1 else w.contiguous(), fmt)
        self.gamma, self.beta = _f32(gamma, d), _f32(beta, d)
        heads = {}
        if epilogue == "qkv":
            if w.shape[0] % 64 or rope is None or q_weight is None or k_weight is None:
                raise RuntimeError("Fp4Linear: qkv needs heads of 64 rows, rope tables and q and k norm weights")
            total = w.shape[0] // 64
            q_heads = total // 3 if q_heads is None else q_heads
            if q_heads < 0 or (total - q_heads) % 2 or total < q_heads:
                raise RuntimeError(f"Fp4Linear: {total} heads do not split into {q_heads} q heads and as many k as v heads")
            tensors = (_f32(t, d) for t in (q_weight, k_weight, q_bias, k_bias, *rope))
            heads = dict(zip(("q_weight", "k_weight", "q_bias", "k_bias", "rope_cos", "rope_sin"), tensors))
            heads |= dict(norm=norm, q_heads=q_heads, k_heads=(total - q_heads) // 2, qk_eps=qk_eps)
        self._kind, self._heads = EPILOGUES[epilogue], heads
        self.bias = bias

    @property
    def fmt(self) -> str:
        return self.weight.fmt

    @property
    def bias(self) -> torch.Tensor | None:
        """[rows] f32 (swiglu: in the order of the weight's rows), or None."""
        return self._bias

    @bias.setter
    def bias(self, bias: torch.Tensor | None) -> None:
        self._epilogue = ops.fp4_epilogue(self._kind, self.rows, self.weight.codes.device, bias=bias, **self._heads)  # refuses bad arguments
        self._bias = bias

    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k != "_epilogue"}  # addresses do not travel

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self.bias = state["_bias"]

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
        """x [M, in_features] -> [M, out_features]: `out`, or a new tensor of x's type whose rows start 16 bytes apart or more. Only the
        bias epilogue writes f32: for an f32 x the others' new tensors are fp16 (give an `out` in bf16 for its range)."""
        w = self.weight
        if x.get_device() != w.codes.get_device():
            raise RuntimeError(f"Fp4Linear: x is on {x.device}, the weight on {w.codes.device}")
        if w.rows != self.rows or w.cols != self.in_features:
            raise RuntimeError(f"Fp4Linear: the weight is [{w.rows}, {w.cols}], the layer's [{self.rows}, {self.in_features}]")
        if out is None:
            pitch = (self.out_features + 7) // 8 * 8
            dtype = torch.float16 if x.dtype == torch.float32 and self._kind != _lib.EPI_BIAS else x.dtype
            out = torch.empty(x.shape[0], pitch, dtype=dtype, device=x.device)[:, : self.out_features]
        if out.shape[-1] != self.out_features:
            raise RuntimeError(f"Fp4Linear: out must have {self.out_features} columns, got {list(out.shape)}")
        ops._linear(x, (w.codes, w.scales, w.row_scale), FORMATS[w.fmt], self.rows, self.in_features, self.gamma, self.beta, self.eps, self._epilogue, out, residual)
        return out


def _interleave(t: torch.Tensor, h: int) -> torch.Tensor:
    """Rows [h gates | h ups] -> [gate 16 | up 16] groups, zero rows past h (the SwiGLU epilogue's layout)."""
    pad = -h % 16
    z = t.new_zeros(pad, *t.shape[1:])
    g, u = torch.cat([t[:h], z]), torch.cat([t[h:], z])
    n = (h + pad) // 16
    return torch.stack([g.reshape(n, 16, *t.shape[1:]), u.reshape(n, 16, *t.shape[1:])], 1).reshape(2 * (h + pad), *t.shape[1:]).contiguous()


class Fp4Block:
    """One pre-norm transformer block of a tagger with 4-bit products and normalised queries and keys:

        x -> LayerNorm, qkv product, q/k head norm and rotation -> attention -> proj product + x
          -> LayerNorm, up product with SwiGLU (EVA02) or GELU (PixAI) -> (hidden LayerNorm), down product + x

    in four calls of a linear layer (a quantisation, with its LayerNorm, and a product each) and one of attention. `raw` holds the
    block's f32 weights under `prefix` with the names of `weights.random_raw` (norm1, qkv, proj, norm2, fc1, mlp_norm,
    fc2); q_weight and k_weight [64] are the head norms' weights; rope the angle-major tables (cos, sin), [32, tokens].
    """

    def __init__(
        self,
        raw: dict[str, torch.Tensor],
        prefix: str,
        cfg: ModelConfig,
        *,
        q_weight: torch.Tensor,
        k_weight: torch.Tensor,
        rope: tuple[torch.Tensor, torch.Tensor],
        fmt: str = "nv",
        device: torch.device | str = "cuda",
    ) -> None:
        if cfg.head_dim != 64:
            raise RuntimeError(f"Fp4Block: heads of {cfg.head_dim} columns (the attention takes 64)")
        w = {k[len(prefix) :]: v.to(device) for k, v in raw.items() if k.startswith(prefix)}
        eva = cfg.arch == "eva02"

        def linear(name: str, epilogue: str, norm: str | None, **kw) -> Fp4Linear:
            g, b = (w[norm + ".weight"], w[norm + ".bias"]) if norm else (None, None)
            return Fp4Linear(w[name + ".weight"], w[name + ".bias"], fmt=fmt, epilogue=epilogue, gamma=g, beta=b, eps=cfg.ln_eps, **kw)

        self.heads, self.tokens = cfg.heads, rope[0].shape[1]
        self.qkv = linear("qkv", "qkv", "norm1", rope=rope, q_weight=q_weight, k_weight=k_weight, qk_eps=cfg.ln_eps)
        self.proj = linear("proj", "residual", None)
        self.fc1 = linear("fc1", "swiglu" if eva else "gelu", "norm2")
        self.fc2 = linear("fc2", "residual", "mlp_norm" if eva else None)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """x [sequences * tokens, dim] fp16 -> the same; x itself is left as it is."""
        qkv = self.qkv(x)
        o = torch.empty_like(x)
        ops.attention(qkv, o, self.tokens, self.heads, scale=0.125)
        y = self.proj(o, residual=x)
        return self.fc2(self.fc1(y), out=y, residual=y)
