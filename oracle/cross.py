"""64-bit definitions of the operators for tokens that read an image's: rotation by positions, the end of a block, cross
attention. Each also gives what its kernel's tolerance is made of (magnitudes that roundings are relative to)."""

from __future__ import annotations

import torch


def rope(x, positions, frequencies, *, heads, head_dim, start, pairing, scale):
    """x [T, heads * head_dim] -> (rotated, sum of both partners' magnitudes, largest angle), f64."""
    T, r = x.shape[0], 2 * frequencies.numel()
    pos = positions.double().reshape(T, -1)
    axes = pos.shape[1]
    angle = pos.repeat_interleave(r // 2 // axes, 1) * frequencies.double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    y = x.double().reshape(T, heads, head_dim).clone()
    size = torch.zeros_like(y)
    part = y[..., start : start + r]
    i0 = torch.arange(0, r, 2) if pairing == "pairs" else torch.arange(r // 2)
    i1 = i0 + 1 if pairing == "pairs" else i0 + r // 2
    a, b = part[..., i0].clone(), part[..., i1].clone()
    part[..., i0], part[..., i1] = scale * (a * c - b * s), scale * (a * s + b * c)
    size[..., start + i0] = size[..., start + i1] = scale * (a.abs() + b.abs())
    top = angle.abs().max().item() if angle.numel() else 0.0
    return y.reshape(T, -1), size.reshape(T, -1), top


def norm(x, kind, w, b, eps):
    """(norm of x's rows, reciprocal deviation)"""
    d = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    rstd = (d.square().mean(-1, keepdim=True) + eps) ** -0.5
    y = d * rstd * (1.0 if w is None else w.double())
    return (y if b is None else y + b.double()), rstd


def block_end(x, y, *, alpha=1.0, post=None, post_weight=None, post_bias=None, gate=None, gate_act=None, gate_rows=1, scale=None, pre=None,
              pre_weight=None, pre_bias=None, eps=1e-6, pre_eps=None):
    """-> (out, bound of its error in f32, normed, bound of its error in f32), before the outputs' own rounding."""
    # A sum of n <= 16384 values goes through at most 32 values per lane, 5 steps in a warp and 5 across warps: 42 roundings.
    sums, step = 42 * 2.0**-24, 2.0**-24
    T = x.shape[0]
    v = y.double()
    err = torch.zeros_like(v)
    if post is not None:
        size = v.abs().mean(-1, keepdim=True)
        w = 1.0 if post_weight is None else post_weight.double().abs()
        n, rstd = norm(v, post, post_weight, post_bias, eps)
        plain = n if post_bias is None else n - post_bias.double()
        err = plain.abs() * (2 * sums + 8 * step) + 2 * sums * size * rstd * w + n.abs() * step
        v = n
    if gate is not None:
        g = gate.double()
        g = {None: lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[gate_act](g)
        g = g[torch.arange(T) // gate_rows]
        v, err = v * g, (err + v.abs() * 8 * step) * g.abs()
    if scale is not None:
        s = scale.double()
        v, err = v * s, (err + v.abs() * step) * s.abs()
    out = alpha * x.double() + v
    err = err + (out.abs() + v.abs() + (alpha * x.double()).abs()) * 2 * step
    if pre is None:
        return out, err, None, None
    n, rstd = norm(out, pre, pre_weight, pre_bias, eps if pre_eps is None else pre_eps)
    w = 1.0 if pre_weight is None else pre_weight.double().abs()
    most = err.amax(-1, keepdim=True) if err.shape[1] else err
    size = out.abs().mean(-1, keepdim=True)
    plain = n if pre_bias is None else n - pre_bias.double()
    n_err = plain.abs() * (2 * sums + 8 * step + 2 * most * rstd) + (2 * most + 2 * sums * size) * rstd * w + n.abs() * step
    return out, err, n, n_err


def attention(q, k, v, *, heads, kv_heads, head_dim, pieces, scale, out=None):
    """pieces: for every sequence (its rows of q, its rows of k that take part), as slices or index tensors. -> (out [Tq, heads *
    head_dim] (rows of no sequence 0), sum of p |v|, largest sum of |q k| * scale, longest number of keys), f64."""
    Tq = q.shape[0]
    o = torch.zeros(Tq, heads, head_dim, dtype=torch.float64)
    size = torch.zeros_like(o)
    dot, longest = 0.0, 0
    qd, kd, vd = q.double().reshape(Tq, heads, head_dim), k.double().reshape(-1, kv_heads, head_dim), v.double().reshape(-1, kv_heads, head_dim)
    for qi, ki in pieces:
        qs, ks, vs = qd[qi], kd[ki].repeat_interleave(heads // kv_heads, 1), vd[ki].repeat_interleave(heads // kv_heads, 1)
        if qs.shape[0] == 0 or ks.shape[0] == 0:
            continue
        p = torch.softmax(torch.einsum("qhd,khd->hqk", qs, ks) * scale, -1)
        o[qi] = torch.einsum("hqk,khd->qhd", p, vs)
        size[qi] = torch.einsum("hqk,khd->qhd", p, vs.abs())
        dot = max(dot, scale * torch.einsum("qhd,khd->hqk", qs.abs(), ks.abs()).max().item())
        longest = max(longest, ks.shape[0])
    return o.reshape(Tq, -1), size.reshape(Tq, -1), dot, longest
