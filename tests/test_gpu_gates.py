"""The gates of the block end by themselves: x = 0 and y = 1, so that out is the activated gate. Bounds as derived at `activate` in
csrc/norm_residual.cu: f32 results within 2^-20 of their value; 16-bit ones within 2^-17 before half a unit of rounding."""

from __future__ import annotations

import pytest
import torch

from foidfinder_b200 import ops

pytestmark = pytest.mark.gpu


def _gates():
    g = torch.Generator().manual_seed(0)
    sizes = torch.tensor([86.9, 1.0, 1e-3], dtype=torch.float64)[:, None]  # bf16 rounds 86.9 to 87
    return ((torch.rand(3, 1 << 17, generator=g, dtype=torch.float64) * 2 - 1) * sizes).float().reshape(-1, 1024)


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize(("xt", "yt"), [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16)])
def test_gates_are_close(cuda_device, xt, yt, act):
    gate = _gates().to(yt)
    x, y = torch.zeros(gate.shape, dtype=xt, device="cuda"), torch.ones(gate.shape, dtype=yt, device="cuda")
    out = torch.empty_like(x)
    ops.norm_residual(x, y, out, gate=gate.cuda(), gate_act=act)
    want = getattr(torch, act)(gate.double())
    err = want.abs() * 2.0**-20 if xt is torch.float32 else want.abs() * (2.0**-17 + torch.finfo(xt).eps / 2 * 1.001) + torch.finfo(xt).tiny
    assert ((out.double().cpu() - want).abs() <= err).all()


def test_sigmoids_below_the_smallest_normal_number_are_zero(cuda_device):
    gate = torch.tensor([-88.0, -100.0, -1e4, -torch.inf]).repeat(4, 1)
    x, y = torch.zeros(4, 4, device="cuda"), torch.ones(4, 4, device="cuda")
    ops.norm_residual(x, y, x, gate=gate.cuda(), gate_act="sigmoid")
    assert (x == 0).all()
