"""Rotation by positions, block end and cross attention without a GPU: the struct's layout, frequencies, and the
host-side argument checks, which return FF_ERR_INVALID_ARGUMENT with a message before any CUDA call."""

from __future__ import annotations

import ctypes as C
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from foidfinder_b200 import _lib, ops

ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "foidfinder_b200.h").read_text()
DEFINES = {k: int(v) for k, v in re.findall(r"#define (FF_\w+) (\d+)", HEADER)}
FAKE = 0x10000  # an aligned address the host checks accept; never dereferenced by the failing calls
BAD = DEFINES["FF_ERR_INVALID_ARGUMENT"]


def _err() -> str:
    return _lib.lib().ff_last_error().decode()


def test_constants_match_the_header():
    for name in ("NORM_NONE", "GATE_PLAIN", "GATE_SIGMOID", "GATE_TANH"):
        assert DEFINES["FF_" + name] == getattr(_lib, name), name


def test_arguments_layout_matches_ctypes(tmp_path):
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "foidfinder_b200.h"', "int main(void) {",
             '  printf("size %zu\\n", sizeof(ff_norm_residual_args));']
    lines += [f'  printf("{f} %zu\\n", offsetof(ff_norm_residual_args, {f}));' for f, _ in _lib.NormResidualArgs._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == C.sizeof(_lib.NormResidualArgs)
    for f, _ in _lib.NormResidualArgs._fields_:
        assert int(got[f]) == getattr(_lib.NormResidualArgs, f).offset, f


# ---------------------------------------------------------------- rotation
ROPE = dict(x=FAKE, dtype=0, ldx=256, out=FAKE, ldo=256, rows=4, heads=4, head_dim=64, start=0, rotary=64, pairing=0, positions=FAKE,
            position_bytes=4, axes=1, frequencies=FAKE, frequency_bytes=8, scale=1.0, stream=None)


@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=3), "type"), (dict(pairing=2), "pairing"), (dict(rows=-1), "shape"), (dict(heads=-1), "shape"), (dict(head_dim=1025), "shape"),
    (dict(rotary=0), "pairs"), (dict(rotary=63), "pairs"), (dict(start=1), "pairs"), (dict(start=-2, rotary=8), "pairs"), (dict(axes=3), "axes"), (dict(axes=0), "axes"),
    (dict(position_bytes=2), "bytes"), (dict(frequency_bytes=2), "bytes"), (dict(ldx=255), "strides"), (dict(ldo=8), "strides"), (dict(x=None), "NULL"),
    (dict(positions=None), "NULL"), (dict(frequencies=None), "NULL"), (dict(x=FAKE + 1), "misaligned"), (dict(frequencies=FAKE + 4), "misaligned"),
    (dict(positions=FAKE + 2), "misaligned"), (dict(ldo=264), "in place"), (dict(dtype=2, out=FAKE + 2), "misaligned")])
def test_rope_refusals(change, message):
    assert _lib.lib().ff_rope(*(ROPE | change).values()) == BAD
    assert message in _err()


def test_rope_nothing_to_do():
    assert _lib.lib().ff_rope(*(ROPE | dict(rows=0, x=None)).values()) == 0
    assert _lib.lib().ff_rope(*(ROPE | dict(heads=0)).values()) == 0


@pytest.mark.parametrize("rotary", [2, 4, 32, 64, 128])
@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_frequencies(rotary, scaling):
    f, scale = ops.rope_frequencies(rotary, 10000.0, scaling=scaling, factor=8.0, trained=4096)
    plain = torch.tensor([10000.0 ** (-2 * i / rotary) for i in range(rotary // 2)], dtype=torch.float64)
    assert f.dtype == torch.float64 and f.shape == plain.shape
    assert scale == (0.1 * math.log(8) + 1 if scaling == "yarn" else 1.0)
    if scaling is None:
        torch.testing.assert_close(f, plain, rtol=1e-14, atol=0)
    elif scaling == "linear":
        torch.testing.assert_close(f, plain / 8, rtol=1e-14, atol=0)
    elif scaling == "ntk":
        assert f[0] == 1
        if rotary > 2:
            torch.testing.assert_close(f[-1], plain[-1] / 8, rtol=1e-12, atol=0)
    else:
        turns = plain * 4096 / (2 * math.pi)
        assert ((f <= plain) & (f >= plain / 8 * (1 - 1e-15))).all()
        if rotary >= 32:
            assert torch.equal(f[turns > 32 * 2], plain[turns > 32 * 2])
            torch.testing.assert_close(f[turns < 0.5], plain[turns < 0.5] / 8, rtol=1e-14, atol=0)


@pytest.mark.parametrize("kw", [dict(rotary=0), dict(rotary=7), dict(rotary=8, base=1.0), dict(rotary=8, factor=0.5), dict(rotary=8, scaling="other"),
                                dict(rotary=8, scaling="yarn", factor=2.0), dict(rotary=8, scaling="yarn", factor=2.0, trained=64, fast=1.0, slow=2.0)])
def test_frequency_refusals(kw):
    with pytest.raises(RuntimeError, match="rope_frequencies"):
        ops.rope_frequencies(**kw)


# ---------------------------------------------------------------- block end
END = dict(x=FAKE, ldx=64, y=FAKE + 4096, ldy=64, out=FAKE + 8192, ldo=64, normed=FAKE + 12288, ldn=64, x_type=0, y_type=0, rows=4, cols=64, alpha=1.0, post=1,
           post_eps=1e-6, pre=2, pre_eps=1e-6)


@pytest.mark.parametrize(("change", "message"), [
    (dict(x_type=3), "type"), (dict(x_type=0, y_type=1), "alike"), (dict(x_type=0, y_type=2), "alike"), (dict(rows=-1), "shape"), (dict(cols=16385), "shape"),
    (dict(post=3), "norm"), (dict(pre=-1), "norm"), (dict(pre=0), "together"), (dict(normed=None), "together"), (dict(ldx=63), "strides"), (dict(ldn=1), "strides"),
    (dict(x=None), "NULL"), (dict(out=None), "NULL"), (dict(gate=FAKE, gate_cols=64, gate_rows=1, gate_type=1), "gate"),
    (dict(gate=FAKE, gate_cols=2, gate_rows=1, gate_type=2), "columns"), (dict(gate=FAKE, gate_cols=1, gate_rows=0, gate_type=2), "rows"),
    (dict(gate=FAKE, gate_cols=1, gate_rows=1, gate_type=2, ldg=-1), "stride"), (dict(gate=FAKE, gate_cols=1, gate_rows=1, gate_type=2, gate_act=3), "unknown gate"),
    (dict(y=FAKE + 4097), "misaligned"), (dict(post_w=FAKE + 2), "misaligned"), (dict(scale=FAKE + 1), "misaligned"), (dict(out=FAKE, ldo=72), "in place"),
    (dict(normed=FAKE + 4096, ldn=72), "in place"), (dict(normed=FAKE + 8192), "one tensor"), (dict(normed=FAKE), "only out may be x"),
    (dict(out=FAKE + 4096), "only out may be x")])
def test_block_end_refusals(change, message):
    assert _lib.lib().ff_norm_residual(C.byref(_lib.NormResidualArgs(**(END | change))), None) == BAD
    assert message in _err()


def test_block_end_nothing_to_do():
    for change in (dict(rows=0, x=None), dict(cols=0)):
        assert _lib.lib().ff_norm_residual(C.byref(_lib.NormResidualArgs(**(END | change))), None) == 0
    assert _lib.lib().ff_norm_residual(None, None) == BAD


# ---------------------------------------------------------------- cross attention
CROSS = dict(q=FAKE, ldq=256, k=FAKE, ldk=128, v=FAKE, ldv=128, out=2 * FAKE, ldo=256, dtype=0, q_rows=8, k_rows=100, sequences=2, q_start=None, k_start=None, k_len=None,
             mask=None, heads=4, kv_heads=2, head_dim=64, scale=0.125, workspace=None, workspace_bytes=0, stream=None)


@pytest.mark.parametrize(("change", "message"), [
    (dict(dtype=2), "type"), (dict(heads=0), "heads"), (dict(kv_heads=3), "heads"), (dict(heads=2048), "heads"), (dict(head_dim=24), "head_dim"), (dict(head_dim=144), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(q_rows=-1), "shape"), (dict(k_rows=-1), "shape"), (dict(sequences=-1), "shape"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(q_rows=7), "equal pieces"), (dict(k_rows=99), "equal pieces"), (dict(q=None), "NULL"), (dict(v=None), "NULL"), (dict(out=FAKE), "an input"),
    (dict(q=FAKE + 8), "aligned"), (dict(k=FAKE + 2), "aligned"), (dict(out=FAKE + 2), "aligned"), (dict(k_start=FAKE + 2), "misaligned"), (dict(k_len=FAKE + 1), "misaligned"),
    (dict(ldq=255), "strides"), (dict(ldk=120), "strides"), (dict(ldv=129), "strides"), (dict(ldo=260), "strides"), (dict(q_rows=1 << 30, ldq=1 << 12), "each key head")])
def test_cross_attention_refusals(change, message):
    assert _lib.lib().ff_cross_attention(*(CROSS | change).values()) == BAD
    assert message in _err()


def test_cross_attention_nothing_to_do():
    for change in (dict(q_rows=0, q=None), dict(sequences=0)):
        assert _lib.lib().ff_cross_attention(*(CROSS | change).values()) == 0


def test_cross_attention_workspace():
    lib = _lib.lib()
    need = lib.ff_cross_attention_workspace_bytes(1, 1 << 16, 1, 16, 16, 64)
    assert need > 0 and need % 8 == 0
    one = CROSS | dict(q_rows=1, k_rows=1 << 16, sequences=1, heads=16, kv_heads=16, ldk=1024, ldv=1024)
    for change in (dict(), dict(workspace=FAKE, workspace_bytes=need - 1), dict(workspace=FAKE + 8, workspace_bytes=need)):
        assert lib.ff_cross_attention(*(one | change).values()) == BAD
        assert "workspace" in _err()
    assert lib.ff_cross_attention_workspace_bytes(1 << 16, 1 << 12, 64, 16, 16, 64) == 0  # enough sequences, nothing to join
    assert lib.ff_cross_attention_workspace_bytes(0, 0, 0, 0, 0, 0) == 0


# ---------------------------------------------------------------- Python checks
def test_python_refuses_host_tensors():
    x = torch.zeros(2, 64, dtype=torch.float16)
    f = ops.rope_frequencies(64)[0]
    with pytest.raises(RuntimeError, match="rope: expected a 2-D CUDA tensor"):
        ops.rope(x, x, torch.zeros(2, dtype=torch.int32), f, heads=1, head_dim=64)
    with pytest.raises(RuntimeError, match="norm_residual: expected a 2-D CUDA tensor"):
        ops.norm_residual(x, x, x)
    with pytest.raises(RuntimeError, match="cross_attention: expected a 2-D CUDA tensor"):
        ops.cross_attention(x, x, x, x, heads=1, head_dim=64)


@pytest.mark.parametrize("trained", [1, 3, 6, 40, 300, 4096])
def test_stretched_frequencies_of_short_contexts(trained):
    """yarn: pairs that turn less than once within the trained context are divided, the first one too, and those that turn more than
    `fast` times are not."""
    f, _ = ops.rope_frequencies(64, scaling="yarn", factor=8.0, trained=trained)
    plain = ops.rope_frequencies(64)[0]
    turns = plain * trained / (2 * math.pi)
    torch.testing.assert_close(f[turns < 1], plain[turns < 1] / 8, rtol=1e-14, atol=0)
    assert torch.equal(f[turns > 32], plain[turns > 32])
    assert ((f <= plain) & (f >= plain / 8 * (1 - 1e-15))).all()
