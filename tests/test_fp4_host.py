"""The 4-bit operators without a GPU: buffer sizes, the struct's layout, and the host-side argument checks, which
return FF_ERR_INVALID_ARGUMENT with a message before any CUDA call."""

from __future__ import annotations

import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from foidfinder_b200 import _lib, fp4, ops
from oracle import fp4 as O

ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "foidfinder_b200.h").read_text()
DEFINES = {k: int(v) for k, v in re.findall(r"#define (FF_\w+) (\d+)", HEADER)}
FAKE = 0x10000  # an aligned address the host checks accept; never dereferenced by the failing calls
BAD = DEFINES["FF_ERR_INVALID_ARGUMENT"]


def _err() -> str:
    return _lib.lib().ff_last_error().decode()


def test_constants_match_the_header():
    for name in ("FP4_NV", "FP4_MX", "F16", "BF16", "F32", "EPI_QKV_NORM_ROPE", "NORM_RMS", "NORM_LAYER", "ROPE_PAIRS", "ROPE_HALVES"):
        assert DEFINES["FF_" + name] == getattr(_lib, name), name


def test_epilogue_layout_matches_ctypes(tmp_path):
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "foidfinder_b200.h"', "int main(void) {",
             '  printf("size %zu\\n", sizeof(ff_fp4_epilogue));']
    lines += [f'  printf("{f} %zu\\n", offsetof(ff_fp4_epilogue, {f}));' for f, _ in _lib.Fp4Epilogue._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == C.sizeof(_lib.Fp4Epilogue)
    for f, _ in _lib.Fp4Epilogue._fields_:
        assert int(got[f]) == getattr(_lib.Fp4Epilogue, f).offset, f


@pytest.mark.parametrize("fmt", ["nv", "mx"])
@pytest.mark.parametrize(("rows", "cols"), [(1, 1), (128, 256), (129, 257), (1025, 1024), (300, 2730)])
def test_buffer_sizes(rows, cols, fmt):
    codes, scales = ops.fp4_sizes(rows, cols, fp4.FORMATS[fmt])
    lib = _lib.lib()
    assert (codes, scales) == (lib.ff_fp4_code_bytes(rows, cols), lib.ff_fp4_scale_bytes(rows, cols, fp4.FORMATS[fmt]))
    assert ops._linear_workspace(rows, cols, fp4.FORMATS[fmt]) == lib.ff_linear_fp4_workspace_bytes(rows, cols, fp4.FORMATS[fmt])
    assert codes == rows * (-(-cols // 32) * 16)
    tiles = -(-rows // 128) * 128
    assert scales == tiles * (-(-cols // 256) * 256 // O.BLOCK[fmt])
    idx = O.scale_index(rows, cols, fmt)
    assert idx.max() < scales and idx.unique().numel() == idx.numel()
    assert _lib.lib().ff_linear_fp4_workspace_bytes(rows, cols, fp4.FORMATS[fmt]) >= codes + scales


def test_buffer_sizes_of_bad_arguments_are_zero():
    lib = _lib.lib()
    assert lib.ff_fp4_code_bytes(-1, 5) == lib.ff_fp4_code_bytes(5, 0) == 0
    assert lib.ff_fp4_scale_bytes(5, 5, 2) == lib.ff_linear_fp4_workspace_bytes(5, 0, 0) == 0


def test_long_buffers_do_not_wrap():
    assert ops.fp4_sizes(1 << 20, 1 << 14, 0)[0] == 1 << 33
    assert ops.fp4_sizes(1 << 20, 1 << 14, 0)[1] == 1 << 30
    assert _lib.lib().ff_fp4_code_bytes(1 << 20, 1 << 14) == 1 << 33


@pytest.mark.parametrize(("args", "msg"), [
    ((FAKE, 0, 64, None, None, 1e-6, 4, 64, 7, FAKE, FAKE, FAKE, None), "format 7"),
    ((FAKE, 3, 64, None, None, 1e-6, 4, 64, 0, FAKE, FAKE, FAKE, None), "type 3"),
    ((FAKE, 0, 63, None, None, 1e-6, 4, 64, 0, FAKE, FAKE, FAKE, None), "row stride 63"),
    ((FAKE, 0, 64, None, None, 1e-6, -1, 64, 0, FAKE, FAKE, FAKE, None), "bad shape"),
    ((FAKE, 0, 64, None, None, 1e-6, 4, 0, 0, FAKE, FAKE, FAKE, None), "bad shape"),
    ((None, 0, 64, None, None, 1e-6, 4, 64, 0, FAKE, FAKE, FAKE, None), "NULL"),
    ((FAKE, 0, 64, None, None, 1e-6, 4, 64, 0, FAKE, FAKE, None, None), "needs row_scale"),
    ((FAKE, 0, 64, FAKE, None, 1e-6, 4, 64, 0, FAKE, FAKE, FAKE, None), "both gamma and beta"),
    ((FAKE + 1, 0, 64, None, None, 1e-6, 4, 64, 0, FAKE, FAKE, FAKE, None), "aligned to its type"),
    ((FAKE, 0, 64, None, None, 1e-6, 4, 64, 0, FAKE + 8, FAKE, FAKE, None), "16-byte aligned"),
])
def test_quantize_host_checks(args, msg):
    assert _lib.lib().ff_quantize_fp4(*args) == BAD
    assert msg in _err()


def test_rows_that_indices_cannot_step_over():
    rows = (1 << 30) + 1
    f = _lib.lib()
    assert f.ff_quantize_fp4(FAKE, 0, 64, None, None, 1e-6, rows, 64, 0, FAKE, FAKE, FAKE, None) == BAD
    assert f.ff_dequantize_fp4(FAKE, FAKE, FAKE, rows, 64, 0, FAKE, 0, 64, None) == BAD
    assert f.ff_qk_norm_rope(FAKE, 0, 128, FAKE, 128, rows, 1, 1, 64, 1, FAKE, None, FAKE, None, 1e-6, FAKE, FAKE, 4, 0, None) == BAD
    assert "bad shape" in _err()


def test_quantize_and_dequantize_of_no_rows():
    assert _lib.lib().ff_quantize_fp4(None, 0, 64, None, None, 1e-6, 0, 64, 0, None, None, None, None) == 0
    assert _lib.lib().ff_dequantize_fp4(None, None, None, 0, 64, 0, None, 0, 64, None) == 0


@pytest.mark.parametrize(("args", "msg"), [
    ((FAKE, FAKE, FAKE, 4, 64, 9, FAKE, 0, 64, None), "format 9"),
    ((FAKE, FAKE, FAKE, 4, 64, 0, FAKE, 5, 64, None), "type 5"),
    ((FAKE, FAKE, FAKE, 4, 64, 0, FAKE, 0, 60, None), "row stride 60"),
    ((FAKE, FAKE, None, 4, 64, 0, FAKE, 0, 64, None), "needs row_scale"),
    ((FAKE, None, FAKE, 4, 64, 0, FAKE, 0, 64, None), "NULL"),
    ((FAKE, FAKE, FAKE, 4, 64, 0, FAKE + 2, 2, 64, None), "aligned to its type"),
])
def test_dequantize_host_checks(args, msg):
    assert _lib.lib().ff_dequantize_fp4(*args) == BAD
    assert msg in _err()


def _epi(**kw):
    e = _lib.Fp4Epilogue(kind=_lib.EPI_BIAS, out_dtype=_lib.F16, out=FAKE, ldo=4096)
    for k, v in kw.items():
        setattr(e, k, v)
    return e


QKV = dict(kind=_lib.EPI_QKV_NORM_ROPE, norm=1, q_heads=1, k_heads=1, tokens=4, q_w=FAKE, k_w=FAKE, rope_cos=FAKE, rope_sin=FAKE)


@pytest.mark.parametrize(("N", "kw", "msg"), [
    (128, dict(kind=0), "unknown epilogue 0"),
    (128, dict(kind=5), "unknown epilogue 5"),
    (128, dict(out_dtype=3), "output type 3"),
    (128, dict(kind=_lib.EPI_GELU, out_dtype=_lib.F32), "not available for epilogue"),
    (144, dict(kind=_lib.EPI_SWIGLU), "N % 32"),
    (128, dict(kind=_lib.EPI_SWIGLU, out_cols=65), "at most N / 2"),
    (128, dict(ldo=120), "row stride 120"),
    (128, dict(ldo=129), "16-byte aligned rows"),
    (128, dict(out=FAKE + 8), "16-byte aligned rows"),
    (128, dict(out=None), "NULL"),
    (128, dict(out=FAKE + 2, out_dtype=_lib.F32), "aligned to its type"),
    (128, dict(kind=_lib.EPI_RESIDUAL), "needs the residual"),
    (128, dict(kind=_lib.EPI_RESIDUAL, residual=FAKE, ldr=120), "needs the residual"),
    (128, dict(kind=_lib.EPI_RESIDUAL, residual=FAKE + 4, ldr=128), "residual rows"),
    (128, {**QKV, "norm": 0}, "unknown head norm"),
    (128, {**QKV, "q_heads": 2}, "do not fit"),
    (130, QKV, "do not fit"),
    (128, {**QKV, "rope_sin": None}, "rotation tables"),
    (128, {**QKV, "tokens": 0}, "tokens"),
    (0, {}, "bad shape"),
])
def test_gemm_host_checks(N, kw, msg):
    rc = _lib.lib().ff_gemm_fp4(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 4, N, 256, C.byref(_epi(**kw)), 0, None)
    assert rc == BAD
    assert msg in _err()


def test_gemm_operand_checks():
    f = _lib.lib().ff_gemm_fp4
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 4, 128, 256, C.byref(_epi()), 0, None) == BAD and "format 2" in _err()
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 4, 128, 256, None, 0, None) == BAD and "NULL epilogue" in _err()
    assert f(FAKE, FAKE, None, FAKE, FAKE, FAKE, 0, 4, 128, 256, C.byref(_epi()), 0, None) == BAD and "row and column scales" in _err()
    assert f(FAKE, FAKE + 4, FAKE, FAKE, FAKE, FAKE, 0, 4, 128, 256, C.byref(_epi()), 0, None) == BAD and "16-byte aligned" in _err()
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 4, 128, 256, C.byref(_epi()), 256, None) == BAD and "tile" in _err()
    e = _epi(**QKV)
    assert f(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, 4, 128, 256, C.byref(e), 512, None) == BAD and "no pair tiles" in _err()
    assert f(None, None, None, FAKE, FAKE, FAKE, 0, 0, 128, 256, C.byref(_epi()), 0, None) == 0  # no rows


def test_linear_workspace_check():
    f = _lib.lib().ff_linear_fp4
    args = (FAKE, 0, 256, None, None, 1e-6, FAKE, FAKE, FAKE, 0, 4, 128, 256, C.byref(_epi()))
    assert f(*args, FAKE, 16, None) == BAD and "workspace" in _err()
    assert f(*args, None, 1 << 30, None) == BAD and "workspace" in _err()


@pytest.mark.parametrize(("kw", "msg"), [
    (dict(dtype=2), "not fp16 or bf16"),
    (dict(head_dim=48), "head_dim 48"),
    (dict(norm=0), "unknown norm"),
    (dict(pairing=2), "unknown pairing"),
    (dict(tokens=0), "bad shape"),
    (dict(rows=-1), "bad shape"),
    (dict(ldx=120), "row strides"),
    (dict(ldo=132), "row strides"),
    (dict(q_w=None), "NULL"),
    (dict(cos=None), "NULL"),
    (dict(x=FAKE + 4), "16-byte aligned"),
    (dict(out=FAKE, ldo=136), "in place"),
])
def test_qk_norm_rope_host_checks(kw, msg):
    a = dict(x=FAKE, dtype=0, ldx=128, out=2 * FAKE, ldo=128, rows=4, q_heads=1, k_heads=1, head_dim=64, norm=1, q_w=FAKE, q_b=None, k_w=FAKE, k_b=None,
             eps=1e-6, cos=FAKE, sin=FAKE, tokens=4, pairing=0, stream=None) | kw
    assert _lib.lib().ff_qk_norm_rope(*a.values()) == BAD
    assert msg in _err()


def test_python_checks_refuse_cpu_tensors_and_bad_names():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quantize_fp4(torch.zeros(4, 64), torch.zeros(1), torch.zeros(1), None, _lib.FP4_MX)
    with pytest.raises(RuntimeError, match="unknown format"):
        fp4.Fp4Tensor.empty(4, 64, "fp8", device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        fp4.Fp4Linear(torch.zeros(64, 64))
    with pytest.raises(RuntimeError, match="epilogue"):
        fp4.Fp4Linear(torch.zeros(64, 64), epilogue="tanh")
    q = fp4.Fp4Tensor.empty(4, 64, "nv", device="cpu")
    with pytest.raises(RuntimeError, match="out is"):
        fp4.quantize(torch.zeros(4, 65), out=q)


def test_interleave_groups_gates_and_ups():
    w = torch.arange(2 * 100, dtype=torch.float32)[:, None].expand(200, 3)
    t = fp4._interleave(w, 100)
    assert t.shape == (224, 3)
    for i in range(6):
        assert torch.equal(t[32 * i : 32 * i + 16, 0], w[16 * i : 16 * i + 16, 0])
        assert torch.equal(t[32 * i + 16 : 32 * i + 32, 0], w[100 + 16 * i : 100 + 16 * i + 16, 0])
    assert torch.equal(t[192:196, 0], w[96:100, 0]) and (t[196:208] == 0).all()
    assert torch.equal(t[208:212, 0], w[196:200, 0]) and (t[212:] == 0).all()


def test_the_extension_module_leaves_cpu_tensors_alone():
    c = ops._calls()
    assert c is not ops._NoCalls, "build it with python -m foidfinder_b200.build"
    x, b, f = torch.zeros(2, 32), torch.zeros(64, dtype=torch.uint8), torch.zeros(2)
    assert c.quantize(x, b, b, f, 0, None, None, 1e-6) is None
    assert c.dequantize(b, b, f, x, 0) is None
    assert c.linear(x, (1, 2, 3), 0, 32, 32, None, None, 1e-6, _lib.Fp4Epilogue(), x, None) is None
    assert c.qk_norm_rope(x, x, 1, 0, 32, 1, f, None, f, None, 1e-6, f, f, 0) is None
    with pytest.raises(TypeError):
        c.bind(1, 2)


class _OnGpu:
    """A CPU tensor that says it is on cuda:0, for host checks that come before any CUDA call."""

    def __init__(self, t):
        self._t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self._t, name)


def test_an_output_of_no_columns_is_refused():
    """For SwiGLU the library takes out_cols = 0 as N / 2, which a view of no columns does not hold."""
    out = _OnGpu(torch.zeros(4, 64, dtype=torch.float16)[:, :0])
    with pytest.raises(RuntimeError, match="out is"):
        ops._bind(_lib.Fp4Epilogue(kind=_lib.EPI_SWIGLU), 4, 128, out, None, 0, "gemm_fp4")
    with pytest.raises(RuntimeError, match="out is"):
        ops._bind(_lib.Fp4Epilogue(kind=_lib.EPI_BIAS), 4, 128, out, None, 0, "gemm_fp4")


def test_a_prepared_epilogue_holds_its_tensors():
    """Each call reads their addresses anew, so that they may be let go, or move, in between."""
    import gc
    import weakref

    bias = _OnGpu(torch.zeros(128))
    e = ops.fp4_epilogue(_lib.EPI_BIAS, 128, torch.device("cuda", 0), bias=bias)
    alive = weakref.ref(bias)
    at = bias.data_ptr()
    del bias
    gc.collect()
    assert alive() is not None and e.bias == at
    alive()._t = torch.ones(128)
    copy = ops._copy(e)
    ops._bind(copy, 4, 128, _OnGpu(torch.zeros(4, 128, dtype=torch.float16)), None, 0, "gemm_fp4")
    assert copy.bias == alive().data_ptr() != at


def _build_in(tmp_path, monkeypatch, cxx_status):
    """foidfinder_b200.build in a folder of its own, with compilers that write an empty file or fail; the commands it ran."""
    from types import SimpleNamespace

    from foidfinder_b200 import build as B

    ran = []

    def run(cmd, **_):
        ran.append(cmd[0])
        ok = cmd[0] == "nvcc" or cxx_status == 0
        if ok:
            Path(cmd[cmd.index("-o") + 1]).write_text("")
        return SimpleNamespace(returncode=0 if ok else cxx_status, stdout="", stderr="no such header")

    for name in ("csrc", "include"):
        (tmp_path / name).mkdir()
    (tmp_path / "csrc" / "calls.cpp").write_text("")
    for name, value in dict(CSRC=tmp_path / "csrc", INCLUDE=tmp_path / "include", BUILD=tmp_path / "o", LIB_DIR=tmp_path / "lib", LIB=tmp_path / "lib" / "l.so",
                            CALLS=tmp_path / "calls.so", nvcc=lambda: "nvcc", subprocess=SimpleNamespace(run=run), shutil=SimpleNamespace(which=lambda _: "cxx")).items():
        monkeypatch.setattr(B, name, value)
    return B, ran


def test_the_library_is_built_where_the_extension_module_cannot_be(tmp_path, monkeypatch, capsys):
    B, ran = _build_in(tmp_path, monkeypatch, 1)
    B.CALLS.write_text("built from other sources")
    assert B.build(force=True) == B.LIB and B.LIB.exists() and "cxx" in ran
    assert not B.CALLS.exists() and "no such header" in capsys.readouterr().err


def test_the_extension_module_is_built_again_for_another_torch(tmp_path, monkeypatch):
    B, ran = _build_in(tmp_path, monkeypatch, 0)
    assert B.build() == B.LIB and ran.count("cxx") == 1
    B.build()
    assert ran.count("cxx") == 1
    monkeypatch.setattr(B, "version", lambda _: "0.0")
    B.build()
    assert ran.count("cxx") == 2


def test_an_extension_module_for_another_torch_is_not_used(monkeypatch):
    load = ops._calls.__wrapped__
    assert load().built_for == torch.__version__
    monkeypatch.setattr(torch, "__version__", "0.0")
    with pytest.warns(UserWarning, match="built for torch"):
        assert load() is ops._NoCalls


def test_tables_of_no_angles():
    """Heads of no columns are left to the library's check, which names them."""
    t = _OnGpu(torch.zeros(0, 5))
    assert ops._tables(t, t, 0, 0, "qk_norm_rope")[2] == 5
    args = (FAKE, 0, 128, FAKE, 128, 4, 1, 1, 0, 1, FAKE, None, FAKE, None, 1e-6, FAKE, FAKE, 5, 0, None)
    assert _lib.lib().ff_qk_norm_rope(*args) == BAD and "head_dim 0" in _err()
