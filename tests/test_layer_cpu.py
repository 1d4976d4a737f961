"""The layer operators without a GPU: their arguments' layout, the refusals made
before any device work, the workspace queries, and the tests' own restatement."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest

from ferrograd_b200 import _lib
from layer_ref import ACTS, act, drop, keep_mask, linear, linear_grad, philox4x32, slope

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_structs_match_the_header(tmp_path):
    names = {"fg_linear_args": _lib.LinearArgsC, "fg_linear_grad_args": _lib.LinearGradArgsC,
             "fg_dropout_spec": _lib.DropoutC}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "ferro_cuda.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    got = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for c, py in names.items():
        assert int(got[c]) == ctypes.sizeof(py)
        for f in py._fields_:
            assert int(got[f"{c}.{f[0]}"]) == getattr(py, f[0]).offset, (c, f[0])


def test_constants_match_the_header():
    text = open(os.path.join(ROOT, "include", "ferro_cuda.h")).read()
    for name in ("ACT_NONE", "ACT_RELU", "ACT_GELU", "ACT_GELU_TANH", "ACT_SILU", "BF16", "F16"):
        assert f"FG_{name} = {getattr(_lib, name)}" in text


BASE = 0x100000  # stands for device memory: refused calls never touch it


def linear_args(**kw):
    a = _lib.LinearArgsC(dtype=_lib.BF16, M=8, N=16, K=32, x=BASE, x_row=32, x_col=1,
                         w=BASE + 0x10000, w_row=32, w_col=1, out=BASE + 0x20000, ld_out=16)
    for k, v in kw.items():
        if k == "p":
            a.drop.p = v
        else:
            setattr(a, k, v)
    return a


def grad_args(**kw):
    a = _lib.LinearGradArgsC(dtype=_lib.BF16, M=8, N=16, K=32, dy=BASE, dy_row=16, dy_col=1,
                             x=BASE + 0x10000, x_row=32, x_col=1, w=BASE + 0x20000, w_row=32,
                             w_col=1, dx=BASE + 0x30000, ld_dx=32, dw=BASE + 0x40000, ld_dw=32,
                             db=BASE + 0x50000)
    for k, v in kw.items():
        if k == "p":
            a.drop.p = v
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=_lib.I32), "not f32"),
    (dict(dtype=9), "not f32"),
    (dict(M=-1), "lie in"),
    (dict(K=0x7fffffff), "lie in"),
    (dict(act=7), "activation"),
    (dict(act=-1), "activation"),
    (dict(p=1.25), "probability"),
    (dict(p=-0.5), "probability"),
    (dict(p=math.nan), "probability"),
    (dict(x=None), "null"),
    (dict(out=None), "null"),
    (dict(ld_out=15), "pitch"),
    (dict(pre=BASE + 0x30000, ld_pre=8), "pitch"),
    (dict(out=BASE + 64, ld_out=16), "overlaps an operand"),
    (dict(pre=BASE + 0x10000, ld_pre=16), "overlaps an operand"),
    (dict(bias=BASE + 0x20000), "overlaps an operand"),
    (dict(residual=BASE + 0x20000, ld_residual=32), "residual"),
    (dict(residual=BASE + 0x20010, ld_residual=16), "residual"),
    (dict(pre=BASE + 0x20000, ld_pre=16), "overlaps pre"),
])
def test_linear_refusals(kw, word):
    L = _lib.lib()
    need = ctypes.c_size_t()
    a = linear_args(**kw)
    for rc in (L.fg_linear(ctypes.byref(a), None),
               L.fg_linear_workspace(ctypes.byref(a), ctypes.byref(need))):
        assert rc == 1  # FG_ERR_INVALID
        assert word in L.fg_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=_lib.BOOL), "not f32"),
    (dict(N=-4), "lie in"),
    (dict(act=5), "activation"),
    (dict(p=2.0), "probability"),
    (dict(dy=None), "null dy"),
    (dict(act=_lib.ACT_GELU), "pre-activations"),
    (dict(act=_lib.ACT_RELU, pre=BASE + 0x60000, ld_pre=4), "pre-activations"),
    (dict(w=None), "needs w"),
    (dict(x=None), "needs x"),
    (dict(ld_dx=31), "pitch"),
    (dict(ld_dw=8), "pitch"),
    (dict(dx=BASE, ld_dx=32), "overlaps an operand"),
    (dict(dw=BASE + 0x30100), "overlaps"),
    (dict(db=BASE + 0x40000), "overlaps"),
    (dict(dx_residual=BASE + 0x30010, ld_dx_residual=32), "dx_residual"),
    (dict(dx_residual=BASE + 0x40000, ld_dx_residual=32), "dx_residual"),
])
def test_grad_refusals(kw, word):
    L = _lib.lib()
    need = ctypes.c_size_t()
    a = grad_args(**kw)
    for rc in (L.fg_linear_grad(ctypes.byref(a), None),
               L.fg_linear_grad_workspace(ctypes.byref(a), ctypes.byref(need))):
        assert rc == 1
        assert word in L.fg_last_error().decode()


def test_null_and_short_workspace():
    L = _lib.lib()
    need = ctypes.c_size_t()
    assert L.fg_linear(None, None) == 1 and L.fg_linear_grad(None, None) == 1
    assert L.fg_linear_workspace(None, ctypes.byref(need)) == 1
    assert L.fg_linear_grad_workspace(None, ctypes.byref(need)) == 1
    a = linear_args(dtype=_lib.F32, M=64, w_row=32)
    assert L.fg_linear_workspace(ctypes.byref(a), ctypes.byref(need)) == 0
    assert need.value >= (64 + 16) * 32 * 6  # three bf16 planes of each operand
    assert L.fg_linear(ctypes.byref(a), None) == 1
    assert "workspace" in L.fg_last_error().decode()
    a.workspace, a.workspace_bytes = BASE + 0x80000, need.value - 1
    assert L.fg_linear(ctypes.byref(a), None) == 1
    g = grad_args(act=_lib.ACT_SILU, pre=BASE + 0x60000, ld_pre=16)
    assert L.fg_linear_grad_workspace(ctypes.byref(g), ctypes.byref(need)) == 0
    assert need.value >= 8 * 16 * 2  # dz
    assert L.fg_linear_grad(ctypes.byref(g), None) == 1
    # 16-bit operands on 16-byte rows are read in place
    assert L.fg_linear_workspace(ctypes.byref(linear_args(M=64)), ctypes.byref(need)) == 0
    assert need.value == 0


def test_dropout_refusals():
    L = _lib.lib()

    def run(dtype=_lib.F32, rows=4, cols=8, x=BASE, ldx=8, r=None, ldr=0, out=BASE + 0x1000, ldo=8,
            p=0.5):
        spec = _lib.DropoutC(p, 1, 2)
        return L.fg_dropout(dtype, rows, cols, x, ldx, r, ldr, out, ldo, ctypes.byref(spec), None)

    for kw in (dict(dtype=_lib.I32), dict(x=None), dict(out=None), dict(ldo=7), dict(p=-1.0),
               dict(p=math.inf), dict(rows=1 << 40), dict(cols=1 << 31), dict(out=BASE + 32),
               dict(r=BASE + 0x1010, ldr=8)):
        assert run(**kw) == 1, kw
    assert run(rows=0) == 0 and run(cols=0, ldo=0) == 0  # nothing to do, no device work


# ---- the restatement the GPU tests compare with ----------------------------------------


def test_philox_known_answers():
    """Published vectors of Philox4x32-10: zeros, ones, pi's digits."""
    ones = 0xFFFFFFFF
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in philox4x32(ctr, key)) == want


def test_mask_depends_on_row_column_seed_and_offset_alone():
    big = keep_mask(40, 100, 0.3, 7, 9)
    assert np.array_equal(keep_mask(12, 33, 0.3, 7, 9), big[:12, :33])
    for seed, offset in ((8, 9), (7, 10), (7 + (1 << 32), 9), (7, 9 + (1 << 32))):
        assert not np.array_equal(keep_mask(40, 100, 0.3, seed, offset), big)


@pytest.mark.parametrize("name", ACTS)
def test_slopes_are_derivatives(name):
    """Central differences of the restated activations: h^2 |f'''| / 6 + 2^-52 / h."""
    z = np.linspace(-6, 6, 401) + 0.0137
    h = 1e-5
    num = (act(z + h, name) - act(z - h, name)) / (2 * h)
    assert np.abs(num - slope(z, name)).max() <= 1e-9


def test_gradients_are_derivatives():
    rng = np.random.default_rng(0)
    x, w, b = rng.standard_normal((5, 4)), rng.standard_normal((6, 4)), rng.standard_normal(6)
    c, spec, h = rng.standard_normal((5, 6)), (0.25, 3, 4), 1e-6

    def loss(x):
        return float((c * linear(x, w, b, "gelu", spec, None)[0]).sum())

    dx = linear_grad(c, x, w, x @ w.T + b, "gelu", spec)[0]
    for i in np.ndindex(x.shape):
        d = np.zeros_like(x)
        d[i] = h
        assert abs((loss(x + d) - loss(x - d)) / (2 * h) - dx[i]) <= 1e-8
    assert not drop(np.full((3, 9), np.nan), (1.0, 0, 0)).any()
