"""Refusals of the layer operators' C entry points that no device has to see."""
import ctypes

import pytest

from ferrograd_b200 import _lib
from test_layer_cpu import BASE, grad_args, linear_args

DTYPES = [(_lib.F32, 4), (_lib.BF16, 2), (_lib.F16, 2)]


def refused(rc, word):
    assert rc == 1  # FG_ERR_INVALID
    assert word in _lib.lib().fg_last_error().decode()


@pytest.mark.parametrize("dtype,size", DTYPES)
def test_addresses_are_multiples_of_the_element(dtype, size):
    L = _lib.lib()
    need = ctypes.c_size_t()
    for name in ("x", "w", "bias", "residual", "pre", "out"):
        for off in range(1, size):
            a = linear_args(dtype=dtype, ld_pre=16, ld_residual=16)
            setattr(a, name, BASE + 0x70000 + off)
            refused(L.fg_linear(ctypes.byref(a), None), "multiple")
            refused(L.fg_linear_workspace(ctypes.byref(a), ctypes.byref(need)), "multiple")
    for name in ("dy", "x", "w", "pre", "dx", "dx_residual", "dw", "db"):
        a = grad_args(dtype=dtype, act=_lib.ACT_GELU, pre=BASE + 0x60000, ld_pre=16,
                      ld_dx_residual=32)
        setattr(a, name, BASE + 0x70000 + 1)
        refused(L.fg_linear_grad(ctypes.byref(a), None), "multiple")
        refused(L.fg_linear_grad_workspace(ctypes.byref(a), ctypes.byref(need)), "multiple")
    spec = _lib.DropoutC(0.5, 1, 2)
    for x, r, out in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        refused(L.fg_dropout(dtype, 4, 8, BASE + x, 8, BASE + 0x1000 + r, 8, BASE + 0x2000 + out, 8,
                             ctypes.byref(spec), None), "multiple")


def test_workspace_boundary():
    L = _lib.lib()
    need = ctypes.c_size_t()
    for a, ask, call in ((linear_args(dtype=_lib.F32, M=64), L.fg_linear_workspace, L.fg_linear),
                         (grad_args(act=_lib.ACT_SILU, pre=BASE + 0x60000, ld_pre=16),
                          L.fg_linear_grad_workspace, L.fg_linear_grad)):
        assert ask(ctypes.byref(a), ctypes.byref(need)) == 0 and need.value > 0
        a.workspace_bytes = need.value + 256
        for off in (1, 2, 4, 8, 16, 128):
            a.workspace = BASE + 0x80000 + off
            refused(call(ctypes.byref(a), None), "boundary")


def test_nothing_overlaps_an_empty_array():
    """No bytes are shared with an array of no elements, wherever it points.  (Past
    the refusals the call asks for a device, which is another error, or has one.)"""
    L = _lib.lib()
    need = ctypes.c_size_t()
    a = linear_args(K=0, x=BASE + 0x20010, w=BASE + 0x20020)
    assert L.fg_linear_workspace(ctypes.byref(a), ctypes.byref(need)) == 0
    for kw in (dict(N=0, dy=BASE + 0x30010, db=BASE + 0x30020, dw=BASE + 0x30030),
               dict(K=0, x=BASE + 0x50000, w=BASE + 0x50002, dx=BASE + 0x50004),
               dict(M=0, dy=BASE + 0x40010, x=BASE + 0x40020, dx=BASE + 0x40040)):
        g = grad_args(**kw)
        assert L.fg_linear_grad_workspace(ctypes.byref(g), ctypes.byref(need)) == 0, kw
