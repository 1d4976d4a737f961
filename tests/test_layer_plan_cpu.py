"""The layer products' shared-memory layout over every form and row count, and what
their kernels may not use."""
import ctypes
import os
import subprocess

from ferrograd_b200 import _lib
from test_layer_cpu import linear_args

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_layout_fits(tmp_path):
    exe = tmp_path / "sweep"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror",
                    "-I" + os.path.join(ROOT, "ferrograd_b200", "csrc"),
                    os.path.join(ROOT, "tests", "layer_plan_sweep.cpp"), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout
    assert int(got.stdout.split()[0]) > 10000


def test_no_constant_loads_in_kernels_that_start_early():
    """The layer's kernels may start before the stream's previous kernel has
    ended, so their inputs are not constant over the kernels' life: neither
    __ldg nor the compiler's own choice of it (const __restrict__) is allowed."""
    csrc = os.path.join(ROOT, "ferrograd_b200", "csrc")
    for name in ("fg_layer.cu", "fg_layer.cuh", "fg_layer_gemm.cu"):
        with open(os.path.join(csrc, name)) as f:
            lines = [line.split("//")[0] for line in f]
        for word in ("__ldg", "__restrict__", "ld.global.nc"):
            assert not any(word in line for line in lines), (name, word)


def test_unaligned_rows_go_where_they_are_faster():
    """Three and four 16-bit rows off 16-byte boundaries take the tensor cores, whose
    copy of the weight shows as workspace (4 x 4095 -> 4096: 28.5 us, 46 row by row)."""
    L = _lib.lib()
    need = ctypes.c_size_t()
    for rows, staged in ((1, False), (2, False), (3, True), (4, True), (5, True)):
        a = linear_args(M=rows, N=64, K=33, x_row=33, w_row=33, ld_out=64)
        assert L.fg_linear_workspace(ctypes.byref(a), ctypes.byref(need)) == 0
        assert (need.value > 0) == staged
    for rows, staged in ((8, False), (9, True)):
        a = linear_args(dtype=_lib.F32, M=rows)
        assert L.fg_linear_workspace(ctypes.byref(a), ctypes.byref(need)) == 0
        assert (need.value > 0) == staged
