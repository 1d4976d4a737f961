"""The layer products' shared-memory layout over every form and row count, and what
their kernels may not use."""
import ctypes
import os
import subprocess

from ferrograd_b200 import _lib
from test_layer_cpu import linear_args

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def compiled(tmp_path, source):
    exe = tmp_path / "plan"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror",
                    "-I" + os.path.join(ROOT, "ferrograd_b200", "csrc"),
                    os.path.join(ROOT, "tests", source), "-o", str(exe)], check=True)
    return str(exe)


def test_every_layout_fits(tmp_path):
    got = subprocess.run([compiled(tmp_path, "layer_plan_sweep.cpp")], capture_output=True, text=True)
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


# Gradients of M x K -> N: microseconds with dx and dw in one launch and in two (one
# B200, a CUDA graph of calls on inputs that do not fit L2).
JOINT = [("bf16", 256, 784, 128, 9.9, 13.8), ("bf16", 256, 1024, 1024, 14.0, 17.5),
         ("bf16", 1024, 512, 512, 13.1, 18.9), ("bf16", 8192, 128, 128, 34.7, 21.5),
         ("bf16", 2048, 256, 1024, 18.9, 23.8), ("bf16", 64, 1024, 1024, 10.1, 14.6),
         ("bf16", 512, 512, 512, 12.5, 17.5), ("bf16", 128, 128, 128, 8.4, 13.0),
         ("bf16", 512, 1024, 1024, 16.2, 20.7), ("bf16", 16384, 64, 64, 49.9, 21.3),
         ("f16", 1024, 256, 2048, 18.5, 24.2), ("bf16", 768, 768, 768, 13.6, 19.9),
         ("f32", 64, 256, 256, 12.1, 16.8), ("f32", 128, 128, 128, 12.1, 19.6),
         ("f32", 4096, 256, 64, 67.8, 28.6), ("f32", 512, 784, 128, 19.9, 24.9),
         ("f32", 8192, 64, 64, 67.5, 33.1), ("f32", 256, 784, 128, 15.0, 21.0),
         ("f32", 512, 256, 256, 16.8, 29.7), ("f32", 512, 512, 512, 21.5, 28.3),
         ("f32", 16384, 128, 64, 260.3, 58.0), ("f32", 128, 64, 8192, 68.2, 34.8)]


def test_two_products_share_a_launch_where_that_is_faster(tmp_path):
    """Every measured gradient whose two ways differ by a fifth takes the faster."""
    chains = {"bf16": (1, 256), "f16": (1, 64), "f32": (3, 2)}
    text = "".join("%d %d %d %d %d\n" % (*chains[dt], m, k, n) for dt, m, k, n, _, _ in JOINT)
    got = subprocess.run([compiled(tmp_path, "layer_forms.cpp")], input=text, capture_output=True,
                         text=True, check=True).stdout.split()
    for case, way in zip(JOINT, got):
        one, two = case[4:]
        assert max(one, two) > 1.2 * min(one, two)
        assert way == ("1" if one < two else "0"), case
