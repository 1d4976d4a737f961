"""The layer products' shared-memory layout over every form and row count, and what
their kernels may not use."""
import os
import subprocess

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
