"""The layer products' shared-memory layout over every form and row count."""
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
