"""When the layer operators' binding is compiled."""
import os
import subprocess
import sys

import torch

from ferrograd_b200 import build


def test_another_torch_rebuilds_the_binding(monkeypatch, tmp_path):
    build.build_layer()
    ran = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, check: ran.append(cmd))
    build.build_layer()
    assert not ran  # up to date
    with open(os.path.join(build.OBJDIR, "layer_torch")) as f:
        (tmp_path / "layer_torch").write_text(f.read())
    monkeypatch.setattr(build, "OBJDIR", str(tmp_path))  # the record of the build alone
    build.build_layer()
    assert not ran
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".other")
    build.build_layer()
    assert len(ran) == 1 and any(a.endswith("layer_py.cpp") for a in ran[0])
    build.build_layer()
    assert len(ran) == 1


def test_the_libraries_build_without_torch():
    code = ("import sys; sys.modules['torch'] = None; from ferrograd_b200 import build; "
            "print(build.build())")
    got = subprocess.run([sys.executable, "-c", code], cwd=build.ROOT, capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    assert got.stdout.strip() == build.LIB
