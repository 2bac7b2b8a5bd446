"""CPU: the library builds where torch is not there; only the operators' torch binding is left out, with a word."""
import os
import subprocess
import sys

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusers_amd", "csrc")


def plan(tmp_path, python):
    """What make would run, nothing being built yet."""
    r = subprocess.run(["make", "-n", "-C", CSRC, f"PYTHON={python}", f"OUT={tmp_path}/libsdengine.so", f"OBJDIR={tmp_path}/obj", f"TORCH_OPS={tmp_path}/_torch_ops.so"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_with_torch(tmp_path):
    out = plan(tmp_path, sys.executable)
    assert "torch_ops.cpp" in out and "op_xattn.hip" in out and "left out" not in out


@pytest.mark.parametrize("script", ["exit 127", f'exec "{sys.executable}" -S "$@"', 'echo /nowhere'])
def test_without_torch(tmp_path, script):
    """No Python, a Python without torch, a torch without headers."""
    python = tmp_path / "python"
    python.write_text(f"#!/bin/sh\n{script}\n")
    python.chmod(0o755)
    out = plan(tmp_path, python)
    assert "torch_ops.cpp" not in out and "op_xattn.hip" in out and f"{tmp_path}/libsdengine.so" in out and "left out" in out
