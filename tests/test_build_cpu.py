"""What the build needs: the library neither torch nor its headers, the binding of the digital operators a rebuild when torch
changes.  Compilers are replaced by a record of their calls."""

import os
import subprocess
import sys

import pytest

from aihwkit_b200 import build as B


def test_the_library_is_built_without_torch(tmp_path):
    """The build as a script in an interpreter that has no torch; stand-ins for nvcc write empty files."""
    nvcc = tmp_path / "nvcc"
    nvcc.write_text("#!/bin/sh\nwhile [ $# -gt 0 ]; do if [ \"$1\" = -o ]; then : > \"$2\"; fi; shift; done\n")
    nvcc.chmod(0o755)
    code = f"""
import runpy, sys
sys.modules["torch"] = None
m = runpy.run_path({B.__file__!r}, run_name="library_build")
g = m["build"].__globals__
g["OBJ"], g["OUT"] = {str(tmp_path / "obj")!r}, {str(tmp_path / "lib.so")!r}
print(m["build"](force=True))
"""
    env = dict(os.environ, NVCC=str(nvcc))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, env=env, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == str(tmp_path / "lib.so"), run.stderr[-1000:]


def test_the_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    import torch

    calls = []

    class Done:
        returncode = 0

    def compiler(cmd, **kw):
        calls.append(cmd)
        open(tmp_path / "binding.so", "w").close()
        return Done()

    monkeypatch.setattr(B, "DIGITAL_OUT", str(tmp_path / "binding.so"))
    monkeypatch.setattr(B, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(B.subprocess, "run", compiler)
    build = lambda **kw: (B.build_digital(**kw), len(calls))[1]
    assert build() == 1 and build() == 1 and build(force=True) == 2
    with monkeypatch.context() as m:
        m.setattr(torch, "__version__", "99.0")
        assert build() == 3 and build() == 3
    assert build() == 4
    os.remove(tmp_path / "binding.so")
    assert build() == 5


def test_a_failing_compiler_is_reported(monkeypatch, tmp_path):
    class Failed:
        returncode, stdout, stderr = 1, "", "no such header"

    monkeypatch.setattr(B, "DIGITAL_OUT", str(tmp_path / "binding.so"))
    monkeypatch.setattr(B, "OBJ", str(tmp_path / "obj"))
    monkeypatch.setattr(B.subprocess, "run", lambda cmd, **kw: Failed())
    with pytest.raises(RuntimeError, match="no such header"):
        B.build_digital()
    assert not os.path.exists(tmp_path / "obj" / "ab200_digital.txt")
