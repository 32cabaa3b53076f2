"""When the build compiles a source again: after a change of it or of any header, .h or .cuh."""
from __future__ import annotations

import importlib.util
import os
import subprocess
import time
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("changed,again", [(None, False), ("k.cu", True), ("a.h", True), ("b.cuh", True)])
def test_a_changed_header_compiles_its_sources_again(tmp_path, monkeypatch, changed, again):
    spec = importlib.util.spec_from_file_location("pk_build_test", ROOT / "parakeet.wgsl_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    csrc, out = tmp_path / "csrc", tmp_path / "out"
    csrc.mkdir()
    out.mkdir()
    now = time.time()
    for name in ("k.cu", "a.h", "b.cuh"):
        (csrc / name).write_text("")
        os.utime(csrc / name, (now + (20 if name == changed else 0),) * 2)
    (out / "k.o").write_text("")
    os.utime(out / "k.o", (now + 10,) * 2)
    ran = []
    monkeypatch.setattr(build, "CSRC", csrc)
    monkeypatch.setattr(build, "BUILD", out)
    monkeypatch.setattr(build, "nvcc", lambda: "nvcc")
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or subprocess.CompletedProcess(cmd, 0, "", ""))
    build._compile(csrc / "k.cu", False)
    assert bool(ran) == again
