"""Every HIP source is compiled without packed fp32 instructions."""
import os
import shutil
import subprocess
from types import SimpleNamespace

import pytest

from midiseq import _build


def test_every_hip_source_has_the_flag(monkeypatch, tmp_path):
    seen = []
    monkeypatch.setattr(_build, "OBJ", str(tmp_path))
    monkeypatch.setattr(subprocess, "run", lambda cmd, **kw: seen.append(cmd) or SimpleNamespace(returncode=0))
    sources = [s for s in _build._sources() if s.endswith(".hip")]
    for src in sources:
        _build._compile(src)
    assert len(seen) == len(sources) > 20
    for cmd in seen:
        at = [i for i, w in enumerate(cmd) if w == "-packed-fp32-ops"]
        assert at and cmd[at[0] - 3:at[0]] == ["-Xclang", "-target-feature", "-Xclang"], os.path.basename(cmd[-3])


def test_no_packed_fp32_in_the_library(tmp_path):
    """the gfx950 code of the built library, disassembled"""
    objdump = "/opt/rocm/llvm/bin/llvm-objdump"
    if not (os.path.exists(objdump) and os.path.exists(_build.LIB)):
        pytest.skip("needs the built library and llvm-objdump")
    lib = shutil.copy(_build.LIB, tmp_path / "lib.so")
    subprocess.run([objdump, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    parts = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    assert len(parts) > 15
    for f in parts:
        asm = subprocess.run([objdump, "-d", f], cwd=tmp_path, check=True, capture_output=True).stdout
        assert b"v_pk_add_f32" not in asm and b"v_pk_mul_f32" not in asm and b"v_pk_fma_f32" not in asm, f
