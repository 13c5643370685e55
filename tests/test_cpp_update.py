"""Builds and runs the C++ mirror test of the operators between logits and an
update (tests/cpp/update_test.cpp)."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
LIBDIR = ROOT / "kernix_b200"


def _build(tmp_path) -> Path:
    exe = tmp_path / "update_test"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", str(ROOT / "include"),
           str(ROOT / "tests/cpp/update_test.cpp"), "-L", str(LIBDIR), "-lkernix_b200", f"-Wl,-rpath,{LIBDIR}", "-o",
           str(exe)]
    subprocess.run(cmd, check=True)
    return exe


def test_cpp_update_compiles(tmp_path):
    assert _build(tmp_path).exists()


@pytest.mark.gpu
def test_cpp_update_gpu(tmp_path):
    out = subprocess.run([str(_build(tmp_path))], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr
    assert "update_test ok" in out.stdout
