"""The paged-cache calls of the C++17 host seam: build tests/cpp/test_paged.cpp against libvox_cuda.so and run it on the GPU."""

from __future__ import annotations

import os
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def build_cpp(tmp: Path) -> Path:
    from vox_b200 import build

    build.build()
    exe = tmp / "test_paged"
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O2", "-Wall", f"-I{ROOT / 'include'}", str(ROOT / "tests/cpp/test_paged.cpp"),
                    str(build.LIB), f"-Wl,-rpath,{build.LIB.parent}", "-o", str(exe)], check=True, capture_output=True, text=True)
    return exe


def test_paged_seam_compiles_and_links(tmp_path):
    assert build_cpp(tmp_path).exists()


@pytest.mark.gpu
def test_paged_seam_on_gpu(tmp_path, vox):
    r = subprocess.run([str(build_cpp(tmp_path))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "OK" in r.stdout
