"""Ranges of tokens that attention behind shared prompts splits its work into:
the header that the kernels take them from, on the host."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_ranges_cpp_cases(tmp_path):
    binary = tmp_path / "test_ranges"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-fconstexpr-ops-limit=500000000",
                    f"-I{ROOT / 'cuda_force_amd' / 'csrc'}", str(ROOT / "tests" / "cpp" / "test_ranges.cpp"), "-o",
                    str(binary)], check=True, capture_output=True, text=True)
    result = subprocess.run([str(binary)], capture_output=True, text=True, timeout=120)
    assert result.returncode == 0, result.stderr
