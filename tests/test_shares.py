"""The arithmetic by which kernels cut work into shares (CPU): compiles tests/shares_check.cc with the header and runs it."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_shares_and_pieces_are_those_of_whole_numbers(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = tmp_path / "shares"
    subprocess.run([cxx, "-O2", "-I", str(HERE.parent / "asterlm-frontier_b200" / "csrc"), "-o", str(exe), str(HERE / "shares_check.cc")],
                   check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "0\n"
