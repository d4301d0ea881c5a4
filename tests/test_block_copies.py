"""What the tiles of the block products copy (novann_amd/csrc/novaq_block_copies.h): inside
the operands and all that is multiplied, for every tiling.  CPU only (the header is built
with g++); the kernel runs the same functions."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_every_copy_lies_in_its_operand(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "block_copies_run")
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", "-Werror", "-o", exe,
                    os.path.join(HERE, "native", "block_copies_run.cpp")], check=True)
    r = subprocess.run([exe, "3000"], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    ok, cases, past = r.stdout.split()
    # sets of 64 rows that all lie past the operand occur, from later blocks on too
    assert ok == "ok" and int(cases) == 3000 and int(past) > 10000
