"""The attention half of include/fns/kernels.h from a hipcc-compiled C++ program (tests/cpp/attn_half_caller.cpp, built by
build()): residual add and norm, append, read back and attention, checked inside that program."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

BIN = Path(__file__).resolve().parent / "cpp" / "attn_half_caller"


def test_attn_half_caller_cpp():
    assert BIN.exists(), "tests/cpp/attn_half_caller is not built: run __graft_entry__.build() first"
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "ATTN_HALF_CALLER_OK" in r.stdout, r.stdout[-4000:] + r.stderr[-2000:]
