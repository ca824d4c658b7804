"""Trees of drafted tokens and bounded caches of include/fns/kernels.h from a hipcc-compiled C++ program
(tests/cpp/kv_tree_caller.cpp, built by build()): plan, append, attention, weights, the accepted path and eviction, checked inside
that program."""
from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

BIN = Path(__file__).resolve().parent / "cpp" / "kv_tree_caller"


def test_kv_tree_caller_cpp():
    assert BIN.exists(), "tests/cpp/kv_tree_caller is not built: run __graft_entry__.build() first"
    r = subprocess.run([str(BIN)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and "KV_TREE_CALLER_OK" in r.stdout, r.stdout[-4000:] + r.stderr[-2000:]
