"""Host-side limits of the attention calls and their wrappers, on the CPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from flintnsteel_amd import _lib, ops

P, BUF = ctypes.c_void_p, 0x1000  # never dereferenced: the checks come first


@pytest.mark.parametrize("n_tok,n_head", [(1 << 24, 1 << 15), ((1 << 24) + 3, 1 << 15), (2 ** 31 - 1, 65535)])
def test_calls_of_more_row_tiles_than_a_grid_has_are_refused(n_tok, n_head):
    """Also where the number of tiles of 128 rows passes 32 bits (2^24 tokens of 2^15 heads over one: 2^32 of them)."""
    cache = ops.KvCacheDesc(1, 64, 16, 4, BUF)
    batch = ops.KvBatchDesc(1, n_tok, n_tok, 100, 2, BUF, BUF, BUF)
    att = ops.AttnDesc(0, n_head, 0, 1.0, None, n_head * 64, n_head * 64)
    L, r = _lib.lib(), ctypes.byref
    assert L.fns_hip_attn(r(cache), r(batch), r(att), P(BUF), P(2 * BUF), P(3 * BUF), 1 << 50, None) == -2
    assert b"too many" in L.fns_hip_last_error()
