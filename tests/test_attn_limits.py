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


def test_a_workspace_has_to_be_contiguous(monkeypatch):
    """Its elements are counted, and the kernels write that many bytes from its address on."""
    calls = []
    monkeypatch.setattr(ops, "_here", lambda what, *ts: 0)
    monkeypatch.setattr(ops, "call", lambda name, *args: calls.append(name))
    cache = ops.KvCache(4, 16, 1, 64, pages=torch.zeros(4, ops.lib().fns_hip_kv_page_bytes(1, 64, 16), dtype=torch.uint8))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    batch = ops.KvBatch(i32(0, 1), i32(10), i32(0).view(1, 1), 1, 1)
    q = torch.zeros(1, 2, 64)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 20, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="contiguous"):
            ops.attn(cache, batch, q, ws=ws)
    assert not calls
    ops.attn(cache, batch, q, ws=torch.zeros(1 << 10, dtype=torch.uint8))
    assert calls == ["fns_hip_attn"]
