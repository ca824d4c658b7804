"""Argument checks of the attention-half entry points, on the host before any launch."""
from __future__ import annotations

import ctypes

import pytest

from flintnsteel_amd import _lib, ops

P = ctypes.c_void_p
BUF = 0x1000  # never dereferenced: the checks come first


def cache(**kw):
    d = dict(n_head_kv=2, head_dim=128, page_size=64, n_pages=4, pages=BUF)
    return ops.KvCacheDesc(**{**d, **kw})


def batch(**kw):
    d = dict(n_seq=1, max_q=1, n_tok=1, max_kv=100, table_stride=2, q_start=BUF, kv_len=BUF, page_table=BUF)
    return ops.KvBatchDesc(**{**d, **kw})


def app(**kw):
    d = dict(dtype=0, rope=0, rope_dim=0, n_head=4, inv_freq=None, k=BUF, v=BUF, q=BUF, q_out=2 * BUF, k_stride=256,
             v_stride=256, q_stride=512, q_out_stride=512)
    return ops.KvAppendDesc(**{**d, **kw})


def att(**kw):
    d = dict(dtype=0, n_head=4, window=0, scale=1.0, sinks=None, q_stride=512, out_stride=512)
    return ops.AttnDesc(**{**d, **kw})


def _append(c=None, b=None, x=None):
    c, b, x = c or cache(), b or batch(), x or app()
    return _lib.lib().fns_hip_kv_append(ctypes.byref(c), ctypes.byref(b), ctypes.byref(x), None)


def _attn(c=None, b=None, x=None, q=BUF, out=2 * BUF, ws=BUF, size=1 << 40):
    c, b, x = c or cache(), b or batch(), x or att()
    return _lib.lib().fns_hip_attn(ctypes.byref(c), ctypes.byref(b), ctypes.byref(x), P(q), P(out), P(ws), size, None)


BAD_CACHES = [dict(head_dim=96), dict(head_dim=0), dict(page_size=48), dict(page_size=8), dict(page_size=8192),
              dict(n_head_kv=0), dict(n_head_kv=2000), dict(n_pages=0), dict(n_pages=1 << 31), dict(pages=None),
              dict(pages=BUF + 8)]
BAD_BATCHES = [dict(n_seq=-1), dict(n_tok=-1), dict(max_q=-1), dict(max_kv=-1), dict(table_stride=-1), dict(n_tok=1 << 31),
               dict(q_start=None), dict(kv_len=None), dict(page_table=None), dict(n_seq=40000)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches(kw):
    assert _append(c=cache(**kw)) == -2 and _attn(c=cache(**kw)) == -2
    assert _lib.lib().fns_hip_kv_read(ctypes.byref(cache(**kw)), ctypes.byref(batch()), P(BUF), P(BUF), None) == -2


@pytest.mark.parametrize("kw", BAD_BATCHES)
def test_bad_batches(kw):
    assert _append(b=batch(**kw)) == -2 and _attn(b=batch(**kw)) == -2
    assert _lib.lib().fns_hip_kv_read(ctypes.byref(cache()), ctypes.byref(batch(**kw)), P(BUF), P(BUF), None) == -2


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=1), -1), (dict(rope=3), -2), (dict(rope=1, rope_dim=64), -2), (dict(rope=1, rope_dim=24, inv_freq=BUF), -2),
    (dict(rope=2, rope_dim=0, inv_freq=BUF), -2), (dict(rope=2, rope_dim=144, inv_freq=BUF), -2), (dict(n_head=3), -2),
    (dict(n_head=-2), -2), (dict(k=None), -2), (dict(v=None), -2), (dict(q=None), -2), (dict(q_out=None), -2),
    (dict(k_stride=255), -2), (dict(v_stride=0), -2), (dict(q_stride=511), -2), (dict(q_out_stride=-512), -2),
    (dict(q_out=BUF, q_out_stride=600), -2)])
def test_append_arguments(kw, rc):
    assert _append(x=app(**kw)) == rc
    assert b"kv_append" in _lib.lib().fns_hip_last_error()


@pytest.mark.parametrize("kw,rc", [(dict(dtype=1), -1), (dict(n_head=5), -2), (dict(n_head=0), -2), (dict(window=-1), -2),
                                   (dict(q_stride=511), -2), (dict(out_stride=0), -2), (dict(n_head=65538), -2)])
def test_attn_arguments(kw, rc):
    assert _attn(x=att(**kw)) == rc
    size = ctypes.c_size_t()
    assert _lib.lib().fns_hip_attn_workspace(ctypes.byref(cache()), ctypes.byref(batch()), ctypes.byref(att(**kw)),
                                             ctypes.byref(size)) == rc


def test_null_arguments():
    L, r = _lib.lib(), ctypes.byref
    assert L.fns_hip_kv_append(None, r(batch()), r(app()), None) == -2
    assert L.fns_hip_kv_append(r(cache()), None, r(app()), None) == -2
    assert L.fns_hip_kv_append(r(cache()), r(batch()), None, None) == -2
    assert L.fns_hip_attn(r(cache()), r(batch()), None, P(BUF), P(BUF), P(BUF), 0, None) == -2
    assert L.fns_hip_attn_workspace(r(cache()), r(batch()), r(att()), None) == -2
    assert _attn(q=None) == -2 and _attn(out=None) == -2
    assert L.fns_hip_kv_read(r(cache()), r(batch()), None, P(BUF), None) == -2
    assert L.fns_hip_add_rms_norm_q8_1(P(BUF), None, P(BUF), P(BUF), P(BUF), P(BUF), 64, 1e-6, 1, None) == -2
    assert L.fns_hip_dequantize_q8_1(None, 0, P(BUF), None, 64, 1, None) == -2


def test_empty_batches_are_noops():
    for kw in (dict(n_seq=0, q_start=None, kv_len=None, page_table=None), dict(n_tok=0), dict(max_q=0)):
        assert _append(b=batch(**kw)) == 0 and _attn(b=batch(**kw), ws=None, size=0) == 0
    assert _lib.lib().fns_hip_add_rms_norm_q8_1(None, None, None, None, None, None, 64, 1e-6, 0, None) == 0


@pytest.mark.parametrize("n,rows,xq", [(33, 1, BUF), (0, 1, BUF), (64, -1, BUF), (64, 1, BUF + 2)])
def test_add_rms_norm_arguments(n, rows, xq):
    assert _lib.lib().fns_hip_add_rms_norm_q8_1(P(BUF), P(BUF), P(BUF), P(BUF), P(BUF), P(xq), n, 1e-6, rows, None) == -2


def test_dequantize_arguments():
    L = _lib.lib()
    assert L.fns_hip_dequantize_q8_1(P(BUF), 30, P(BUF), None, 64, 1, None) == -1
    assert L.fns_hip_dequantize_q8_1(P(BUF), 0, P(BUF), None, 33, 1, None) == -2
    assert L.fns_hip_dequantize_q8_1(P(BUF + 1), 0, P(BUF), None, 64, 1, None) == -2


def test_page_bytes():
    L = _lib.lib()
    # codes of K and V, 4 bits each, and a scale byte per 32 channels of either
    assert L.fns_hip_kv_page_bytes(8, 128, 64) == 8 * 64 * (64 + 64 + 4 + 4)
    assert L.fns_hip_kv_page_bytes(1, 256, 16) == 16 * (128 + 128 + 8 + 8)
    assert L.fns_hip_kv_page_bytes(8, 100, 64) == 0 and L.fns_hip_kv_page_bytes(8, 128, 24) == 0


def test_attn_overlap_workspace_and_limits():
    L, r = _lib.lib(), ctypes.byref
    assert _attn(out=BUF, q=BUF) == -2

    def need(c, b, x):
        size = ctypes.c_size_t()
        assert L.fns_hip_attn_workspace(r(c), r(b), r(x), r(size)) == 0
        return size.value

    # one token over a long context is split; a long prompt leaves a note a wave of every 128 rows; short ones need nothing
    long, prompt = batch(max_kv=100000, table_stride=2000), batch(n_tok=32768, max_q=32768, max_kv=32768, table_stride=512)
    assert need(cache(), batch(), att()) == 0
    assert need(cache(), prompt, att()) == 2 * (32768 * 2 // 128) * 4
    for b in (long, prompt):
        n = need(cache(), b, att())
        assert n > 0
        for ws, size in ((None, n), (BUF, n - 1), (BUF + 8, n), (BUF, 0)):
            assert _attn(b=b, out=3 * BUF, ws=ws, size=size) == -4
    # more row tiles than a grid has
    assert _attn(c=cache(n_head_kv=1), b=batch(n_tok=1 << 30, max_q=1 << 30), x=att(n_head=16, q_stride=1 << 14, out_stride=1 << 14),
                 out=3 * BUF) == -2
