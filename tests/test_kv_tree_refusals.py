"""Argument checks of the tree and eviction entry points, on the host before any launch; the scaled frequencies."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from flintnsteel_amd import _lib, ops
from test_attn_half_refusals import BAD_BATCHES, BAD_CACHES, BUF, P, app, att, batch, cache

r = ctypes.byref


def L():
    return _lib.lib()


def tree(**kw):
    return ops.KvTreeDesc(**{**dict(sees=BUF, words=1), **kw})


def evict(**kw):
    return ops.KvEvictDesc(**{**dict(budget=8, first=2, recent=3, weights=BUF, weights_out=BUF, to_table=None, to_stride=0,
                                     kept=BUF, new_len=2 * BUF, workspace=None, workspace_bytes=0), **kw})


def keep(**kw):
    return ops.KvKeepDesc(**{**dict(kept=BUF, n_kept=BUF, stride=4, weights=None, new_len=2 * BUF), **kw})


def _plan(b=None, parents=BUF, base=None, words=1, sees=BUF, pos=BUF):
    b = b or batch()
    return L().fns_hip_tree_plan(r(b), P(parents), P(base), words, P(sees), P(pos), None)


def _attn(c=None, b=None, x=None, t=None, q=BUF, out=2 * BUF, lse=BUF, ws=BUF, size=1 << 40):
    c, b, x, t = c or cache(), b or batch(), x or att(), t or tree()
    return L().fns_hip_attn_tree(r(c), r(b), r(x), r(t), P(q), P(out), P(lse), P(ws), size, None)


def _weigh(c=None, b=None, x=None, t=None, q=BUF, lse=BUF, w=BUF, ws=BUF, size=1 << 40):
    c, b, x, t = c or cache(), b or batch(), x or att(), t or tree()
    return L().fns_hip_kv_weigh(r(c), r(b), r(x), r(t), P(q), P(lse), None, P(w), P(ws), size, None)


def _evict(c=None, b=None, x=None):
    c, b, x = c or cache(), b or batch(), x or evict()
    return L().fns_hip_kv_evict(r(c), r(b), r(x), None)


def _keep(c=None, b=None, x=None):
    c, b, x = c or cache(), b or batch(), x or keep()
    return L().fns_hip_kv_keep(r(c), r(b), r(x), None)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches(kw):
    c = cache(**kw)
    x = app()
    assert _attn(c=c) == _weigh(c=c) == _evict(c=c) == _keep(c=c) == -2
    assert L().fns_hip_kv_append_at(r(c), r(batch()), r(x), P(BUF), 1.0, None) == -2


@pytest.mark.parametrize("kw", BAD_BATCHES)
def test_bad_batches(kw):
    if kw == dict(n_seq=40000):  # too many for two kv heads; a plan has none
        kw = dict(n_seq=70000)
    b = batch(**kw)
    assert _attn(b=b) == _weigh(b=b) == _evict(b=b) == _keep(b=b) == _plan(b=b) == -2


@pytest.mark.parametrize("kw,rc", [(dict(dtype=1), -1), (dict(n_head=5), -2), (dict(n_head=0), -2), (dict(window=-1), -2), (dict(q_stride=511), -2)])
def test_attention_arguments(kw, rc):
    assert _attn(x=att(**kw)) == rc and _weigh(x=att(**kw)) == rc
    size = ctypes.c_size_t()
    assert L().fns_hip_kv_weigh_workspace(r(cache()), r(batch()), r(att(**kw)), r(size)) == rc


@pytest.mark.parametrize("kw", [dict(words=0), dict(words=17), dict(sees=None)])
def test_trees(kw):
    assert _attn(t=tree(**kw)) == -2 and _weigh(t=tree(**kw)) == -2


@pytest.mark.parametrize("kw", [dict(parents=None), dict(sees=None), dict(words=0), dict(words=17), dict(b=batch(n_tok=200, max_q=65))])
def test_plan_arguments(kw):
    assert _plan(**kw) == -2
    assert b"tree_plan" in L().fns_hip_last_error()


@pytest.mark.parametrize("magnitude", [0.0, -1.0, float("inf"), float("nan")])
def test_magnitudes(magnitude):
    x = app(rope=1, rope_dim=64, inv_freq=BUF)
    assert L().fns_hip_kv_append_at(r(cache()), r(batch()), r(x), P(BUF), magnitude, None) == -2


@pytest.mark.parametrize("kw", [dict(budget=0), dict(budget=(1 << 30) + 1), dict(first=-1), dict(recent=-1), dict(first=6), dict(weights=None),
                                dict(weights_out=None), dict(kept=None), dict(new_len=None), dict(weights=BUF + 4, weights_out=BUF + 4),
                                dict(weights_out=2 * BUF), dict(new_len=BUF), dict(to_table=BUF, to_stride=4),
                                dict(to_table=2 * BUF), dict(to_table=2 * BUF, to_stride=-1)])
def test_evict_arguments(kw):
    assert _evict(x=evict(**kw)) == -2
    assert b"kv_evict" in L().fns_hip_last_error()


@pytest.mark.parametrize("kw", [dict(stride=0), dict(stride=1025), dict(kept=None), dict(n_kept=None), dict(new_len=None), dict(new_len=BUF)])
def test_keep_arguments(kw):
    assert _keep(x=keep(**kw)) == -2
    assert b"kv_keep" in L().fns_hip_last_error()


def test_null_arguments_overlap_and_workspaces():
    assert _attn(q=None) == _attn(out=None) == _attn(out=BUF) == -2
    assert _weigh(q=None) == _weigh(lse=None) == _weigh(w=None) == -2
    assert L().fns_hip_attn_tree(None, r(batch()), r(att()), None, P(BUF), P(2 * BUF), None, P(BUF), 0, None) == -2
    assert L().fns_hip_attn_tree(r(cache()), r(batch()), None, None, P(BUF), P(2 * BUF), None, P(BUF), 0, None) == -2
    assert L().fns_hip_kv_weigh(r(cache()), None, r(att()), None, P(BUF), P(BUF), None, P(BUF), P(BUF), 0, None) == -2
    assert L().fns_hip_kv_evict(r(cache()), r(batch()), None, None) == -2
    assert L().fns_hip_kv_keep(r(cache()), r(batch()), None, None) == -2
    assert L().fns_hip_kv_weigh_workspace(r(cache()), r(batch()), r(att()), None) == -2
    assert L().fns_hip_kv_weigh_workspace(r(cache()), r(batch()), None, None) == -2
    size = ctypes.c_size_t()
    assert L().fns_hip_kv_evict_workspace(r(cache()), r(batch()), None) == -2
    assert L().fns_hip_kv_evict_workspace(r(cache()), r(batch(table_stride=512)), r(size)) == 0 and size.value == 0
    wide = batch(table_stride=513)
    assert L().fns_hip_kv_evict_workspace(r(cache()), r(wide), r(size)) == 0 and size.value > 0
    for kw in (dict(), dict(workspace=BUF, workspace_bytes=size.value - 1), dict(workspace=BUF + 8, workspace_bytes=size.value)):
        assert _evict(b=wide, x=evict(**kw)) == -4
    b = batch(n_tok=1000, max_q=1000)
    assert L().fns_hip_kv_weigh_workspace(r(cache()), r(b), r(att()), r(size)) == 0 and size.value > 0
    for ws, n in ((None, size.value), (BUF, size.value - 1), (BUF + 8, size.value), (BUF, 0)):
        assert _weigh(b=b, ws=ws, size=n) == -4
    long = batch(max_kv=100000, table_stride=2000)
    assert L().fns_hip_attn_workspace(r(cache()), r(long), r(att()), r(size)) == 0 and size.value > 0
    assert _attn(b=long, ws=BUF, size=size.value - 1) == -4
    many = batch(n_tok=1 << 30, max_q=1 << 30)
    assert _weigh(c=cache(n_head_kv=1), b=many, x=att(n_head=16, q_stride=1 << 14), size=1 << 62) == -2


def test_empty_batches_are_noops():
    for kw in (dict(n_tok=0), dict(max_q=0), dict(n_seq=0, q_start=None, kv_len=None, page_table=None)):
        b = batch(**kw)
        assert _attn(b=b, ws=None, size=0) == _weigh(b=b, ws=None, size=0) == _plan(b=b) == 0
    b = batch(n_seq=0, q_start=None, kv_len=None, page_table=None)
    assert _evict(b=b) == _keep(b=b) == 0


@pytest.mark.parametrize("dim,base,factor,original,fast,slow", [(128, 500000.0, 16.0, 8192, 32.0, 1.0), (64, 10000.0, 4.0, 4096, 32.0, 1.0),
                                                                (2, 10000.0, 2.0, 100, 32.0, 1.0), (96, 1e6, 40.0, 32768, 16.0, 2.0),
                                                                (128, 10000.0, 1.0, 2048, 32.0, 1.0)])
def test_scaled_frequencies(dim, base, factor, original, fast, slow):
    out, m = (ctypes.c_float * (dim // 2))(), ctypes.c_float()
    assert L().fns_hip_rope_scaled(dim, base, factor, original, fast, slow, out, r(m)) == 0
    i = np.arange(dim // 2)
    f = base ** (-2.0 * i / dim)
    turns = original * f / (2 * np.pi)
    at = lambda t: dim * np.log(original / (t * 2 * np.pi)) / (2 * np.log(base))  # noqa: E731
    lo, hi = max(np.floor(at(fast)), 0), min(np.ceil(at(slow)), dim // 2 - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
    got = np.array(out, np.float64)
    assert np.allclose(got, f * (1 - ramp) + f / factor * ramp, rtol=2.0 ** -23, atol=0)
    assert abs(m.value - (0.1 * np.log(factor) + 1)) <= 2.0 ** -23
    # what the rule is for: fast pairs as they were, slow ones divided (a pair beside either border belongs to the ramp)
    assert np.allclose(got[(turns >= fast) & (i <= lo)], f[(turns >= fast) & (i <= lo)], rtol=2.0 ** -23)
    assert np.allclose(got[i >= max(hi, lo + 1)], (f / factor)[i >= max(hi, lo + 1)], rtol=2.0 ** -23)


@pytest.mark.parametrize("args", [(0, 1e4, 2.0, 100.0, 32.0, 1.0), (3, 1e4, 2.0, 100.0, 32.0, 1.0), (64, 1.0, 2.0, 100.0, 32.0, 1.0),
                                  (64, 1e4, 0.5, 100.0, 32.0, 1.0), (64, 1e4, 2.0, 0.0, 32.0, 1.0), (64, 1e4, 2.0, 100.0, 1.0, 1.0),
                                  (64, 1e4, 2.0, 100.0, 32.0, 0.0), (64, float("nan"), 2.0, 100.0, 32.0, 1.0),
                                  (64, 1e4, float("inf"), 100.0, 32.0, 1.0)])
def test_scaled_frequencies_refusals(args):
    out, m = (ctypes.c_float * 64)(), ctypes.c_float()
    assert L().fns_hip_rope_scaled(*args, out, r(m)) == -2
    assert L().fns_hip_rope_scaled(64, 1e4, 2.0, 100.0, 32.0, 1.0, None, r(m)) == -2


@pytest.mark.parametrize("dim,base,factor,original,fast,slow", [
    (128, 1e4, 4.0, 65536, 32.0, 1.0), (128, 1e4, 4.0, 131072, 32.0, 1.0), (64, 1e4, 16.0, 262144, 32.0, 1.0),  # no pair is slow
    (16, 100.0, 4.0, 500, 32.0, 1.0), (128, 1e4, 4.0, 1e12, 32.0, 1.0), (64, 1e4, 4.0, 1e9, 32.0, 1.0),
    (64, 1e4, 2.0, 6, 32.0, 1.0), (64, 1e4, 16.0, 1, 32.0, 1.0), (2, 1e4, 8.0, 2, 32.0, 1.0),                      # every pair is
    (2, 1e4, 2.0, 100, 32.0, 1.0), (64, 1e4, 8.0, 100, 32.0, 1.0), (128, 5e5, 16.0, 8192, 32.0, 1.0), (96, 1e6, 40.0, 32768, 16.0, 2.0)])
def test_scaled_frequencies_by_turns(dim, base, factor, original, fast, slow):
    """From the pairs' turns over the original positions: kept, divided, or strictly between and linear in the index."""
    out, m = (ctypes.c_float * (dim // 2))(), ctypes.c_float()
    assert L().fns_hip_rope_scaled(dim, base, factor, original, fast, slow, out, r(m)) == 0
    i = np.arange(dim // 2)
    f = base ** (-2.0 * i / dim)
    turns = original * f / (2 * np.pi)
    kept, cut = turns >= fast, turns <= slow
    if not kept.any() and not cut[0]:
        kept[0] = True  # then the ramp starts at the first pair
    part = np.array(out, np.float64) / f  # (f32: off by half a step, 2^-24, and f by less)
    assert np.all(np.abs(part[kept] - 1) <= 2.0 ** -23)
    assert np.all(np.abs(part[cut] * factor - 1) <= 2.0 ** -23)
    between = part[~kept & ~cut]
    assert np.all((between > 1 / factor + 2.0 ** -23) & (between < 1 - 2.0 ** -23))
    # from the last kept pair to the first divided one (indices go on behind the last pair, up to dim - 1), in equal steps
    first, last = kept.sum() - 1, int(cut.argmax()) if cut.any() else 0
    while not cut.any() and last < dim - 1 and original * base ** (-2.0 * last / dim) / (2 * np.pi) > slow:
        last += 1
    for j in np.flatnonzero(~kept & ~cut):
        assert abs(part[j] - (1 + (1 / factor - 1) * (j - first) / (last - first))) <= 2.0 ** -23


@pytest.mark.parametrize("args,part", [((128, 1e4, 4.0, 65536.0), 1 - 3 / 4 * 23 / 25),
                                       ((128, 1e4, 4.0, 131072.0), 1 - 3 / 4 * 18 / 25), ((64, 1e4, 16.0, 262144.0), 1 - 15 / 16 * 7 / 13)])
def test_scaled_frequencies_where_no_pair_is_slow(args, part):
    """The last pair's share by hand: the ramp ends at index 65, 70 and 37 and starts at 40, 45 and 24."""
    n = args[0] // 2
    out, m = (ctypes.c_float * n)(), ctypes.c_float()
    assert L().fns_hip_rope_scaled(*args, 32.0, 1.0, out, r(m)) == 0
    assert abs(out[n - 1] / args[1] ** (-2.0 * (n - 1) / args[0]) - part) <= 2.0 ** -23


@pytest.mark.parametrize("dim,tiles", [(256, 65535), (256, 40000), (256, 4000), (128, 65535), (64, 65535), (64, 4000)])
def test_steps_of_many_rows_fit_their_plan(dim, tiles):
    """kv_weigh counts the steps (16 rows, a block of keys) of a kv head in int32: row tiles times planned blocks stay below 2^31
    at the longest context. What a plan of `blocks` takes is read off the workspace: 4 (blocks + 1) bytes, up to 256's multiple."""
    def size(kv):
        n, b = ctypes.c_size_t(), batch(n_tok=16 * tiles, max_q=16 * tiles, max_kv=kv, table_stride=1 << 20)
        x = att(n_head=1, q_stride=dim)
        assert L().fns_hip_kv_weigh_workspace(r(cache(n_head_kv=1, head_dim=dim)), r(b), r(x), r(n)) == 0
        return n.value

    most = (size(2 ** 31 - 1) - size(1) + 256) // 4 - 1  # (images and partial sums are as many; one block's plan takes 256 bytes)
    assert most > 1000 and tiles * (most - 63) <= 2 ** 31 - 1


def test_eviction_states_are_aligned():
    """kv_evict's states of the kv heads lie beside each other in the 16-byte aligned workspace, before 8 bytes a chunk: of a kv
    head's bytes at room for 65536 and 131072 positions, twice the first less the second is a state."""
    def size(heads, room):
        n = ctypes.c_size_t()
        assert L().fns_hip_kv_evict_workspace(r(cache(n_head_kv=heads)), r(batch(table_stride=room // 64)), r(n)) == 0
        return n.value

    for heads in (1, 2, 3):
        state = 2 * size(heads, 65536) - size(heads, 131072)
        assert state % heads == 0 and state // heads % 16 == 0


@pytest.mark.parametrize("kw", [dict(first=1 << 32), dict(recent=(1 << 32) + 2), dict(first=-(1 << 32)), dict(budget=(1 << 32) + 5)])
def test_eviction_numbers_beyond_32_bits(kw):
    """Refused before they become others in the call's ints."""
    c = SimpleNamespace(desc=cache(), n_head_kv=2, page_size=64, pages=torch.empty(0, dtype=torch.uint8))
    b = SimpleNamespace(desc=batch(n_seq=0), kv_len=torch.zeros(0, dtype=torch.int32))
    w = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="budget"):
        ops.kv_evict(c, b, w, **{**dict(budget=8), **kw})


def test_eviction_workspace_of_the_wrapper_is_the_librarys():
    """ops asks the library only where it expects a workspace: the same tables."""
    n = ctypes.c_size_t()
    for page in (16, 64, 4096):
        c = cache(page_size=page)
        for pages in (1, 32768 // page, 32768 // page + 1, 5 * 32768 // page):
            d = batch(table_stride=pages)
            b = SimpleNamespace(desc=d, _for=lambda _, d=d: r(d))
            got = ops.kv_evict_workspace(SimpleNamespace(ref=r(c), page_size=page, pages=torch.empty(0)), b)
            assert L().fns_hip_kv_evict_workspace(r(c), r(d), r(n)) == 0
            assert (0 if got is None else got.numel()) == n.value
