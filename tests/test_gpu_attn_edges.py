"""Attention over the paged 4-bit cache where sizes of values, windows and divided contexts go to their ends, against the 64-bit
definitions of kv_data.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_data as kd
from flintnsteel_amd import ops
from test_gpu_attn_half import MANY_ROWS, Setup, _check_attn, _rand

pytestmark = pytest.mark.gpu


def _upload(s: Setup) -> None:
    s.cache.pages.copy_(torch.from_numpy(s.host.raw.copy()).view(s.cache.pages.shape))
    s.batch.page_table.copy_(torch.from_numpy(s.table))


# ---- windows ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 4, 2 ** 30, 3])
def test_windows_of_any_width_where_a_sequence_has_fewer_positions_than_new_tokens(window, many, dtype):
    """Tokens before position 0 see nothing, the others what the window leaves them."""
    s = Setup([20, 70], [20, 70], 16, 1, 64, seed=83, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else 70
    s.kv_lens = [5, 67]
    s.batch.kv_len.copy_(torch.tensor(s.kv_lens, dtype=torch.int32))
    _, out = _check_attn(s, 1, dtype, window=window)
    assert (out[:15] == 0).all() and (out[15:20] != 0).any(-1).all()
    assert (out[20:23] == 0).all() and (out[23:90] != 0).any(-1).all()


# ---- blocks of V of all sizes -----------------------------------------------------------------------------------------

def _v_scales(h: kd.Pages, head: int) -> np.ndarray:
    """View of V's scale bytes, [pages][positions][blocks]."""
    o = head * h.head_bytes + h.page * (h.dim + h.dim // 32)
    return h.raw[:, o: o + h.page * (h.dim // 32)].reshape(h.n_pages, h.page, h.dim // 32)


def _check_relative(s: Setup, group: int, dtype: str, window: int = 0) -> None:
    """As _check_attn, without its absolute part: 2^-145 is left, for sums of parts that f32 holds as subnormals."""
    q, qh = _rand(s.rng, (s.n_tok, s.heads_kv * group, s.dim), dtype)
    got = ops.attn(s.cache, s.batch, q, window=window)[: s.tok].double().cpu().numpy()
    ref, ax, vm = kd.attention(s.host, s.table, s.q_lens, s.kv_lens, qh[: s.tok], s.dim ** -0.5, window)
    far = np.abs(ref) >= 2.0 ** 128  # f32's infinity
    assert np.array_equal(got[far], np.copysign(np.inf, ref[far]))
    tol = kd.attn_tolerance(dtype, s.dim, max(s.kv_lens), ref, ax, vm) - 1e-37 + 2.0 ** -145
    bad = ~far & ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, rows {np.unique(np.nonzero(bad)[0])}"


FORMS = [(64, 32, 3, False), (128, 64, 20, False), (64, 16, 50, False), (256, 32, 12, False), (128, 16, 100, False),
         (128, 64, 140, True), (64, 32, 150, True), (256, 128, 70, True)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,q,many", FORMS)
@pytest.mark.parametrize("least", [104, 60, 20])
def test_rows_keep_what_they_see_beside_a_huge_block_that_they_do_not_see(least, dim, page, q, many, dtype):
    """Everything at 2^(least - 127) and a few blocks of the largest scales, which rows before them and windows behind them do
    not see."""
    s = Setup([q, 2], [q + 90, 200], page, 1, dim, seed=least + dim, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    v = _v_scales(s.host, 0)
    v[:] = s.rng.integers(least, least + 4, v.shape)
    for seq, pos, block, e in ((0, q + 89 - q // 2, 0, 254), (0, 40, 1, 253), (1, 199, dim // 32 - 1, 250)):
        v[s.table[seq, pos // page], pos % page, block] = e
    _upload(s)
    _check_relative(s, 2, dtype)
    _check_relative(s, 2, dtype, window=q // 3 + 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,q,many", FORMS)
@pytest.mark.parametrize("least,most", [(100, 250), (20, 200), (60, 175), (112, 213), (75, 111), (74, 110)])
def test_rows_keep_what_they_saw_before_a_tile_of_huge_blocks(least, most, dim, page, q, many, dtype):
    """All blocks of the last positions (from 65 tokens on a whole tile) far above all others; rows before them see the small
    ones only."""
    kv = (q + 70) // 64 * 64 + 384  # the last new token sits at the end of a tile; more tiles than waves
    s = Setup([q], [kv], page, 1, dim, seed=least + dim, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    v = _v_scales(s.host, 0)
    first = kv - min(q - 1, 64)
    for pos in range(kv):
        v[s.table[0, pos // page], pos % page] = least if pos < first else most
    _upload(s)
    _check_relative(s, 2, dtype)


@pytest.mark.parametrize("dim,page,q,many", FORMS)
@pytest.mark.parametrize("least,dtype", [(1, "f32"), (5, "f32"), (30, "f32"), (72, "f32"), (108, "f32"), (30, "bf16"), (72, "bf16")])
def test_small_values_keep_their_bits(least, dim, page, q, many, dtype):
    s = Setup([q], [q + 90], page, 1, dim, seed=least + dim, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    v = _v_scales(s.host, 0)
    v[:] = s.rng.integers(least, least + 4, v.shape)
    _upload(s)
    _check_relative(s, 2, dtype)


# ---- sizes of queries and keys ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,q,many", FORMS)
def test_powers_of_two_between_queries_and_keys(dim, page, q, many, dtype):
    """q 2^-n and K 2^n give the bits of q and K, as long as scale * log2(e) * q reaches 2^-100; below, a score is off by up to
    2^-125 sum |K| of log2 units."""
    s = Setup([q], [q + 90], page, 1, dim, seed=101 + dim, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    x, _ = _rand(s.rng, (s.n_tok, 2, dim), dtype)
    want = ops.attn(s.cache, s.batch, x)[: s.tok]
    k = s.host.raw[:, page * dim: page * dim + page * (dim // 32)]
    keep = k.copy()
    for n in (-100, 50, 95, 118):
        k[:] = keep.astype(int) + n
        _upload(s)
        small = x * 2.0 ** -n
        got = ops.attn(s.cache, s.batch, small)[: s.tok]
        if n < 100:
            assert torch.equal(got, want), n
            continue
        ref, ax, vm = kd.attention(s.host, s.table, s.q_lens, s.kv_lens, small.double().cpu().numpy()[: s.tok], dim ** -0.5)
        most = np.abs(s.host.get(np.repeat(np.arange(s.host.n_pages), page), np.tile(np.arange(page), s.host.n_pages), 0)[0]).sum(-1).max()
        tol = kd.attn_tolerance(dtype, dim, q + 90, ref, ax, vm)
        tol = tol + 2 * np.log(2) * 2.0 ** -125 * most * vm[..., None] * (1 if dtype == "f32" else 2 ** 10)
        assert (np.abs(got.double().cpu().numpy() - ref) <= tol).all()


@pytest.mark.parametrize("dim,page,q,many", FORMS + [(128, 64, 1, False)])
def test_sinks_and_queries_beyond_f32(dim, page, q, many):
    """Sinks of +infinity and NaN make their heads NaN, of -infinity are none; a row whose scale * q is beyond f32 is NaN; the
    other heads and rows keep their bits."""
    kv = q + 90 if q > 1 else 3000  # (divided)
    s = Setup([q], [kv], page, 1, dim, seed=103 + dim, pad=MANY_ROWS // 4 if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    x, _ = _rand(s.rng, (s.n_tok, 4, dim))
    inf, some = float("inf"), torch.tensor([0.5, -1.0, 2.0, 0.0], device="cuda")
    want, none = (ops.attn(s.cache, s.batch, x, sinks=t)[: s.tok] for t in (some, None))
    odd = some.clone()
    odd[0], odd[2], odd[3] = inf, -inf, float("nan")
    got = ops.attn(s.cache, s.batch, x, sinks=odd)[: s.tok]
    assert torch.isnan(got[:, [0, 3]]).all() and torch.equal(got[:, 1], want[:, 1]) and torch.equal(got[:, 2], none[:, 2])
    x[q // 2, 1, dim - 1] = 3e38
    got = ops.attn(s.cache, s.batch, x, scale=2.0)[: s.tok]
    assert torch.isnan(got[q // 2, 1]).all()
    x[q // 2, 1, dim - 1] = 0.0
    want = ops.attn(s.cache, s.batch, x, scale=2.0)[: s.tok]
    got[q // 2, 1] = want[q // 2, 1]
    assert torch.equal(got, want)


# ---- contexts divided among workgroups --------------------------------------------------------------------------------

def _splits(s: Setup, group: int, dtype: str) -> int:
    """From the size of the workspace: a row of f32 and two numbers a split, token and head."""
    H = s.heads_kv * group
    q = torch.empty(s.n_tok, H, s.dim, dtype=torch.float32 if dtype == "f32" else torch.bfloat16, device="cuda")
    return ops.attn_workspace(s.cache, s.batch, q).numel() // (s.n_tok * H * (4 * s.dim + 8))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,q_lens,kv_lens,window,sinks,least", [
    (16, [1], [5003], 0, False, 17),          # joined a workgroup a row, 20 splits with keys
    (64, [1], [16384], 0, True, 64),          # 64
    (32, [1], [9000], 3000, False, 17),       # a window's edge inside a split, and splits without keys
    (16, [4, 1, 0, 3], [900, 70, 5, 700], 0, True, 2),  # joined a wave a row, sequences of other lengths
    (128, [3, 5], [2500, 1900], 1000, False, 2),
    (32, [20], [3000], 0, False, 2),          # more than a tile of rows
    (16, [2], [4100], 77, True, 2),           # the window in one split
])
def test_divided_contexts(page, q_lens, kv_lens, window, sinks, least, dim, dtype):
    s = Setup(q_lens, kv_lens, page, 1 if max(kv_lens) > 9000 else 2, dim, seed=89 + dim, pad=1)
    assert _splits(s, 4, dtype) >= least
    _check_attn(s, 4, dtype, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("q,window", [(1, 0), (5, 0), (5, 2000), (40, 0)])
def test_divided_contexts_with_odd_places(q, window, dim, page, dtype):
    """Missing pages, a huge block of V and a tiny one in one split each; then a NaN in V and one in K."""
    s = Setup([q, 1], [4000, 2600], page, 1, dim, seed=97 + dim)
    assert _splits(s, 3, dtype) >= 4
    v = _v_scales(s.host, 0)
    for seq, pos, block, e in ((0, 3999 - q // 2, 0, 170), (0, 1000, 1, 60), (1, 2599, 1, 180), (1, 30, 0, 50)):
        v[s.table[seq, pos // page], pos % page, block] = e
    s.table[0, [3500 // page, 2222 // page]] = [-1, s.host.n_pages]
    _upload(s)
    _check_attn(s, 3, dtype, window)
    v[s.table[0, 3100 // page], 3100 % page, 0] = 255
    page_of = s.table[1, 77 // page]
    s.host.raw[page_of, page * dim + 77 % page * (dim // 32)] = 255
    _upload(s)
    _check_attn(s, 3, dtype, window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("q,kv", [(1, 300), (1, 5121), (3, 4097), (20, 3009)])  # (the last key in a split of its own)
def test_values_of_v_beyond_f32_with_small_weights(q, kv, dim, page, dtype):
    """Codes of the largest scales stand for up to 6 * 2^127; a weight of one in a thousand makes them ordinary f32 numbers, divided
    or not."""
    s = Setup([q], [kv], page, 1, dim, seed=107 + dim)
    v = _v_scales(s.host, 0)
    for pos in (kv // 2, kv // 2 + 1, kv - 1):
        v[s.table[0, pos // page], pos % page] = 254
    _upload(s)
    _check_attn(s, 3, dtype, std=0.1)
