"""Trees of drafted tokens and caches of a bounded length on the device: bits and positions from parents, append at positions of
their own, attention with denominators, attention weights, eviction, accepted paths, against the 64-bit definitions of
kv_data.py and tree_data.py; and a run of them together, captured."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import kv_data as kd
import tree_data as td
from flintnsteel_amd import ops
from flintnsteel_amd._lib import FnsError
from test_gpu_attn_half import MANY_ROWS, Setup, _rand, _rounded_ok

pytestmark = pytest.mark.gpu


def dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def trees_of(s: Setup, seed: int = 0, pads: bool = True):
    rng = np.random.default_rng(seed)
    return [td.random_parents(rng, n, n // 5 if pads and i % 2 else 0) for i, n in enumerate(s.q_lens)]


def kv_tree(s: Setup, rows, words=None):
    """The batch's KvTree of token rows [sequence][token] -> seen; rows of padding tokens see everything (they must not count)."""
    words = words or max(1, (max(s.q_lens + [1]) + 63) // 64)
    bits = td.words_of([row for seq in rows for row in seq], words)
    bits = np.concatenate([bits, np.full((s.n_tok - s.tok, words), -1, np.int64)])
    return ops.KvTree(torch.from_numpy(bits).cuda())


# ---- bits and positions ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("q_lens,words", [([1], 1), ([5, 0, 64, 3], 1), ([65, 2], 2), ([200, 256, 1], 4), ([1000], 16), ([30, 7], 3)])
def test_tree_plan(q_lens, words):
    s = Setup(q_lens, [n + 50 * (i + 1) for i, n in enumerate(q_lens)], 16, 1, 64, pad=2)
    parents = trees_of(s, seed=words)
    if len(parents[0]) > 60:  # a line, and a token whose parent is itself or behind it: no token, nor what follows from it
        parents[0] = list(range(-1, len(parents[0]) - 1))
        parents[0][40] = 40
    if len(parents[-1]) > 6:
        parents[-1][5] = 6
        parents[-1][3] = -2 ** 31
    flat = [p for seq in parents for p in seq]
    rows = [td.seen_by(p) for p in parents]
    want = td.words_of([row for seq in rows for row in seq], words)
    for base in (None, [7, -3, 2 ** 30, 0][: len(q_lens)]):
        t = ops.tree_plan(s.batch, dev(flat + [-1, 0]), base=None if base is None else dev(base), words=words)
        assert np.array_equal(t.sees.cpu().numpy()[: s.tok], want)
        at = base or [kv - n for n, kv in zip(s.q_lens, s.kv_lens)]
        pos = [at[i] + max(len(row) - 1, 0) for i, seq in enumerate(rows) for row in seq]
        assert t.pos.cpu().tolist()[: s.tok] == pos


# ---- append ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rope,rope_dim,magnitude", [(1, 128, 1.0), (2, 64, 1.3), (1, 32, 0.7), (0, 0, 1.5)])
def test_append_at_positions(rope, rope_dim, magnitude, dtype):
    s = Setup([5, 0, 17, 33], [37, 12, 17, 80], 16, 2, 128, seed=3 + rope, pad=2)
    freq = ops.rope_freqs(rope_dim, 10000.0) if rope else None
    pos = s.rng.integers(-5, 2 ** 20, s.n_tok)
    pos[:4] = [0, 2 ** 31 - 1, -2 ** 31, 1]
    k, kh = _rand(s.rng, (s.n_tok, 2, 128), dtype, 2.0)
    v, vh = _rand(s.rng, (s.n_tok, 2, 128), dtype)
    q, qh = _rand(s.rng, (s.n_tok, 6, 128), dtype)
    m = float(np.float32(magnitude))
    qo = ops.kv_append(s.cache, s.batch, k, v, q=q, rope=rope, inv_freq=freq, pos=dev(pos), magnitude=magnitude)

    def turn(x):
        y = kd.rotate(x[: s.tok], pos[: s.tok], rope, None if freq is None else freq.cpu().numpy())
        if rope:
            y[..., :rope_dim] *= m
        return y

    s.put(turn(kh), vh[: s.tok])
    assert s.same_bytes()
    ref = turn(qh)
    # An angle is a product of three numbers in 64 bits (position, frequency, 1 / 2 pi), each operation and the constant off by
    # 2^-53 of it at most; it turns a pair, whose sum is at most twice the row's largest value. (kd.rotate's own sum of two
    # products may cancel: 1e-11.)
    step = kd.F32_STEP if dtype == "f32" else kd.BF16_STEP * (1 + 2.0 ** -15)
    angle = 3 * 2.0 ** -53 * np.abs(pos[: s.tok].astype(np.float64))[:, None, None]  # (the largest frequency is 1)
    tol = np.abs(ref) * step + (1 + step) * angle * 2 * np.abs(qh[: s.tok]).max(-1, keepdims=True) * m + 1e-11
    assert (np.abs(qo[: s.tok].double().cpu().numpy() - ref) <= tol).all()


def test_append_at_its_own_places_is_append():
    s = Setup([20, 3], [55, 9], 32, 2, 64, seed=5)
    t = Setup([20, 3], [55, 9], 32, 2, 64, seed=5)
    k, v, q = (_rand(s.rng, (s.tok, n, 64))[0] for n in (2, 2, 4))
    freq, one = ops.rope_scaled(64, 10000.0, 1.0, 4096)
    assert one == 1.0
    a = ops.kv_append(s.cache, s.batch, k, v, q=q, rope=ops.ROPE_PAIRS, inv_freq=freq)
    b = ops.kv_append(t.cache, t.batch, k, v, q=q, rope=ops.ROPE_PAIRS, inv_freq=freq, pos=dev(s.positions()))
    assert torch.equal(a, b) and torch.equal(s.cache.pages, t.cache.pages)


# ---- attention ------------------------------------------------------------------------------------------------------

def _check_tree(s: Setup, group: int, dtype: str, window: int = 0, sinks: bool = False, std: float = 1.0, rows="random", words=None, scale=None):
    H = s.heads_kv * group
    q, qh = _rand(s.rng, (s.n_tok, H, s.dim), dtype, std)
    sk, skh = _rand(s.rng, (H,)) if sinks else (None, None)
    out = torch.full_like(q, 7.0)
    lse = torch.full((s.n_tok, H), 7.0, device="cuda")
    if rows == "random":
        rows = [td.seen_by(p) for p in trees_of(s, seed=s.dim + group)]
    tree = None if rows is None else kv_tree(s, rows, words)
    scale = s.dim ** -0.5 if scale is None else scale
    ops.attn(s.cache, s.batch, q, window=window, sinks=sk, out=out, scale=scale, tree=tree, lse=lse)
    ref, ref_lse, ax, vm = td.attention(s.host, s.table, s.q_lens, s.kv_lens, qh[: s.tok], scale, window, skh, rows)
    assert (out[s.tok:] == 7.0).all() and (lse[s.tok:] == 7.0).all()
    got, got_lse = out.double().cpu().numpy()[: s.tok], lse.double().cpu().numpy()[: s.tok]
    n = max(s.kv_lens + [1])
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(np.isnan(got_lse), np.isnan(ref_lse))
    tol = kd.attn_tolerance(dtype, s.dim, n, ref, ax, vm)
    if dtype == "bf16":  # contexts that are divided are weighted by sums of p before it is cut to 11 bits
        tol = tol + 2 * 2.0 ** -11 * vm[..., None]
    fine = ~np.isnan(ref)
    bad = fine & ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"out: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - ref) / tol):.3g} of the tolerance"
    low = np.isneginf(ref_lse)
    assert np.array_equal(low, np.isneginf(got_lse)) and (got[low] == 0).all()
    tol = td.lse_tolerance(dtype, s.dim, n, ref_lse, ax)
    fine = ~np.isnan(ref_lse) & ~low
    bad = np.zeros(fine.shape, bool)
    bad[fine] = ~(np.abs(got_lse[fine] - ref_lse[fine]) <= tol[fine])
    assert not bad.any(), f"lse: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got_lse - ref_lse)[fine] / tol[fine]):.3g} of the tolerance"
    return q, out, lse, sk


SHAPES = [
    (128, 64, 2, 4, [7], [7], 0, False),
    (128, 64, 1, 4, [26], [726], 0, False),
    (64, 32, 2, 8, [63, 0, 17, 1], [200, 30, 64, 5], 0, True),
    (128, 16, 2, 1, [64, 65], [64 + 63, 300], 0, False),
    (256, 32, 1, 3, [40, 90], [90, 157], 30, False),
    (64, 16, 1, 2, [130, 150], [150, 1000], 100, True),
    (128, 128, 1, 5, [33], [1500], 9, False),
    (64, 64, 1, 17, [20, 5], [83, 5], 1, True),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,heads_kv,group,q_lens,kv_lens,window,sinks", SHAPES)
def test_attn_tree(dim, page, heads_kv, group, q_lens, kv_lens, window, sinks, dtype):
    _check_tree(Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim + group, pad=1), group, dtype, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,heads_kv,group,q_lens,kv_lens,window,sinks", SHAPES[1:])
def test_attn_tree_in_a_prompts_workgroups(dim, page, heads_kv, group, q_lens, kv_lens, window, sinks, dtype):
    s = Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim + group, pad=MANY_ROWS // group)
    s.batch.desc.max_q = s.n_tok
    _check_tree(s, group, dtype, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,q,kv,window", [(128, 64, 6, 9000, 0), (64, 16, 30, 6000, 5000), (256, 128, 3, 7001, 0), (128, 32, 1, 12000, 0)])
def test_attn_tree_over_divided_contexts(dim, page, q, kv, window, dtype):
    s = Setup([q], [kv], page, 1, dim, seed=q)
    x = _check_tree(s, 4, dtype, window, True)[0]
    assert ops.attn_workspace(s.cache, s.batch, x).numel() > 0


def test_attn_tree_any_bits():
    """Masks that are no tree: rows without bits, without themselves, of all new tokens, behind a sequence's tokens, in words
    that are not needed."""
    s = Setup([70, 3], [333, 3], 16, 2, 64, seed=77)
    rng = np.random.default_rng(4)
    rows = [[sorted(rng.choice(n, rng.integers(0, n + 1), replace=False).tolist()) for _ in range(n)] for n in s.q_lens]
    rows[0][0], rows[0][1], rows[0][69], rows[1][2] = list(range(70)), [], [3], []
    for window in (0, 20, 200):
        _check_tree(s, 3, "f32", window, window == 20, rows=rows, words=5)
    q = _rand(s.rng, (s.n_tok, 6, 64))[0]
    t = kv_tree(s, rows, 5)
    more = t.sees.clone()
    more[:70, 1] |= -(1 << 6)   # tokens 70.. of the first sequence
    more[:70, 2:] = -1
    more[70:, 0] |= -(1 << 3)
    more[70:, 1:] = -1
    for window in (0, 20):
        a, b = torch.zeros(2, s.n_tok, 6, device="cuda")
        assert torch.equal(ops.attn(s.cache, s.batch, q, window=window, tree=t, lse=a),
                           ops.attn(s.cache, s.batch, q, window=window, tree=ops.KvTree(more), lse=b))
        assert torch.equal(a, b)


def test_attn_tree_sees_fewer_new_tokens_than_there_are_positions_for():
    """kv_len below the new tokens: those before position 0 are nobody's key."""
    s = Setup([10, 4], [6, 0], 16, 1, 64, seed=9)
    _check_tree(s, 2, "f32", rows=[td.seen_by(list(range(-1, 9))), td.seen_by([-1, 0, 0, 1])])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q,kv,many", [(1, 500, False), (9, 300, False), (5, 9000, False), (80, 200, True)])
def test_denominators_of_plain_attention(q, kv, many, dtype):
    """Without a tree: attn's own output, and its denominators, causal and with a window."""
    s = Setup([q, 2], [kv, 77], 32, 2, 64, seed=q, pad=MANY_ROWS // 4 if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    for window, sinks in ((0, False), (40, True)):
        x, out, _, sk = _check_tree(s, 4, dtype, window, sinks, rows=None)
        plain = torch.full_like(out, 7.0)
        ops.attn(s.cache, s.batch, x, window=window, sinks=sk, out=plain)
        if dtype == "f32":  # (bf16 queries enter with more digits than attn takes)
            assert torch.equal(plain, out)


@pytest.mark.parametrize("many", [False, True])
def test_attn_tree_odd_places(many):
    """NaN blocks of K and V that some rows see and others do not, missing pages, NaN queries, huge scores and V blocks far
    apart (which take the second walk)."""
    q = 40
    s = Setup([q, 2], [300, 64], 16, 1, 64, seed=61, pad=MANY_ROWS // 4 if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    h = s.host
    s.table[0, 3], s.table[0, 5] = -1, h.n_pages
    for pos, off, e in ((300 - 7, 0, 255), (300 - 12, 32, 255), (20, 32, 210), (300 - 2, 32, 200)):  # K, V, V, V scales
        h.raw[s.table[0, pos // 16], 16 * 64 + off + pos % 16 * 2] = e
    s.cache.pages.copy_(torch.from_numpy(h.raw.copy()).view(s.cache.pages.shape))
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    _check_tree(s, 4, "f32", std=10.0)
    _check_tree(s, 4, "bf16", window=100, std=10.0)
    x = _rand(s.rng, (s.n_tok, 4, 64))[0]
    rows = [td.seen_by(p) for p in trees_of(s, 1)]
    t, lse = kv_tree(s, rows), torch.zeros(s.n_tok, 4, device="cuda")
    good, good_lse = ops.attn(s.cache, s.batch, x, tree=t, lse=lse).clone(), lse.clone()
    x[3, 1, 5] = float("nan")
    got = ops.attn(s.cache, s.batch, x, tree=t, lse=lse)
    assert torch.isnan(got[3, 1]).all() and torch.isnan(lse[3, 1])
    got[3, 1], lse[3, 1] = good[3, 1], good_lse[3, 1]
    tok = slice(0, s.tok)
    assert torch.equal(got[tok].nan_to_num(9), good[tok].nan_to_num(9)) and torch.equal(lse[tok].nan_to_num(9), good_lse[tok].nan_to_num(9))


# ---- attention weights ----------------------------------------------------------------------------------------------

def _check_weigh(s: Setup, group: int, dtype: str, window: int = 0, rows=None, past=True, lse=None, q=None, scale=None, in_place=False):
    H = s.heads_kv * group
    q, qh = _rand(s.rng, (s.n_tok, H, s.dim), dtype) if q is None else (q, q.double().cpu().numpy())
    scale = s.dim ** -0.5 if scale is None else scale
    if lse is None:
        lse = td.attention(s.host, s.table, s.q_lens, s.kv_lens, qh[: s.tok], scale, window, None, rows)[1]
        lse = torch.from_numpy(np.concatenate([lse, np.zeros((s.n_tok - s.tok, H))])).float().cuda()
    shape = (s.host.n_pages, s.heads_kv, s.page)
    before = torch.rand(shape, device="cuda") if past else None
    out = before.clone() if in_place else torch.full(shape, 5.0, device="cuda")
    tree = None if rows is None else kv_tree(s, rows)
    ref, tol = td.weigh(s.host, s.table, s.q_lens, s.kv_lens, qh[: s.tok], lse.double().cpu().numpy(),
                        None if before is None else before.double().cpu().numpy(), scale, window, rows, keep=out.double().cpu().numpy())
    ops.kv_weigh(s.cache, s.batch, q, lse, out if in_place else before, scale=scale, window=window, tree=tree, out=out)
    got = out.double().cpu().numpy()
    bad = ~(np.abs(got - ref) <= tol)  # (exactly what was there, where nothing is due)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - ref) / np.maximum(tol, 1e-300)):.3g} of the tolerance"
    return q, lse, out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,heads_kv,group,q_lens,kv_lens,window", [
    (128, 64, 2, 4, [1], [1], 0),
    (128, 64, 2, 4, [1, 1, 0, 1], [700, 3, 50, 257], 0),
    (64, 16, 1, 3, [1, 1], [500, 65], 70),
    (256, 32, 2, 5, [1, 7], [129, 333], 0),
    (128, 16, 1, 4, [33, 90, 1], [200, 90, 64], 0),
    (64, 128, 2, 2, [130], [300], 40),
    (128, 32, 1, 17, [20], [400], 1),
    (64, 64, 1, 1, [257], [257], 0),
    (256, 64, 1, 2, [130, 300], [700, 300], 0),
    (256, 16, 2, 1, [150], [400], 90),
])
def test_weigh(dim, page, heads_kv, group, q_lens, kv_lens, window, dtype):
    s = Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim + group, pad=2)
    _check_weigh(s, group, dtype, window)
    _check_weigh(s, group, dtype, window, past=False)
    _check_weigh(s, group, dtype, window, in_place=True)


@pytest.mark.parametrize("longest", [None, 1 << 21])  # (work is divided by it: 65 to 256 rows in one launch, or by their images)
@pytest.mark.parametrize("dim,page,group,q_lens,kv_lens,window", [
    (128, 64, 4, [26, 0, 3], [200, 9, 3], 0), (64, 16, 2, [130, 70], [150, 400], 100), (256, 32, 1, [64], [127], 9),
    (128, 128, 4, [60, 20, 1], [1500, 20, 777], 0), (256, 64, 2, [60, 33], [60, 1100], 0), (64, 32, 8, [32, 31, 5], [1030, 513, 300], 200),
    (128, 16, 1, [256, 65], [700, 65], 0), (256, 16, 1, [128, 81], [128, 600], 60), (128, 64, 3, [170, 90], [300, 1400], 0)])
def test_weigh_of_a_tree(dim, page, group, q_lens, kv_lens, window, longest):
    s = Setup(q_lens, kv_lens, page, 2, dim, seed=dim, pad=1)
    if longest:
        s.batch.desc.max_kv = longest
    rows = [td.seen_by(p) for p in trees_of(s, seed=group)]
    q, lse, out = _check_weigh(s, group, "f32", window, rows)
    # a rejected token's rows are left out by their lse
    lse[1], lse[s.tok - 1] = float("inf"), float("nan")
    _check_weigh(s, group, "f32", window, rows, lse=lse, q=q)


def test_weigh_of_many_heads():
    """More heads than workgroups that run at once: each takes several steps of keys."""
    n = 70
    s = Setup([10 + i % 3 for i in range(n)], [1300 - 17 * i for i in range(n)], 64, 2, 64, seed=9)
    _check_weigh(s, 8, "f32")
    _check_weigh(s, 8, "bf16", in_place=True)


@pytest.mark.parametrize("new,longest", [(60, 10), (60, 1 << 21), (150, 10), (150, 2000)])
def test_weigh_odd_places(new, longest):
    """NaN blocks, missing pages, queries that are no numbers, lengths beyond the batch's longest and a prompt's many rows."""
    s = Setup([new, 1], [300, 2000], 16, 2, 64, seed=61)
    s.batch.desc.max_kv = longest
    h = s.host
    s.table[0, 3], s.table[0, 5] = -1, h.n_pages
    for pos, off in ((300 - 7, 0), (300 - 12, 32), (20, 0)):
        h.raw[s.table[0, pos // 16], 16 * 64 + off + pos % 16 * 2] = 255
    s.cache.pages.copy_(torch.from_numpy(h.raw.copy()).view(s.cache.pages.shape))
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    q = _rand(s.rng, (s.n_tok, 4, 64))[0]
    q[4, 2, 3], q[7, 0, 63] = float("nan"), float("inf")
    lse = torch.rand(s.n_tok, 4, device="cuda") + 6  # (not what attention gives, which is NaN for most of them)
    _check_weigh(s, 2, "f32", q=q, lse=lse)
    _check_weigh(s, 2, "f32", window=33, q=q, lse=lse, scale=-0.2)


def test_weights_of_a_row_add_up():
    """From the operators' own denominators: every row gives one in all."""
    s = Setup([50, 1, 3], [400, 3000, 3], 64, 2, 128, seed=8)
    q = _rand(s.rng, (s.n_tok, 8, 128))[0]
    lse = torch.empty(s.n_tok, 8, device="cuda")
    ops.attn(s.cache, s.batch, q, lse=lse)
    w = ops.kv_weigh(s.cache, s.batch, q, lse, None)
    for i, n in enumerate(s.q_lens):
        got = w[dev(s.lists[i]).long()].double().sum((0, 2))
        # 4 heads a kv head; a row's scores are off by 1e-5 at most at this size of values
        assert torch.allclose(got, torch.full_like(got, 4.0 * n), rtol=3e-5, atol=0)


# ---- eviction -------------------------------------------------------------------------------------------------------

def _check_evict(kv_lens, page, heads_kv, dim, budget, first, recent, to=False, spoil=None, odd=False, seed=0):
    s = Setup([1] * len(kv_lens), kv_lens, page, heads_kv, dim, seed=seed, n_extra=3 + sum((min(n, budget) + page - 1) // page for n in kv_lens))
    rng = s.rng
    w = np.exp(rng.standard_normal((s.host.n_pages, heads_kv, page)) * 2).astype(np.float32)
    w = np.where(rng.random(w.shape) < 0.4, np.round(w * 4) / 4, w).astype(np.float32)  # equal ones, zeros
    if odd:
        for v in (np.nan, np.inf, -np.inf, -0.0, -1.5, 1e-42, -np.nan):
            w[rng.random(w.shape) < 0.03] = v
    if spoil:
        spoil(s)
        s.batch.page_table.copy_(torch.from_numpy(s.table))
    free = [p for p in range(s.host.n_pages) if p not in {q for l in s.lists for q in l}]
    table, dst = s.table, s.table
    if to:
        dst = np.full((len(kv_lens), max([(min(n, budget) + page - 1) // page for n in kv_lens] + [1])), -1, np.int64)
        for i, n in enumerate(kv_lens):
            for j in range((min(n, budget) + page - 1) // page):
                dst[i, j] = free.pop()
    wd = torch.from_numpy(w).cuda()
    wo = torch.full_like(wd, 3.0) if to else wd
    kept, new_len = ops.kv_evict(s.cache, s.batch, wd, budget, first, recent, to_table=dev(dst) if to else None, weights_out=wo if to else None)
    got = s.cache.pages.cpu().numpy().reshape(s.host.raw.shape)
    moves, sure = [], np.zeros(s.host.raw.shape, bool)
    want_w, sure_w = (np.full_like(w, 3.0), np.ones(w.shape, bool)) if to else (w.copy(), np.ones(w.shape, bool))
    sure[:] = True
    kept, new_len = kept.cpu().numpy(), new_len.cpu().numpy()
    for i, n in enumerate(kv_lens):
        n = min(n, table.shape[1] * page)
        j = np.arange(n)
        pg = table[i, j // page]
        there = (pg >= 0) & (pg < s.host.n_pages)
        for h in range(heads_kv):
            keep = td.evicted(np.where(there, w[np.where(there, pg, 0), h, j % page], 0), there, budget, first, recent)
            assert kept[i, h, : len(keep)].tolist() == keep and (kept[i, h, len(keep):] == -1).all()
            assert new_len[i] == len(keep)
            for r, p in enumerate(keep):
                a, b = (table[i, p // page], p % page), (dst[i, r // page], r % page)
                if 0 <= b[0] < s.host.n_pages:
                    moves.append((a, b, h))
                    want_w[b[0], h, b[1]] = w[a[0], h, a[1]]
            if not to:  # what follows is anything
                for p in range(len(keep), n):
                    if there[p]:
                        sure[pg[p], td.slot_bytes(s.host, pg[p], p % page, h)] = False
                        sure_w[pg[p], h, p % page] = False
    want = td.move(s.host, s.host.raw, moves)
    assert np.array_equal(got[sure], want[sure])
    assert np.array_equal(wo.cpu().numpy()[sure_w].view(np.int32), want_w[sure_w].view(np.int32))
    if to:
        assert np.array_equal(wd.cpu().numpy().view(np.int32), w.view(np.int32))


EVICT = [
    ([100], 16, 1, 64, 40, 4, 10),
    ([1, 0, 17, 64], 16, 2, 128, 16, 1, 3),
    ([300, 5], 64, 3, 128, 299, 0, 0),
    ([200], 32, 1, 256, 1, 0, 0),
    ([200], 32, 1, 256, 1, 0, 1),
    ([500, 1000], 128, 2, 64, 2000, 7, 100),
    ([90], 16, 1, 64, 30, 10, 20),
    ([5000, 4097, 4096], 64, 1, 64, 2500, 3, 100),
    ([9000], 4096, 1, 64, 8999, 0, 5),
    ([3500, 100], 16, 2, 128, 1023, 4, 64),
    ([4700, 1025], 64, 2, 128, 4300, 4, 64),
    ([2600, 1500], 32, 2, 256, 2300, 1, 50),
]


@pytest.mark.parametrize("to", [False, True])
@pytest.mark.parametrize("kv_lens,page,heads_kv,dim,budget,first,recent", EVICT)
def test_evict(kv_lens, page, heads_kv, dim, budget, first, recent, to):
    _check_evict(kv_lens, page, heads_kv, dim, budget, first, recent, to, seed=budget)


@pytest.mark.parametrize("to", [False, True])
def test_evict_odd_weights_and_missing_pages(to):
    _check_evict([700, 20], 16, 2, 64, 300, 5, 20, to, odd=True, seed=1)

    def holes(s):
        s.table[0, 2], s.table[0, 9], s.table[1, :] = -1, s.host.n_pages, -5

    _check_evict([400, 30], 16, 1, 64, 100, 40, 30, to, odd=True, spoil=holes, seed=2)
    _check_evict([400, 30], 16, 1, 64, 390, 0, 0, to, spoil=holes, seed=3)


@pytest.mark.parametrize("value", [0.0, 1.0, float("nan"), float("-inf"), float("inf")])
def test_evict_equal_weights_keeps_the_first(value):
    s = Setup([1], [5000], 16, 1, 64)
    w = torch.full((s.host.n_pages, 1, 16), value, device="cuda")
    kept, _ = ops.kv_evict(s.cache, s.batch, w, 3000, first=2, recent=500)
    assert kept[0, 0].tolist() == [*range(2500), *range(4500, 5000)]


@pytest.mark.parametrize("lens,page,heads,budget,first,recent", [
    ([70001], 64, 1, 33333, 4, 1000), ([40000, 5, 0, 32768, 16384], 128, 2, 16000, 0, 0), ([33000], 16, 3, 32999, 1, 1), ([50000, 49152], 256, 1, 1, 0, 0),
    ([36000], 64, 1, 70000, 5, 60)])
@pytest.mark.parametrize("equal", [False, True])
def test_evict_long_sequences(lens, page, heads, budget, first, recent, equal):
    """Selection in chunks: weights of all magnitudes, or few different ones; the lists twice the same."""
    s = Setup([1] * len(lens), lens, page, heads, 64, seed=4)
    w = torch.exp(torch.randn(s.host.n_pages, heads, page, device="cuda") * 8)
    if equal:
        w = torch.randint(0, 3, w.shape, device="cuda").float()
    assert ops.kv_evict_workspace(s.cache, s.batch) is not None
    pages, w0 = s.cache.pages.clone(), w.clone()
    kept, new_len = ops.kv_evict(s.cache, s.batch, w, budget, first=first, recent=recent)
    for i, n in enumerate(lens):
        assert new_len[i].item() == min(n, budget)
        for h in range(heads if n else 0):
            flat = w0[dev(s.lists[i]).long(), h].flatten()[:n].cpu().double()
            flat[: min(first, n)] = float("inf")
            flat[max(0, n - recent):] = float("inf")
            want = torch.sort(flat, descending=True, stable=True).indices[:budget].sort().values
            got = kept[i, h].cpu().long()
            assert torch.equal(got[: len(want)], want) and (got[len(want):] == -1).all()
            pg = dev(s.lists[i]).long()
            assert torch.equal(w[pg, h].flatten()[: len(want)].cpu(), w0[pg, h].flatten()[:n].cpu()[want])
    s.cache.pages.copy_(pages)
    again, _ = ops.kv_evict(s.cache, s.batch, w0, budget, first=first, recent=recent)
    assert torch.equal(kept, again)


@pytest.mark.parametrize("budget,first,recent", [(100, 40, 30), (390, 0, 0), (1, 0, 0), (5000, 3, 2)])
def test_evict_in_chunks_picks_the_same(budget, first, recent):
    """A table with room for more than is there: the same choice as without, of weights of all kinds and with pages missing."""
    s = Setup([1, 1, 1], [400, 30, 0], 16, 2, 64, seed=12)
    s.table[0, 2], s.table[0, 9], s.table[1, 1] = -1, s.host.n_pages, -5
    w = np.round(np.exp(s.rng.standard_normal((s.host.n_pages, 2, 16))) * 4).astype(np.float32)
    for v in (np.nan, np.inf, -np.inf, -0.0, -1.5, 1e-42, -np.nan):
        w[s.rng.random(w.shape) < 0.03] = v
    got = []
    for columns in (s.table.shape[1], 2049):
        table = np.full((3, columns), -1, np.int32)
        table[:, : s.table.shape[1]] = s.table
        batch = ops.KvBatch(s.batch.q_start, s.batch.kv_len, dev(table), 3, 1, 400)
        assert (ops.kv_evict_workspace(s.cache, batch) is None) == (columns < 2049)
        s.cache.pages.copy_(torch.from_numpy(s.host.raw.copy()).view(s.cache.pages.shape))
        wd = torch.from_numpy(w.copy()).cuda()
        got.append([*ops.kv_evict(s.cache, batch, wd, budget, first=first, recent=recent), wd.view(torch.int32), s.cache.pages.clone()])
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---- accepted paths -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,page,heads_kv", [(64, 16, 1), (128, 64, 3), (256, 32, 2)])
def test_keep(dim, page, heads_kv):
    q_lens, kv_lens = [9, 0, 40, 3, 5], [30, 12, 100, 3, 5]
    s = Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim)
    lists = [[0, 2, 5, 8], [1, 2], [39, 3, 3, 0, 17, -1, 40, 38], [0, 1, 2], [4]]
    n_kept = [4, 2, 8, 9, 0]
    stride = 10
    kept = np.full((5, stride), 2 ** 31 - 1, np.int64)
    for i, l in enumerate(lists):
        kept[i, : len(l)] = l
    w = np.random.default_rng(1).random((s.host.n_pages, heads_kv, page)).astype(np.float32)
    wd = torch.from_numpy(w.copy()).cuda()
    new_len = ops.kv_keep(s.cache, s.batch, dev(kept), dev(n_kept), weights=wd)
    moves = []
    for i, l in enumerate(lists):
        f = kv_lens[i] - q_lens[i]
        for r, x in enumerate(l[: n_kept[i]]):
            if q_lens[i] and 0 <= x < q_lens[i]:
                a, b = f + x, f + r
                for h in range(heads_kv):
                    moves.append(((s.table[i, a // page], a % page), (s.table[i, b // page], b % page), h))
    assert np.array_equal(s.cache.pages.cpu().numpy().reshape(s.host.raw.shape), td.move(s.host, s.host.raw, moves))
    for a, b, h in moves:
        assert wd[b[0], h, b[1]].item() == w[a[0], h, a[1]]
    assert int((wd.cpu().numpy() != w).sum()) <= len(moves)
    # (never more than the new tokens)
    assert new_len.tolist() == [25, 12, 68, 3, 0]


def test_keep_outside_the_cache():
    """Missing pages on either side, lengths below the new tokens: what has no place is not moved."""
    s = Setup([20, 6], [40, 3], 16, 1, 64, seed=2)
    s.table[0, 1] = -1
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    kept = np.tile(np.arange(20)[::-1], (2, 1))
    kept[1, :6] = [5, 4, 3, 2, 1, 0]
    new_len = ops.kv_keep(s.cache, s.batch, dev(kept.copy()), dev([20, 6]))
    moves = []
    for i, (q, kv) in enumerate(((20, 40), (6, 3))):
        for r in range(q):
            a, b = kv - q + int(kept[i, r]), kv - q + r
            if a >= 0 and b >= 0 and s.table[i, a // 16] >= 0 and s.table[i, b // 16] >= 0:
                moves.append(((s.table[i, a // 16], a % 16), (s.table[i, b // 16], b % 16), 0))
    assert np.array_equal(s.cache.pages.cpu().numpy().reshape(s.host.raw.shape), td.move(s.host, s.host.raw, moves))
    assert new_len.tolist() == [40, 3]


# ---- anywhere -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q_lens,kv_lens,many", [([9, 2], [300, 41], False), ([70, 40], [500, 90], True)])
def test_strided_queries_and_outputs(q_lens, kv_lens, many, dtype):
    """Queries and outputs as slices of wider rows at odd offsets: the bits of contiguous ones, and the same bits twice."""
    s = Setup(q_lens, kv_lens, 32, 2, 128, seed=13, pad=MANY_ROWS // 4 if many else 0)
    if many:
        s.batch.desc.max_q = s.n_tok
    rows = [td.seen_by(p) for p in trees_of(s, 5)]
    t = kv_tree(s, rows)
    q = _rand(s.rng, (s.n_tok, 8, 128), dtype)[0]
    wide = torch.zeros(s.n_tok * (12 * 128 + 7) + 3, dtype=q.dtype, device="cuda")[3:].view(s.n_tok, 12 * 128 + 7)
    qs, outs = wide[:, 128: 9 * 128].view(s.n_tok, 8, 128), torch.zeros_like(wide)[:, 5: 5 + 8 * 128].view(s.n_tok, 8, 128)
    qs.copy_(q)
    a, b = torch.zeros(2, s.n_tok, 8, device="cuda")
    first = ops.attn(s.cache, s.batch, q, tree=t, lse=a)
    ops.attn(s.cache, s.batch, qs, tree=t, lse=b, out=outs)
    tok = slice(0, s.tok)
    assert torch.equal(first[tok], outs[tok]) and torch.equal(a[tok], b[tok])
    w = ops.kv_weigh(s.cache, s.batch, q, a, None, tree=t)
    for x in (qs, q):
        assert torch.equal(w, ops.kv_weigh(s.cache, s.batch, x, a, None, tree=t))


def test_pages_behind_four_gigabytes():
    """A cache of more bytes than 32 bits count, its sequences in the last pages: what a small cache gives."""
    s = Setup([40, 3], [700, 90], 64, 8, 128, seed=3)
    n = s.host.n_pages
    far = (5 << 30) // s.cache.page_bytes
    pages = torch.empty(far + n, s.cache.page_bytes, dtype=torch.uint8, device="cuda")
    pages[far:] = s.cache.pages
    big = ops.KvCache(far + n, 64, 8, 128, pages=pages)
    there = ops.KvBatch(s.batch.q_start, s.batch.kv_len, torch.where(s.batch.page_table >= 0, s.batch.page_table + far, -1).int(),
                        n_tok=s.tok, max_q=40, max_kv=700)
    parents = dev([p for seq in trees_of(s, 3) for p in seq])
    q, k, v = (_rand(s.rng, (s.tok, h, 128))[0] for h in (16, 8, 8))
    kept, n_kept = dev([[0, 2, 9], [1, 2, 0]]), dev([3, 2])
    freq = ops.rope_freqs(128)
    got = []
    for cache, batch in ((s.cache, s.batch), (big, there)):
        t = ops.tree_plan(batch, parents)
        x = ops.kv_append(cache, batch, k, v, q=q, rope=ops.ROPE_HALVES, inv_freq=freq, pos=t.pos)
        lse = torch.empty(s.tok, 16, device="cuda")
        out = ops.attn(cache, batch, x, tree=t, lse=lse)
        w = ops.kv_weigh(cache, batch, x, lse, ops.kv_weights(cache), tree=t)
        new_len = ops.kv_keep(cache, batch, kept, n_kept, weights=w)
        after = ops.KvBatch(batch.q_start, new_len, batch.page_table, n_tok=s.tok, max_q=40, max_kv=700)
        which, cut = ops.kv_evict(cache, after, w, 300, first=3, recent=50)
        got.append([x, out, lse, new_len, which, cut, w[-n:], cache.pages[-n:]])
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---- together -------------------------------------------------------------------------------------------------------

def test_python_checks():
    s = Setup([4], [20], 16, 2, 64)
    q, lse = torch.zeros(4, 4, 64, device="cuda"), torch.zeros(4, 4, device="cuda")
    w = ops.kv_weights(s.cache)
    assert w.shape == (s.host.n_pages, 2, 16) and not w.any()
    tree = ops.KvTree(torch.zeros(3, 1, dtype=torch.int64, device="cuda"))
    for f in (lambda: ops.attn(s.cache, s.batch, q, tree=tree), lambda: ops.kv_weigh(s.cache, s.batch, q, lse, w, tree=tree),
              lambda: ops.attn(s.cache, s.batch, q, lse=lse.double()), lambda: ops.attn(s.cache, s.batch, q, lse=lse[:, :2]),
              lambda: ops.kv_weigh(s.cache, s.batch, q, lse.t(), w), lambda: ops.kv_weigh(s.cache, s.batch, q, lse, w[:-1]),
              lambda: ops.kv_evict(s.cache, s.batch, w.double(), 4), lambda: ops.kv_keep(s.cache, s.batch, dev([[0]]).long(), dev([1])),
              lambda: ops.kv_keep(s.cache, s.batch, dev([[0]]), dev([1, 2])), lambda: ops.kv_append(s.cache, s.batch, q[:, :2], q[:, :2], rope=1,
              inv_freq=ops.rope_freqs(64), pos=dev([1, 2, 3])), lambda: ops.tree_plan(s.batch, dev([-1, 0])),
              lambda: ops.kv_evict(s.cache, s.batch, w, 4, to_table=dev([0])), lambda: ops.KvTree(torch.zeros(4, 1, device="cuda"))):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(ValueError):
        ops.KvTree(torch.zeros(4, 1, dtype=torch.int64))  # not on the device
    with pytest.raises(FnsError, match="words"):
        ops.tree_plan(s.batch, dev([-1, 0, 0, 1]), words=0)
    with pytest.raises(FnsError, match="budget"):
        ops.kv_evict(s.cache, s.batch, w, 0)
    with pytest.raises(FnsError, match="workspace"):
        many = ops.KvBatch.from_lists([200], [200], [s.lists[0] * 7])
        q, lse = torch.zeros(200, 4, 64, device="cuda"), torch.zeros(200, 4, device="cuda")
        ops.kv_weigh(s.cache, many, q, lse, w, ws=ops.kv_weigh_workspace(s.cache, many, q)[:-16])


class Step:
    """A verify step of a layer with weights, then (every now and then) eviction, as an engine runs it."""

    def __init__(self, seed=0):
        self.s = s = Setup([26, 9, 12], [500, 40, 130], 16, 2, 64, seed=seed)
        self.parents = dev([p for seq in trees_of(s, 3, pads=False) for p in seq])
        self.base = dev([9000, 31, 118])
        self.qkv = _rand(s.rng, (s.tok, 8 + 4, 64))[0]
        self.freq, self.mag = ops.rope_scaled(64, 10000.0, 8.0, 2048)
        self.w = torch.rand(s.host.n_pages, 2, 16, device="cuda")
        self.kept, self.n_kept = dev([[0, 1, 4, 7], [0, 2, 3, 8], [0, 5, -1, -1]]), dev([4, 3, 2])
        self.out, self.lse = torch.empty(s.tok, 8, 64, device="cuda"), torch.empty(s.tok, 8, device="cuda")
        self.ws = ops.attn_workspace(s.cache, s.batch, self.qkv[:, :8])
        self.ws2 = ops.kv_weigh_workspace(s.cache, s.batch, self.qkv[:, :8])
        self.pages0, self.w0 = s.cache.pages.clone(), self.w.clone()
        self.after = ops.KvBatch(s.batch.q_start, dev([478, 34, 120]), s.batch.page_table, n_tok=s.tok, max_q=26, max_kv=500)

    def reset(self):
        self.s.cache.pages.copy_(self.pages0)
        self.w.copy_(self.w0)

    def __call__(self):
        s = self.s
        tree = ops.tree_plan(s.batch, self.parents, base=self.base)
        q = ops.kv_append(s.cache, s.batch, self.qkv[:, 8:10], self.qkv[:, 10:], q=self.qkv[:, :8], rope=ops.ROPE_HALVES,
                          inv_freq=self.freq, pos=tree.pos, magnitude=self.mag)
        ops.attn(s.cache, s.batch, q, out=self.out, ws=self.ws, tree=tree, lse=self.lse)
        ops.kv_weigh(s.cache, s.batch, q, self.lse, self.w, tree=tree, ws=self.ws2)
        new_len = ops.kv_keep(s.cache, s.batch, self.kept, self.n_kept, weights=self.w)
        self.after.kv_len.copy_(new_len)
        kept, cut = ops.kv_evict(s.cache, self.after, self.w, 100, first=2, recent=20)
        return [tree.sees, tree.pos, q, self.out, self.lse, new_len, kept, cut]

    def results(self, outs):
        live = [t.clone() for t in outs]
        k, v = [], []
        for i in range(3):  # what the sequences hold now
            n = int(outs[-1][i])
            b = ops.KvBatch.from_lists([n], [n], [self.s.lists[i]])
            a = ops.kv_read(self.s.cache, b)
            k.append(a[0]), v.append(a[1])
        return live + k + v


def test_a_step_of_a_layer():
    """Every part against its definition, each from what the one before it left on the device."""
    t = Step(1)
    s = t.s
    outs = t()
    sees, pos, q, out, lse, new_len, kept, cut = outs
    host = kd.Pages(s.host.n_pages, 16, 2, 64)
    host.raw = t.pages0.cpu().numpy().reshape(s.host.raw.shape).copy()
    s.host.raw = host.raw
    parents = t.parents.tolist()
    per = [parents[:26], parents[26:35], parents[35:]]
    rows = [td.seen_by(p) for p in per]
    x, f, m = t.qkv.double().cpu().numpy(), t.freq.cpu().numpy(), float(np.float32(t.mag))
    ph = pos.cpu().numpy()
    turn = lambda a: kd.rotate(a, ph, 1, f) * m  # noqa: E731
    s.put(turn(x[:, 8:10]), x[:, 10:])
    qh = q.double().cpu().numpy()
    assert (np.abs(qh - turn(x[:, :8])) <= np.abs(qh) * 2 * kd.F32_STEP + 1e-11).all()
    ref, ref_lse, ax, vm = td.attention(s.host, s.table, s.q_lens, s.kv_lens, qh, 0.125, rows=rows)
    assert (np.abs(out.double().cpu().numpy() - ref) <= kd.attn_tolerance("f32", 64, 500, ref, ax, vm)).all()
    assert (np.abs(lse.double().cpu().numpy() - ref_lse) <= td.lse_tolerance("f32", 64, 500, ref_lse, ax)).all()
    assert new_len.tolist() == [478, 34, 120] and cut.tolist() == [100, 34, 100]
    w, tol = td.weigh(s.host, s.table, s.q_lens, s.kv_lens, qh, lse.double().cpu().numpy(), t.w0.double().cpu().numpy(), 0.125, rows=rows)
    # the accepted paths, then what eviction picks: from the device's own weights, which a tolerance must not decide
    lists = [l[:n] for l, n in zip(t.kept.tolist(), t.n_kept.tolist())]
    s.cache.pages.copy_(torch.from_numpy(s.host.raw.copy()).view(s.cache.pages.shape))
    wd = torch.from_numpy(t.w0.cpu().numpy().copy()).cuda()
    ops.kv_weigh(s.cache, s.batch, q, lse, wd, tree=ops.KvTree(sees))
    assert (np.abs(wd.double().cpu().numpy() - w) <= tol).all()
    wk = wd.cpu().numpy().copy()
    for i, l in enumerate(lists):
        first = s.kv_lens[i] - s.q_lens[i]
        for h in range(2):
            pairs = [((s.table[i, (first + a) // 16], (first + a) % 16), (s.table[i, (first + r) // 16], (first + r) % 16)) for r, a in enumerate(l)]
            vals = [wk[a[0], h, a[1]] for a, _ in pairs]
            for (_, b), v in zip(pairs, vals):
                wk[b[0], h, b[1]] = v
    for i, n in enumerate(new_len.tolist()):
        j = np.arange(n)
        for h in range(2):
            want = td.evicted(wk[s.table[i, j // 16], h, j % 16], np.ones(n, bool), 100, 2, 20)
            assert kept[i, h, : len(want)].tolist() == want


def test_a_step_captured():
    """Replayed with the program's own work between: the eager results every time, also with another tree and other lengths."""
    t = Step(2)
    t()
    t.reset()
    want = t.results(t())
    t.reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = t()
    for _ in range(3):
        t.reset()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(t.results(outs), want))
        t.reset()
        t()  # eager, on the same buffers
    t.parents.copy_(dev([-1, 0, 0, 1] + [2] * 22 + [-1] * 9 + list(range(-1, 11))))
    t.s.batch.kv_len.copy_(dev([400, 40, 99]))
    t.reset()
    want = t.results(t())
    t.reset()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(t.results(outs), want))


def test_two_streams():
    """Two steps at once, a stream and workspaces each."""
    a, b = Step(3), Step(4)
    for t in (a, b):
        t()
        t.reset()
    want = [t.results(t()) for t in (a, b)]
    for t in (a, b):
        t.reset()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for t, st in zip((a, b), streams):
        with torch.cuda.stream(st):
            outs.append(t())
    torch.cuda.synchronize()
    for t, o, w in zip((a, b), outs, want):
        assert all(torch.equal(x, y) for x, y in zip(t.results(o), w))


@pytest.mark.parametrize("many", [False, True])
def test_denominators_of_rows_that_see_nothing(many):
    """The head's sink, minus infinity without sinks: of tokens without bits, and of causal ones in front of the context."""
    s = Setup([70 if many else 5, 3], [200, 2], 16, 1, 64, seed=12)
    q, sinks = _rand(s.rng, (s.n_tok, 4, 64))[0], torch.tensor([0.5, -3.0, 40.0, -200.0], device="cuda")
    rows = [td.seen_by(p) for p in trees_of(s, 2)]
    rows[0][1], rows[0][-1] = [], []
    blind = [1, s.q_lens[0] - 1]
    for tree, dark in ((kv_tree(s, rows), blind), (None, [s.q_lens[0]])):  # (a token at position -1 sees nothing)
        for sink in (sinks, None):
            lse = torch.zeros(s.n_tok, 4, device="cuda")
            out = ops.attn(s.cache, s.batch, q, sinks=sink, tree=tree, lse=lse)
            for t in dark:
                assert not out[t].any()
                want = sinks if sink is not None else torch.full_like(sinks, float("-inf"))
                # to log2 units and back: two half steps each, and one step of the log of a sum that is held 2^8 up
                assert torch.allclose(lse[t], want, rtol=2.0 ** -22, atol=2.0 ** -20)


def test_weigh_behind_the_planned_blocks_of_256_channels():
    """A prompt's rows over a context that is longer than the batch says: blocks behind the plan are gone over whole."""
    for kv in (900, 2100):
        s = Setup([280, 5], [kv, 700], 32, 1, 256, seed=kv)
        s.batch.desc.max_kv = 300
        _check_weigh(s, 2, "f32")
        _check_weigh(s, 2, "bf16", window=77, in_place=True)


def test_plan_of_a_line_of_1024():
    """The deepest plan: every token's path is all tokens before it."""
    s = Setup([1024, 700], [1024, 900], 64, 1, 64)
    plan = ops.tree_plan(s.batch, dev([i - 1 for n in s.q_lens for i in range(n)]), base=dev([5, 7]))
    bits = np.tril(np.ones((1024, 1024), np.uint8))
    want = np.concatenate([np.packbits(bits[:n], axis=1, bitorder="little").view(np.int64) for n in s.q_lens])
    assert np.array_equal(plan.sees.cpu().numpy(), want)
    assert np.array_equal(plan.pos.cpu().numpy(), np.concatenate([5 + np.arange(1024), 7 + np.arange(700)]))


def test_eviction_of_many_heads_in_chunks():
    """States of several kv heads beside each other: the same choice as that of one head at a time."""
    s = Setup([1, 1], [40000, 300], 64, 3, 64, seed=4)
    w = torch.rand(s.host.n_pages, 3, 64, device="cuda")
    kept, new_len = ops.kv_evict(s.cache, s.batch, w.clone(), 500, 3, 7)
    assert new_len.tolist() == [500, 300]
    for i, n in enumerate(s.kv_lens):
        for h in range(3):
            of = w[dev(s.lists[i]).long(), h].reshape(-1)[:n].cpu().numpy()
            want = td.evicted(of, np.ones(n, bool), 500, 3, 7)
            assert kept[i, h].tolist() == want + [-1] * (500 - len(want))
