"""The attention half of a block on the device: residual add + RMSNorm + Q8_1, append to the paged 4-bit cache, attention
over it, against 64-bit computations of their definitions (kv_data.py); tolerances count the roundings."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import kv_data as kd
from flintnsteel_amd import ops, synth
from flintnsteel_amd._lib import FnsError, call
from oracle import oracle as orc

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _rand(rng, shape, dtype="f32", std=1.0):
    """A device tensor and its exact values in f64."""
    t = torch.from_numpy(rng.standard_normal(shape) * std).to(DT[dtype])
    return t.cuda(), t.double().numpy()


# ---- residual add + RMSNorm + Q8_1 ----------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,n", [(1, 32), (1, 2048), (3, 2080), (7, 4096), (2, 4128), (5, 8192), (3, 8224), (300, 512)])
@pytest.mark.parametrize("alias", ["none", "x", "y"])
def test_add_rms_norm_is_add_then_rms_norm(rows, n, alias):
    rng = np.random.default_rng(n + rows)
    (x, xh), (y, yh) = _rand(rng, (rows, n), std=3.0), _rand(rng, (rows, n))
    w, wh = _rand(rng, (n,))
    s0 = ops.add(x, y)
    o0, q0 = ops.rms_norm_q8_1(s0, w, 1e-6)
    x0, y0 = x.clone(), y.clone()
    s, o, q = ops.add_rms_norm_q8_1(x, y, w, 1e-6, sum_out={"none": None, "x": x, "y": y}[alias],
                                    xq=torch.full((rows, ops.q8_1_row_bytes(n)), 255, dtype=torch.uint8, device="cuda"))
    assert torch.equal(s, s0) and torch.equal(o, o0) and torch.equal(q, q0)
    assert alias == "x" or torch.equal(x, x0)
    assert alias == "y" or torch.equal(y, y0)
    sh = (xh + yh)
    ref = sh / np.sqrt((sh ** 2).mean(-1, keepdims=True) + 1e-6) * wh
    # s rounds once; the mean of n squares of non-negative terms by at most (n / 256 + 12) steps, halved by the root
    tol = (n / 512 + 16) * 2 * kd.F32_STEP
    assert (np.abs(o.cpu().numpy() - ref) <= np.abs(ref) * tol + np.abs(xh * wh) * 2 * kd.F32_STEP
            / np.sqrt((sh ** 2).mean(-1, keepdims=True)) + 1e-30).all()


def test_add_rms_norm_unaligned_rows_and_no_f32_output():
    rng = np.random.default_rng(5)
    n, rows = 1056, 4
    base = torch.zeros(3 * rows * n + 16, device="cuda")
    x, y, s = (base[1 + i * rows * n: 1 + (i + 1) * rows * n].view(rows, n) for i in range(3))  # 4-byte aligned only
    x.copy_(_rand(rng, (rows, n))[0])
    y.copy_(_rand(rng, (rows, n))[0])
    w = _rand(rng, (n,))[0]
    ref = ops.add_rms_norm_q8_1(x.clone(), y.clone(), w, 1e-5)
    got = ops.add_rms_norm_q8_1(x, y, w, 1e-5, sum_out=s)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    xq = torch.zeros_like(ref[2])
    xc, yc, sc = x.clone(), y.clone(), torch.empty_like(ref[0])
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    call("fns_hip_add_rms_norm_q8_1", p(xc), p(yc), p(w), p(sc), None, p(xq), n, 1e-5, rows,
         ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(xq, ref[2]) and torch.equal(sc, ref[0])


def test_add_rms_norm_special_rows():
    n = 512
    x, y = torch.zeros(4, n, device="cuda"), torch.zeros(4, n, device="cuda")
    x[1], y[1] = 1e18, 1e18     # squares near the top of f32
    x[2, 3] = float("inf")
    y[3] = float("nan")
    w = torch.ones(n, device="cuda")
    s0 = ops.add(x, y)
    o0, q0 = ops.rms_norm_q8_1(s0, w, 1e-6)
    s, o, q = ops.add_rms_norm_q8_1(x, y, w, 1e-6)
    assert torch.equal(o.view(torch.int32), o0.view(torch.int32)) and torch.equal(q, q0)
    assert torch.equal(s.view(torch.int32), s0.view(torch.int32))
    assert (o[0] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,n", [(1, 32), (5, 96), (3, 1024), (130, 2080)])
def test_dequantize_q8_1(rows, n, dtype):
    rng = np.random.default_rng(rows)
    x, _ = _rand(rng, (rows, n), std=2.0)
    x[0, :32] = 0
    xq = ops.quantize_q8_1(x)
    v, sums = ops.dequantize_q8_1(xq, n, dtype)
    b = xq.cpu().numpy()[:, : n // 32 * 36].reshape(rows, n // 32, 36)
    d = b[..., :2].copy().view(np.float16).astype(np.float32)
    want = (b[..., 4:].view(np.int8).astype(np.float32) * d).reshape(rows, n)
    np_t = np.float32 if dtype == torch.float32 else np.float16
    assert np.array_equal(v.cpu().numpy(), want.astype(np_t))
    assert np.array_equal(sums.cpu().numpy(), b[..., 2:4].copy().view(np.float16)[..., 0].astype(np_t))


# ---- a batch over a cache -------------------------------------------------------------------------------------------

class Setup:
    """Sequences with scattered pages; the host's copy of the cache beside the device's."""

    def __init__(self, q_lens, kv_lens, page, heads_kv, dim, seed=0, pad=0, n_extra=3):
        rng = self.rng = np.random.default_rng(seed)
        self.q_lens, self.kv_lens, self.page, self.heads_kv, self.dim = list(q_lens), list(kv_lens), page, heads_kv, dim
        per = [(kv + page - 1) // page for kv in kv_lens]
        n_pages = sum(per) + n_extra
        perm = list(rng.permutation(n_pages)[: sum(per)])
        self.lists = [[int(perm.pop()) for _ in range(n)] for n in per]
        self.table = np.full((len(per), max(per + [1])), -1, np.int64)
        for i, p in enumerate(self.lists):
            self.table[i, : len(p)] = p
        self.host = kd.Pages(n_pages, page, heads_kv, dim, fill=seed).sane(seed)
        self.cache = ops.KvCache(n_pages, page, heads_kv, dim, pages=torch.from_numpy(self.host.raw.copy()).cuda())
        self.tok = sum(q_lens)
        self.n_tok = self.tok + pad
        self.batch = ops.KvBatch.from_lists(self.q_lens, self.kv_lens, self.lists, n_tok=self.n_tok)

    def positions(self):
        return np.concatenate([np.arange(kv - q, kv) for q, kv in zip(self.q_lens, self.kv_lens)] or [np.zeros(0, int)]).astype(int)

    def sequences(self):
        return np.repeat(np.arange(len(self.q_lens)), self.q_lens)

    def put(self, k, v):
        for t, (s, p) in enumerate(zip(self.sequences(), self.positions())):
            i = p // self.page
            page = self.table[s, i] if 0 <= i < self.table.shape[1] else -1
            if 0 <= page < self.host.n_pages and p >= 0:
                for h in range(self.heads_kv):
                    self.host.put(page, p % self.page, h, k[t, h], v[t, h])

    def same_bytes(self):
        got = self.cache.pages.cpu().numpy().reshape(self.host.raw.shape)
        return np.array_equal(got, self.host.raw)


def _rounded_ok(got: torch.Tensor, ref: np.ndarray, dtype: str) -> bool:
    # one rounding of the 64-bit result (bf16: through f32)
    step = kd.F32_STEP if dtype == "f32" else kd.BF16_STEP * (1 + 2.0 ** -15)
    return bool((np.abs(got.double().cpu().numpy() - ref) <= np.abs(ref) * (step + 1e-12) + 1e-38).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rope,rope_dim", [(0, 0), (1, 0), (2, 0), (1, 32), (2, 48)])
@pytest.mark.parametrize("dim,page,heads_kv,group,q_lens,kv_lens", [
    (128, 64, 2, 4, [1], [1]),
    (64, 16, 1, 1, [1, 1, 1, 0, 1], [5, 16, 17, 9, 100]),
    (128, 16, 3, 3, [5, 17, 0, 33], [5, 40, 12, 48]),
    (256, 32, 2, 1, [3, 16, 31], [77, 16, 64]),
    (64, 128, 2, 16, [20, 1], [149, 128]),
])
def test_append(dim, page, heads_kv, group, q_lens, kv_lens, rope, rope_dim, dtype):
    s = Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim + rope, pad=2)
    rope_dim = rope_dim or dim
    freq = ops.rope_freqs(rope_dim, 10000.0) if rope else None
    fh = freq.cpu().numpy() if rope else None
    H = heads_kv * group
    k, kh = _rand(s.rng, (s.n_tok, heads_kv, dim), dtype, 2.0)
    v, vh = _rand(s.rng, (s.n_tok, heads_kv, dim), dtype)
    q, qh = _rand(s.rng, (s.n_tok, H, dim), dtype)
    qo = torch.full_like(q, 7.0)
    ops.kv_append(s.cache, s.batch, k, v, q=q, rope=rope, inv_freq=freq, q_out=qo)
    pos = s.positions()
    s.put(kd.rotate(kh[: s.tok], pos, rope, fh), vh[: s.tok])
    assert s.same_bytes()  # the tokens' blocks, and no other byte
    assert _rounded_ok(qo[: s.tok], kd.rotate(qh[: s.tok], pos, rope, fh), dtype)
    assert (qo[s.tok:] == 7.0).all()  # padding rows are left alone
    kr, vr = ops.kv_read(s.cache, s.batch)
    for t, (sq, p) in enumerate(zip(s.sequences(), pos)):
        for h in range(heads_kv):
            K, V = s.host.get(s.table[sq, p // page][None], np.array([p % page]), h)
            assert np.array_equal(kr[t, h].double().cpu().numpy(), K[0]) and np.array_equal(vr[t, h].double().cpu().numpy(), V[0])


def test_append_slices_of_a_fused_projection_in_place():
    s = Setup([7, 18], [30, 18], 16, 2, 128, seed=3)
    H, Hk, D = 6, 2, 128
    flat = torch.zeros(s.tok * ((H + 2 * Hk) * D + 3) + 1, device="cuda")  # rows at odd offsets
    qkv = flat[1:].view(s.tok, (H + 2 * Hk) * D + 3)[:, : (H + 2 * Hk) * D].view(s.tok, H + 2 * Hk, D)
    full, fh = _rand(s.rng, (s.tok, H + 2 * Hk, D))
    qkv.copy_(full)
    freq = ops.rope_freqs(D, 500000.0, factors=1 + np.arange(D // 2) / 16)
    got = ops.kv_append(s.cache, s.batch, qkv[:, H:H + Hk], qkv[:, H + Hk:], q=qkv[:, :H], rope=ops.ROPE_HALVES,
                        inv_freq=freq, q_out=qkv[:, :H])
    assert got.data_ptr() == qkv.data_ptr()
    pos, f = s.positions(), freq.cpu().numpy()
    s.put(kd.rotate(fh[:, H:H + Hk], pos, 1, f), fh[:, H + Hk:])
    assert s.same_bytes() and _rounded_ok(qkv[:, :H], kd.rotate(fh[:, :H], pos, 1, f), "f32")
    assert torch.equal(qkv[:, H:], full[:, H:])


@pytest.mark.parametrize("last", [131072, (1 << 24) + 5])
def test_append_far_positions(last):
    """Only the pages that are written have to exist: the table points every position at two pages."""
    page, D = 4096, 64
    s = Setup([3], [3], page, 1, D, seed=9)
    n = (last + page - 1) // page
    s.table = np.zeros((1, n), np.int64)
    s.kv_lens = [last]
    s.batch = ops.KvBatch.from_lists([3], [last], [[0] * n])
    freq = ops.rope_freqs(D, 1.0001)  # every angle large
    k, kh = _rand(s.rng, (3, 1, D))
    v, vh = _rand(s.rng, (3, 1, D))
    ops.kv_append(s.cache, s.batch, k, v, rope=ops.ROPE_PAIRS, inv_freq=freq)
    s.put(kd.rotate(kh, s.positions(), 2, freq.cpu().numpy()), vh)
    assert s.same_bytes()


def test_append_odd_values_and_missing_pages():
    s = Setup([16, 4, 2], [40, 4, 10], 16, 1, 64, seed=4)
    k, kh = _rand(s.rng, (22, 1, 64))
    v, vh = _rand(s.rng, (22, 1, 64))
    k[0, 0, 5], v[1, 0, 40], k[2, 0, 33] = float("nan"), float("inf"), float("-inf")
    k[3], v[4, 0, :32] = 0.0, 0.0
    k[5], v[5] = 3.0e38, -1e-41
    v[6, 0, 7], k[6, 0, 0] = 7.0, -0.0
    v[7, 0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    v[7, 0, 8:] = 0
    s.table[0, 2], s.table[2, 0] = s.host.n_pages, -7  # no pages of the cache
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    ops.kv_append(s.cache, s.batch, k, v)
    s.put(k.double().cpu().numpy(), v.double().cpu().numpy())
    assert s.same_bytes()
    kr, vr = ops.kv_read(s.cache, s.batch)
    assert torch.isnan(kr[0, 0, :32]).all() and torch.isfinite(kr[0, 0, 32:]).all() and torch.isnan(vr[1, 0, 32:]).all()
    assert torch.isnan(kr[8:16]).all() and torch.isnan(vr[20:]).all()  # positions 32.. of sequence 0, all of sequence 2
    assert torch.isfinite(kr[16:20]).all()


def test_batches_that_make_no_sense_touch_nothing():
    """Ranges of tokens outside the batch, descending, lengths below the new tokens, tables too short: no write elsewhere."""
    s = Setup([4, 4, 4, 4], [4, 4, 4, 4], 16, 1, 64, seed=6)
    k, _ = _rand(s.rng, (16, 1, 64))
    q, _ = _rand(s.rng, (16, 2, 64))
    s.batch.q_start.copy_(torch.tensor([-3, 4, 2, 20, 16], dtype=torch.int32))
    out = torch.full_like(q, 5.0)
    ops.kv_append(s.cache, s.batch, k, k)
    ops.attn(s.cache, s.batch, q, out=out)
    assert s.same_bytes() and (out == 5.0).all()
    s.batch.q_start.copy_(torch.tensor([0, 4, 8, 12, 16], dtype=torch.int32))
    s.batch.kv_len.copy_(torch.tensor([-5, 2, 0, 2 ** 31 - 1], dtype=torch.int32))
    ops.kv_append(s.cache, s.batch, k, k)
    s.q_lens, s.kv_lens = [0, 2, 0, 0], [0, 2, 0, 0]
    kh = k.double().cpu().numpy()[6:8]  # the last two of sequence 1's tokens have positions
    s.put(kh, kh)
    assert s.same_bytes()
    ops.attn(s.cache, s.batch, q, window=100, out=out)
    assert (out[:6] == 0).all() and (out[8:] == 0).all() and (out[6:8] != 0).any()


# ---- attention ------------------------------------------------------------------------------------------------------

def _check_attn(s: Setup, group: int, dtype: str, window: int = 0, sinks: bool = False, std: float = 1.0, **kw):
    H = s.heads_kv * group
    q, qh = _rand(s.rng, (s.n_tok, H, s.dim), dtype, std)
    sk, skh = _rand(s.rng, (H,)) if sinks else (None, None)
    out = torch.full_like(q, 7.0)
    scale = s.dim ** -0.5
    ops.attn(s.cache, s.batch, q, window=window, sinks=sk, out=out, **kw)
    ref, ax, vm = kd.attention(s.host, s.table, s.q_lens, s.kv_lens, qh[: s.tok], scale, window, skh)
    got = out.double().cpu().numpy()
    assert (got[s.tok:] == 7.0).all()
    got = got[: s.tok]
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    tol = kd.attn_tolerance(dtype, s.dim, max(s.kv_lens + [1]), ref, ax, vm)
    far = np.abs(ref) >= 2.0 ** 128  # codes of scale 254 stand for up to 6 * 2^127, which f32 has as an infinity
    assert np.array_equal(got[far], np.copysign(np.inf, ref[far]))
    bad = ~np.isnan(ref) & ~far & ~(np.abs(got - ref) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - ref) / tol):.3g} of the tolerance"
    return q, out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv", [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 500])
def test_attn_decode_lengths(kv, dim, dtype):
    _check_attn(Setup([1], [kv], 16 if kv % 2 else 64, 2, dim, seed=kv), 4, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("group", [1, 3, 5, 8, 16, 17, 33])
@pytest.mark.parametrize("window,sinks", [(0, False), (0, True), (1, True), (70, False)])
def test_attn_decode_ragged(group, window, sinks, dtype):
    s = Setup([1, 1, 0, 1, 1, 1], [700, 3, 50, 64, 257, 1], 32, 2, 128, seed=group, pad=3)
    _check_attn(s, group, dtype, window, sinks)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,heads_kv,group,q_lens,kv_lens,window,sinks", [
    (128, 16, 2, 4, [4, 2, 3], [4, 130, 67], 0, False),
    (64, 32, 1, 8, [5, 8, 1, 0], [300, 8, 64, 20], 33, True),
    (256, 64, 1, 3, [7], [200], 0, True),
    (128, 128, 1, 1, [16, 3], [16, 260], 5, False),
    (64, 64, 2, 8, [70], [70], 0, False),
    (128, 64, 1, 4, [65, 1, 130], [65, 900, 401], 0, True),
    (128, 16, 1, 7, [33, 90], [200, 90], 40, False),
    (256, 32, 2, 2, [100], [333], 64, True),
    (64, 16, 1, 1, [257], [300], 0, False),
    (128, 256, 1, 40, [9], [77], 0, False),
])
def test_attn_many_tokens(dim, page, heads_kv, group, q_lens, kv_lens, window, sinks, dtype):
    _check_attn(Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim + group, pad=1), group, dtype, window, sinks)


MANY_ROWS = 65536  # rows a sequence at most, by the batch's numbers: what a prompt's workgroups are for


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,heads_kv,group,q_lens,kv_lens,window,sinks", [
    (128, 16, 2, 4, [4, 2, 3], [4, 130, 67], 0, False),
    (64, 32, 1, 8, [5, 8, 1, 0], [300, 8, 64, 20], 33, True),
    (256, 64, 1, 3, [7, 60], [200, 60], 0, True),
    (64, 64, 2, 8, [70], [70], 0, False),
    (128, 64, 1, 4, [65, 1, 130], [65, 900, 401], 0, True),
    (128, 16, 1, 7, [33, 90], [200, 90], 40, False),
    (256, 32, 2, 2, [100], [333], 64, True),
    (64, 16, 1, 1, [257], [300], 0, False),
    (128, 256, 1, 40, [9], [77], 1, False),
])
def test_attn_in_a_prompts_workgroups(dim, page, heads_kv, group, q_lens, kv_lens, window, sinks, dtype):
    """The same sequences in a batch that is padded to many rows."""
    s = Setup(q_lens, kv_lens, page, heads_kv, dim, seed=dim + group, pad=MANY_ROWS // group)
    s.batch.desc.max_q = s.n_tok
    _check_attn(s, group, dtype, window, sinks)


@pytest.mark.parametrize("q,many", [(4, False), (50, False), (50, True), (150, True)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attn_odd_places_in_a_prompts_workgroups(q, many, dtype):
    """NaNs, missing pages and freed ones before a window, and scores of hundreds, in either form."""
    s = Setup([q, 1], [400, 64], 16, 1, 64, seed=61, pad=MANY_ROWS // 4 if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    h, first = s.host, 400 - q - 100 + 1
    s.table[0, : first // 16] = np.array([-1, 1 << 30, h.n_pages] * 20)[: first // 16]
    s.table[0, 20] = -1
    for pos, off in ((399 - q // 2, 0), (399 - q // 3, 32), (first - 1, 0), (first - 1, 32)):
        page = s.table[0, pos // 16]
        if 0 <= page < h.n_pages:
            h.raw[page, 16 * 64 + off + pos % 16 * 2] = 255
    s.cache.pages.copy_(torch.from_numpy(h.raw.copy()).view(s.cache.pages.shape))
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    _check_attn(s, 4, dtype, window=100, std=20.0)


@pytest.mark.parametrize("scale", [160, 166, 200, 250, 254])
@pytest.mark.parametrize("q,many", [(3, False), (50, False), (50, True), (140, True)])
def test_attn_a_huge_block_of_v_is_nothing_to_rows_that_do_not_see_it(q, many, scale):
    """V of two tokens in the middle far above everything else, and of one block far below: the rows before them, and with
    the window those behind, keep the precision of what they see."""
    s = Setup([q, q], [q + 30, q + 200], 32, 2, 64, seed=scale, pad=MANY_ROWS // 4 if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    h = s.host
    for seq in (0, 1):
        for pos, block, e in ((s.kv_lens[seq] - 1 - q // 2, 0, scale), (s.kv_lens[seq] - 2 - q // 2, 1, scale - 20), (3, 1, 60)):
            for head in (0, 1):
                at = head * h.head_bytes + 32 * 64 + 32 * 2 + pos % 32 * 2 + block
                h.raw[s.table[seq, pos // 32], at] = e
    s.cache.pages.copy_(torch.from_numpy(h.raw.copy()).view(s.cache.pages.shape))
    _check_attn(s, 4, "f32")
    _check_attn(s, 4, "f32", window=q // 4 + 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,page,q,many", [(128, 64, 5, False), (128, 64, 90, True), (128, 16, 40, False), (256, 128, 6, False),
                                             (256, 16, 70, True), (64, 256, 130, True)])
def test_attn_huge_blocks_of_v_in_every_form(dim, page, q, many, dtype):
    s = Setup([q, 2], [q + 100, 300], page, 1, dim, seed=67, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    h = s.host
    for seq, back, e in ((0, 1, 250), (0, q // 2, 200), (1, 1, 180)):
        pos = s.kv_lens[seq] - back
        at = page * dim + page * (dim // 32) + pos % page * (dim // 32) + back % (dim // 32)
        h.raw[s.table[seq, pos // page], at] = e
    s.cache.pages.copy_(torch.from_numpy(h.raw.copy()).view(s.cache.pages.shape))
    _check_attn(s, 2, dtype)
    _check_attn(s, 2, dtype, window=q // 3 + 1, sinks=True)


@pytest.mark.parametrize("q,many", [(1, False), (20, False), (80, True)])
def test_attn_odd_queries_scales_windows_and_sinks(q, many):
    """Rows of q with NaNs and infinities are NaN, their neighbours are not; scales of zero and below; windows beyond any
    length; sinks of either infinity."""
    s = Setup([q], [q + 70], 64, 1, 64, seed=71, pad=MANY_ROWS if many else 0)
    s.batch.desc.max_q = s.n_tok if many else q
    x, xh = _rand(s.rng, (s.n_tok, 2, 64))
    for scale, window in ((0.0, 0), (-0.3, 0), (0.2, 2 ** 31 - 1), (0.125, 2 ** 30)):
        got = ops.attn(s.cache, s.batch, x, scale=scale, window=window)[: s.tok].double().cpu().numpy()
        ref, ax, vm = kd.attention(s.host, s.table, s.q_lens, s.kv_lens, xh[: s.tok], scale, 0)
        assert (np.abs(got - ref) <= kd.attn_tolerance("f32", 64, q + 70, ref, np.abs(ax), vm)).all()
    good = ops.attn(s.cache, s.batch, x)[: s.tok]
    low = ops.attn(s.cache, s.batch, x, sinks=torch.tensor([float("-inf"), 0.5], device="cuda"))[: s.tok]
    assert torch.equal(low[:, 0], good[:, 0])
    bad = x.clone()
    bad[0, 0, 63], bad[q // 2, 1, 0] = float("nan"), float("-inf")
    got = ops.attn(s.cache, s.batch, bad)[: s.tok]
    assert torch.isnan(got[0, 0]).all() and torch.isnan(got[q // 2, 1]).all()
    got[0, 0], got[q // 2, 1] = good[0, 0], good[q // 2, 1]
    assert torch.equal(got, good)
    tiny = ops.attn(s.cache, s.batch, x * 1e-36)[: s.tok]  # scores of nothing: the mean of V
    assert torch.equal(tiny, ops.attn(s.cache, s.batch, x, scale=0.0)[: s.tok])


def test_sequences_may_share_pages_and_workspaces_are_checked():
    """A common prefix, in order and twice in one table; a workspace that is too small is refused before anything runs."""
    s = Setup([1, 3], [2000, 2040], 64, 2, 128, seed=73)
    s.table[1, :30] = s.table[0, :30]
    s.table[0, 7] = s.table[0, 6]
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    q, out = _check_attn(s, 4, "f32")
    ws = ops.attn_workspace(s.cache, s.batch, q)
    assert ws.numel() > 0
    with pytest.raises(FnsError, match="workspace"):
        ops.attn(s.cache, s.batch, q, out=out, ws=ws[:-16])
    with pytest.raises(FnsError, match="overlap"):
        ops.attn(s.cache, s.batch, q, out=q, ws=ws)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("q", [1, 3, 40])
def test_attn_large_scores(q, dtype):
    """Scores of hundreds: a softmax that is nearly one-hot, its maximum moving from tile to tile."""
    _check_attn(Setup([q, q], [400, 130], 64, 1, 128, seed=11), 4, dtype, std=40.0)


@pytest.mark.parametrize("q", [1, 40])
def test_attn_blocks_of_all_sizes(q):
    """Scales over 2^-120 .. 2^100 in one cache; the largest decide the result."""
    s = Setup([q], [300], 32, 1, 64, seed=13)
    P, D = 32, 64
    o = P * D
    s.host.raw[:, o: o + P * 2] = s.rng.integers(90, 128, (s.host.n_pages, P * 2))   # K
    s.host.raw[:, o + P * 2:] = s.rng.integers(7, 228, (s.host.n_pages, P * 2))      # V
    s.cache.pages.copy_(torch.from_numpy(s.host.raw.copy()).view(s.cache.pages.shape))
    _check_attn(s, 4, "f32")


@pytest.mark.parametrize("q", [1, 4, 50])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attn_nan_blocks_reach_the_rows_that_see_them(q, dtype):
    """A NaN in K of one position and in V of another: rows behind them or past the window stay finite; so do all rows
    when the positions belong to no row (behind the end, or before the window)."""
    s = Setup([q, 1], [200, 64], 16, 1, 64, seed=17)
    h = s.host

    def poison(seq, pos, off):
        page = s.table[seq, pos // 16]
        h.raw[page, 16 * 64 + off + (pos % 16) * 2] = 255

    poison(0, 200 - (q + 1) // 2, 0)       # K, seen by half of the new tokens
    poison(0, 70, 32)                      # V, inside nobody's window of 100
    poison(1, 40, 32)                      # V, seen by the other sequence
    s.cache.pages.copy_(torch.from_numpy(h.raw.copy()).view(s.cache.pages.shape))
    _check_attn(s, 2, dtype, window=100 if q < 50 else 60)


@pytest.mark.parametrize("q", [1, 3, 70])
def test_attn_freed_pages_behind_the_window(q):
    """Pages before the window may be gone: entries of any value; the page that the window starts in holds NaNs before it."""
    s = Setup([q], [500], 32, 2, 64, seed=19)
    window = 90
    first = 500 - q - window + 1
    s.table[0, : first // 32] = np.array([-1, 1 << 30, s.host.n_pages] * 20)[: first // 32]
    for h in range(2):
        o = h * s.host.head_bytes + 32 * 64
        s.host.raw[s.table[0, first // 32], o: o + first % 32 * 2] = 255
        s.host.raw[s.table[0, first // 32], o + 64: o + 64 + first % 32 * 2] = 255
    s.cache.pages.copy_(torch.from_numpy(s.host.raw.copy()).view(s.cache.pages.shape))
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    _check_attn(s, 4, "f32", window=window)


@pytest.mark.parametrize("q", [1, 5, 80])
def test_attn_missing_pages_are_left_out(q):
    s = Setup([q], [260], 16, 1, 128, seed=23)
    s.table[0, [1, 4, 5, 16]] = [-1, s.host.n_pages, -5, 1 << 30]
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    _check_attn(s, 3, "f32")
    s.table[:] = -1
    s.batch.page_table.copy_(torch.from_numpy(s.table))
    out = ops.attn(s.cache, s.batch, torch.ones(q, 2, 128, device="cuda"))
    assert (out == 0).all()


@pytest.mark.parametrize("q,kv", [(1, 2000), (40, 600)])
def test_attn_split_hint_does_not_matter(q, kv):
    """max_kv only divides the work: far too small and far too large, within the tolerances; and the same call twice has the
    same bits."""
    s = Setup([q, q], [kv, kv // 3], 64, 1, 128, seed=29)
    for hint in (1, kv, 1 << 20):
        s.batch.desc.max_kv = hint
        q1, out = _check_attn(s, 4, "f32")
        assert torch.equal(out[: s.tok], ops.attn(s.cache, s.batch, q1)[: s.tok])


def test_attn_strides():
    s = Setup([1, 9], [90, 100], 16, 2, 64, seed=31)
    H, D = 6, 64
    flat = torch.zeros(s.tok * (3 * H * D + 5) + 3, device="cuda")
    wide = flat[3:].view(s.tok, 3 * H * D + 5)
    q = wide[:, : H * D].view(s.tok, H, D)
    o = wide[:, H * D + 1: 2 * H * D + 1].view(s.tok, H, D)
    qc, qh = _rand(s.rng, (s.tok, H, D))
    q.copy_(qc)
    ops.attn(s.cache, s.batch, q, out=o)
    assert torch.equal(o, ops.attn(s.cache, s.batch, qc)) and torch.equal(q, qc)
    assert (wide[:, H * D] == 0).all() and (wide[:, 2 * H * D + 1:] == 0).all()


def test_pages_beyond_4_gib():
    page, Hk, D = 4096, 8, 128
    size = ops.KvCache(1, page, Hk, D).page_bytes
    n = (9 << 30) // size + 2
    pages = torch.zeros(n, size, dtype=torch.uint8, device="cuda")
    cache = ops.KvCache(n, page, Hk, D, pages=pages)
    s = Setup([60], [60], 64, Hk, D, seed=37)
    batch = ops.KvBatch.from_lists([60], [60], [[n - 1]])
    k, kh = _rand(s.rng, (60, Hk, D))
    v, vh = _rand(s.rng, (60, Hk, D))
    q, qh = _rand(s.rng, (60, Hk * 2, D))
    ops.kv_append(cache, batch, k, v)
    kr, vr = ops.kv_read(cache, batch)
    ops.kv_append(s.cache, s.batch, k, v)
    kr2, vr2 = ops.kv_read(s.cache, s.batch)
    assert torch.equal(kr, kr2) and torch.equal(vr, vr2)
    assert torch.equal(ops.attn(cache, batch, q), ops.attn(s.cache, s.batch, q))
    one, two = ops.KvBatch.from_lists([1], [60], [[n - 1]]), ops.KvBatch.from_lists([1], [60], [s.lists[0]])
    assert torch.equal(ops.attn(cache, one, q[:1]), ops.attn(s.cache, two, q[:1]))
    assert not pages[: n - 1].any()


def test_rows_per_call_do_not_change_a_kv_append():
    """Token by token or at once: the same bytes."""
    a, b = (Setup([37], [50], 16, 2, 64, seed=41) for _ in range(2))
    k, _ = _rand(a.rng, (37, 2, 64))
    v, _ = _rand(a.rng, (37, 2, 64))
    freq = ops.rope_freqs(64)
    ops.kv_append(a.cache, a.batch, k, v, rope=ops.ROPE_HALVES, inv_freq=freq)
    for i in range(37):
        one = ops.KvBatch.from_lists([1], [14 + i], b.lists)
        ops.kv_append(b.cache, one, k[i:i + 1], v[i:i + 1], rope=ops.ROPE_HALVES, inv_freq=freq)
    assert torch.equal(a.cache.pages, b.cache.pages)


# ---- graphs, streams, a whole block ---------------------------------------------------------------------------------

@pytest.mark.parametrize("q", [1, 20])
def test_graph_of_a_growing_sequence(q):
    """Append and attention captured once, replayed while the lengths in device memory grow, eager calls and
    synchronisations between the replays; two graphs that share a workspace, replayed in turn."""
    H, Hk, D, page = 8, 2, 128, 16
    a, b = (Setup([q, q], [40 + 6 * q, 30 + 6 * q], page, Hk, D, seed=43) for _ in range(2))
    freq = ops.rope_freqs(D)
    k, v, x = (torch.empty(2 * q, n, D, device="cuda") for n in (Hk, Hk, H))
    qr, out = torch.empty_like(x), torch.empty_like(x)
    start = torch.tensor([40, 30], dtype=torch.int32, device="cuda")
    batch = ops.KvBatch(a.batch.q_start, a.batch.kv_len, a.batch.page_table, 2 * q, q)
    ws = ops.attn_workspace(a.cache, batch, x)

    def step(cache, bt, o):
        ops.kv_append(cache, bt, k, v, q=x, rope=ops.ROPE_HALVES, inv_freq=freq, q_out=qr)
        ops.attn(cache, bt, qr, out=o, ws=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a.cache, batch, out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(a.cache, batch, out)
        graphs.append(g)
    a.cache.pages.copy_(b.cache.pages)
    eager = ops.KvBatch(b.batch.q_start, b.batch.kv_len, b.batch.page_table, 2 * q, q)
    for i in range(5):
        for t in (k, v, x):
            t.normal_()
        a.batch.kv_len.copy_(start + (i + 1) * q)
        b.batch.kv_len.copy_(start + (i + 1) * q)
        graphs[i % 2].replay()
        got = out.clone()
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        step(b.cache, eager, want)
        assert torch.equal(got, want)
        assert torch.equal(a.cache.pages, b.cache.pages)


def test_graphs_of_prompts_that_share_a_workspace():
    """Two graphs of a prompt's workgroups over one workspace, replayed in turn while blocks that send rows to the second pass
    come and go, eager calls between."""
    s = Setup([70, 33], [70, 140], 64, 1, 128, seed=79, pad=MANY_ROWS)
    s.batch.desc.max_q = s.n_tok
    q = _rand(s.rng, (s.n_tok, 2, 128))[0]
    ws, outs, graphs = ops.attn_workspace(s.cache, s.batch, q), [torch.zeros_like(q) for _ in range(2)], []
    ops.attn(s.cache, s.batch, q, out=outs[0], ws=ws)
    torch.cuda.synchronize()
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.attn(s.cache, s.batch, q, out=o, ws=ws)
        graphs.append(g)
    page, row = int(s.table[0, 0]), 64 * 128 + 64 * 4 + 40 * 4
    keep = s.cache.pages[page, row].clone()
    for i in range(6):
        s.cache.pages[page, row] = keep if i % 3 == 0 else torch.full_like(keep, 200 + i)
        q.normal_()
        graphs[i % 2].replay()
        graphs[(i + 1) % 2].replay()
        want = ops.attn(s.cache, s.batch, q)
        torch.cuda.synchronize()
        assert torch.equal(outs[0][: s.tok], want[: s.tok]) and torch.equal(outs[1][: s.tok], want[: s.tok])
        assert torch.isfinite(want[:40]).all() and (want[:40].abs() < 100).all()


def test_two_streams_with_workspaces_of_their_own():
    s = Setup([1, 1], [3000, 2500], 64, 2, 128, seed=47)
    qs = [_rand(s.rng, (2, 16, 128))[0] for _ in range(2)]
    want = [ops.attn(s.cache, s.batch, q) for q in qs]
    outs, streams = [torch.empty_like(q) for q in qs], [torch.cuda.Stream() for _ in qs]
    wss = [ops.attn_workspace(s.cache, s.batch, q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, q, o, w in zip(streams, qs, outs, wss):
            with torch.cuda.stream(st):
                ops.attn(s.cache, s.batch, q, out=o, ws=w)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_decode_block_end_to_end():
    """Two tokens of a block as an engine runs them: projections on Q8_1 rows, append, attention, output projection, residual
    add + norm, routed experts - every stage against 64 bits fed with the device's own inputs to it."""
    hidden, H, Hk, D, page, Q4_K = 512, 4, 2, 128, 16, 12
    s = Setup([1, 1], [70, 33], page, Hk, D, seed=53)
    x, xh = _rand(s.rng, (2, hidden))
    norm_w, nw2 = _rand(s.rng, (hidden,))[0], _rand(s.rng, (hidden,))[0]
    width = (H + 2 * Hk) * D
    wqkv = ops.quantize_weights(Q4_K, _rand(s.rng, (width, hidden), std=0.05)[0])
    wo = ops.quantize_weights(Q4_K, _rand(s.rng, (hidden, H * D), std=0.05)[0])
    freq = ops.rope_freqs(D)
    h, xq = ops.rms_norm_q8_1(x, norm_w, 1e-6)
    qkv = ops.mmvq(Q4_K, wqkv, hidden, width, xq, 2).view(2, H + 2 * Hk, D)
    qkv_h = qkv.double().cpu().numpy()
    q = ops.kv_append(s.cache, s.batch, qkv[:, H:H + Hk], qkv[:, H + Hk:], q=qkv[:, :H], rope=ops.ROPE_HALVES, inv_freq=freq)
    pos, f = s.positions(), freq.cpu().numpy()
    s.put(kd.rotate(qkv_h[:, H:H + Hk], pos, 1, f), qkv_h[:, H + Hk:])
    assert s.same_bytes() and _rounded_ok(q, kd.rotate(qkv_h[:, :H], pos, 1, f), "f32")
    att = ops.attn(s.cache, s.batch, q)
    ref, ax, vm = kd.attention(s.host, s.table, s.q_lens, s.kv_lens, q.double().cpu().numpy(), D ** -0.5)
    assert (np.abs(att.double().cpu().numpy() - ref) <= kd.attn_tolerance("f32", D, 70, ref, ax, vm)).all()
    y = ops.mmvq(Q4_K, wo, H * D, hidden, ops.quantize_q8_1(att.view(2, H * D)), 2)
    resid, h2, xq2 = ops.add_rms_norm_q8_1(x, y, nw2, 1e-6)
    assert torch.equal(resid, ops.add(x, y)) and np.array_equal(orc.quantize_q8_1(h2.cpu().numpy()), xq2.cpu().numpy())
    layer = synth.build_layer(hidden, 256, 16, 4, Q4_K, Q4_K, seed=7)
    ids, w = ops.route_topk(ops.gemv_router(layer.router_w, h2), 4)
    sl = layer.slots
    act = ops.mmvq_experts_swiglu(Q4_K, sl.table, sl.gate_off, sl.up_off, hidden, 256, xq2, 2, ids)
    down = ops.mmvq_experts(Q4_K, sl.table, sl.down_off, 256, hidden, ops.quantize_q8_1(act), 8, ids)
    got = ops.moe_combine(down.view(2, 4, hidden), w, x=resid)
    want = layer(h2, x_resid=resid)
    assert (got - want).abs().max() <= 1e-3 * want.abs().max()  # the layer's own chain (its Q8_1 codes may move by one)


def test_refusals_of_the_wrappers():
    s = Setup([2], [20], 16, 2, 64, seed=59)
    q, k = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    with pytest.raises(ValueError, match="kv heads"):
        ops.kv_append(s.cache, s.batch, q, q)
    with pytest.raises(ValueError, match="expected"):
        ops.kv_append(s.cache, s.batch, k, k.bfloat16())
    with pytest.raises(ValueError, match="expected"):
        ops.attn(s.cache, s.batch, q[:1])
    with pytest.raises(ValueError, match="expected"):
        ops.attn(s.cache, s.batch, q.half())
    with pytest.raises(ValueError, match="contiguous"):
        ops.attn(s.cache, s.batch, torch.zeros(2, 64, 4, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError, match="inv_freq"):
        ops.kv_append(s.cache, s.batch, k, k, rope=ops.ROPE_HALVES)
    with pytest.raises(ValueError, match="sinks"):
        ops.attn(s.cache, s.batch, q, sinks=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError, match="device"):
        ops.attn(s.cache, s.batch, q.cpu())
    with pytest.raises(FnsError, match="multiple"):
        ops.attn(s.cache, s.batch, torch.zeros(2, 3, 64, device="cuda"))
    with pytest.raises(FnsError, match="rope_dim"):
        ops.kv_append(s.cache, s.batch, k, k, rope=ops.ROPE_PAIRS, inv_freq=torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="pages"):
        ops.KvCache(3, 16, 2, 64, pages=torch.zeros(7, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError, match="int32"):
        ops.KvBatch(torch.zeros(2, device="cuda"), s.batch.kv_len, s.batch.page_table, 2, 2)
    with pytest.raises(ValueError, match="weights"):
        ops.add_rms_norm_q8_1(q.view(2, 256), q.view(2, 256), torch.zeros(64, device="cuda"), 1e-6)
    assert s.same_bytes()
