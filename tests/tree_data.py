"""Trees of drafted tokens, attention weights and eviction from their definitions, in 64 bits on the CPU: what the tests of
fns_hip_attn_tree, fns_hip_kv_weigh, fns_hip_kv_evict and fns_hip_kv_keep hold the kernels to."""
from __future__ import annotations

import numpy as np

import kv_data as kd


def random_parents(rng, n: int, pads: int = 0) -> list[int]:
    """n new tokens of which the last `pads` are no token of the tree."""
    rows = [-1] + [int(rng.integers(max(-1, i - 6), i)) for i in range(1, n - pads)]
    return (rows[: n - pads] + [-2] * pads)[:n]


def seen_by(parents: list[int]) -> list[list[int]]:
    """Of every token the new tokens that it sees: itself and its ancestors; nothing if it is no token of the tree."""
    rows: list = []
    for i, p in enumerate(parents):
        up = None if p < -1 or p >= i else [] if p == -1 else rows[p]
        rows.append(None if up is None else [*up, i])
    return [r or [] for r in rows]


def words_of(rows: list[list[int]], words: int) -> np.ndarray:
    out = np.zeros((len(rows), words), np.uint64)
    for i, row in enumerate(rows):
        for j in row:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def mask(n: int, kv: int, window: int, rows=None) -> np.ndarray:
    """[n][kv]: whether new token i sees position j. rows: of a tree; None: causal."""
    j, first = np.arange(kv), kv - n
    see = np.zeros((n, kv), bool)
    for i in range(n):
        if rows is None:
            p = first + i
            see[i] = (j <= p) & ((j > p - window) if window else True)
        elif rows[i]:
            see[i] = j < first
            if window:
                see[i] &= j >= first - max(0, window - len(rows[i]))
            new = np.array([first + t for t in rows[i]])
            see[i, new[(new >= 0) & (new < kv)]] = True
    return see


def _keys(cache: kd.Pages, table: np.ndarray, s: int, kv: int, h: int):
    if kv == 0:
        return np.zeros((0, cache.dim)), np.zeros((0, cache.dim)), np.zeros(0, bool), np.zeros(0, int)
    pos = np.arange(kv)
    idx = pos // cache.page
    pg = np.where(idx < table.shape[1], table[s, np.minimum(idx, table.shape[1] - 1)], -1)
    there = (pg >= 0) & (pg < cache.n_pages)
    K, V = cache.get(np.where(there, pg, 0), pos % cache.page, h)
    return K, V, there, pg


def attention(cache: kd.Pages, table, q_lens, kv_lens, q, scale, window=0, sinks=None, rows=None):
    """(out, lse, ax, vm) as kv_data.attention, and the logarithms of the denominators; rows: of every sequence, or None."""
    H = q.shape[1]
    G = H // cache.heads
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    ax, vm, t = np.zeros((*q.shape[:2], 2)), np.zeros(q.shape[:2]), 0
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        see = mask(n, kv, window, None if rows is None else rows[s])
        for h in range(cache.heads if n else 0):
            K, V, there, _ = _keys(cache, table, s, kv, h)
            for i in range(n):
                on = see[i] & there
                for g in range(G):
                    hh = h * G + g
                    if not on.any():
                        if sinks is not None:
                            lse[t + i, hh] = sinks[hh]
                        continue
                    k, v = K[on], V[on]
                    x = k @ q[t + i, hh] * scale
                    m = max(x.max(), sinks[hh]) if sinks is not None else x.max()
                    w = np.exp(x - m)
                    den = w.sum() + (np.exp(sinks[hh] - m) if sinks is not None else 0.0)
                    out[t + i, hh], lse[t + i, hh] = w @ v / den, m + np.log(den)
                    if np.isnan(k).any() or np.isnan(v).any():
                        out[t + i, hh] = lse[t + i, hh] = np.nan
                    aq, ak = np.abs(q[t + i, hh]), np.abs(k)
                    ax[t + i, hh] = abs(scale) * (ak @ aq).max(), abs(scale) * aq.max() * ak.sum(-1).max()
                    vm[t + i, hh] = np.abs(v).max()
        t += n
    return out, lse, ax, vm


def lse_tolerance(dtype: str, D: int, n: int, lse: np.ndarray, ax: np.ndarray) -> np.ndarray:
    """A score is off as kv_data.attn_tolerance says (queries as digits, f32 sums of products), a term of the sum by exp2's 4 half
    steps and (f32) p's 2^-21; n terms are summed in f32. The logarithm moves by those relative errors. It is taken in log2 units
    (of up to |lse| log2(e) and the running maximum, bounded by ax[0], plus log2 of a sum that is carried 2^8 up, below 64),
    each of its four operations within two half steps of what it handles."""
    h = kd.F32_STEP
    x = ax[..., 0] * (D + 14) * h + ax[..., 1] * 2.0 ** -24  # (queries of either type enter as f32 does)
    return x + 4 * h + n * h + 2.0 ** -21 + 8 * h * (np.abs(np.where(np.isfinite(lse), lse, 0)) + ax[..., 0] + 64)


def weigh(cache: kd.Pages, table, q_lens, kv_lens, q, lse, past, scale, window=0, rows=None, keep=None):
    """(weights, tolerance) f64 [n_pages][heads][page], with what `past` (or `keep`, where positions are left alone) has
    elsewhere. A pair's score is off by D + 14 half steps of scale * sum |q_i K_i|, 2^-24 of scale * max |q_i| * sum |K_i| (the
    digits), and by half steps of the start -lse in log2 units (two roundings) and of the running sums, bounded by both; exp2
    adds 4 half steps. The rows are summed in f32, at most one half step a term at worst."""
    h2 = kd.F32_STEP
    H, D = q.shape[1:]
    G, t = H // cache.heads, 0
    w = np.array(past if keep is None else keep, np.float64)
    tol = np.zeros(w.shape)
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        see = mask(n, kv, window, None if rows is None else rows[s])
        for h in range(cache.heads if n else 0):
            K, _, there, pg = _keys(cache, table, s, kv, h)
            bad = np.isnan(K).any(-1)
            k = np.where(bad[:, None], 0.0, K)
            for j in np.flatnonzero(there):
                old = 0.0 if past is None or j >= kv - n else float(past[pg[j], h, j % cache.page])
                w[pg[j], h, j % cache.page] = old
                tol[pg[j], h, j % cache.page] = abs(old) * h2
            total, off = np.zeros(kv), np.zeros(kv)
            for g in range(G):
                hh = h * G + g
                for i in range(n):
                    z, qq = lse[t + i, hh], q[t + i, hh]
                    if not np.isfinite(z) or not np.isfinite(qq).all():
                        continue
                    on = see[i] & there & ~bad
                    x = k @ qq * scale
                    size = np.abs(k) @ np.abs(qq) * abs(scale)
                    p = np.where(on, np.exp(np.where(on, x - z, -np.inf)), 0.0)
                    e = size * (D + 14) * h2 + abs(scale) * np.abs(qq).max() * np.abs(k).sum(-1) * 2.0 ** -24
                    total += p
                    off += p * np.expm1(e + 8 * h2 * (abs(z) + size) + 6 * h2)
            off += total * h2 * (n * G + 8) + 1e-37
            for j in np.flatnonzero(there):
                w[pg[j], h, j % cache.page] += total[j]
                tol[pg[j], h, j % cache.page] += off[j] + h2 * total[j]
        t += n
    return w, tol


def evicted(w: np.ndarray, there: np.ndarray, budget: int, first: int, recent: int) -> list[int]:
    """Positions that a kv head keeps of weights w [n] (f32 values), in order."""
    n = len(w)
    key = [(0 if j < first or j >= n - recent else 1, 0 if np.isnan(w[j]) else 1, -w[j] if not np.isnan(w[j]) else 0.0, j) for j in range(n) if there[j]]
    return sorted(k[-1] for k in sorted(key)[:budget])


def slot_bytes(cache: kd.Pages, page: int, row: int, head: int) -> np.ndarray:
    """Indices, within a page, of the bytes that hold one position of one kv head."""
    P, D, o = cache.page, cache.dim, head * cache.head_bytes
    nb = D // 32
    return o + np.concatenate([row * (D // 2) + np.arange(D // 2), P * D // 2 + np.arange(D // 2) * P + row,
                               P * D + row * nb + np.arange(nb), P * (D + nb) + row * nb + np.arange(nb)])


def move(cache: kd.Pages, raw: np.ndarray, moves) -> np.ndarray:
    """raw with positions copied, all reads first: moves of ((page, row) from, (page, row) to, head)."""
    out = raw.copy()
    for (a, i), (b, k), h in moves:
        out[b, slot_bytes(cache, b, k, h)] = raw[a, slot_bytes(cache, a, i, h)]
    return out
