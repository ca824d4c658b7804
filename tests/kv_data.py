"""The paged 4-bit cache and attention over it from their definitions, in 64 bits on the CPU: what the tests of
fns_hip_kv_append, fns_hip_kv_read and fns_hip_attn hold the kernels to."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
F32_STEP, BF16_STEP, F16_STEP = 2.0 ** -24, 2.0 ** -8, 2.0 ** -11  # half a step, relative to the value


def codes_of(x: np.ndarray):
    """(codes [..., D], scale bytes [..., D / 32]) of f64 x: the least scale with max <= 7 units, nearest code, ties to even."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    m, k = np.frexp(top)
    e = np.clip(k - 3 + (m > 0.875) + 127, 1, 254)
    e = np.where(top == 0, 0, e)
    a = np.ldexp(np.abs(b), (127 - e)[..., None])
    dist = np.abs(a[..., None] - LEVELS)
    hit = dist == dist.min(-1, keepdims=True)
    first = hit.argmax(-1)
    code = first + (hit.sum(-1) > 1) * (first % 2)  # of two levels at the same distance, the even one
    code = code + 8 * (b < 0)
    code = np.where(bad[..., None], 0, code)
    e = np.where(bad, 255, e)
    return code.reshape(x.shape).astype(np.uint8), e.astype(np.uint8)


def values_of(code: np.ndarray, e: np.ndarray) -> np.ndarray:
    v = (LEVELS[code & 7] * np.where(code > 7, -1, 1)).reshape(*code.shape[:-1], -1, 32)
    v = np.ldexp(v, (e.astype(np.int64) - 127)[..., None])
    v = np.where((e == 255)[..., None], np.nan, v)
    return v.reshape(code.shape)


def rotate(x: np.ndarray, pos: np.ndarray, rope: int, inv_freq) -> np.ndarray:
    """x [n][heads][D] f64 at positions pos [n]; rope 0 none, 1 halves, 2 pairs."""
    x = np.array(x, np.float64)
    if rope == 0:
        return x
    half = len(inv_freq)
    t = pos.astype(np.longdouble)[:, None] * np.asarray(inv_freq, np.float32).astype(np.longdouble)[None, :]
    c, s = np.cos(t).astype(np.float64)[:, None], np.sin(t).astype(np.float64)[:, None]
    i = np.arange(half)
    u, w = (i, i + half) if rope == 1 else (2 * i, 2 * i + 1)
    a, b = x[..., u].copy(), x[..., w].copy()
    x[..., u], x[..., w] = a * c - b * s, a * s + b * c
    return x


class Pages:
    """A cache as bytes [n_pages][page_bytes] on the host."""

    def __init__(self, n_pages: int, page: int, heads: int, dim: int, fill=None):
        self.n_pages, self.page, self.heads, self.dim = n_pages, page, heads, dim
        self.head_bytes = page * (dim + dim // 16)
        rng = np.random.default_rng(0 if fill is None else fill)
        self.raw = rng.integers(0, 256, (n_pages, heads * self.head_bytes)).astype(np.uint8)

    def put(self, page: int, row: int, head: int, k: np.ndarray, v: np.ndarray) -> None:
        P, D, o = self.page, self.dim, head * self.head_bytes
        r = self.raw[page]
        code, e = codes_of(k)
        r[o + row * D // 2: o + (row + 1) * D // 2] = code[0::2] | (code[1::2] << 4)
        r[o + P * D + row * (D // 32): o + P * D + (row + 1) * (D // 32)] = e
        code, e = codes_of(v)
        for j in range(D // 2):
            c = j // 16 * 32 + j % 16
            r[o + P * D // 2 + j * P + row] = code[c] | (code[c + 16] << 4)
        s = o + P * D + P * (D // 32) + row * (D // 32)
        r[s: s + D // 32] = e

    def get(self, pages: np.ndarray, rows: np.ndarray, head: int):
        """K, V f64 [n][D] of positions given by page and row."""
        P, D, o = self.page, self.dim, head * self.head_bytes
        ch = np.arange(D)[None, :]
        p, r = pages[:, None], rows[:, None]
        k = (self.raw[p, o + r * (D // 2) + ch // 2] >> (4 * (ch % 2))) & 15
        v = (self.raw[p, o + P * D // 2 + (ch // 32 * 16 + ch % 16) * P + r] >> (4 * (ch % 32 // 16))) & 15
        b = np.arange(D // 32)[None, :]
        ke = self.raw[p, o + P * D + r * (D // 32) + b]
        ve = self.raw[p, o + P * D + P * (D // 32) + r * (D // 32) + b]
        return values_of(k.astype(np.uint8), ke), values_of(v.astype(np.uint8), ve)

    def sane(self, seed: int = 1) -> "Pages":
        """Scale bytes of ordinary values everywhere (the random bytes of a fresh cache reach 2^127)."""
        rng = np.random.default_rng(seed)
        P, D = self.page, self.dim
        for h in range(self.heads):
            o = h * self.head_bytes + P * D
            self.raw[:, o: o + P * D // 16] = rng.integers(120, 128, (self.n_pages, P * D // 16))
        return self


def attention(cache: Pages, table: np.ndarray, q_lens, kv_lens, q: np.ndarray, scale: float, window: int = 0, sinks=None):
    """(out f64 [sum q][H][D], ax [sum q][H][2], vm): the result, and for the tolerances per row scale * max_j sum_i |q_i K_ji|
    and scale * max_i |q_i| * max_j sum_i |K_ji|, and max |V|, over what the row sees."""
    H, D = q.shape[1], q.shape[2]
    G = H // cache.heads
    out, ax, vm, t = np.zeros(q.shape), np.zeros((*q.shape[:2], 2)), np.zeros(q.shape[:2]), 0
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        for h in range(cache.heads if n else 0):
            pos = np.arange(kv)
            idx = pos // cache.page
            pg = np.where(idx < table.shape[1], table[s, np.minimum(idx, table.shape[1] - 1)], -1)
            there = (pg >= 0) & (pg < cache.n_pages)
            K, V = cache.get(np.where(there, pg, 0), pos % cache.page, h)
            for i in range(n):
                p = kv - n + i
                see = there & (pos <= p) & ((pos > p - window) if window else True)
                for g in range(G):
                    hh = h * G + g
                    if not see.any():
                        continue
                    k, v = K[see], V[see]
                    x = k @ q[t + i, hh] * scale
                    m = max(x.max(), sinks[hh]) if sinks is not None else x.max()
                    w = np.exp(x - m)
                    out[t + i, hh] = w @ v / (w.sum() + (np.exp(sinks[hh] - m) if sinks is not None else 0.0))
                    if np.isnan(k).any() or np.isnan(v).any():
                        out[t + i, hh] = np.nan
                    aq, ak = np.abs(q[t + i, hh]), np.abs(k)
                    ax[t + i, hh] = scale * (ak @ aq).max(), scale * aq.max() * ak.sum(-1).max()
                    vm[t + i, hh] = np.abs(v).max()
        t += n
    return out, ax, vm


def attn_tolerance(dtype: str, D: int, n: int, ref: np.ndarray, ax: np.ndarray, vm: np.ndarray) -> np.ndarray:
    """What rounding allows, per element. A query row enters the products as a sum of 5 (f32) or 3 (bf16) e2m3 digits, each 32
    times finer than the one before: with the largest element in [2, 4) the first digit leaves 1/8 (half of a step of 1/4),
    each further one 1/32 of that, so 2^-3 2^-20 <= 2^-24 of the largest (2^-3 2^-10 <= 2^-14): a score is off by that times
    scale * max |q_i| * sum |K_i| = ax[1]. Multiplying the row by scale * log2(e) costs two half steps, its products are exact,
    and their f32 sums, one instruction a digit and 128 channels, are given D + 8 half steps of scale * sum |q_i K_i| = ax[0]
    (which bounds the running maximum that they start from, too); exp2's argument and result add 4 half steps of |x| <= ax[0]
    and of 1. A probability that is off by the factor 1 + r moves the output by at most 2 r vmax (numerator and denominator).
    p itself is carried to 2^-21 (f32) or 2^-10 (bf16: 11 bits, toward zero; the sum of p counts the same values, which
    leaves what differs from key to key), sums over n keys by n half steps at worst; the result is rounded to its type."""
    h, bf16 = F32_STEP, dtype == "bf16"
    x = ax[..., 0] * (D + 14) * h + ax[..., 1] * 2.0 ** (-14 if bf16 else -24)
    r = x + 4 * h + n * h + 2.0 ** (-11 if bf16 else -21)
    out = BF16_STEP if bf16 else 4 * h
    return 2 * (r * vm)[..., None] + np.abs(ref) * out + 1e-37
