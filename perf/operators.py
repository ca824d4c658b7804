"""The attention half of a decoder block as cases that can be timed and checked.

Three operators join the FFN half that the framework runs (perf/cases.py):
  norm    the residual stream takes a sub-layer's output, its RMSNorm feeds the next sub-layer in f32 and in Q8_1 blocks
  append  new tokens' keys and values go into a paged cache held in 4 bits, keys and queries rotated on the way
  attn    grouped-query attention of the new tokens over that cache (causal, sliding window, sinks)

The cache. A page holds `page` positions of every kv head; a head's part of it is
  K codes [page][dim / 2]      byte b of a row: channels 2 b (low half) and 2 b + 1
  V codes [dim / 2][page]      byte column j = 16 i + r, r < 16: channels 32 i + r (low half) and 32 i + 16 + r
  K scales [page][dim / 32], V scales [page][dim / 32]   one byte e a block of 32 channels
A code is a sign and an index into 0, .5, 1, 1.5, 2, 3, 4, 6; a value is that times 2^(e - 127), e the least with
max |block| <= 7 * 2^(e - 127) (1 at least; 0 for a block of zeros), codes to nearest, ties to the even code.

A case is a dict: op; norm: rows, n; append and attn: dtype (of q, k, v, out), n_seq sequences of which every one
brings `q` new tokens (ragged: 0 to q) and then has `kv` positions (ragged: down to a sixteenth, but not below its new
tokens), heads, kv_heads, dim, page, rope (append: "none", "halves", "pairs") over rope_dim channels, window (0: none),
sinks.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
BASE = 500000.0  # of the rotation's frequencies
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed() -> list[dict]:
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 64}
    return [
        # a decode step's residual stream between attention and FFN
        {"name": "norm-1x2048", "op": "norm", "rows": 1, "n": 2048},
        # a ragged prompt end of a model with an uncommon width
        {"name": "norm-213x2880", "op": "norm", "rows": 213, "n": 2880},
        # a long prompt at once
        {"name": "norm-4096x4096", "op": "norm", "rows": 4096, "n": 4096},
        # one user's decode step
        {"name": "append-decode-1", "op": "append", "dtype": "f32", "n_seq": 1, "q": 1, "kv": 5000, "ragged": False,
         "rope": "halves", "rope_dim": 128, **gqa},
        # a server's step over many users, part of each head rotated, 16-bit activations
        {"name": "append-decode-61-bf16", "op": "append", "dtype": "bf16", "n_seq": 61, "q": 1, "kv": 4000,
         "ragged": True, "rope": "pairs", "rope_dim": 64, "heads": 16, "kv_heads": 2, "dim": 128, "page": 16},
        # a long prompt of odd length
        {"name": "append-prefill-4001", "op": "append", "dtype": "f32", "n_seq": 1, "q": 4001, "kv": 4001,
         "ragged": False, "rope": "halves", "rope_dim": 128, **gqa},
        # the start of a chat: one token over a short context, where launches count
        {"name": "attn-decode-500", "op": "attn", "dtype": "f32", "n_seq": 1, "q": 1, "kv": 500, "ragged": False,
         "window": 0, "sinks": False, **gqa},
        # a server's step: many users with contexts of all lengths
        {"name": "attn-decode-48x16k", "op": "attn", "dtype": "f32", "n_seq": 48, "q": 1, "kv": 16000, "ragged": True,
         "window": 0, "sinks": False, **gqa},
        # one user with a book in the context
        {"name": "attn-decode-1x131k", "op": "attn", "dtype": "bf16", "n_seq": 1, "q": 1, "kv": 131072, "ragged": False,
         "window": 0, "sinks": False, **gqa},
        # speculative decoding: four tokens checked at once, wide groups, learned sinks
        {"name": "attn-verify4-8x4k-sinks", "op": "attn", "dtype": "f32", "n_seq": 8, "q": 4, "kv": 4096,
         "ragged": False, "heads": 64, "kv_heads": 8, "dim": 64, "page": 32, "window": 0, "sinks": True},
        # prompts of several users, ragged, in a layer with a sliding window
        {"name": "attn-prefill-5x1021-window", "op": "attn", "dtype": "f32", "n_seq": 5, "q": 1021, "kv": 2500,
         "ragged": True, "window": 513, "sinks": True, **gqa},
        # the second chunk of a long prompt, over a cache that holds the first
        {"name": "attn-prefill-4096-at-4096", "op": "attn", "dtype": "bf16", "n_seq": 1, "q": 4096, "kv": 8192,
         "ragged": False, "window": 0, "sinks": False, **gqa},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng) -> dict:
    op = rng.choice(["norm", "append", "append", "attn", "attn", "attn"])
    if op == "norm":
        return {"op": op, "rows": _log_int(rng, 1, 8192), "n": 32 * _log_int(rng, 8, 256)}
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    c = {"op": op, "dtype": rng.choice(["f32", "f32", "bf16"]), "kv_heads": kv_heads, "dim": dim,
         "heads": kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 16]), "page": rng.choice([16, 32, 64, 128])}
    form = rng.choice(["decode", "decode", "verify", "prefill"])
    n_seq = _log_int(rng, 1, 64) if form != "prefill" else _log_int(rng, 1, 8)
    q = {"decode": 1, "verify": rng.randint(2, 8), "prefill": _log_int(rng, 9, 4096)}[form]
    past = _log_int(rng, 1, 131072 if op == "attn" else 20000) - 1
    c.update(n_seq=n_seq, q=q, kv=q + past, ragged=n_seq > 1 and rng.random() < 0.7)
    if op == "append":
        c["rope"] = rng.choice(["none", "halves", "halves", "pairs"])
        c["rope_dim"] = rng.choice([dim, dim, dim // 2])
    else:
        c["window"] = rng.choice([0, 0, _log_int(rng, 16, 4096)])
        c["sinks"] = rng.random() < 0.4
    return c


def draw(rng) -> dict:
    """A case of the same ranges that costs no more (bytes, products, cache to make) than the listed ones."""
    works = [work(c) for c in listed()]
    top = {key: max(w[key] for w in works) for key in ("bytes", "flops")}
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] > top["bytes"] or w["flops"] > top["flops"]:
            continue
        if c["op"] != "norm" and sum(_lens(c)[1]) * c["kv_heads"] * c["dim"] > 48 * 16000 * 1024:
            continue
        return c


def _lens(c: dict) -> tuple[list[int], list[int]]:
    """New tokens and positions (with them) of every sequence: a matter of the case, not of the seed."""
    if not c["ragged"]:
        return [c["q"]] * c["n_seq"], [c["kv"]] * c["n_seq"]
    rng = random.Random(c["n_seq"] * 1000003 + c["kv"] * 31 + c["q"])
    qs, kvs = [], []
    for i in range(c["n_seq"]):
        q = c["q"] if i == 0 else rng.randint(0, c["q"]) if c["q"] > 1 else int(i != 2)
        kv = c["kv"] if i == 0 else _log_int(rng, max(1, c["kv"] // 16), c["kv"])
        qs.append(q)
        kvs.append(max(q, kv))
    return qs, kvs


def _pairs(q: int, kv: int, window: int) -> tuple[int, int]:
    """(query, key) pairs that a sequence's mask leaves, and positions that any of its queries sees."""
    if q == 0:
        return 0, 0
    first = kv - q
    if not window:
        return q * first + q * (q + 1) // 2, kv
    lo = max(0, first - window + 1)
    return sum(min(p + 1, window) for p in range(first, kv)), kv - lo


def work(case: dict) -> dict:
    c = case
    if c["op"] == "norm":
        e = c["rows"] * c["n"]
        # x and y in; the sum, the norm, its codes with two 16-bit numbers a block out; the weights
        return {"bytes": e * 16 + e // 32 * 36 + 4 * c["n"], "flops": 10 * e}
    size = 2 if c["dtype"] == "bf16" else 4
    qs, kvs = _lens(c)
    tok, H, Hk, D = sum(qs), c["heads"], c["kv_heads"], c["dim"]
    row = Hk * (D // 2 + D // 32)  # a token's K or V in the cache
    if c["op"] == "append":
        return {"bytes": tok * ((2 * H + 2 * Hk) * D * size + 2 * row), "flops": tok * D * (3 * H + 10 * Hk)}
    pairs, seen = (sum(v) for v in zip(*(_pairs(q, kv, c["window"]) for q, kv in zip(qs, kvs))))
    return {"bytes": 2 * tok * H * D * size + seen * 2 * row, "flops": 4 * pairs * H * D}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _normal(shape, gen, std: float = 1.0) -> torch.Tensor:
    return torch.empty(*shape, device="cuda").normal_(0.0, std, generator=gen)


def _hold(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (uint8 [..., dim]) and block scales (uint8 [..., dim / 32]) of x; decided in x's own type."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    m, k = torch.frexp(amax)  # amax = m * 2^k, m in [.5, 1): at most 7 * 2^e for e = k - 3 where m <= 7 / 8
    e = (k + 124 + (m > 0.875).to(k.dtype)).clamp(1, 254)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    a = torch.ldexp(b.abs(), (127 - e).unsqueeze(-1))
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte())
    return (code + 8 * (b < 0).byte()).flatten(-2), e.byte()


def _values(st: dict, codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """f32 values of codes [..., dim] with scales [..., dim / 32]."""
    v = st["levels"][codes.int()].unflatten(-1, (-1, 32))
    return torch.ldexp(v, (scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _parts(c: dict, pages: torch.Tensor):
    """Views of pages [n][bytes]: K codes [n][Hk][page][dim / 2], V codes [n][Hk][dim / 2][page], the scales."""
    P, D, Hk = c["page"], c["dim"], c["kv_heads"]
    h = pages.view(pages.shape[0], Hk, P * (D + D // 16))
    a, s = P * D // 2, P * D // 32
    return (h[..., :a].unflatten(-1, (P, D // 2)), h[..., a:2 * a].unflatten(-1, (D // 2, P)),
            h[..., 2 * a:2 * a + s].unflatten(-1, (P, D // 32)), h[..., 2 * a + s:].unflatten(-1, (P, D // 32)))


def _k_bytes(code):  # [..., dim] -> [..., dim / 2]
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _k_codes(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _v_bytes(code):  # [..., dim] -> [..., dim / 2]
    h = code.unflatten(-1, (-1, 2, 16))
    return (h[..., 0, :] | (h[..., 1, :] << 4)).flatten(-2)


def _v_codes(b):
    h = b.unflatten(-1, (-1, 16))
    return torch.stack((h & 15, h >> 4), -2).flatten(-3)


def prepare(case: dict, seed: int) -> dict:
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed & 0x7FFFFFFFFFFFFFFF)
    if c["op"] == "norm":
        n = c["n"]
        return {"case": c, "x": _normal((c["rows"], n), gen, 3.0), "y": _normal((c["rows"], n), gen),
                "w": _normal((n,), gen, 0.1) + 1.0}
    qs, kvs = _lens(c)
    tok, H, Hk, D, P = sum(qs), c["heads"], c["kv_heads"], c["dim"], c["page"]
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    per = [(kv + P - 1) // P for kv in kvs]  # pages of a sequence, handed out in no order
    n_pages = sum(per) + 3
    perm = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed & 0x7FFFFFFF))[:sum(per)].int()
    table = torch.full((c["n_seq"], max(per)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = perm[at:at + n]
        at += n
    start = [0]
    for q in qs:
        start.append(start[-1] + q)
    pages = torch.zeros(n_pages, Hk * P * (D + D // 16), dtype=torch.uint8, device="cuda")
    kb, vb, ks, vs = _parts(c, pages)
    step = max(1, (1 << 25) // (Hk * P * D))
    for p in range(0, n_pages, step):  # what earlier calls appended: every position, a channel's size its own
        n = min(step, n_pages - p)
        size = 0.2 + torch.rand(Hk, 1, D, device="cuda", generator=gen) ** 4 * 4
        code, e = _hold(_normal((n, Hk, P, D), gen) * size)
        kb[p:p + n], ks[p:p + n] = _k_bytes(code), e
        code, e = _hold(_normal((n, Hk, P, D), gen))
        vb[p:p + n], vs[p:p + n] = _v_bytes(code).transpose(-1, -2), e
    st = {"case": c, "qs": qs, "kvs": kvs, "pages": pages, "table": table.cuda(),
          "start": torch.tensor(start, dtype=torch.int32, device="cuda"),
          "kv_len": torch.tensor(kvs, dtype=torch.int32, device="cuda"),
          "q": _normal((tok, H, D), gen).to(dt), "levels": torch.tensor(LEVELS + tuple(-v for v in LEVELS)).cuda()}
    if c["op"] == "append":
        st["k"], st["v"] = _normal((tok, Hk, D), gen, 2.0).to(dt), _normal((tok, Hk, D), gen).to(dt)
        r = c["rope_dim"]
        st["freq"] = (BASE ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)).float().cuda()
    else:
        st["scale"] = D ** -0.5
        st["sinks"] = _normal((H,), gen) if c["sinks"] else None
    if own:
        from flintnsteel_amd import ops
        st["cache"] = ops.KvCache(n_pages, P, Hk, D, pages=pages)
        st["batch"] = ops.KvBatch(st["start"], st["kv_len"], st["table"], n_tok=tok, max_q=max(qs), max_kv=max(kvs))
        if c["op"] == "attn":
            st["out"] = torch.empty_like(st["q"])
            st["ws"] = ops.attn_workspace(st["cache"], st["batch"], st["q"])
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st: dict):
    from flintnsteel_amd import ops
    c = st["case"]
    if c["op"] == "norm":
        s, h, xq = ops.add_rms_norm_q8_1(st["x"], st["y"], st["w"], EPS)
        return (s, h, *ops.dequantize_q8_1(xq, c["n"], dtype=torch.float16))  # the type of a block's scale and sum
    if c["op"] == "append":
        rope = {"none": ops.ROPE_NONE, "halves": ops.ROPE_HALVES, "pairs": ops.ROPE_PAIRS}[c["rope"]]
        q = ops.kv_append(st["cache"], st["batch"], st["k"], st["v"], q=st["q"], rope=rope,
                          inv_freq=st["freq"] if rope else None)
        return (q, *ops.kv_read(st["cache"], st["batch"]))
    return ops.attn(st["cache"], st["batch"], st["q"], scale=st["scale"], window=c["window"], sinks=st["sinks"],
                    out=st["out"], ws=st["ws"])


def _rotated(c: dict, x: torch.Tensor, pos: torch.Tensor, freq: torch.Tensor) -> torch.Tensor:
    x = x.double()  # a far position's angle, and codes next to a border
    if c["rope"] == "none":
        return x
    r = c["rope_dim"]
    t = (pos.double()[:, None] * freq.double())[:, None, :]
    cos, sin = t.cos(), t.sin()
    head, rest = x[..., :r], x[..., r:]
    if c["rope"] == "halves":
        a, b = head[..., :r // 2], head[..., r // 2:]
        head = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((head, rest), -1)


def _places(st: dict):
    """Position, page and row in the page of every new token."""
    c, table = st["case"], st["table"]
    dev = table.device
    pos = torch.cat([torch.arange(kv - q, kv, device=dev) for q, kv in zip(st["qs"], st["kvs"])])
    seq = torch.cat([torch.full((q,), i, device=dev) for i, q in enumerate(st["qs"])])
    return pos, table[seq, pos // c["page"]].long(), pos % c["page"]


def _run_plain(st: dict):
    c = st["case"]
    if c["op"] == "norm":
        s = st["x"] + st["y"]
        h = (s * torch.rsqrt((s * s).double().mean(-1, keepdim=True) + EPS).float() * st["w"])
        b = h.unflatten(-1, (-1, 32))
        d = b.abs().amax(-1, keepdim=True) / 127.0
        v = torch.where(d > 0, b / d, torch.zeros_like(b))
        q = torch.sign(v) * torch.floor(v.abs() + 0.5)
        return s, h, (q * d.half().float()).flatten(-2).half(), b.sum(-1).half()
    pages = st["pages"]
    kb, vb, ks, vs = _parts(c, pages)
    if c["op"] == "append":
        pos, page, row = _places(st)
        q = _rotated(c, st["q"], pos, st["freq"]).to(st["q"].dtype)
        code, e = _hold(_rotated(c, st["k"], pos, st["freq"]))
        kb[page, :, row], ks[page, :, row] = _k_bytes(code), e
        code, e = _hold(st["v"].float())
        vb[page, :, :, row], vs[page, :, row] = _v_bytes(code), e
        return (q, _values(st, _k_codes(kb[page, :, row]), ks[page, :, row]),
                _values(st, _v_codes(vb[page, :, :, row]), vs[page, :, row]))
    H, Hk, D, P = c["heads"], c["kv_heads"], c["dim"], c["page"]
    G, at, outs = H // Hk, 0, []
    for i, (n, kv) in enumerate(zip(st["qs"], st["kvs"])):
        if n == 0:
            continue
        lo = max(0, kv - n - c["window"] + 1) // P * P if c["window"] else 0
        page = st["table"][i, lo // P:(kv + P - 1) // P].long()
        q = st["q"][at:at + n].float().view(n, Hk, G, D)
        at += n
        qpos = torch.arange(kv - n, kv, device=q.device)[:, None]
        kpos = torch.arange(lo, kv, device=q.device)[None, :]
        off = (kpos > qpos) | ((kpos <= qpos - c["window"]) if c["window"] else torch.zeros_like(kpos > qpos))
        out = torch.empty(n, Hk, G, D, device=q.device)
        for h in range(Hk):  # a kv head and its group of query heads at a time
            K = _values(st, _k_codes(kb[page, h]), ks[page, h]).flatten(0, 1)[:kv - lo]
            V = _values(st, _v_codes(vb[page, h].transpose(-1, -2)), vs[page, h]).flatten(0, 1)[:kv - lo]
            s = torch.matmul(q[:, h].reshape(n * G, D), K.t().contiguous()).view(n, G, -1) * st["scale"]
            s = s.masked_fill_(off[:, None, :], -math.inf)
            m = s.amax(-1, keepdim=True)
            extra = torch.zeros_like(m)
            if st["sinks"] is not None:
                sink = st["sinks"][h * G:(h + 1) * G][None, :, None]
                m = torch.maximum(m, sink)
                extra = (sink - m).exp()
            p = (s - m).exp_()
            p = p / (p.sum(-1, keepdim=True) + extra)
            out[:, h] = torch.matmul(p.view(n * G, -1), V).view(n, G, D)
        outs.append(out.view(n, H, D))
    return torch.cat(outs).to(st["q"].dtype)


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------

def _nearest(x: torch.Tensor) -> torch.Tensor:
    """What the cache's 4 bits hold of x (f64 [..., dim]), as f64."""
    lv = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 7))
    e = torch.where(torch.pow(2.0, e - 1) * 7 >= top, e - 1, e)  # the logarithm may be off next to a whole number
    e = torch.where(torch.pow(2.0, e) * 7 < top, e + 1, e).clamp(-126, 127)
    unit = torch.pow(2.0, e)
    a = (b / unit).abs()
    up = torch.bucketize(a, lv).clamp(max=7)      # the level not below a, and the one before it
    dn = (up - 1).clamp_min(0)
    du, dd = lv[up] - a, a - lv[dn]
    pick = torch.where((du < dd) | ((du == dd) & (up % 2 == 0)), up, dn)
    return (torch.sign(b) * lv[pick] * unit).reshape(x.shape)


def _turn(c: dict, x: torch.Tensor, pos: torch.Tensor, freq: torch.Tensor) -> torch.Tensor:
    x = x.to(torch.float64)
    if c["rope"] == "none":
        return x
    out, half = x.clone(), c["rope_dim"] // 2
    i = torch.arange(half, device=x.device)
    first, second = (i, i + half) if c["rope"] == "halves" else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., first], x[..., second])
    angle = pos.to(torch.float64)[:, None, None] * freq.to(torch.float64)[None, None, :]
    z = z * torch.polar(torch.ones_like(angle), angle)
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _cached(c: dict, pages: torch.Tensor, table: torch.Tensor, lo: int, hi: int, head: int):
    """K and V (f64 [hi - lo][dim]) of positions lo .. hi - 1 of one kv head, read byte by byte from their places."""
    P, D, dev = c["page"], c["dim"], pages.device
    pos = torch.arange(lo, hi, device=dev)
    base = (table[pos // P].long() * pages.shape[1] + head * P * (D + D // 16))[:, None]
    row, ch = (pos % P)[:, None], torch.arange(D, device=dev)[None, :]
    flat = pages.reshape(-1)
    k = (flat[base + row * (D // 2) + ch // 2] >> (4 * (ch % 2)).byte()) & 15
    v = (flat[base + P * D // 2 + (ch // 32 * 16 + ch % 16) * P + row] >> (ch % 32 // 16 * 4).byte()) & 15
    ke = flat[base + P * D + row * (D // 32) + ch // 32]
    ve = flat[base + P * D + P * D // 32 + row * (D // 32) + ch // 32]
    lv = torch.tensor(LEVELS, dtype=torch.float64, device=dev)
    val = lambda code, e: (lv[(code & 7).long()] * torch.where(code > 7, -1.0, 1.0)  # noqa: E731
                           * torch.pow(2.0, e.double() - 127))
    return val(k, ke), val(v, ve)


def exact(case: dict, seed: int):
    c, st = case, prepare(case, seed)
    if c["op"] == "norm":
        s = st["x"].double() + st["y"].double()
        h = s / torch.sqrt(s.pow(2).mean(-1, keepdim=True) + EPS) * st["w"].double()
        b = h.reshape(c["rows"], -1, 32)
        d = b.abs().max(-1, keepdim=True).values / 127
        v = b / d.clamp_min(1e-300)
        v = torch.where(v < 0, torch.ceil(v - 0.5), torch.floor(v + 0.5))
        return s, h, (v * d.half().double()).reshape(h.shape), b.sum(-1)
    if c["op"] == "append":
        pos = torch.cat([torch.arange(kv - q, kv) for q, kv in zip(st["qs"], st["kvs"])]).cuda()
        return (_turn(c, st["q"], pos, st["freq"]), _nearest(_turn(c, st["k"], pos, st["freq"])),
                _nearest(st["v"].double()))
    H, Hk, D = c["heads"], c["kv_heads"], c["dim"]
    G, out, t = H // Hk, torch.zeros(sum(st["qs"]), H, D, dtype=torch.float64, device="cuda"), 0
    for i, (n, kv) in enumerate(zip(st["qs"], st["kvs"])):
        for h in range(Hk if n else 0):
            K, V = _cached(c, st["pages"], st["table"][i], 0, kv, h)
            for a in range(0, n, 512):  # some queries of every head of the group at a time
                m = min(512, n - a)
                p = torch.arange(kv - n + a, kv - n + a + m, device="cuda")
                j = torch.arange(kv, device="cuda")
                see = j[None, :] <= p[:, None]
                if c["window"]:
                    see = see & (j[None, :] > p[:, None] - c["window"])
                for g in range(G):
                    x = st["q"][t + a:t + a + m, h * G + g].double() @ K.T * st["scale"]
                    x = torch.where(see, x, torch.full_like(x, -math.inf))
                    if st["sinks"] is not None:
                        x = torch.cat((x, st["sinks"][h * G + g].double().expand(m, 1)), 1)
                    w = torch.softmax(x, -1)[:, :kv]
                    out[t + a:t + a + m, h * G + g] = w @ V
        t += n
    return out
