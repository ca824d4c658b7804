"""Drafted trees and bounded caches over the 4-bit paged cache, as cases that can be timed and checked.

  append  new tokens go into the cache at rotary positions of their own (a tree's depths, a cache that has lost tokens),
          with frequencies and a magnitude scaled for long contexts
  tree    attention of a tree of drafted tokens over the cache, with the logarithms of the rows' denominators
  weigh   the attention weight that every cached position gets from the new tokens, added to what it got before
  evict   each kv head keeps the first, the last and the heaviest positions of a sequence, in order, on other pages
  verify  a layer's whole step: the tree's masks from parents, append, attention, the accepted path made the sequence's own

The cache. A page holds `page` positions of every kv head; a head's part of it is
  K codes [page][dim / 2]      byte b of a row: channels 2 b (low half) and 2 b + 1
  V codes [dim / 2][page]      byte column j = 16 i + r, r < 16: channels 32 i + r (low half) and 32 i + 16 + r
  K scales [page][dim / 32], V scales [page][dim / 32]   one byte e a block of 32 channels
A code is a sign and an index into 0, .5, 1, 1.5, 2, 3, 4, 6; a value is that times 2^(e - 127), e the least with
max |block| <= 7 * 2^(e - 127) (1 at least; 0 for a block of zeros), codes to nearest, ties to the even code. Weights
are f32 [pages][kv_heads][page].

A tree. Bit j of a token's mask: it sees the j-th new token of its sequence. It sees all earlier positions too, with a
window only as many of the last ones as the mask leaves of it; a token with an empty mask sees nothing.

A case is a dict: op; n_seq sequences of which every one brings `q` new tokens (ragged: fewer, 0 among them) and then has
`kv` positions (ragged: down to a sixteenth, but not below its new tokens), heads, kv_heads, dim, page; form of the new
tokens ("chain" or "tree"); dtype of q, k, v, out; append and verify: rope over rope_dim channels, scale (of the context),
ahead (how far a text's position is in front of its place in the cache); tree: window, sinks; evict: budget, first, recent.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BASE = 500000.0  # of the rotation's frequencies
ORIGINAL = 8192  # positions that they were made for, before scaling
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed() -> list[dict]:
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128, "page": 64}
    wide = {"heads": 64, "kv_heads": 8, "dim": 64, "page": 32}
    return [
        # one user's drafted tree, far into a text of which the cache holds a part
        {"name": "append-tree-26", "op": "append", "dtype": "f32", "n_seq": 1, "q": 26, "kv": 5026, "ragged": False,
         "form": "tree", "rope": "halves", "rope_dim": 128, "scale": 16.0, "ahead": 90000, **gqa},
        # a long prompt of odd length, part of each head rotated, 16-bit activations
        {"name": "append-prompt-3877", "op": "append", "dtype": "bf16", "n_seq": 1, "q": 3877, "kv": 3877,
         "ragged": False, "form": "chain", "rope": "pairs", "rope_dim": 64, "scale": 4.0, "ahead": 0, **gqa},
        # one user's tree over a short context, where launches count
        {"name": "tree-26-at-700", "op": "tree", "dtype": "f32", "n_seq": 1, "q": 26, "kv": 726, "ragged": False,
         "form": "tree", "window": 0, "sinks": False, **gqa},
        # a server's step: trees of several users, wide groups, learned sinks
        {"name": "tree-8x63-at-4k-sinks", "op": "tree", "dtype": "bf16", "n_seq": 8, "q": 63, "kv": 4200, "ragged": True,
         "form": "tree", "window": 0, "sinks": True, **wide},
        # one user with a book in the context
        {"name": "tree-60-at-100k", "op": "tree", "dtype": "f32", "n_seq": 1, "q": 60, "kv": 100000, "ragged": False,
         "form": "tree", "window": 0, "sinks": False, **gqa},
        # one user's decode step in a chat
        {"name": "weigh-decode-1x1500", "op": "weigh", "dtype": "f32", "n_seq": 1, "q": 1, "kv": 1500, "ragged": False,
         "form": "chain", **gqa},
        # a server's decode step
        {"name": "weigh-decode-24x16k", "op": "weigh", "dtype": "bf16", "n_seq": 24, "q": 1, "kv": 16000, "ragged": True,
         "form": "chain", **gqa},
        # a prompt, whose tokens weigh each other
        {"name": "weigh-prompt-2801", "op": "weigh", "dtype": "f32", "n_seq": 1, "q": 2801, "kv": 2801, "ragged": False,
         "form": "chain", **gqa},
        # one user's cache, a page over its bound
        {"name": "evict-1x4160", "op": "evict", "n_seq": 1, "q": 1, "kv": 4160, "ragged": False, "budget": 4096,
         "first": 4, "recent": 512, "form": "chain", "dtype": "f32", **gqa},
        # prompts of several users cut to what decoding keeps
        {"name": "evict-16x20k", "op": "evict", "n_seq": 16, "q": 1, "kv": 20000, "ragged": True, "budget": 2048,
         "first": 4, "recent": 256, "form": "chain", "dtype": "f32", **gqa},
        # a layer of one user's verify step
        {"name": "verify-1x26-at-2k", "op": "verify", "dtype": "f32", "n_seq": 1, "q": 26, "kv": 2074, "ragged": False,
         "form": "tree", "rope": "halves", "rope_dim": 128, "scale": 1.0, "ahead": 0, "window": 0, "sinks": False, **gqa},
        # the same for a server's users
        {"name": "verify-24x32-at-3k", "op": "verify", "dtype": "bf16", "n_seq": 24, "q": 32, "kv": 2900, "ragged": True,
         "form": "tree", "rope": "halves", "rope_dim": 64, "scale": 8.0, "ahead": 1000, "window": 0, "sinks": False,
         **wide},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng) -> dict:
    op = rng.choice(["append", "tree", "tree", "weigh", "weigh", "evict", "verify"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    c = {"op": op, "dtype": rng.choice(["f32", "f32", "bf16"]), "kv_heads": kv_heads, "dim": dim,
         "heads": kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8]), "page": rng.choice([16, 32, 64, 128]), "form": "chain"}
    past = _log_int(rng, 1, 131072) - 1
    if op == "evict":
        kv = _log_int(rng, 2, 131072)
        budget = max(1, min(_log_int(rng, 1, 65536), kv + 40))
        first = min(budget, rng.choice([0, 1, 4, 100]))
        c.update(n_seq=_log_int(rng, 1, 32), q=1, kv=kv, budget=budget, first=first,
                 recent=rng.randint(0, budget - first) // rng.choice([1, 4, 16]))
        c["ragged"] = c["n_seq"] > 1 and rng.random() < 0.7
        return c
    form = {"append": ["tree", "decode", "prompt"], "tree": ["tree"], "verify": ["tree"],
            "weigh": ["tree", "decode", "decode", "prompt"]}[op]
    form = rng.choice(form)
    q = {"tree": _log_int(rng, 2, 150), "decode": 1, "prompt": _log_int(rng, 9, 4096)}[form]
    c.update(n_seq=_log_int(rng, 1, 6 if form == "prompt" else 48), q=q, kv=q + past, form="tree" if form == "tree" else "chain")
    c["ragged"] = c["n_seq"] > 1 and rng.random() < 0.7
    if op in ("append", "verify"):
        c.update(rope=rng.choice(["halves", "pairs"]), rope_dim=rng.choice([dim, dim // 2]),
                 scale=rng.choice([1.0, 4.0, 16.0, 40.0]), ahead=rng.choice([0, 0, _log_int(rng, 1, 900000)]))
    if op in ("tree", "verify"):
        c.update(window=rng.choice([0, 0, _log_int(rng, 16, 4096)]), sinks=rng.random() < 0.4)
    return c


def _load(c: dict) -> int:
    """Scores that a plain form holds at once: what of it has to fit beside the states."""
    return c["n_seq"] * c["heads"] * c["q"] * c["kv"] if c["op"] in ("tree", "weigh", "verify") else 0


def draw(rng) -> dict:
    """A case of the same ranges that costs no more (bytes, products, cache to make) than the listed ones."""
    works = [work(c) for c in listed()]
    top = {key: max(w[key] for w in works) for key in ("bytes", "flops")}
    cells = max(sum(_lens(c)[1]) * c["kv_heads"] * c["dim"] for c in listed())
    load = max(_load(c) for c in listed())
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and _load(c) <= load:
            if c["n_seq"] * c["kv"] * c["kv_heads"] * c["dim"] <= 2 * cells:  # (lengths filled up to the longest)
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


def _parents(c: dict) -> list[list[int]]:
    """Of every new token its parent among its sequence's (-1: none, -2: no token of the tree)."""
    rng = random.Random(c["n_seq"] * 7919 + c["kv"] * 131 + c["q"])
    found = []
    for q in _lens(c)[0]:
        if c["form"] == "chain":
            found.append(list(range(-1, q - 1)))
            continue
        n = q - rng.choice([0, 0, q // 8])  # the rest fills up a plan of fixed size
        rows = [-1] + [max(-1, i - 1 - int(rng.expovariate(0.25))) for i in range(1, n)]
        found.append((rows[:n] + [-2] * (q - n))[:q])
    return found


def _seen(parents: list[int]) -> list[list[int]]:
    """The new tokens that each of them sees."""
    rows: list[list[int]] = []
    for i, p in enumerate(parents):
        rows.append([] if p < -1 else [*(rows[p] if p >= 0 else []), i])
    return rows


def _visits(c: dict) -> tuple[int, int]:
    """(token, position) pairs that the masks leave, and positions that any token sees."""
    pairs = seen = 0
    for q, kv, parents in zip(*_lens(c), _parents(c)):
        first, widest = kv - q, 0
        for row in _seen(parents):
            n = min(first, max(0, c["window"] - len(row))) if c.get("window") else first
            pairs += (n + len(row)) if row else 0
            widest = max(widest, n if row else 0)
        seen += (widest + q) if q else 0
    return pairs, seen


def work(case: dict) -> dict:
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    qs, kvs = _lens(c)
    tok, H, Hk, D = sum(qs), c["heads"], c["kv_heads"], c["dim"]
    row = Hk * (D // 2 + D // 32)  # a token's K or V in the cache
    if c["op"] == "evict":
        kept = sum(min(kv, c["budget"]) for kv in kvs)
        # the weights once; what is kept, its weights too, from one place to another; its list
        return {"bytes": 4 * Hk * sum(kvs) + kept * (4 * row + 4 * Hk + 4 * Hk), "flops": 0}
    turned = {"bytes": tok * ((2 * H + 2 * Hk) * D * size + 2 * row + 4), "flops": tok * D * (4 * H + 11 * Hk)}
    if c["op"] == "append":
        return turned
    pairs, seen = _visits(c)
    if c["op"] == "weigh":
        return {"bytes": tok * H * (D * size + 4) + seen * (row + 8 * Hk), "flops": 2 * pairs * H * D}
    words = (max(qs) + 63) // 64
    attn = {"bytes": tok * (2 * H * D * size + 4 * H + 8 * words) + seen * 2 * row, "flops": 4 * pairs * H * D}
    if c["op"] == "tree":
        return attn
    moved = sum(_accepted(c)[1])
    return {"bytes": turned["bytes"] + attn["bytes"] - 4 * H * tok + 4 * tok + moved * 4 * row,
            "flops": turned["flops"] + attn["flops"]}


def _accepted(c: dict) -> tuple[list[list[int]], list[int]]:
    """The path that verification takes over, of every sequence: the new tokens on it, and how many."""
    rng = random.Random(c["n_seq"] + c["kv"] * 17 + c["q"] * 5)
    paths = [rng.choice([r for r in _seen(p) if r]) if p else [] for p in _parents(c)]
    return paths, [len(p) for p in paths]


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _normal(shape, gen, std: float = 1.0) -> torch.Tensor:
    return torch.empty(*shape, device="cuda").normal_(0.0, std, generator=gen)


def _ints(rows, dtype=torch.int32) -> torch.Tensor:
    return torch.tensor(rows, dtype=dtype, device="cuda")


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


def _frequencies(c: dict) -> tuple[torch.Tensor, float]:
    """Frequencies of the rotation and its magnitude, scaled: those that turn 32 times and more over the original
    context stay, those that do not turn once are divided by the scale, a ramp lies between."""
    r, s = c["rope_dim"], c["scale"]
    f = BASE ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if s <= 1.0:
        return f.float().cuda(), 1.0
    at = lambda turns: r * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(BASE))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r // 2 - 1)
    stay = 1.0 - ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    return (f * stay + f / s * (1.0 - stay)).float().cuda(), 0.1 * math.log(s) + 1.0


def prepare(case: dict, seed: int) -> dict:
    c = case
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed & 0x7FFFFFFFFFFFFFFF)
    qs, kvs = _lens(c)
    tok, H, Hk, D, P, S = sum(qs), c["heads"], c["kv_heads"], c["dim"], c["page"], c["n_seq"]
    per = [(kv + P - 1) // P for kv in kvs]  # pages of a sequence, handed out in no order
    keep = [min(kv, c["budget"]) for kv in kvs] if c["op"] == "evict" else []
    per_to = [(n + P - 1) // P for n in keep]
    used, n_pages = sum(per) + 3, sum(per) + 3 + sum(per_to)
    host = torch.Generator().manual_seed(seed & 0x7FFFFFFF)

    def table_of(counts, pool):
        t, at = torch.full((S, max(counts)), -1, dtype=torch.int32), 0
        for i, n in enumerate(counts):
            t[i, :n] = pool[at:at + n]
            at += n
        return t.cuda()

    table = table_of(per, torch.randperm(used, generator=host).int())
    start = [0]
    for q in qs:
        start.append(start[-1] + q)
    pages = torch.zeros(n_pages, Hk * P * (D + D // 16), dtype=torch.uint8, device="cuda")
    kb, vb, ks, vs = _parts(c, pages)
    step = max(1, (1 << 25) // (Hk * P * D))
    for p in range(0, used, step):  # what earlier calls appended: every position, a channel's size its own
        n = min(step, used - p)
        size = 0.2 + torch.rand(Hk, 1, D, device="cuda", generator=gen) ** 4 * 4
        code, e = _hold(_normal((n, Hk, P, D), gen) * size)
        kb[p:p + n], ks[p:p + n] = _k_bytes(code), e
        code, e = _hold(_normal((n, Hk, P, D), gen))
        vb[p:p + n], vs[p:p + n] = _v_bytes(code).transpose(-1, -2), e
    st = {"case": c, "qs": qs, "kvs": kvs, "pages": pages, "table": table, "start": _ints(start), "kv_len": _ints(kvs),
          "levels": torch.tensor(LEVELS + tuple(-v for v in LEVELS)).cuda()}
    if own:
        from flintnsteel_amd import ops
        st["cache"] = ops.KvCache(n_pages, P, Hk, D, pages=pages)
        st["batch"] = ops.KvBatch(st["start"], st["kv_len"], table, n_tok=tok, max_q=max(qs), max_kv=max(kvs))
    if c["op"] == "evict":
        # what attention leaves: few heavy positions, many light ones, some that nothing has looked at, equal ones
        w = torch.exp(_normal((n_pages, Hk, P), gen, 2.0))
        w = torch.where(torch.rand(n_pages, Hk, P, device="cuda", generator=gen) < 0.5, w, (w * 64).round() / 64)
        st.update(weights=w, keep=_ints(keep), used=used, to=table_of(per_to, used + torch.randperm(sum(per_to), generator=host).int()),
                  most=max(keep))
        return st
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    parents = _parents(c)
    words = (max(qs) + 63) // 64
    bits = torch.zeros(tok, words * 64, dtype=torch.bool)
    depth, t = torch.zeros(tok, dtype=torch.int32), 0
    for rows in map(_seen, parents):
        for row in rows:
            bits[t, row] = True
            depth[t] = max(len(row) - 1, 0)
            t += 1
    # what a row sees of its sequence's new tokens, as bits
    bits = bits.cuda().unflatten(-1, (words, 64))
    sees = (bits[..., :63].long() << torch.arange(63, device="cuda")).sum(-1) + bits[..., 63].long() * (-2 ** 63)
    seq = torch.repeat_interleave(torch.arange(S), torch.tensor(qs)).cuda()
    first = (st["kv_len"] - torch.tensor(qs).cuda()).long()
    st.update(q=_normal((tok, H, D), gen).to(dt), sees=sees, seq=seq, words=words, first=first,
              nth=torch.cat([torch.arange(q) for q in qs]).cuda())
    if c["op"] in ("append", "verify"):
        st["k"], st["v"] = _normal((tok, Hk, D), gen, 2.0).to(dt), _normal((tok, Hk, D), gen).to(dt)
        st["freq"], st["magnitude"] = _frequencies(c)
        st["base"] = (first + c["ahead"]).int()
        st["pos"] = (st["base"][seq] + depth.cuda()).int()
        st["parents"] = _ints([p for rows in parents for p in rows])
    if c["op"] in ("tree", "verify"):
        st["sinks"] = _normal((H,), gen) if c["sinks"] else None
    if c["op"] == "verify":
        paths, counts = _accepted(c)
        most = max(counts)
        st["kept"], st["n_kept"] = _ints([p + [-1] * (most - len(p)) for p in paths]), _ints(counts)
        ends = [0]
        for n in counts:
            ends.append(ends[-1] + n)
        st["kept_start"], st["kept_len"] = _ints(ends), first.int() + st["n_kept"]
        st["kept_seq"] = torch.repeat_interleave(torch.arange(S), torch.tensor(counts)).cuda()
        st["kept_nth"] = torch.cat([torch.arange(n) for n in counts]).cuda()
        if own:
            st["after"] = ops.KvBatch(st["kept_start"], st["kept_len"], table, n_tok=ends[-1], max_q=most, max_kv=max(kvs))
    if c["op"] == "weigh":
        st["past"] = torch.exp(_normal((n_pages, Hk, P), gen, 2.0)) / c["kv"]  # of the few steps before
        st["weights"] = torch.zeros_like(st["past"])
        st["lse"] = _plain_attn(st, values=False)[1]  # attention's, of the same step
    if own:
        st["tree"] = ops.KvTree(st["sees"]) if c["form"] == "tree" else None
        if c["op"] in ("tree", "verify"):
            st["out"], st["lse"] = torch.empty_like(st["q"]), torch.empty(tok, H, device="cuda")
            st["ws"] = ops.attn_workspace(st["cache"], st["batch"], st["q"])
        elif c["op"] == "weigh":
            st["ws"] = ops.kv_weigh_workspace(st["cache"], st["batch"], st["q"])
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st: dict):
    from flintnsteel_amd import ops
    c, cache, batch = st["case"], st["cache"], st["batch"]
    if c["op"] == "evict":
        kept, new_len = ops.kv_evict(cache, batch, st["weights"], c["budget"], first=c["first"], recent=c["recent"], to_table=st["to"])
        # (the bytes are moved as they are, so they are compared as they are)
        return kept[..., :st["most"]], new_len, st["weights"][st["used"]:], st["pages"][st["used"]:]
    if c["op"] == "weigh":
        ops.kv_weigh(cache, batch, st["q"], st["lse"], st["past"], tree=st["tree"], out=st["weights"], ws=st["ws"])
        return st["weights"]
    if c["op"] == "tree":
        ops.attn(cache, batch, st["q"], window=c["window"], sinks=st["sinks"], out=st["out"], ws=st["ws"], tree=st["tree"], lse=st["lse"])
        return st["out"], st["lse"]
    rope = {"halves": ops.ROPE_HALVES, "pairs": ops.ROPE_PAIRS}[c["rope"]]
    if c["op"] == "append":
        q = ops.kv_append(cache, batch, st["k"], st["v"], q=st["q"], rope=rope, inv_freq=st["freq"], pos=st["pos"], magnitude=st["magnitude"])
        return (q, *ops.kv_read(cache, batch))
    tree = ops.tree_plan(batch, st["parents"], base=st["base"])
    q = ops.kv_append(cache, batch, st["k"], st["v"], q=st["q"], rope=rope, inv_freq=st["freq"], pos=tree.pos, magnitude=st["magnitude"])
    ops.attn(cache, batch, q, window=c["window"], sinks=st["sinks"], out=st["out"], ws=st["ws"], tree=tree)
    new_len = ops.kv_keep(cache, batch, st["kept"], st["n_kept"])
    return (tree.sees, tree.pos, st["out"], new_len, *ops.kv_read(cache, st["after"]))


def _turned(c: dict, x: torch.Tensor, pos: torch.Tensor, freq: torch.Tensor, magnitude: float) -> torch.Tensor:
    x, r = x.double(), c["rope_dim"]  # a far position's angle, and codes next to a border
    t = (pos.double()[:, None] * freq.double())[:, None, :]
    cos, sin = t.cos() * magnitude, t.sin() * magnitude
    head, rest = x[..., :r], x[..., r:]
    if c["rope"] == "halves":
        a, b = head[..., :r // 2], head[..., r // 2:]
        head = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    return torch.cat((head, rest), -1)


def _place(st: dict, seq: torch.Tensor, pos: torch.Tensor):
    """Page and row in the page of positions of sequences."""
    P = st["case"]["page"]
    return st["table"][seq, pos // P].long(), pos % P


def _plain_append(st: dict, pos: torch.Tensor) -> torch.Tensor:
    c = st["case"]
    kb, vb, ks, vs = _parts(c, st["pages"])
    page, row = _place(st, st["seq"], st["first"][st["seq"]] + st["nth"])
    code, e = _hold(_turned(c, st["k"], pos, st["freq"], st["magnitude"]))
    kb[page, :, row], ks[page, :, row] = _k_bytes(code), e
    code, e = _hold(st["v"].float())
    vb[page, :, :, row], vs[page, :, row] = _v_bytes(code), e
    return _turned(c, st["q"], pos, st["freq"], st["magnitude"]).to(st["q"].dtype)


def _plain_read(st: dict, seq: torch.Tensor, pos: torch.Tensor):
    kb, vb, ks, vs = _parts(st["case"], st["pages"])
    page, row = _place(st, seq, pos)
    return (_values(st, _k_codes(kb[page, :, row]), ks[page, :, row]),
            _values(st, _v_codes(vb[page, :, :, row]), vs[page, :, row]))


def _plain_scores(st: dict, q: torch.Tensor, sees: torch.Tensor):
    """scale * q . K of every sequence's tokens (filled up to the most) and positions (to the longest), -infinity where
    the mask leaves nothing: [n_seq][kv_heads][tokens][group][positions]; the pages."""
    c, dev = st["case"], q.device
    S, Q, H, Hk, D = c["n_seq"], max(st["qs"]), c["heads"], c["kv_heads"], c["dim"]
    kb, _, ks, _ = _parts(c, st["pages"])
    page = st["table"].clamp_min(0).long()
    K = _values(st, _k_codes(kb[page]), ks[page]).transpose(1, 2).flatten(2, 3)  # [S][Hk][positions][D]
    full = torch.zeros(S, Q, H, D, device=dev)
    full[st["seq"], st["nth"]] = q.float()
    full = full.view(S, Q, Hk, H // Hk, D).transpose(1, 2).flatten(2, 3)
    x = torch.matmul(full.contiguous(), K.transpose(-1, -2).contiguous()).view(S, Hk, Q, H // Hk, -1) * D ** -0.5
    j = torch.arange(x.shape[-1], device=dev)
    bits = ((sees[..., None] >> torch.arange(64, device=dev)) & 1).flatten(1).bool()
    mask = torch.zeros(S, Q, bits.shape[1], dtype=torch.bool, device=dev)
    mask[st["seq"], st["nth"]] = bits
    count = mask.sum(-1)
    nth = j - st["first"][:, None]  # of a position among the new tokens
    new = torch.gather(mask, 2, nth[:, None, :].clamp(0, mask.shape[2] - 1).expand(S, Q, -1))
    see = torch.where((nth < 0)[:, None, :], (count > 0)[..., None], new & (nth < mask.shape[2])[:, None, :])
    if c.get("window"):
        see = see & ((nth >= 0)[:, None, :] | (nth[:, None, :] >= (count - c["window"])[..., None]))
    return x.masked_fill_(~see[:, None, :, None, :], -math.inf), page


def _plain_attn(st: dict, q: torch.Tensor | None = None, sees: torch.Tensor | None = None, values: bool = True):
    c = st["case"]
    q, sees = st["q"] if q is None else q, st["sees"] if sees is None else sees
    H, Hk = c["heads"], c["kv_heads"]
    x, page = _plain_scores(st, q, sees)
    m = x.amax(-1, keepdim=True)
    sinks = st.get("sinks")
    if sinks is not None:
        sinks = sinks.view(1, Hk, 1, H // Hk, 1)
        m = torch.maximum(m, sinks)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = (x - m).exp_()
    den = p.sum(-1, keepdim=True)
    if sinks is not None:
        den = den + (sinks - m).exp()
    lse = (m + den.log()).squeeze(-1).permute(0, 2, 1, 3).flatten(2)[st["seq"], st["nth"]]
    if not values:
        return None, lse
    _, vb, _, vs = _parts(c, st["pages"])
    V = _values(st, _v_codes(vb[page].transpose(-1, -2)), vs[page]).transpose(1, 2).flatten(2, 3).contiguous()
    p = torch.where(den == 0, torch.zeros_like(p), p / den)
    out = torch.matmul(p.flatten(2, 3), V).unflatten(2, (-1, H // Hk))  # [S][Hk][tokens][group][D]
    return out.transpose(1, 2).flatten(2, 3)[st["seq"], st["nth"]].to(st["q"].dtype), lse


def _plain_evict(st: dict):
    c = st["case"]
    P, Hk, S, dev = c["page"], c["kv_heads"], c["n_seq"], st["table"].device
    w = st["weights"][st["table"].clamp_min(0).long()].transpose(1, 2).flatten(2)  # [S][Hk][positions]
    j, n = torch.arange(w.shape[-1], device=dev), st["kv_len"].long()[:, None, None]
    w = torch.where((j < c["first"]) | (j >= n - c["recent"]), torch.full_like(w, math.inf), w)
    w = torch.where(j >= n, torch.full_like(w, -1.0), w)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :st["most"]]
    rank, keep = torch.arange(order.shape[-1], device=dev), st["keep"].long()[:, None, None]
    kept = torch.where(rank < keep, order, torch.full_like(order, 2 ** 30)).sort(-1).values
    s, h, r = torch.nonzero(kept < 2 ** 30, as_tuple=True)
    src = kept[s, h, r]
    a, i, b, k = st["table"][s, src // P].long(), src % P, st["to"][s, r // P].long(), r % P
    for part in _parts(c, st["pages"])[0::2] + _parts(c, st["pages"])[3:]:
        part[b, h, k] = part[a, h, i]
    vb = _parts(c, st["pages"])[1]
    vb[b, h, :, k] = vb[a, h, :, i]
    st["weights"][b, h, k] = st["weights"][a, h, i]
    return (torch.where(kept < 2 ** 30, kept, torch.full_like(kept, -1)).int(), st["keep"], st["weights"][st["used"]:],
            st["pages"][st["used"]:])


def _plain_weigh(st: dict):
    c = st["case"]
    H, Hk, P = c["heads"], c["kv_heads"], c["page"]
    x, page = _plain_scores(st, st["q"], st["sees"])
    lse = torch.full((c["n_seq"], max(st["qs"]), H), math.inf, device=x.device)
    lse[st["seq"], st["nth"]] = torch.where(st["lse"].isfinite(), st["lse"], torch.full_like(st["lse"], math.inf))
    w = (x - lse.unflatten(2, (Hk, -1)).transpose(1, 2)[..., None]).exp_().flatten(2, 3).sum(2)  # [S][Hk][positions]
    j = torch.arange(w.shape[-1], device=x.device)
    past = st["past"][page].transpose(1, 2).flatten(2)
    w = w + torch.where(j < st["first"][:, None, None], past, torch.zeros_like(past))
    at = torch.tensor(st["qs"], device=x.device)
    s, j = torch.nonzero((j < st["kv_len"][:, None]) & (at > 0)[:, None], as_tuple=True)
    page, row = _place(st, s, j)
    st["weights"][page, :, row] = w[s, :, j]
    return st["weights"]


def _plain_plan(st: dict):
    """Masks and positions from parents: paths double in length until no tree is deeper."""
    c, dev = st["case"], st["parents"].device
    S, Q = c["n_seq"], max(st["qs"])
    parent = torch.full((S, Q), -2, device=dev)
    parent[st["seq"], st["nth"]] = st["parents"].long()
    i = torch.arange(Q, device=dev)
    reach = (i[:, None] == i) & (parent >= -1)[..., None]
    up = (parent[..., None] == i).float()  # a step to the parent
    for _ in range(max(1, Q - 1).bit_length()):
        reach = reach | (torch.matmul(up, reach.float()) > 0)
        up = (torch.matmul(up, up) > 0).float()
    bits = torch.zeros(S, Q, st["words"] * 64, dtype=torch.bool, device=dev)
    bits[..., :Q] = reach
    bits = bits[st["seq"], st["nth"]]
    pos = st["base"][st["seq"]] + (bits.sum(-1) - 1).clamp_min(0)
    w = bits.unflatten(-1, (-1, 64))
    sees = (w[..., :63].long() << torch.arange(63, device=dev)).sum(-1) + w[..., 63].long() * (-2 ** 63)
    return sees, pos.int()


def _run_plain(st: dict):
    c = st["case"]
    if c["op"] == "evict":
        return _plain_evict(st)
    if c["op"] == "weigh":
        return _plain_weigh(st)
    if c["op"] == "tree":
        return _plain_attn(st)
    if c["op"] == "append":
        q = _plain_append(st, st["pos"])
        return (q, *_plain_read(st, st["seq"], st["first"][st["seq"]] + st["nth"]))
    sees, pos = _plain_plan(st)
    q = _plain_append(st, pos)
    out = _plain_attn(st, q, sees)[0]
    kb, vb, ks, vs = _parts(c, st["pages"])
    first = st["first"][st["kept_seq"]]
    a, i = _place(st, st["kept_seq"], first + st["kept"][st["kept_seq"], st["kept_nth"]])
    b, k = _place(st, st["kept_seq"], first + st["kept_nth"])
    got = kb[a, :, i], vb[a, :, :, i], ks[a, :, i], vs[a, :, i]
    kb[b, :, k], vb[b, :, :, k], ks[b, :, k], vs[b, :, k] = got
    return (sees, pos, out, st["first"].int() + st["n_kept"], *_plain_read(st, st["kept_seq"], first + st["kept_nth"]))


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


def _rotor(c: dict, x: torch.Tensor, pos: list[int], freq: torch.Tensor, magnitude: float) -> torch.Tensor:
    x = x.to(torch.float64)
    out, half = x.clone(), c["rope_dim"] // 2
    i = torch.arange(half, device=x.device)
    u, w = (i, i + half) if c["rope"] == "halves" else (2 * i, 2 * i + 1)
    angle = torch.tensor(pos, dtype=torch.float64, device=x.device)[:, None, None] * freq.to(torch.float64)[None, None, :]
    z = torch.complex(x[..., u], x[..., w]) * torch.polar(torch.full_like(angle, magnitude), angle)
    out[..., u], out[..., w] = z.real, z.imag
    return out


def _cached(c: dict, pages: torch.Tensor, table: torch.Tensor, n: int, head: int):
    """K and V (f64 [n][dim]) of positions 0 .. n - 1 of one kv head, read byte by byte from their places."""
    P, D, dev = c["page"], c["dim"], pages.device
    pos = torch.arange(n, device=dev)
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


def _exact_rows(c: dict, st: dict, q: torch.Tensor, new=None):
    """Of every sequence and kv head with tokens: (sequence, head, first token, scores f64 [tokens][group][positions]
    with -infinity where nothing is seen, V). new: K and V of the new tokens in the place of what the cache has."""
    H, Hk, D, t = c["heads"], c["kv_heads"], c["dim"], 0
    for s, (n, kv, parents) in enumerate(zip(*_lens(c), _parents(c))):
        see = torch.zeros(n, kv, dtype=torch.bool)
        for i, row in enumerate(_seen(parents)):
            if row:
                see[i, max(0, kv - n - max(0, c["window"] - len(row))) if c.get("window") else 0:kv - n] = True
                see[i, torch.tensor(row) + (kv - n)] = True
        for h in range(Hk if n else 0):
            K, V = _cached(c, st["pages"], st["table"][s], kv, h)
            if new is not None:
                K[kv - n:], V[kv - n:] = new[0][t:t + n, h], new[1][t:t + n, h]
            x = torch.stack([q[t:t + n, h * (H // Hk) + g].double() @ K.T for g in range(H // Hk)], 1) * D ** -0.5
            yield s, h, t, torch.where(see.cuda()[:, None, :], x, torch.full_like(x, -math.inf)), V
        t += n


def _exact_attn(c: dict, st: dict, q: torch.Tensor, new=None):
    G = c["heads"] // c["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for _, h, t, x, V in _exact_rows(c, st, q, new):
        if st["sinks"] is not None:
            x = torch.cat((x, st["sinks"][h * G:(h + 1) * G].double()[None, :, None].expand(len(x), G, 1)), -1)
        den = torch.logsumexp(x, -1)
        p = torch.exp(x - torch.where(den == -math.inf, 0.0, den)[..., None])[..., :len(V)]
        out[t:t + len(x), h * G:(h + 1) * G], lse[t:t + len(x), h * G:(h + 1) * G] = p @ V, den
    return out, lse


def exact(case: dict, seed: int):
    c, st = case, prepare(case, seed)
    if c["op"] == "tree":
        return _exact_attn(c, st, st["q"])
    qs, kvs = _lens(c)
    if c["op"] == "weigh":
        w = torch.zeros(st["past"].shape, dtype=torch.float64, device="cuda")
        G = c["heads"] // c["kv_heads"]
        for s, h, t, x, _ in _exact_rows(c, st, st["q"]):
            den = st["lse"][t:t + len(x), h * G:(h + 1) * G].double()
            den = torch.where(den.isfinite(), den, math.inf)
            j = torch.arange(kvs[s], device="cuda")
            page, row = st["table"][s, j // c["page"]].long(), j % c["page"]
            before = torch.where(j < kvs[s] - qs[s], st["past"][page, h, row].double(), 0.0)
            w[page, h, row] = before + torch.exp(x - den[..., None]).sum((0, 1))
        return w
    if c["op"] == "evict":  # whole numbers and moved ones, but for the weights
        moved = torch.zeros(st["weights"].shape, dtype=torch.float64, device="cuda")
        moved += st["weights"].double()
        for s, n in enumerate(kvs):
            j = torch.arange(n, device="cuda")
            w = st["weights"][st["table"][s, j // c["page"]].long(), :, j % c["page"]].double()
            w[:min(c["first"], n)] = math.inf
            w[max(0, n - c["recent"]):] = math.inf
            for h in range(c["kv_heads"]):
                best = torch.sort(w[:, h], descending=True, stable=True).indices[:c["budget"]].sort().values
                r = torch.arange(len(best), device="cuda")
                moved[st["to"][s, r // c["page"]].long(), h, r % c["page"]] = \
                    st["weights"][st["table"][s, best // c["page"]].long(), h, best % c["page"]].double()
        return None, None, moved[st["used"]:], None
    pos = [kv - q + c["ahead"] + max(len(row) - 1, 0)
           for q, kv, parents in zip(qs, kvs, _parents(c)) for row in _seen(parents)]
    q = _rotor(c, st["q"], pos, st["freq"], st["magnitude"])
    K, V = _nearest(_rotor(c, st["k"], pos, st["freq"], st["magnitude"])), _nearest(st["v"].double())
    if c["op"] == "append":
        return q, K, V
    paths, _ = _accepted(c)
    at = [sum(qs[:s]) + i for s, p in enumerate(paths) for i in p]
    return None, None, _exact_attn(c, st, q.to(st["q"].dtype), (K, V))[0], None, K[at], V[at]
