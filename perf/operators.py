"""The operators around a key/value cache that is held in 4 bits, as cases that can be timed and compared.

Three kinds: norms of queries and keys for each head with the position rotation in the same pass, which with a cache also
writes keys and values into its pages ("rope"); attention over the paged cache, from one query token per sequence to whole
prompts ("attention"); and copies of pages, as forking and compacting sequences need them ("pages").

The cache's format.  32 neighbouring values of a head share a scale: scale = fp16(bf16(absmax / 7)), code =
clamp(round(x / scale), -7, 7) + 8, and a value is scale * (code - 8), which always is an fp16 number.  16 tokens of
a head are a tile of 18 * head_dim bytes: codes of K, codes of V, scales of K, scales of V ([16][head_dim / 32] fp16).  A page
is [kv_heads][page_tokens / 16] tiles.  Where a code lies within its tile: `_order`.

Heads of 128 in groups of four to a key/value head, blocks of 32 values, caches of 2048 tokens and a 32-layer decoder are this
repository's own sizes; the others are generic.
"""
import functools
import importlib
import math
import random

import numpy as np
import torch

own = False

NEIGHBOURS = {"halves": 0, "neighbours": 1}
MIN_TIMESCALE, MAX_TIMESCALE, EPS = 1.0, 1.0e6, 1e-6


def _mld():
    return importlib.import_module("ml-drift_b200")


# ------------------------------------------------------------------------------------------------------------ cases
def _rope(tokens, heads, kv_heads, head_dim, rotary, pairs, axes, type_, cache, longest):
    return {"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rotary,
            "pairs": pairs, "axes": axes, "type": type_, "cache": cache, "longest": longest, "page": 64}


def _attention(batch, longest, shortest, queries, heads, kv_heads, head_dim, window, page):
    """Sequences of `shortest` to `longest` cached tokens, each with 1 to `queries` (one of them with all) new ones."""
    return {"kind": "attention", "batch": batch, "longest": longest, "shortest": shortest, "queries": queries, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "window": window, "page": page}


def _pages(layers, pages, copies, kv_heads, head_dim, page):
    return {"kind": "pages", "layers": layers, "pages": pages, "copies": copies, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": page}


def listed():
    return [
        # One generated token of one sequence: the smallest call, nothing but latency.
        {"name": "rope_token", **_rope(1, 32, 8, 128, 128, "halves", 1, "f16", True, 2048)},
        # fp32 tensors, an odd number of tokens, neighbouring values paired over half of a head; no cache: keys are returned.
        {"name": "rope_f32_509", **_rope(509, 8, 1, 256, 128, "neighbours", 1, "f32", False, 4096)},
        # A long prompt of text and pictures: positions with three axes.
        {"name": "rope_prompt8192", **_rope(8192, 32, 8, 128, 128, "halves", 3, "f16", True, 131072)},
        # Early in a conversation: one sequence, one token, a few hundred cached ones.
        {"name": "attention_chat300", **_attention(1, 300, 300, 1, 32, 8, 128, 0, 64)},
        # The benchmark's geometry: as many key/value heads as heads, 2048 cached tokens.
        {"name": "attention_2048", **_attention(1, 2048, 2048, 1, 32, 32, 128, 0, 64)},
        # One token over a very long document.
        {"name": "attention_131071", **_attention(1, 131071, 131071, 1, 32, 8, 128, 0, 64)},
        # A server's batch, one token each, lengths from none (a sequence that has not begun) to 8191; small pages.
        {"name": "attention_batch64", **_attention(64, 8191, 0, 1, 32, 8, 128, 0, 16)},
        # Up to five drafted tokens checked at once, small heads, a sliding window.
        {"name": "attention_draft5", **_attention(16, 3001, 1, 5, 16, 4, 64, 1024, 32)},
        # A whole prompt against itself, already in the cache.
        {"name": "attention_prompt2048", **_attention(1, 2048, 2048, 2048, 32, 8, 128, 0, 64)},
        # Chunks of ragged prompts behind long histories, five heads to a key/value head.
        {"name": "attention_chunks", **_attention(4, 16384, 1000, 1023, 40, 8, 128, 0, 64)},
        # A sequence forked: its last page copied, in one layer ...
        {"name": "pages_fork", **_pages(1, 64, 1, 8, 128, 64)},
        # ... and a 32-layer cache compacted.
        {"name": "pages_compact", **_pages(32, 256, 101, 8, 128, 64)},
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))


def draw(rng):
    kind = rng.choice(("rope", "attention", "attention", "attention", "pages"))
    head_dim = rng.choice((64, 128, 128, 256))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 16))
    group = rng.choice((1, 2, 3, 4, 5, 8, 16))
    page = rng.choice((16, 32, 64, 128, 48))
    if kind == "rope":
        while kv_heads * group > 64:
            group = rng.choice((1, 2, 4))
        most = 8192 * 48 * 128 // ((kv_heads * group + 2 * kv_heads) * head_dim)
        type_ = rng.choice(("f16", "f16", "f32"))
        return {**_rope(_log(rng, 1, min(8192, most)), kv_heads * group, kv_heads, head_dim, head_dim // rng.choice((1, 1, 2, 4)),
                        rng.choice(("halves", "neighbours")), rng.choice((1, 1, 2, 3, 4)), type_,
                        type_ == "f16" and rng.random() < 0.7, _log(rng, 64, 1 << 20)), "page": page}
    if kind == "pages":
        layers = rng.choice((1, 2, 16, 32, 48))
        size = layers * kv_heads * head_dim * page * 18 // 16
        pages = max(8, min(_log(rng, 8, 2048), (600 << 20) // size))
        return _pages(layers, pages, _log(rng, 1, max(1, pages * 2 // 5)), kv_heads, head_dim, page)
    while kv_heads * group > 48:
        group = rng.choice((1, 2, 3))
    queries = rng.choice((1, 1, 1, _log(rng, 2, 8), _log(rng, 9, 128), _log(rng, 129, 2048)))
    batch = _log(rng, 1, 128 if queries < 9 else 8)
    longest = _log(rng, 16, 131071)
    # no more cached values, scores and products than the listed cases have
    while batch * longest * kv_heads * head_dim > 64 * 8191 * 8 * 128 or \
            batch * queries * longest * kv_heads * group * max(head_dim, 128) > 4 * 1023 * 16384 * 40 * 128 // 2:
        if batch > 1 and rng.random() < 0.5:
            batch = (batch + 1) // 2
        else:
            longest = (longest + 1) // 2
    return _attention(batch, longest, rng.choice((0, longest // 2, longest)), min(queries, longest), kv_heads * group, kv_heads,
                      head_dim, rng.choice((0, 0, 0, _log(rng, 16, 4096))), page)


def _lengths(case):
    """(cached tokens, new tokens among them) of every sequence: the same for every seed, since work() has to know them."""
    rng = random.Random(1000 * case["longest"] + case["batch"])
    lens, news = [], []
    for b in range(case["batch"]):
        lens.append(case["longest"] if b == 0 else rng.randint(case["shortest"], case["longest"]))
        news.append(case["queries"] if b == 0 or case["queries"] == 1 else rng.randint(1, case["queries"]))
    if case["shortest"] == 0 and case["batch"] > 1:
        lens[-1] = 0
    return lens, news


def _visible(case):
    """Per sequence: (query, key) pairs that the mask leaves, and keys that any query sees."""
    window, got = case["window"], []
    for n, m in zip(*_lengths(case)):
        at = np.arange(n - m, n, dtype=np.int64)  # negative: a query ahead of the first token, which sees nothing
        seen = np.clip(at + 1, 0, None)
        first = max(0, n - m + 1 - window) if window else 0
        got.append((int(np.minimum(seen, window).sum() if window else seen.sum()), max(0, n - first)))
    return got


def work(case):
    d, hk = case["head_dim"], case["kv_heads"]
    row = hk * d * 18 // 16  # bytes of a token's keys and values in the cache
    if case["kind"] == "rope":
        n, size, h = case["tokens"], 2 if case["type"] == "f16" else 4, case["heads"]
        values = n * (h + hk) * d
        data = 2 * n * h * d * size + n * hk * d * size + 4 * n * case["axes"]
        # keys out; or values in, the cache written, read again and returned
        data += n * hk * d * size if not case["cache"] else n * hk * d * size + 2 * n * row + 2 * n * hk * d * 2 + 8 * n
        return {"bytes": data, "flops": 8 * values}
    if case["kind"] == "pages":
        return {"bytes": 2 * case["copies"] * case["layers"] * case["page"] * row, "flops": 0}
    tokens = sum(_lengths(case)[1])
    pairs, keys = (sum(x) for x in zip(*_visible(case)))
    return {"bytes": keys * row + 2 * tokens * case["heads"] * d * 2, "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------------------------------------- the cache's layout
@functools.lru_cache(None)
def _order(d):
    """Where the codes of a tile's K and V lie: two arrays [16][d] of positions in units of 4 bits from the start of each."""
    tau, e = np.arange(16)[:, None], np.arange(d)[None, :]
    group, r = e // 32, e % 32
    words = min(4, d // 32)
    unit = group // words * 4 + r // 8
    if d == 256:
        unit = unit ^ (tau & 1) * 4
    k = (tau * (d // 8) + unit * words + group % words) * 8 + 4 * (r % 2) + r % 8 // 2
    row = 8 * (tau // 8) + (tau % 8 // 2) + 4 * (tau % 2)
    piece = r // 4 ^ {64: 0 * row, 128: row // 2 % 2 * 4, 256: row % 4 * 2}[d]
    v = row * d + piece * (d // 8) + group * 4 + r % 4
    return k, v


@functools.lru_cache(None)
def _order_on_gpu(d):
    return tuple(torch.from_numpy(np.ascontiguousarray(x).reshape(-1)).cuda() for x in _order(d))


def _codes(x):
    """Values [..., d] -> (codes 1 to 15 as uint8, scales [..., d / 32] fp16)."""
    g = x.half().float().unflatten(-1, (-1, 32))
    scale = (g.abs().amax(-1) / 7).bfloat16().half()
    steps = torch.where(scale > 0, scale.float(), float("inf"))[..., None]
    return (torch.clamp(torch.round(g / steps), -7, 7) + 8).to(torch.uint8).flatten(-2), scale


def _tiles(kc, ks, vc, vs):
    """Codes [n, 16, d] and scales [n, 16, d / 32] of n tiles as bytes [n, 18 d]."""
    d = kc.shape[-1]
    out = []
    for c, order in zip((kc, vc), _order_on_gpu(d)):
        nibbles = torch.empty_like(c).flatten(1)
        nibbles[:, order] = c.flatten(1)
        out.append(nibbles[:, 0::2] | nibbles[:, 1::2] << 4)
    return torch.cat(out + [s.contiguous().view(torch.uint8).flatten(1) for s in (ks, vs)], 1)


def _values(tiles):
    """Bytes [n, 18 d] of n tiles -> K and V [n, 16, d] in fp32."""
    d = tiles.shape[1] // 18
    got = []
    for i, order in enumerate(_order_on_gpu(d)):
        packed = tiles[:, 8 * d * i:8 * d * (i + 1)]
        codes = torch.stack((packed & 15, packed >> 4), -1).flatten(1)[:, order].view(-1, 16, d // 32, 32)
        scales = tiles[:, 16 * d + d * i:17 * d + d * i].contiguous().view(torch.float16).view(-1, 16, d // 32, 1)
        got.append(((codes.float() - 8) * scales.float()).flatten(-2))
    return got


# ------------------------------------------------------------------------------------- what a program has in hand
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _sections(case):
    """Pairs of a head that each axis of the positions turns."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    return [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)


def prepare(case, seed):
    return {"rope": _prepare_rope, "attention": _prepare_attention, "pages": _prepare_pages}[case["kind"]](case, _generator(seed))


def _prepare_rope(case, gen):
    n, h, hk, d = (case[k] for k in ("tokens", "heads", "kv_heads", "head_dim"))
    dtype = torch.float16 if case["type"] == "f16" else torch.float32
    # what the projections leave, one row per token; some channels are larger than the others
    channels = torch.exp(0.5 * _randn(gen, h + 2 * hk, d))
    qkv = (_randn(gen, n, h + 2 * hk, d) * channels).to(dtype)
    first = torch.randint(0, max(1, case["longest"] - n), (case["axes"], 1), generator=gen, device="cuda")
    step = torch.arange(n, device="cuda") // torch.tensor([[1], [3], [7], [2]], device="cuda")[:case["axes"]]
    s = {"case": case, "q": qkv[:, :h], "k": qkv[:, h:h + hk], "v": qkv[:, h + hk:], "positions": (first + step).int(),
         "q_weight": (1 + 0.1 * _randn(gen, d)).to(dtype), "k_weight": (1 + 0.1 * _randn(gen, d)).to(dtype),
         "q_out": torch.empty(n, h, d, dtype=dtype, device="cuda")}
    if case["cache"]:
        pages = -(-n // case["page"]) + 3
        s["slots"] = torch.randperm(pages, generator=gen, device="cuda").repeat_interleave(case["page"])[:n].int() * case["page"] + \
            torch.arange(n, device="cuda", dtype=torch.int32) % case["page"]
        s["pool"] = torch.zeros(1, pages, hk, case["page"] // 16, 18 * d, dtype=torch.uint8, device="cuda")
        s["k_read"], s["v_read"] = (torch.empty(n, hk, d, dtype=torch.float16, device="cuda") for _ in range(2))
    else:
        s["k_out"] = torch.empty(n, hk, d, dtype=dtype, device="cuda")
    if own:
        m = _mld()
        s["plan"] = m.QkNormRope(h, hk, d, rotary_dim=case["rotary"], pairing=NEIGHBOURS[case["pairs"]], sections=_sections(case),
                                 min_timescale=MIN_TIMESCALE, max_timescale=MAX_TIMESCALE, rms_eps=EPS, f16=case["type"] == "f16")
        s["cache"] = m.Kv4Cache(hk, d, case["page"], pages, pool=s["pool"]) if case["cache"] else None
    return s


def _prepare_attention(case, gen):
    b, h, hk, d, page = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim", "page"))
    lens, news = _lengths(case)
    per = [-(-n // page) for n in lens]
    pages = max(1, sum(per)) + 5
    # Keys as a norm and a rotation leave them, values with channels of their own size and a mean.  What lies behind a
    # sequence's end, and in pages that nobody holds, is whatever was there before: NaN scales here.
    pool = torch.full((pages * hk * (page // 16), 18 * d), 0x7E, dtype=torch.uint8, device="cuda")
    ids = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.zeros(b, max(1, max(per)), dtype=torch.int32, device="cuda")
    k_size, v_size = 1 + 0.1 * _randn(gen, hk, 1, d), 0.5 * torch.exp(0.4 * _randn(gen, hk, 1, d))
    v_mean = 0.3 * _randn(gen, hk, 1, d)
    pool = pool.view(pages, hk, page // 16, 18 * d)
    at = 0
    for i, (n, p) in enumerate(zip(lens, per)):
        mine = ids[at:at + p]
        at += p
        table[i, :p] = mine
        done = 0
        while done < p:  # a long sequence in pieces, so that their 32-bit values stay small
            some = min(p - done, max(1, (1 << 25) // (page * hk * d)))
            (kc, ks), (vc, vs) = _codes(_randn(gen, hk, some * page, d) * k_size), _codes(_randn(gen, hk, some * page, d) * v_size + v_mean)
            gone = torch.arange(done * page, (done + some) * page, device="cuda") >= n
            ks[:, gone] = float("nan")
            vs[:, gone] = float("nan")
            tiles = _tiles(*(x.reshape(hk * some * page // 16, 16, -1) for x in (kc, ks, vc, vs)))
            pool[mine[done:done + some].long()] = tiles.view(hk, some, page // 16, 18 * d).transpose(0, 1)
            done += some
    starts = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device="cuda")
    s = {"case": case, "q": _randn(gen, sum(news), h, d).mul_(1.5).half(), "pool": pool.unsqueeze(0), "table": table,
         "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "starts": starts,
         "out": torch.empty(sum(news), h, d, dtype=torch.float16, device="cuda")}
    if own:
        m = _mld()
        s["cache"] = m.Kv4Cache(hk, d, page, pages, pool=s["pool"])
        s["plan"] = m.Kv4Attention(s["cache"], h, max_batch=b, max_pages=table.shape[1], window=case["window"])
    return s


def _prepare_pages(case, gen):
    layers, pages, n = case["layers"], case["pages"], case["copies"]
    shape = (layers, pages, case["kv_heads"], case["page"] // 16, 18 * case["head_dim"])
    pool = torch.randint(0, 256, shape, generator=gen, dtype=torch.uint8, device="cuda")
    ids = torch.randperm(pages, generator=gen, device="cuda").tolist()
    s = {"case": case, "pool": pool, "src": ids[:n], "dst": ids[n:2 * n]}  # a pager's answer: page numbers on the host
    if own:
        s["cache"] = _mld().Kv4Cache(case["kv_heads"], case["head_dim"], case["page"], pages, layers=layers, pool=pool)
    return s


# ------------------------------------------------------------------------------------------------------- one pass
def run(s):
    return {"rope": _run_rope, "attention": _run_attention, "pages": _run_pages}[s["case"]["kind"]](s)


def _run_rope(s):
    if own:
        if "cache" in s and s["cache"] is not None:
            s["plan"].run(s["q"], s["k"], s["positions"], s["q_out"], q_weight=s["q_weight"], k_weight=s["k_weight"], v=s["v"],
                          cache=s["cache"], slots=s["slots"])
            s["cache"].read(s["slots"], s["k_read"], s["v_read"])
            return {"q": s["q_out"], "k": s["k_read"], "v": s["v_read"]}
        s["plan"].run(s["q"], s["k"], s["positions"], s["q_out"], k_out=s["k_out"], q_weight=s["q_weight"], k_weight=s["k_weight"])
        return {"q": s["q_out"], "k": s["k_out"]}
    case = s["case"]
    turns = _turns(case, s["positions"])
    q = _norm_rotate(case, s["q"], s["q_weight"], turns).to(s["q"].dtype)
    k = _norm_rotate(case, s["k"], s["k_weight"], turns).to(s["k"].dtype)
    if not case["cache"]:
        return {"q": q, "k": k}
    _write(s, k, s["v"])
    k, v = _read(s)
    return {"q": q, "k": k, "v": v}


def _turns(case, positions):
    """Angles in turns, -0.5 to 0.5.  The product of position and frequency is taken in integers of 2^-64 turns, of which the
    wrap-around leaves what counts: in 32-bit floats a position of 100000 would leave no more than two decimals."""
    pairs = case["rotary"] // 2
    steps = [round((MIN_TIMESCALE * (MAX_TIMESCALE / MIN_TIMESCALE) ** (i / pairs) * 2 * math.pi) ** -1 * 2.0 ** 64) for i in range(pairs)]
    steps = torch.tensor(steps, device="cuda")
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"), torch.tensor(_sections(case), device="cuda"))
    return ((positions.long()[axis].T * steps) >> 32).float() * 2.0 ** -32


def _norm_rotate(case, x, weight, turns):
    x = x.float()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    c, s = torch.cos(2 * math.pi * turns)[:, None], torch.sin(2 * math.pi * turns)[:, None]
    r = case["rotary"]
    if case["pairs"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((turned, x[..., r:]), -1)


def _places(s):
    """Positions of the tokens' codes (in units of 4 bits) and scales (in units of 2 bytes) in the pool: K [n][heads][d], V, ..."""
    page, hk, d = (s["case"][k] for k in ("page", "kv_heads", "head_dim"))
    slots = s["slots"].long()[:, None]
    tile = (slots // page * hk + torch.arange(hk, device="cuda")) * (page // 16) + slots % page // 16
    at = tile[..., None] * (36 * d)
    tau = (slots % 16)[:, 0]
    k, v = (at + o.view(16, d)[tau][:, None] for o in _order_on_gpu(d))
    ks = tile[..., None] * (9 * d) + 8 * d + (tau * (d // 32))[:, None, None] + torch.arange(d // 32, device="cuda")
    return k, v + 16 * d, ks, ks + d // 2


def _write(s, k, v):
    pool = s["pool"].view(-1)
    nibbles = torch.stack((pool & 15, pool >> 4), -1).view(-1)
    places = _places(s)
    scales = {}
    for i, x in enumerate((k, v)):
        codes, scales[i] = _codes(x)
        nibbles[places[i]] = codes
    nibbles = nibbles.view(-1, 2)
    pool.copy_(nibbles[:, 0] | nibbles[:, 1] << 4)
    for i in range(2):
        pool.view(torch.float16)[places[2 + i]] = scales[i]


def _read(s):
    pool = s["pool"].view(-1)
    places = _places(s)
    got = []
    for i in range(2):
        codes = pool[places[i] // 2] >> (4 * (places[i] % 2)).to(torch.uint8) & 15
        scales = pool.view(torch.float16)[places[2 + i]].float()
        got.append(((codes.float() - 8).unflatten(-1, (-1, 32)) * scales[..., None]).flatten(-2).half())
    return got


def _run_attention(s):
    case = s["case"]
    if own:
        if case["queries"] == 1:
            s["plan"].run(s["q"], s["table"], s["lens"], s["out"])
        else:
            s["plan"].run(s["q"], s["table"], s["lens"], s["out"], q_starts=s["starts"], max_queries=case["queries"])
        return s["out"]
    h, hk, d, m = case["heads"], case["kv_heads"], case["head_dim"], case["queries"]
    k, v = _cached(s["pool"][0], s["table"])
    b, t = k.shape[0], k.shape[2]
    starts, lens = s["starts"].long(), s["lens"].long()
    news = starts[1:] - starts[:-1]
    i = torch.arange(m, device="cuda")
    rows = torch.minimum(starts[:-1, None] + i, starts[1:, None] - 1)  # [b][m]; beyond a sequence's queries the last again
    at = (lens - news)[:, None] + torch.minimum(i, news[:, None] - 1)
    key = torch.arange(t, device="cuda")
    sees = (key <= at[..., None]) & (key < lens[:, None, None])
    if case["window"]:
        sees &= key > at[..., None] - case["window"]
    sees = sees[:, None, None]                                            # [b][1][1][m][t]
    q = s["q"].float()[rows].view(b, m, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    exists = key < lens[:, None]
    k = torch.where(exists[:, None, :, None], k, 0.0)
    v = torch.where(exists[:, None, :, None], v, 0.0)
    score = q @ k[:, :, None].transpose(-1, -2)
    score *= d ** -0.5
    score.masked_fill_(~sees, float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    o = (score @ v[:, :, None]) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, m, h, d).half()
    token = torch.arange(s["q"].shape[0], device="cuda")
    seq = (starts[1:, None] <= token).sum(0)
    return o[seq, token - starts[seq]]


def _cached(pool, table):
    """K and V [batch][kv_heads][tokens][d] of the pages in `table`."""
    b, p = table.shape
    _, hk, per, size = pool.shape
    tiles = pool[table.long()].transpose(1, 2).reshape(-1, size)  # [b][hk][p][per]
    return [x.view(b, hk, p * per * 16, -1) for x in _values(tiles)]


def _run_pages(s):
    if own:
        s["cache"].copy_pages(s["src"], s["dst"])
    else:
        s["pool"][:, torch.tensor(s["dst"], device="cuda")] = s["pool"][:, torch.tensor(s["src"], device="cuda")]
    return s["pool"].view(torch.int32)


# ----------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    if case["kind"] == "pages":
        return None
    s = prepare(case, seed)
    return _exact_rope(case, s) if case["kind"] == "rope" else _exact_attention(case, s)


def _exact_rope(case, s):
    d, r = case["head_dim"], case["rotary"]
    half = r // 2
    scale_of = MIN_TIMESCALE * (MAX_TIMESCALE / MIN_TIMESCALE) ** (2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / r)
    axis = [a for a, n in enumerate(_sections(case)) for _ in range(n)]
    angle = s["positions"].double()[axis] / scale_of[:, None]  # [pairs][tokens]
    # which value of a head is a pair's first and second
    first = torch.arange(half, device="cuda") if case["pairs"] == "halves" else 2 * torch.arange(half, device="cuda")
    second = first + (half if case["pairs"] == "halves" else 1)

    def turned(x, w):
        x = x.double()
        x = x * w.double() / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt()
        z = torch.polar(torch.ones_like(angle), angle).T[:, None] * torch.complex(x[..., first], x[..., second])
        x[..., first], x[..., second] = z.real, z.imag
        return x

    q = turned(s["q"], s["q_weight"])
    if not case["cache"]:
        return {"q": q, "k": turned(s["k"], s["k_weight"])}
    # The keys in the cache have no value of this kind: which code a key gets goes by its value rounded to fp16.
    v = s["v"].double().unflatten(-1, (-1, 32))
    step = (v.abs().amax(-1, keepdim=True) / 7).bfloat16().half().double()
    v = torch.where(step > 0, step * torch.round(v / step).clamp(-7, 7), 0.0)
    return {"q": q, "k": None, "v": v.flatten(-2)}


def _exact_attention(case, s):
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    g = h // hk
    lens, news = _lengths(case)
    out = torch.zeros(sum(news), h, d, dtype=torch.float64, device="cuda")
    pool = s["pool"][0]
    where_k, where_v = (torch.from_numpy(x).cuda() for x in _order(d))
    start = 0
    for b, (n, m) in enumerate(zip(lens, news)):
        lo = max(0, n - m - case["window"]) // 16 * 16 if case["window"] else 0
        for j in range(hk if n > lo else 0):
            tiles = pool[s["table"][b, :-(-n // case["page"])].long(), j].reshape(-1, 18 * d)[lo // 16:-(-n // 16)]
            part = []
            for codes, scales, where in ((tiles[:, :8 * d], tiles[:, 16 * d:17 * d], where_k),
                                         (tiles[:, 8 * d:16 * d], tiles[:, 17 * d:], where_v)):
                c = (codes[:, where // 2] >> (where % 2 * 4).to(torch.uint8) & 15).double() - 8
                f = scales.contiguous().view(torch.float16).view(-1, 16, d // 32).double()
                part.append((c * f.repeat_interleave(32, -1)).reshape(-1, d)[:n - lo])
            k, v = part
            key = torch.arange(lo, n, device="cuda")
            for i0 in range(0, m, 256):
                i1 = min(m, i0 + 256)
                at = torch.arange(n - m + i0, n - m + i1, device="cuda")[:, None]
                sees = key <= at
                if case["window"]:
                    sees &= key > at - case["window"]
                q = s["q"][start + i0:start + i1, j * g:(j + 1) * g].double()
                w = torch.einsum("mgd,td->gmt", q, k) / math.sqrt(d)
                w = torch.softmax(w.masked_fill(~sees, -math.inf), -1).nan_to_num_(0.0)
                out[start + i0:start + i1, j * g:(j + 1) * g] = torch.einsum("gmt,td->mgd", w, v)
        start += m
    return out
