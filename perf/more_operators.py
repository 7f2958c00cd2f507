"""Measured cases of rotary positions, appends that rotate on the way, and
attention over a paged cache of latent rows.

A latent row of a token is ``latent`` values that keys and values of every head
are made from, and ``rope`` values that hold its position.  The arena keeps a
layer's rows as 16-bit ``[pages, page_tokens, latent + rope]``; a request's
tokens lie in the pages that its row of the block table names.

* ``rotate``   rotary positions put on rows of several heads, or taken off
* ``append``   a step's rows written into their pages with the keys rotated on the
               way: keys and values of 8 bits with one scale for each page and kv
               head (``arena="codes"``), or latent rows (``arena="latent"``)
* ``absorbed`` attention whose queries are in the latent space already: scores and
               results are taken from the cached rows themselves
* ``expanded`` attention whose keys and values of each head are made from the
               cached rows by the head's weights first

A case names its sizes; the requests' lengths follow from them and from the
case's own ``shape`` number, so that ``work`` needs no inputs.
"""

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
SCALINGS = ("none", "linear", "ntk", "yarn", "factors")


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # Queries of one decode step whose heads end in a positional part, with a
        # factor for each frequency.
        dict(name="rotate_step_r61", op="rotate", tokens=61, heads=40, head_dim=96, offset=64,
             dim=32, layout="half", scaling="factors", position_max=32768, inverse=False,
             type="bf16", shape=1),
        # Queries of long prompts, far positions, the whole head.
        dict(name="rotate_prompts", op="rotate", tokens=8449, heads=32, head_dim=128, offset=0,
             dim=128, layout="half", scaling="yarn", position_max=131072, inverse=False,
             type="bf16", shape=2),
        # Keys read back for a harvest: positions taken off half of each head.
        dict(name="rotate_harvest", op="rotate", tokens=2047, heads=8, head_dim=128, offset=0,
             dim=64, layout="interleaved", scaling="linear", position_max=16384, inverse=True,
             type="f32", shape=3),
        # One decode step's keys and values of 61 conversations, 8 bits.
        dict(name="append_step_r61", op="append", arena="codes", page=64, requests=61,
             cached_min=1, cached_max=4000, fresh_min=1, fresh_max=1, kv_heads=8, head_dim=128,
             dim=128, layout="half", scaling="none", type="bf16", shape=4),
        # Ragged prompts of a model with few wide heads, part of the head rotated.
        dict(name="append_prompts", op="append", arena="codes", page=32, requests=11,
             cached_min=0, cached_max=900, fresh_min=37, fresh_max=4096, kv_heads=8,
             head_dim=128, dim=64, layout="interleaved", scaling="yarn", type="f16", shape=5),
        # Latent rows of ragged prompts: the projection's row holds both parts.
        dict(name="append_latent", op="append", arena="latent", page=64, requests=23,
             cached_min=0, cached_max=5000, fresh_min=1, fresh_max=2048, latent=256, rope=32,
             layout="half", scaling="factors", type="bf16", shape=6),
        # One short conversation: latency alone.
        dict(name="absorbed_step_short", op="absorbed", page=64, requests=1, length_min=333,
             length_max=333, fresh_min=1, fresh_max=1, heads=40, latent=256, rope=32,
             causal=True, type="bf16", shape=7),
        # A full decode batch of ragged conversations.
        dict(name="absorbed_step_batch", op="absorbed", page=64, requests=64, length_min=200,
             length_max=16384, fresh_min=1, fresh_max=1, heads=40, latent=256, rope=32,
             causal=True, type="bf16", shape=8),
        # One very long conversation over wide rows.
        dict(name="absorbed_step_long", op="absorbed", page=32, requests=1, length_min=250007,
             length_max=250007, fresh_min=1, fresh_max=1, heads=16, latent=512, rope=64,
             causal=True, type="f16", shape=9),
        # Several proposed tokens of each request checked at once.
        dict(name="absorbed_verify", op="absorbed", page=16, requests=16, length_min=100,
             length_max=8192, fresh_min=5, fresh_max=5, heads=40, latent=256, rope=32,
             causal=True, type="bf16", shape=10),
        # Ragged prompts that start from nothing, wide heads.
        dict(name="expanded_fresh", op="expanded", page=32, requests=7, length_min=19,
             length_max=1500, fresh_min=1500, fresh_max=1500, heads=16, latent=512, rope=64,
             nope=128, value=128, causal=True, type="f16", shape=11),
        # Pieces of prompts on top of what is cached: bound by arithmetic.
        dict(name="expanded_prompt", op="expanded", page=64, requests=3, length_min=5000,
             length_max=16000, fresh_min=1000, fresh_max=4000, heads=40, latent=256, rope=32,
             nope=64, value=64, causal=True, type="bf16", shape=12),
    ]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        for k in ("bytes", "flops"):
            most[k] = max(most.get(k, 0), w[k])
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _draw(rng):
    op = rng.choice(["rotate", "append", "append", "absorbed", "absorbed", "absorbed", "expanded",
                     "expanded"])
    c = dict(op=op, shape=rng.randrange(1 << 30), type=rng.choice(["bf16", "f16"]))
    if op in ("rotate", "append"):
        c.update(layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(SCALINGS))
    if op == "rotate":
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        before, after = rng.choice([(0, 0), (0, 0), (64, 0), (0, 32), (128, 0), (0, 128)])
        c.update(tokens=_log_between(rng, 1, 9000), heads=rng.choice([1, 2, 5, 8, 16, 32, 40]),
                 head_dim=before + dim + after, offset=before, dim=dim,
                 position_max=_log_between(rng, 100, 1 << 20), inverse=rng.random() < 0.3,
                 type=rng.choice(["bf16", "f16", "f32"]))
        return c
    c["page"] = rng.choice([16, 32, 64, 128])
    if op == "append":
        c["requests"] = _log_between(rng, 1, 200)
        c.update(cached_min=0, cached_max=_log_between(rng, 1, 6000), fresh_min=1,
                 fresh_max=rng.choice([1, _log_between(rng, 2, 300), _log_between(rng, 100, 4000)]))
        if sum(lengths(c)[1]) > 12000:
            return _draw(rng)
        c["arena"] = rng.choice(["codes", "codes", "latent"])
        if c["arena"] == "codes":
            c["head_dim"] = rng.choice([64, 128, 128, 256])
            c["kv_heads"] = rng.choice([1, 2, 4, 5, 8])
            c["dim"] = rng.choice([d for d in (32, 64, 96, 128, 256) if d <= c["head_dim"]])
        else:
            c["latent"], c["rope"] = rng.choice([128, 256, 256, 512]), rng.choice([32, 64])
        return c
    c["latent"], c["rope"] = rng.choice([128, 256, 256, 512]), rng.choice([32, 64])
    c["heads"] = rng.choice([1, 5, 8, 16, 16, 32, 40, 40, 128])
    kind = rng.choice(["step", "step", "verify", "memory"] if op == "absorbed" else
                      ["prompt", "prompt", "fresh", "memory"])
    c["causal"] = kind != "memory"
    if op == "absorbed":
        c["requests"] = _log_between(rng, 1, 100)
        top = _log_between(rng, rng.choice([1, 300]), 60000)
        c.update(length_min=rng.choice([1, top]) if c["causal"] else 0, length_max=top, fresh_min=1,
                 fresh_max=1 if kind == "step" else rng.randrange(2, 17))
    else:
        c["nope"] = c["value"] = rng.choice([64, 128])
        c["requests"] = _log_between(rng, 1, 8)
        top = _log_between(rng, 100, 12000)
        rows = top if kind == "fresh" else _log_between(rng, 2, 3000)
        c.update(length_min=rng.choice([1, top]) if c["causal"] else 0, length_max=top,
                 fresh_min=rows if kind == "fresh" else 1, fresh_max=rows)
    return c


def lengths(case):
    """(cached, fresh) of every request: tokens already in the arena and the
    step's new rows.  The first request takes the upper ends."""
    rng = random.Random(case["shape"])

    def one(what, top):
        lo, hi = case[what + "_min"], case[what + "_max"]
        if top or lo == hi:
            return hi
        if lo == 0 and rng.random() < 0.15:
            return 0
        return _log_between(rng, max(lo, 1), hi)

    cached, fresh = [], []
    for r in range(case["requests"]):
        n = one("fresh", r == 0)
        if case["op"] != "append":
            total = one("length", r == 0)
            if case["causal"]:  # the rows are the last ones of the cached tokens
                n = min(n, total)
                total -= n
            cached.append(total)
        else:
            cached.append(one("cached", r == 0))
        fresh.append(n)
    return cached, fresh


def _grows(case):
    return case["op"] == "append" or case["causal"]


def _after(case):
    cached, fresh = lengths(case)
    return [c + n if _grows(case) else c for c, n in zip(cached, fresh)]


def _pages(n, page):
    return -(-n // page)


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["head_dim"] * size + 4 * case["tokens"],
                "flops": 3 * n * case["dim"]}
    cached, fresh = lengths(case)
    after, page, tokens = _after(case), case["page"], sum(fresh)
    if case["op"] == "append":
        if case["arena"] == "latent":
            return {"bytes": 2 * tokens * (case["latent"] + case["rope"]) * size + 12 * tokens,
                    "flops": 3 * tokens * case["rope"]}
        H, D = case["kv_heads"], case["head_dim"]
        span = [(c // page * page, a) for c, a, n in zip(cached, after, fresh) if n]
        touched = sum(a - f for f, a in span)
        pages = sum(_pages(a - f, page) for f, a in span)
        return {"bytes": 2 * H * (tokens * D * (2 + 1) + touched * D * (1 + 2) + 8 * pages),
                "flops": 2 * H * D * (3 * tokens + touched) + 3 * H * case["dim"] * tokens}
    H, C, R = case["heads"], case["latent"], case["rope"]
    seen = 0
    for c, n in zip(cached, fresh):
        seen += n * c + (n * (n + 1) // 2 if case["causal"] else 0)
    held = sum(a for a, n in zip(after, fresh) if n)
    pages = sum(_pages(a, page) for a, n in zip(after, fresh) if n)
    read = held * (C + R) * 2 + 4 * pages
    if case["op"] == "absorbed":
        return {"bytes": read + tokens * H * ((C + R) * 2 + C * 2 + 4),
                "flops": 2 * (2 * C + R) * H * seen}
    N, V = case["nope"], case["value"]
    return {"bytes": read + H * (N + V) * C * 2 + tokens * H * ((N + R) * 2 + V * 2 + 4),
            "flops": 2 * C * H * (N + V) * held + 2 * (N + R + V) * H * seen}


# ------------------------------------------------------------ rotary frequencies

def _scaling(kind, dim):
    """The scaling that a case names, as a user writes it."""
    if kind == "linear":
        return dict(kind="linear", factor=4.0)
    if kind == "ntk":
        return dict(kind="ntk", factor=8.0)
    if kind == "yarn":
        return dict(kind="yarn", factor=16.0, original=4096)
    if kind == "factors":
        return dict(kind="factors", amplitude=1.19,
                    factors=[1.0 + 0.05 * i * i for i in range(dim // 2)])
    return None


def _frequencies(kind, dim, base=10000.0):
    """Radians a position of each pair, in 64 bits, and the amplitude."""
    i = np.arange(dim // 2, dtype=np.float64)
    s = _scaling(kind, dim) or {}
    if kind == "ntk":  # the base that leaves the first pair alone and slows the last by `factor`
        base = base * s["factor"] ** (dim / (dim - 2))
    f = base ** (-2.0 * i / dim)
    if kind == "linear":
        return f / s["factor"], 1.0
    if kind == "factors":
        return f / np.array(s["factors"]), s["amplitude"]
    if kind == "yarn":  # pairs that turn often keep their frequency, slow ones are interpolated
        def pair(turns):
            return dim * math.log(s["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
        slow = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f * (1 - slow) + f / s["factor"] * slow, 0.1 * math.log(s["factor"]) + 1.0
    return f, 1.0


# ------------------------------------------------------------------ the inputs

def _tables(case, seed):
    """Block table of the cached tokens, ring of free pages and its cursor."""
    cached, _ = lengths(case)
    after, page = _after(case), case["page"]
    rng = np.random.default_rng(seed)
    have = [_pages(c, page) for c in cached]
    need = [_pages(a, page) for a in after]
    pool = sum(need) + 7  # a few pages stay free
    order = rng.permutation(pool).astype(np.int32)
    table = np.full((case["requests"], max(max(need), 1) + 2), -1, np.int32)
    at = 0
    for r, h in enumerate(have):
        table[r, :h] = order[at:at + h]
        at += h
    first = int(rng.integers(0, pool))  # the ring has turned before
    ring = np.full(pool, -1, np.int32)
    left = order[at:]
    ring[(first + np.arange(len(left))) % pool] = left
    cursor = np.array([first, first + len(left)], np.int64)
    full = table.copy()  # with the step's new pages in it
    for r, (h, n) in enumerate(zip(have, need)):
        full[r, h:n] = left[:n - h]
        left = left[n - h:]
    return table, full, ring, cursor, pool


def _normal(shape, gen, kind, spread=1.0):
    return (torch.randn(shape, device=DEVICE, generator=gen) * spread).to(kind)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, op = TYPES[case["type"]], case["op"]
    st = {"case": case}
    if op in ("rotate", "append"):
        dim = case["rope"] if case.get("arena") == "latent" else case["dim"]
        f, st["amplitude"] = _frequencies(case["scaling"], dim)
        st["frequencies"] = torch.from_numpy(f).to(DEVICE)
    if op == "rotate":
        T = case["tokens"]
        st["x"] = _normal((T, case["heads"], case["head_dim"]), gen, kind)
        st["positions"] = torch.randint(0, case["position_max"], (T,), device=DEVICE,
                                        generator=gen, dtype=torch.int32)
        if own:
            st["rotary"] = _own_rotary(case, case["dim"], case["offset"])
        return st
    cached, fresh = lengths(case)
    after, page, T = _after(case), case["page"], sum(fresh)
    table, full, ring, cursor, pool = _tables(case, seed)
    rows = np.concatenate([np.full(n, r, np.int64) for r, n in enumerate(fresh)])
    positions = np.concatenate([np.arange(c, c + n) for c, n in zip(cached, fresh)])
    if _grows(case):
        slots = full[rows, positions // page].astype(np.int64) * page + positions % page
    else:
        slots = np.full(T, -1, np.int64)
    put = lambda x: torch.from_numpy(x).to(DEVICE)
    st.update(host=(cached, fresh, after), tokens=T, table=put(full), slots=put(slots),
              positions=put(positions.astype(np.int32)))
    if op == "append" and case["arena"] == "codes":
        H, D = case["kv_heads"], case["head_dim"]
        st["codes"], st["scales"] = [], []
        for _ in range(2):  # codes and scales as an earlier store leaves them
            s = torch.exp(0.3 * torch.randn((pool, H), device=DEVICE, generator=gen)) * 0.03
            st["scales"].append(s)
            st["codes"].append(torch.randint(-127, 128, (pool, H, page, D), device=DEVICE,
                                             generator=gen, dtype=torch.int8))
        # rows as a fused projection leaves them: keys beside values
        kv = torch.randn((T, 2, H, D), device=DEVICE, generator=gen)
        kv *= torch.exp(0.3 * torch.randn((1, 2, H, D), device=DEVICE, generator=gen))
        kv = kv.to(kind)
        st["k"], st["v"] = kv[:, 0], kv[:, 1]
        st["touched"] = _touched(st, page)
    else:
        C, R = case["latent"], case["rope"]
        cache = torch.empty((pool, page, C + R), dtype=kind, device=DEVICE)
        step = max(1, (1 << 26) // (page * (C + R)))
        for a in range(0, pool, step):
            cache[a:a + step] = _normal((min(pool, a + step) - a, page, C + R), gen, kind)
        st["cache"] = cache
        if op == "append":
            kv = _normal((T, C + R), gen, kind)
            st["latent"], st["rope"] = kv[:, :C], kv[:, C:]
        elif op == "absorbed":
            # as a head's weights take a query of unit values to the latent space
            st["q_latent"] = _normal((T, case["heads"], C), gen, kind, 8 / math.sqrt(C))
            st["q_rope"] = _normal((T, case["heads"], R), gen, kind)
            st["scale"] = (64 + R) ** -0.5
        else:
            N, V, H = case["nope"], case["value"], case["heads"]
            st["q"] = _normal((T, H, N + R), gen, kind)
            st["weights"] = _normal((H, N + V, C), gen, kind, C ** -0.5)
            st["scale"] = (N + R) ** -0.5
    if own:
        _prepare_own(st, table, ring, cursor, pool)
    return st


def _touched(st, page):
    """Slots of every token in the pages that the step writes."""
    cached, fresh, after = st["host"]
    r = np.concatenate([np.full(a - c // page * page, i) for i, (c, a, n)
                        in enumerate(zip(cached, after, fresh)) if n])
    pos = np.concatenate([np.arange(c // page * page, a) for c, a, n
                          in zip(cached, after, fresh) if n])
    r, pos = torch.from_numpy(r).to(DEVICE), torch.from_numpy(pos).to(DEVICE)
    return st["table"][r, pos // page].long() * page + pos % page


def _own_rotary(case, dim, offset):
    from graftrepository_b200.rotary import Rotary

    return Rotary(dim, offset=offset, layout=case["layout"],
                  scaling=_scaling(case["scaling"], dim), device=DEVICE)


def _prepare_own(st, table, ring, cursor, pool):
    from graftrepository_b200 import latent_arena, paged_arena

    case = st["case"]
    cached, fresh, after = st["host"]
    tables = paged_arena.PageTables(case["requests"], pool, table.shape[1],
                                    page_tokens=case["page"], device=DEVICE)
    tables.table.copy_(torch.from_numpy(table))
    tables.lens.copy_(torch.tensor(cached, dtype=torch.int32))
    tables.ring.copy_(torch.from_numpy(ring))
    tables.cursor.copy_(torch.from_numpy(cursor))
    kind, most = TYPES[case["type"]], max(fresh)
    if case.get("arena") == "codes":
        plan = tables.make_plan(st["tokens"], kv_heads=case["kv_heads"],
                                query_heads=case["kv_heads"], head_dim=case["head_dim"],
                                max_fresh=most)
        arena = paged_arena.PagedArena(1, pool, case["kv_heads"], case["head_dim"],
                                       page_tokens=case["page"], device=DEVICE)
        (k, v), (ks, vs) = st.pop("codes"), st.pop("scales")
        for to, x in ((arena.k_codes, k), (arena.v_codes, v), (arena.k_scales, ks),
                      (arena.v_scales, vs)):
            to[0].copy_(x)
        st["rotary"] = _own_rotary(case, case["dim"], 0)
    else:
        C, R = case["latent"], case["rope"]
        arena = latent_arena.LatentArena(1, pool, C, R, page_tokens=case["page"], dtype=kind,
                                         device=DEVICE)
        arena.rows[0].copy_(st.pop("cache"))
        sizes = dict(heads=case.get("heads", 1), max_fresh=most)
        if case["op"] == "expanded":
            held = sum(_pages(a, 64) * 64 for a, n in zip(after, fresh) if n)
            sizes.update(nope=case["nope"], value=case["value"], expand_tokens=held)
        plan = arena.make_plan(tables, st["tokens"], **sizes)
        if case["op"] == "append":
            st["rotary"] = _own_rotary(case, R, 0)
    tables.plan(plan, torch.tensor(fresh, dtype=torch.int32, device=DEVICE), grow=_grows(case))
    st["tables"], st["plan"], st["arena"] = tables, plan, arena


# ------------------------------------------------------------- the plain forms

def _turn(x, positions, frequencies, amplitude, layout, inverse=False):
    """Rows x [T, heads, dim] turned by their positions: angles in 64 bits, values in 32."""
    angle = positions.double()[:, None] * frequencies[None]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    gain = amplitude
    if inverse:
        sin, gain = -sin, 1.0 / amplitude
    x, half = x.float(), x.shape[2] // 2
    a, b = (x[..., :half], x[..., half:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    c, d = (a * cos - b * sin) * gain, (b * cos + a * sin) * gain
    if layout == "half":
        return torch.cat([c, d], 2)
    return torch.stack([c, d], 3).flatten(2)


def _rotate_plain(st):
    case, x = st["case"], st["x"]
    a, b = case["offset"], case["offset"] + case["dim"]
    y = _turn(x[:, :, a:b], st["positions"], st["frequencies"], st["amplitude"], case["layout"],
              case["inverse"])
    return torch.cat([x[:, :, :a], y.to(x.dtype), x[:, :, b:]], 2)


def _store_plain(st, x, codes, scales):
    """Quantises x [T, H, D] (32 bits) into codes and scales, in place."""
    page, slots = st["case"]["page"], st["slots"]
    T, H, D = x.shape
    first = torch.ones(T, dtype=torch.bool, device=DEVICE)  # first row of its page
    first[1:] = (slots[1:] // page) != (slots[:-1] // page)
    unit = torch.cumsum(first, 0) - 1
    n = int(unit[-1]) + 1
    begin = torch.full((n,), 1 << 60, dtype=torch.int64, device=DEVICE)
    begin.scatter_reduce_(0, unit, slots, "amin")
    pages, off = begin // page, begin % page
    top = torch.zeros((n, H), device=DEVICE)
    top.scatter_reduce_(0, unit[:, None].expand(T, H), x.abs().amax(2), "amax")
    old = torch.where((off > 0)[:, None], scales[pages], 0.0)
    s = torch.maximum(old, top / 127.0)
    safe = torch.where(s > 0, s, 1.0)
    moved = torch.round(codes[pages].float() * old[:, :, None, None] / safe[:, :, None, None])
    keep = torch.arange(page, device=DEVICE)[None, :] < off[:, None]
    codes[pages] = torch.where(keep[:, None, :, None], moved.to(torch.int8), codes[pages])
    codes[slots // page, :, slots % page] = torch.round(x / safe[unit][:, :, None]).to(torch.int8)
    scales[pages] = s


def _values(codes, scales, slots, page):
    at = slots // page
    return codes[at, :, slots % page].float() * scales[at][:, :, None]


def _append_plain(st):
    case = st["case"]
    turned = lambda x: _turn(x, st["positions"], st["frequencies"], st["amplitude"],
                             case["layout"])
    if case["arena"] == "latent":
        rows, C = st["cache"].view(-1, st["cache"].shape[2]), case["latent"]
        rows[st["slots"], :C] = st["latent"]
        rows[st["slots"], C:] = turned(st["rope"][:, None])[:, 0].to(rows.dtype)
        return [st["cache"]]
    d, got = case["dim"], []
    k = torch.cat([turned(st["k"][:, :, :d]), st["k"][:, :, d:].float()], 2)
    for x, codes, scales in zip((k, st["v"].float()), st["codes"], st["scales"]):
        _store_plain(st, x, codes, scales)
        got += [_values(codes, scales, st["touched"], case["page"]).to(st["v"].dtype), scales]
    return got


def _softmax_plain(st, i, n, s, v, out, lse, head, c, a):
    """Scores s [rows, L] of `n` tokens' rows (several heads a token) and values v
    [L, V]: results into out and lse at tokens a.., heads `head`."""
    per = s.shape[0] // n
    if st["case"]["causal"]:
        last = c + i + torch.arange(n, device=DEVICE).repeat_interleave(per)
        s.masked_fill_(torch.arange(s.shape[1], device=DEVICE)[None, :] > last[:, None], -math.inf)
    top = s.amax(1, keepdim=True)
    s = torch.exp(s - top)
    total = s.sum(1, keepdim=True)
    y = (s @ v) / total
    out[a + i:a + i + n, head] = y.view(n, per, -1).to(out.dtype)
    lse[a + i:a + i + n, head] = (top + torch.log(total)).view(n, per)


def _held(st, r, L):
    """The rows that request r holds, in token order, in 32 bits."""
    page = st["case"]["page"]
    pages = st["table"][r, :_pages(L, page)].long()
    return st["cache"][pages].view(-1, st["cache"].shape[2])[:L].float()


def _attend_plain(st):
    case = st["case"]
    cached, fresh, after = st["host"]
    H, C, T = case["heads"], case["latent"], st["tokens"]
    wide = C if case["op"] == "absorbed" else case["value"]
    kind = st["cache"].dtype
    out = torch.zeros((T, H, wide), dtype=kind, device=DEVICE)
    lse = torch.full((T, H), -math.inf, device=DEVICE)
    a = 0
    for r, (c, n, L) in enumerate(zip(cached, fresh, after)):
        if n and L:
            rows = _held(st, r, L)
            if case["op"] == "absorbed":
                most = max(1, (1 << 28) // (H * L))  # tokens whose scores fit at once
                for i in range(0, n, most):
                    m = min(most, n - i)
                    q = torch.cat([st["q_latent"][a + i:a + i + m].float(),
                                   st["q_rope"][a + i:a + i + m].float()], 2).view(m * H, -1)
                    _softmax_plain(st, i, m, (q @ rows.T) * st["scale"], rows[:, :C], out, lse,
                                   slice(None), c, a)
            else:
                N, w = case["nope"], st["weights"]
                for h in range(H):
                    k = torch.cat([rows[:, :C] @ w[h, :N].float().T, rows[:, C:]], 1)
                    v = rows[:, :C] @ w[h, N:].float().T
                    s = (st["q"][a:a + n, h].float() @ k.T) * st["scale"]
                    _softmax_plain(st, 0, n, s, v, out, lse, slice(h, h + 1), c, a)
        a += n
    return [out, lse]


# -------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "rotate":
        return _rotate_plain(state)
    if op == "append":
        return _append_plain(state)
    return _attend_plain(state)


def _run_own(st, op):
    case = st["case"]
    if op == "rotate":
        return st["rotary"].rotate(st["x"], st["positions"], inverse=case["inverse"])
    arena, plan = st["arena"], st["plan"]
    if op == "append":
        if case["arena"] == "latent":
            arena.append(plan, st["latent"], st["rope"], rotary=st["rotary"])
            return [arena.rows[0]]
        arena.append(plan, st["k"], st["v"], rotary=st["rotary"])
        k, v = arena.read(st["touched"], dtype=st["k"].dtype)
        return [k, arena.k_scales[0], v, arena.v_scales[0]]
    if op == "absorbed":
        return list(arena.attend(plan, st["q_latent"], st["q_rope"], scale=st["scale"],
                                 causal=case["causal"]))
    return list(arena.attend_expanded(plan, st["q"], st["weights"], scale=st["scale"],
                                      causal=case["causal"]))


# ------------------------------------------------------ the definitions, 64 bits

def exact(case, seed):
    if case["op"] in ("absorbed", "expanded") and work(case)["flops"] > 8e12:
        return None
    global own
    held, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = held
    if case["op"] == "rotate":
        return _rotate_exact(st)
    if case["op"] == "append":
        return _append_exact(st)
    return _attend_exact(st)


def _complex_turn(st, x, inverse=False):
    """x [T, heads, dim] as complex numbers times amplitude * e^(i angle)."""
    case = st["case"]
    x = x.double()
    if case["layout"] == "half":
        z = torch.complex(*x.chunk(2, 2))
    else:
        z = torch.view_as_complex(x.unflatten(2, (-1, 2)).contiguous())
    w = torch.polar(torch.full_like(st["frequencies"], st["amplitude"])[None],
                    torch.outer(st["positions"].double(), st["frequencies"]))[:, None]
    z = z / w if inverse else z * w
    y = torch.view_as_real(z)
    return torch.cat([y[..., 0], y[..., 1]], 2) if case["layout"] == "half" else y.flatten(2)


def _rotate_exact(st):
    case, y = st["case"], st["x"].double()
    part = slice(case["offset"], case["offset"] + case["dim"])
    y[:, :, part] = _complex_turn(st, st["x"][:, :, part], case["inverse"])
    return y


def _append_exact(st):
    case = st["case"]
    cached, fresh, after = st["host"]
    page, table = case["page"], st["table"].cpu().numpy()
    if case["arena"] == "latent":
        cache = st["cache"].double()
        new = torch.cat([st["latent"].double(), _complex_turn(st, st["rope"][:, None])[:, 0]], 1)
        at = 0
        for r, (c, n) in enumerate(zip(cached, fresh)):
            for p in range(c // page, _pages(c + n, page)):
                lo, hi = max(c, p * page), min(c + n, (p + 1) * page)
                cache[int(table[r, p]), lo - p * page:hi - p * page] = new[at + lo - c:at + hi - c]
            at += n
        return [cache]
    k = st["k"].double()
    k[:, :, :case["dim"]] = _complex_turn(st, st["k"][:, :, :case["dim"]])
    out = []
    for x, codes, scales in zip((k, st["v"].double()), st["codes"], st["scales"]):
        s64, got, at = scales.double(), [], 0
        for r, (c, n) in enumerate(zip(cached, fresh)):
            pos = c
            while pos < c + n:
                p, off = int(table[r, pos // page]), pos % page
                m = min(page - off, c + n - pos)
                new = x[at + pos - c:at + pos - c + m]                      # [m, H, D]
                old = codes[p, :, :off].double()                           # [H, off, D]
                s = new.abs().amax((0, 2)) / 127
                if off:
                    s = torch.maximum(s, s64[p])
                    old = old * s64[p][:, None, None]
                held = torch.cat([old, new.transpose(0, 1)], 1)            # [H, off + m, D]
                step = torch.where(s > 0, s, 1.0)[:, None, None]
                got.append((torch.round(held / step) * s[:, None, None]).transpose(0, 1))
                s64[p] = s
                pos += m
            at += n
        out += [torch.cat(got), s64]
    return out


def _attend_exact(st):
    case, page = st["case"], st["case"]["page"]
    cached, fresh, after = st["host"]
    H, C = case["heads"], case["latent"]
    wide = C if case["op"] == "absorbed" else case["value"]
    ys, zs, a = [], [], 0
    for r in range(case["requests"]):
        n, L = fresh[r], after[r]
        y = torch.zeros((n, H, wide), dtype=torch.float64, device=DEVICE)
        z = torch.full((n, H), -math.inf, dtype=torch.float64, device=DEVICE)
        if n and L:
            t = torch.arange(L, device=DEVICE)
            rows = st["cache"][st["table"][r, t // page].long(), t % page].double()
            unseen = t[None, :] > (cached[r] + torch.arange(n, device=DEVICE))[:, None]
            for h in range(H):
                if case["op"] == "absorbed":
                    q = torch.cat([st["q_latent"][a:a + n, h], st["q_rope"][a:a + n, h]], 1)
                    k, v = rows, rows[:, :C]
                else:
                    kv = rows[:, :C] @ st["weights"][h].double().T
                    q, v = st["q"][a:a + n, h], kv[:, case["nope"]:]
                    k = torch.cat([kv[:, :case["nope"]], rows[:, C:]], 1)
                s = q.double() @ k.T * st["scale"]
                if case["causal"]:
                    s.masked_fill_(unseen, -math.inf)
                z[:, h] = torch.logsumexp(s, 1)
                y[:, h] = torch.exp(s - z[:, h, None]) @ v
        ys.append(y)
        zs.append(z)
        a += n
    return [torch.cat(ys), torch.cat(zs)]
