"""Measured cases of the 8-bit paged arena: the step plan, the store and the attention.

The arena keeps a layer's keys and values as int8 codes ``[pages, kv_heads,
page_tokens, head_dim]`` with one fp32 scale for each (page, kv head); a value
is ``code * scale``.  A request's tokens lie in the pages that its row of the
block table names.

* ``plan``    block table, slots, positions and row ranges of one step, from
              the requests' lengths, with pages taken from a ring of free ones
* ``store``   a step's new key and value rows quantised into their pages (a
              page that needs a larger scale has its older codes rescaled),
              and the pages that it touched read back as values
* ``attend``  attention of a step's query rows over the arena, with the
              logarithm of each row's sum

A case names its sizes; the requests' lengths follow from them and from the
case's own ``shape`` number, so that ``work`` needs no inputs.
"""

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # The plan of one decode step: 64 conversations, one token each.
        dict(name="plan_step_r64", op="plan", page=64, requests=64, cached_min=1, cached_max=8192,
             fresh_min=1, fresh_max=1, shape=1),
        # A step that mixes decoding requests with idle ones and pieces of
        # prompts, small pages, a number of requests that fills no block.
        dict(name="plan_mixed_r1023", op="plan", page=16, requests=1023, cached_min=0,
             cached_max=4096, fresh_min=0, fresh_max=300, shape=2),
        # The largest: a whole queue of prompts planned in one call.
        dict(name="plan_prompts_r4096", op="plan", page=32, requests=4096, cached_min=0,
             cached_max=600, fresh_min=1, fresh_max=400, shape=3),
        # One decode step's rows of 61 conversations; most land in a page that
        # older tokens already share.
        dict(name="store_step_r61", op="store", page=64, requests=61, cached_min=1,
             cached_max=4000, fresh_min=1, fresh_max=1, kv_heads=8, dim=128, type="bf16", shape=4),
        # Prompts of ragged lengths, as a turn with mounted grafts writes them.
        dict(name="store_prompts_f16", op="store", page=32, requests=11, cached_min=0,
             cached_max=900, fresh_min=37, fresh_max=4096, kv_heads=8, dim=128, type="f16", shape=5),
        # Few wide heads and small pages.
        dict(name="store_prompts_d256", op="store", page=16, requests=5, cached_min=0,
             cached_max=100, fresh_min=100, fresh_max=1500, kv_heads=4, dim=256, type="bf16", shape=6),
        # One short conversation: latency alone.
        dict(name="attend_step_short", op="attend", page=64, requests=1, length_min=333,
             length_max=333, fresh_min=1, fresh_max=1, kv_heads=8, group=4, dim=128, type="bf16",
             causal=True, shape=7),
        # A full decode batch of ragged conversations.
        dict(name="attend_step_batch", op="attend", page=64, requests=64, length_min=200,
             length_max=16384, fresh_min=1, fresh_max=1, kv_heads=8, group=4, dim=128, type="bf16",
             causal=True, shape=8),
        # One very long conversation.
        dict(name="attend_step_long", op="attend", page=32, requests=1, length_min=250007,
             length_max=250007, fresh_min=1, fresh_max=1, kv_heads=8, group=4, dim=128, type="f16",
             causal=True, shape=9),
        # Query rows over mounted memory that they do not extend; some
        # requests have nothing mounted, so their rows are empty.
        dict(name="attend_memory_d64", op="attend", page=16, requests=24, length_min=0,
             length_max=3000, fresh_min=1, fresh_max=3, kv_heads=16, group=1, dim=64, type="bf16",
             causal=False, shape=10),
        # Several proposed tokens of each request checked at once, wide heads.
        dict(name="attend_verify_d256", op="attend", page=64, requests=16, length_min=100,
             length_max=8192, fresh_min=5, fresh_max=5, kv_heads=4, group=4, dim=256, type="bf16",
             causal=True, shape=11),
        # Pieces of prompts on top of what is already cached: the one case
        # that is bound by arithmetic.
        dict(name="attend_prompt", op="attend", page=64, requests=3, length_min=5000,
             length_max=16000, fresh_min=1000, fresh_max=4000, kv_heads=8, group=4, dim=128,
             type="bf16", causal=True, shape=12),
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
        op = rng.choice(["plan", "store", "attend", "attend", "attend"])
        c = dict(op=op, page=rng.choice([16, 32, 64, 128]), shape=rng.randrange(1 << 30))
        if op == "plan":
            c["requests"] = _log_between(rng, 1, 4096)
            c.update(cached_min=0, cached_max=_log_between(rng, 1, 8192),
                     fresh_min=rng.choice([0, 1]), fresh_max=_log_between(rng, 1, 2000))
            if sum(lengths(c)[1]) > sum(lengths(listed()[2])[1]):
                continue
        else:
            c["dim"] = rng.choice([64, 128, 128, 256])
            c["kv_heads"] = rng.choice([1, 2, 4, 5, 8, 16])
            c["type"] = rng.choice(["bf16", "f16"])
        if op == "store":
            c["requests"] = _log_between(rng, 1, 200)
            c.update(cached_min=0, cached_max=_log_between(rng, 1, 4000), fresh_min=1,
                     fresh_max=rng.choice([1, _log_between(rng, 2, 300),
                                           _log_between(rng, 100, 4000)]))
            if sum(lengths(c)[1]) > 20000:
                continue
        if op == "attend":
            c["group"] = rng.choice([1, 2, 3, 4, 5, 7, 8, 12])
            kind = rng.choice(["step", "step", "verify", "memory", "prompt", "prompt"])
            c["causal"] = kind != "memory"
            c["requests"] = _log_between(rng, 1, 4 if kind == "prompt" else 100)
            top = _log_between(rng, rng.choice([1, 300]), 16000 if kind == "prompt" else 60000)
            most_rows = {"prompt": _log_between(rng, 2, 4000), "step": 1}
            c.update(length_min=0 if kind == "memory" else rng.choice([1, top]), length_max=top,
                     fresh_min=1, fresh_max=most_rows.get(kind, rng.randrange(2, 17)))
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
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
        if case["op"] == "attend":
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
    return case["op"] != "attend" or case["causal"]


def _after(case):
    cached, fresh = lengths(case)
    return [c + n if _grows(case) else c for c, n in zip(cached, fresh)]


def _pages(n, page):
    return -(-n // page)


def work(case):
    cached, fresh = lengths(case)
    after, page = _after(case), case["page"]
    tokens, R = sum(fresh), case["requests"]
    if case["op"] == "plan":
        taken = sum(_pages(a, page) - _pages(c, page) for a, c in zip(after, cached))
        # lengths in, the partial page's entry in, each page taken in and out;
        # lengths and row ranges out; request, position and slot of each row
        return {"bytes": 8 * R + 4 * R + 8 * taken + 4 * R + 4 * (R + 1) + 16 * tokens,
                "flops": 2 * R + 4 * tokens}
    H, D = case["kv_heads"], case["dim"]
    if case["op"] == "store":
        span = [(c // page * page, a) for c, a, n in zip(cached, after, fresh) if n]
        touched = sum(a - f for f, a in span)
        pages = sum(_pages(a - f, page) for f, a in span)
        return {"bytes": 2 * H * (tokens * D * (2 + 1) + touched * D * (1 + 2) + 8 * pages),
                "flops": 2 * H * D * (3 * tokens + touched)}
    heads = H * case["group"]
    seen = 0
    for c, n in zip(cached, fresh):
        seen += n * c + (n * (n + 1) // 2 if case["causal"] else 0)
    held = sum(a for a, n in zip(after, fresh) if n)
    pages = sum(_pages(a, page) for a, n in zip(after, fresh) if n)
    return {"bytes": 2 * H * (held * D + 4 * pages) + 4 * pages +
            tokens * heads * (2 * D * 2 + 4),
            "flops": 4 * D * heads * seen}


# ------------------------------------------------------------------ the inputs

def _random_pool(pages, H, page, D, gen):
    """Codes and scales as a store leaves them: every page's values normal,
    with a spread of its own for each head."""
    codes = torch.empty((pages, H, page, D), dtype=torch.int8, device=DEVICE)
    scales = torch.empty((pages, H), dtype=torch.float32, device=DEVICE)
    step = max(1, (1 << 26) // (H * page * D))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        x = torch.randn((b - a, H, page, D), device=DEVICE, generator=gen)
        x *= torch.exp(0.3 * torch.randn((b - a, H, 1, 1), device=DEVICE, generator=gen))
        s = x.abs().amax((2, 3)) / 127.0
        codes[a:b] = torch.round(x / s[:, :, None, None]).to(torch.int8)
        scales[a:b] = s
    return codes, scales


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
    return table, ring, np.array([first, first + len(left)], np.int64), pool


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    cached, fresh = lengths(case)
    after, page = _after(case), case["page"]
    table, ring, cursor, pool = _tables(case, seed)
    st = {
        "case": case, "page": page, "pool": pool, "tokens": sum(fresh),
        "cached": torch.tensor(cached, dtype=torch.int32, device=DEVICE),
        "fresh": torch.tensor(fresh, dtype=torch.int32, device=DEVICE),
        "table": torch.from_numpy(table).to(DEVICE),
        "ring": torch.from_numpy(ring).to(DEVICE),
        "cursor": torch.from_numpy(cursor).to(DEVICE),
        "host": (cached, fresh, after),
    }
    if case["op"] != "plan":
        H, D = case["kv_heads"], case["dim"]
        T, kind = st["tokens"], TYPES[case["type"]]
        st["k_codes"], st["k_scales"] = _random_pool(pool, H, page, D, gen)
        st["v_codes"], st["v_scales"] = _random_pool(pool, H, page, D, gen)
        # the step's plan, which a program makes once for all layers
        p = _plan_plain(st)
        st["table"], st["after"], st["starts"] = p[0], p[1], p[2]
        st["positions"], st["slots"], st["rows"] = p[3], p[4], p[5]
        if case["op"] == "store":
            # rows as a fused projection leaves them: keys beside values
            kv = torch.randn((T, 2, H, D), device=DEVICE, generator=gen)
            kv *= torch.exp(0.3 * torch.randn((1, 2, H, D), device=DEVICE, generator=gen))
            kv = kv.to(kind)
            st["k"], st["v"] = kv[:, 0], kv[:, 1]
            st["touched"] = _touched(st)
        else:
            st["q"] = torch.randn((T, H * case["group"], D), device=DEVICE,
                                  generator=gen).to(kind)
    if own:
        _prepare_own(st, table)
    return st


def _touched(st):
    """Slots of every token in the pages that the step writes."""
    cached, fresh, after = st["host"]
    page = st["page"]
    r = np.concatenate([np.full(a - c // page * page, i) for i, (c, a, n)
                        in enumerate(zip(cached, after, fresh)) if n])
    pos = np.concatenate([np.arange(c // page * page, a) for c, a, n
                          in zip(cached, after, fresh) if n])
    r, pos = torch.from_numpy(r).to(DEVICE), torch.from_numpy(pos).to(DEVICE)
    return st["table"][r, pos // page].long() * page + pos % page


def _prepare_own(st, table):
    from graftrepository_b200 import paged_arena

    case = st["case"]
    tables = paged_arena.PageTables(case["requests"], st["pool"], table.shape[1],
                                    page_tokens=st["page"], device=DEVICE)
    tables.table.copy_(torch.from_numpy(table))
    tables.lens.copy_(st["cached"])
    tables.ring.copy_(st["ring"])
    tables.cursor.copy_(st["cursor"])
    H, G = case.get("kv_heads", 8), case.get("group", 1)
    plan = tables.make_plan(st["tokens"], kv_heads=H, query_heads=H * G,
                            head_dim=case.get("dim", 128), max_fresh=max(st["host"][1]))
    st["tables"], st["plan"] = tables, plan
    if case["op"] == "plan":
        return
    tables.plan(plan, st["fresh"], grow=_grows(case))
    arena = paged_arena.PagedArena(1, st["pool"], H, case["dim"], page_tokens=st["page"],
                                   device=DEVICE)
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        getattr(arena, name)[0].copy_(st.pop(name))
    st["arena"] = arena


# ------------------------------------------------------------- the plain forms

def _plan_plain(st):
    page, cached, fresh, table = st["page"], st["cached"], st["fresh"], st["table"].clone()
    ring, cursor, T = st["ring"], st["cursor"], st["tokens"]
    grow = _grows(st["case"])
    after = cached + fresh if grow else cached.clone()
    have, need = (cached + page - 1) // page, (after + page - 1) // page
    take = need - have
    taken = torch.cumsum(take, 0)
    column = torch.arange(table.shape[1], device=DEVICE, dtype=torch.int64)[None, :]
    new = (column >= have[:, None]) & (column < need[:, None])
    at = cursor[0] + (taken - take)[:, None] + column - have[:, None]
    table = torch.where(new, ring[torch.where(new, at % ring.numel(), 0)], table)
    starts = torch.zeros(cached.numel() + 1, dtype=torch.int32, device=DEVICE)
    starts[1:] = torch.cumsum(fresh, 0)
    row = torch.arange(T, device=DEVICE, dtype=torch.int32)
    rows = torch.bucketize(row, starts[1:], right=True)
    positions = cached[rows] + row - starts[rows]
    if grow:
        slots = table[rows, (positions // page).long()].long() * page + positions % page
    else:
        slots = torch.full((T,), -1, dtype=torch.int64, device=DEVICE)
    moved = torch.stack([cursor[0] + take.sum(), cursor[1]])
    return [table, after, starts, positions.int(), slots, rows.int(), moved]


def _store_plain(st, x, codes, scales):
    """Quantises x [T, H, D] into codes and scales, in place."""
    page, slots, x = st["page"], st["slots"], x.float()
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


def _attend_plain(st):
    case, page, q = st["case"], st["page"], st["q"]
    cached, fresh, after = st["host"]
    H, G, D, T = case["kv_heads"], case["group"], case["dim"], st["tokens"]
    out = torch.zeros((T, H * G, D), dtype=q.dtype, device=DEVICE)
    lse = torch.full((T, H * G), -math.inf, device=DEVICE)
    at = 0
    for r, (c, n, L) in enumerate(zip(cached, fresh, after)):
        if n and L:
            pages = st["table"][r, :_pages(L, page)].long()
            x = q[at:at + n].float().view(n, H, G, D)
            for h in range(H):
                k = st["k_codes"][pages, h].float() * st["k_scales"][pages, h][:, None, None]
                v = st["v_codes"][pages, h].float() * st["v_scales"][pages, h][:, None, None]
                k, v = k.view(-1, D)[:L], v.view(-1, D)[:L]
                s = (x[:, h].reshape(n * G, D) @ k.T) / math.sqrt(D)
                if case["causal"]:
                    last = c + torch.arange(n, device=DEVICE).repeat_interleave(G)
                    s.masked_fill_(torch.arange(L, device=DEVICE)[None, :] > last[:, None],
                                   -math.inf)
                top = s.amax(1, keepdim=True)
                s = torch.exp(s - top)
                total = s.sum(1, keepdim=True)
                y = (s @ v) / total
                out[at:at + n, h * G:(h + 1) * G] = y.view(n, G, D).to(q.dtype)
                lse[at:at + n, h * G:(h + 1) * G] = (top + torch.log(total)).view(n, G)
        at += n
    return out, lse


# -------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _run_own(state, op)
    if op == "plan":
        return _plan_plain(state)
    if op == "store":
        got = []
        for x, codes, scales in ((state["k"], state["k_codes"], state["k_scales"]),
                                 (state["v"], state["v_codes"], state["v_scales"])):
            _store_plain(state, x, codes, scales)
            got += [_values(codes, scales, state["touched"], state["page"]).to(x.dtype), scales]
        return got
    return list(_attend_plain(state))


def _run_own(st, op):
    if op == "plan":
        tables, plan = st["tables"], st["plan"]
        tables.plan(plan, st["fresh"])
        return [tables.table, plan.lens, plan.starts, plan.positions, plan.slots, plan.rows,
                plan.cursor]
    arena = st["arena"]
    if op == "store":
        arena.append(st["plan"], st["k"], st["v"])
        k, v = arena.read(st["touched"], dtype=st["k"].dtype)
        return [k, arena.k_scales[0], v, arena.v_scales[0]]
    return list(arena.attend(st["plan"], st["q"], causal=st["case"]["causal"]))


# ------------------------------------------------------ the definitions, 64 bits

def exact(case, seed):
    if case["op"] == "plan":
        return _plan_exact(case, seed)
    global own
    held, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = held
    return _store_exact(st) if case["op"] == "store" else _attend_exact(st)


def _plan_exact(case, seed):
    """Request by request, page by page, on the host."""
    cached, fresh = lengths(case)
    table, ring, cursor, pool = _tables(case, seed)
    page, taken = case["page"], int(cursor[0])
    starts, positions, slots, rows, after = [0], [], [], [], []
    for r, (c, n) in enumerate(zip(cached, fresh)):
        for p in range(_pages(c, page), _pages(c + n, page)):
            table[r, p] = ring[taken % pool]
            taken += 1
        pos = np.arange(c, c + n, dtype=np.int64)
        positions.append(pos)
        slots.append(table[r, pos // page].astype(np.int64) * page + pos % page)
        rows.append(np.full(n, r, np.int64))
        after.append(c + n)
        starts.append(starts[-1] + n)
    as_int = lambda v: torch.from_numpy(np.asarray(v).astype(np.int32))
    return [torch.from_numpy(table), as_int(after), as_int(starts),
            as_int(np.concatenate(positions)), torch.from_numpy(np.concatenate(slots)),
            as_int(np.concatenate(rows)), torch.tensor([taken, int(cursor[1])])]


def _store_exact(st):
    """Page by page: the scale covers the largest value that the page holds."""
    cached, fresh, after = st["host"]
    page, table = st["page"], st["table"].cpu().numpy()
    out = []
    for x, codes, scales in ((st["k"], st["k_codes"], st["k_scales"]),
                             (st["v"], st["v_codes"], st["v_scales"])):
        x, s64 = x.double(), scales.double()
        got, at = [], 0
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
    case, page = st["case"], st["page"]
    cached, fresh, after = st["host"]
    if work(case)["flops"] > 5e12:
        return None
    H, G, D = case["kv_heads"], case["group"], case["dim"]
    rows, sums = [], []
    for r in range(case["requests"]):
        n, L = fresh[r], after[r]
        slot = torch.arange(L, device=DEVICE)
        slot = st["table"][r, slot // page].long() * page + slot % page
        a = sum(fresh[:r])
        k = v = None
        y = torch.zeros((n, H * G, D), dtype=torch.float64, device=DEVICE)
        z = torch.full((n, H * G), -math.inf, dtype=torch.float64, device=DEVICE)
        if n and L:
            for head in range(H * G):
                h = head // G
                if head % G == 0:
                    k = st["k_codes"][slot // page, h, slot % page].double() * \
                        st["k_scales"][slot // page, h].double()[:, None]
                    v = st["v_codes"][slot // page, h, slot % page].double() * \
                        st["v_scales"][slot // page, h].double()[:, None]
                w = st["q"][a:a + n, head].double() @ k.T * D ** -0.5
                if case["causal"]:
                    w += torch.triu(torch.full((n, L), -math.inf, dtype=torch.float64,
                                               device=DEVICE), 1 + L - n)
                z[:, head] = torch.logsumexp(w, 1)
                y[:, head] = torch.exp(w - z[:, head, None]) @ v
        rows.append(y)
        sums.append(z)
    return [torch.cat(rows), torch.cat(sums)]
