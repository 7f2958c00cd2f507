"""The 8-bit paged arena: many requests' keys and values, and attention over them.

``graft_mount`` writes routed grafts as bf16 rows of one request's arena.  This
module holds the keys and values of many requests at 8 bits, in pages that
belong to one request at a time, and answers query rows from them:

* ``PageTables`` -- block table, lengths and the ring of free pages; ``plan``
  lays out one step on the GPU from the requests' new row counts (pages taken,
  slots, positions, work lists), with no length known to the host;
* ``PagedArena.append`` -- quantises the step's key and value rows (mounted
  rows of an arena or a model's projections) into their pages, one fp32 scale
  for each page, kv head and side;
* ``PagedArena.attend`` -- attention of the step's query rows over the pages,
  causal or not, with the log-sum-exp of every row;
* ``PagedArena.read`` -- pages back to rows of values (harvest).

A step::

    plan = tables.make_plan(tokens, kv_heads=8, query_heads=32, head_dim=128)
    tables.plan(plan, fresh)                  # once a step
    for layer in range(layers):               # the same plan for every layer
        arena.append(plan, k, v, layer=layer)
        out, lse = arena.attend(plan, q, layer=layer)
    tables.commit(plan)                       # the new lengths hold from here on
    tables.release(rows)                      # requests that are done give their pages back

Steps whose rows join the arena go one at a time, from ``plan`` to ``commit``,
whatever plans and streams they use: two that are planned side by side take the
same pages.  Planning another step leaves one that is not committed behind; what
is called with it then is refused.

Nothing here synchronises but ``PagePlan.check``; every call runs on ``stream``
(a torch stream or a raw handle; default: the tensors' device's current torch
stream) and can be captured in a CUDA graph.  Plans, tables and arenas follow
the streams that they are used on: the first call on a stream waits for the one
they were made on, and their memory is kept until those calls have ended, so a
plan may be dropped as soon as its step is queued.  That the rows of a call are
there when its stream comes to it, and that calls on several streams come in
order, is the caller's affair, as with torch's own.  (A stream under capture
waits for nothing outside its graph; what a graph uses has to outlive it.)
Results do not depend on the order in which blocks run.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

__all__ = ["PAGE_TOKENS", "HEAD_DIMS", "PageTables", "PagePlan", "PagedArena"]

PAGE_TOKENS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)

PLAN_BAD_LENGTH, PLAN_ROWS, PLAN_TABLE, PLAN_PAGES, PLAN_WAIT, PLAN_STALE = 1, 2, 4, 8, 16, 32
_REASONS = {
    PLAN_BAD_LENGTH: "a negative length, or one past 2^31 - 1024",
    PLAN_ROWS: "more new rows than the plan has room for (tokens, max_fresh)",
    PLAN_TABLE: "a request needs more pages than its block table row has entries",
    PLAN_PAGES: "not enough free pages",
    PLAN_WAIT: "a wait inside attention gave up and left rows of NaN",
    PLAN_STALE: "its requests or free pages have changed since it was planned, and it was not "
                "committed",
}


class _ArenaC(ctypes.Structure):
    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("kv_heads", ctypes.c_int32),
                ("page_tokens", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


class _PlanC(ctypes.Structure):
    _fields_ = [("requests", ctypes.c_int64), ("tokens", ctypes.c_int64),
                ("max_fresh", ctypes.c_int64), ("table_width", ctypes.c_int64),
                ("pages", ctypes.c_int64), ("page_tokens", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("query_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("grow", ctypes.c_int32),
                ("cached", ctypes.c_void_p), ("ring", ctypes.c_void_p),
                ("cursor_in", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("lens", ctypes.c_void_p), ("starts", ctypes.c_void_p),
                ("positions", ctypes.c_void_p), ("rows", ctypes.c_void_p),
                ("slots", ctypes.c_void_p), ("cursor", ctypes.c_void_p),
                ("status", ctypes.c_void_p), ("scratch", ctypes.c_void_p),
                ("scratch_bytes", ctypes.c_int64)]


_TYPES = {torch.float16: _lib.GRM_B200_F16, torch.bfloat16: _lib.GRM_B200_BF16}
_READ_TYPES = {torch.float32: _lib.GRM_B200_F32, **_TYPES}

# A decoding step makes these calls for every layer, so their host side is kept
# short: shapes and entry points are looked up once, and the current stream's
# handle comes straight from torch's binding where it has one.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _torch_stream(stream, index):
    """`stream` (a torch stream or a raw handle) as a torch stream."""
    if hasattr(stream, "cuda_stream"):
        return stream
    if int(stream) == 0:  # torch takes an external stream 0 for a new one
        return torch.cuda.default_stream(index)
    return torch.cuda.ExternalStream(int(stream), device=torch.device("cuda", index))


class _Buffers:
    """Device buffers of an object, made on the torch stream that was current.  The
    first call on any other stream waits for what that stream had queued by then
    (their first contents, and whatever still ran on memory that they took over),
    and the caching allocator learns of the stream, so that it gives none of them
    away while that still runs."""

    def _made(self, *tensors) -> None:
        self._tensors = tensors
        stream = torch.cuda.current_stream(self.device)
        self._streams, self._event = set(), None  # handles
        self._last = stream.cuda_stream  # of the call before
        if not _capturing(stream):
            self._streams.add(stream.cuda_stream)
            self._event = torch.cuda.Event()
            self._event.record(stream)

    def _join(self, stream) -> None:
        # a stream that is being captured cannot wait for work outside the graph
        if not _capturing(stream):
            if self._event is not None:
                stream.wait_event(self._event)
            self._streams.add(stream.cuda_stream)
        for t in self._tensors:
            t.record_stream(stream)


def _capturing(stream) -> bool:
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _handle(stream, index, owners, *tensors) -> int:
    """The raw handle of `stream`, joined by the buffers of `owners`.  Of a stream
    that is given, the allocator learns that `tensors` are used on it; those of the
    current stream are the caller's affair, as with torch's own calls."""
    if stream is None:
        handle = _raw_stream(index)
    else:
        stream = _torch_stream(stream, index)
        handle = stream.cuda_stream
        for t in tensors:
            t.record_stream(stream)
    for x in owners:
        if handle not in x._streams:
            x._join(torch.cuda.current_stream(index) if stream is None else stream)
        x._last = handle
    return handle


def _empty(like, shape, dtype, stream):
    """A result on the device of `like` that belongs to the stream that writes it."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(_torch_stream(stream, like.get_device())):
        return like.new_empty(shape, dtype=dtype)


def _result(pattern, stream):
    """The same of `pattern`'s shape and type, contiguous (1.4 us, where new_empty
    takes 2.0 to 2.7)."""
    if stream is None:
        return torch.empty_like(pattern, memory_format=torch.contiguous_format)
    with torch.cuda.stream(_torch_stream(stream, pattern.get_device())):
        return torch.empty_like(pattern, memory_format=torch.contiguous_format)


def _device(device):
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"the paged arena lives on a CUDA device, not {device!r}")
    return d if d.index is not None else torch.device("cuda", torch.cuda.current_device())


def _call(fn, index, *args) -> None:
    """One library call with device `index` current."""
    if torch.cuda.current_device() == index:
        rc = fn(*args)
    else:
        with torch.cuda.device(index):
            rc = fn(*args)
    if rc:
        _lib.check(rc, _lib.thread_error)


def _check_page(page_tokens: int) -> int:
    if page_tokens not in PAGE_TOKENS:
        raise ValueError(f"page_tokens must be one of {PAGE_TOKENS}, got {page_tokens}")
    return int(page_tokens)


class PagePlan(_Buffers):
    """The buffers of one step (``PageTables.make_plan``), filled by
    ``PageTables.plan``: ``lens`` int32 [requests], ``starts`` int32
    [requests + 1], ``positions`` and ``rows`` int32 [tokens], ``slots`` int64
    [tokens] (-1 past the last row), ``cursor`` int64 [2], ``status`` int32 [1]."""

    def __init__(self, tables: "PageTables", tokens: int, kv_heads: int, query_heads: int,
                 head_dim: int, max_fresh: int | None):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if kv_heads < 1 or query_heads < 1 or query_heads % kv_heads:
            raise ValueError(f"query_heads {query_heads} must be a multiple of kv_heads {kv_heads}")
        if tokens < 1:
            raise ValueError(f"a plan needs room for at least one row, got tokens = {tokens}")
        self.tables, self.tokens = tables, int(tokens)
        self.kv_heads, self.query_heads, self.head_dim = kv_heads, query_heads, head_dim
        self.max_fresh = self.tokens if max_fresh is None else int(max_fresh)
        if self.max_fresh < 1:
            raise ValueError(f"max_fresh must be at least 1, got {max_fresh}")
        self.device, self._index = tables.device, tables._index
        self.query_shape = torch.Size((self.tokens, query_heads, head_dim))
        self.kv_shape = torch.Size((self.tokens, kv_heads, head_dim))

        # shapes and types of attention's results, one element each
        self._out_like = {kind: torch.empty(1, dtype=kind, device=self.device).expand(
            self.query_shape) for kind in _TYPES}
        self._lse_like = torch.empty(1, device=self.device).expand(self.query_shape[:2])

        # the step's outputs, in two allocations
        n, t = tables.requests, self.tokens
        words = torch.zeros(2 * n + 2 * t + 2, dtype=torch.int32, device=self.device)
        self.lens, self.starts, self.positions, self.rows, self.status = words.split(
            [n, n + 1, t, t, 1])
        longs = torch.zeros(t + 2, dtype=torch.int64, device=self.device)
        self.slots, self.cursor = longs.split([t, 2])
        self.c = _PlanC(tables.requests, self.tokens, self.max_fresh, tables.width, tables.pages,
                        tables.page_tokens, kv_heads, query_heads, head_dim, 1)
        need = ctypes.c_int64(0)
        _call(_lib.load().grm_b200_paged_scratch_bytes, self._index, ctypes.byref(self.c),
              ctypes.byref(need))
        self.scratch = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._made(words, longs, self.scratch)
        _handle(None, self._index, (tables,))
        c = self.c
        c.cached, c.cursor_in = tables.lens.data_ptr(), tables.cursor.data_ptr()
        c.ring, c.table = tables.ring.data_ptr(), tables.table.data_ptr()
        c.lens, c.starts = self.lens.data_ptr(), self.starts.data_ptr()
        c.positions, c.rows = self.positions.data_ptr(), self.rows.data_ptr()
        c.slots, c.cursor = self.slots.data_ptr(), self.cursor.data_ptr()
        c.status = self.status.data_ptr()
        c.scratch, c.scratch_bytes = self.scratch.data_ptr(), need.value
        self.planned, self.grow = False, True
        self._turn = None  # of the tables' joining steps, until it is committed
        self._ref = ctypes.byref(c)

    def _join(self, stream) -> None:  # and the tables, for every call that takes a plan
        super()._join(stream)
        if stream.cuda_stream not in self.tables._streams:
            self.tables._join(stream)

    def _in_turn(self) -> None:
        if self._turn is not None and self._turn != self.tables._turn:
            raise ValueError("another step of these tables has been planned since and takes the "
                             "same pages; plan this one again")

    def check(self) -> None:
        """Wait for the plan (and calls that used it, on the stream of the last
        one and on the current one) and raise if the step could not be planned
        (it then took no pages and has no rows), its commit came too late or
        attention gave up on rows.  Speaks of the last step planned."""
        if self._last != _raw_stream(self._index):
            _torch_stream(self._last, self._index).synchronize()
        bits = int(self.status.item())
        if bits:
            why = "; ".join(text for bit, text in _REASONS.items() if bits & bit)
            raise _lib.GrmB200Error(bits, f"the step failed: {why}")


class PageTables(_Buffers):
    """Block table ``table`` int32 [requests, width], lengths ``lens`` int32
    [requests], free pages ``ring`` int32 [pages] and ``cursor`` int64 [2]
    (pages ever taken, pages ever returned).  All pages are free at first."""

    def __init__(self, requests: int, pages: int, width: int, *, page_tokens: int = 64,
                 device="cuda"):
        if requests < 1 or pages < 1 or width < 1:
            raise ValueError(f"requests, pages and width must be positive, got "
                             f"{requests}, {pages}, {width}")
        self.requests, self.pages, self.width = int(requests), int(pages), int(width)
        self.page_tokens = _check_page(page_tokens)
        self.device = _device(device)
        self._index, self._shape = self.device.index, torch.Size((self.requests,))
        self._plan_step = _lib.load().grm_b200_paged_plan_step
        self._turn = 0  # joining steps planned so far, those under capture left out
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=self.device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=self.device)
        self.ring = torch.arange(pages, dtype=torch.int32, device=self.device)
        self.cursor = torch.tensor([0, pages], dtype=torch.int64, device=self.device)
        self._made(self.table, self.lens, self.ring, self.cursor)

    def make_plan(self, tokens: int, *, kv_heads: int, query_heads: int, head_dim: int,
                  max_fresh: int | None = None) -> PagePlan:
        """Buffers for steps of up to `tokens` new rows, at most `max_fresh` of
        one request (default: `tokens`; a step that keeps it small, such as
        max_fresh = 1 for decoding, is served by the kernel made for that).  A
        plan's steps may not overlap on the GPU."""
        return PagePlan(self, tokens, kv_heads, query_heads, head_dim, max_fresh)

    def plan(self, plan: PagePlan, fresh, *, grow: bool = True, stream=None) -> PagePlan:
        """Lay out a step: request r brings ``fresh[r]`` new rows (int32 on the
        device).  `grow`: the rows are tokens that join the requests; without
        it they are query rows that only read what is cached.  A joining step
        leaves behind one that was planned and not committed."""
        if plan.tables is not self:
            raise ValueError("the plan was made for other tables")
        if (not isinstance(fresh, torch.Tensor) or fresh.dtype is not torch.int32 or
                fresh.get_device() != self._index or fresh.shape != self._shape or
                not fresh.is_contiguous()):
            raise ValueError(f"fresh must be int32 [{self.requests}] on {self.device}")
        if grow is not plan.grow:
            plan.grow = bool(grow)
            plan.c.grow = 1 if grow else 0
        _call(self._plan_step, self._index, plan._ref, fresh.data_ptr(),
              _handle(stream, self._index, (plan,), fresh))
        plan.planned, plan._turn = True, None
        # a step that a graph plans again has no turn: the host does not see it
        if grow and not (torch.cuda.is_current_stream_capturing() if stream is None else
                         _capturing(_torch_stream(stream, self._index))):
            plan._turn = self._turn = self._turn + 1
        return plan

    def commit(self, plan: PagePlan, *, stream=None) -> None:
        """Take up the lengths of a planned step: requests with rows in it hold
        `plan.lens` tokens from here on.  The plan stays good for append and
        attend, and a second commit of it does nothing.  Other requests may be
        released between plan and commit; where the step's own requests or the
        pages it takes have changed since, nothing is taken up and
        ``plan.check`` says so."""
        if plan.tables is not self or not plan.planned:
            raise ValueError("commit takes a plan of these tables that has been planned")
        if not plan.grow:
            return
        plan._in_turn()
        _call(_lib.load().grm_b200_paged_commit, self._index, plan._ref, self.lens.data_ptr(),
              self.cursor.data_ptr(), _handle(stream, self._index, (plan,)))
        plan._turn = None

    def release(self, rows, *, stream=None) -> None:
        """Return the pages that the requests ``rows`` (int32 on the device) hold
        to the ring and empty them.  A step that is planned and not committed
        does not hold its pages yet; if it has rows of these requests, its
        commit comes too late."""
        if (not isinstance(rows, torch.Tensor) or rows.dtype != torch.int32 or rows.dim() != 1 or
                rows.device != self.device or not rows.is_contiguous()):
            raise ValueError(f"rows must be int32 [n] on {self.device}")
        if rows.numel() == 0:
            return
        _call(_lib.load().grm_b200_paged_release, self._index, rows.data_ptr(), rows.numel(),
              self.requests, self.width, self.pages, self.page_tokens, self.table.data_ptr(),
              self.lens.data_ptr(), self.ring.data_ptr(), self.cursor.data_ptr(),
              _handle(stream, self._index, (self,), rows))


class PagedArena(_Buffers):
    """Codes int8 [layers, pages, kv_heads, page_tokens, head_dim] and scales
    fp32 [layers, pages, kv_heads] of the keys and of the values."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *,
                 page_tokens: int = 64, device="cuda"):
        if layers < 1 or pages < 1 or kv_heads < 1:
            raise ValueError(f"layers, pages and kv_heads must be positive, got "
                             f"{layers}, {pages}, {kv_heads}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        self.layers, self.pages = int(layers), int(pages)
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.page_tokens = _check_page(page_tokens)
        self.device = _device(device)
        shape = (layers, pages, kv_heads)
        codes = shape + (page_tokens, head_dim)
        self.k_codes = torch.zeros(codes, dtype=torch.int8, device=self.device)
        self.v_codes = torch.zeros(codes, dtype=torch.int8, device=self.device)
        self.k_scales = torch.zeros(shape, dtype=torch.float32, device=self.device)
        self.v_scales = torch.zeros(shape, dtype=torch.float32, device=self.device)
        self._made(self.k_codes, self.v_codes, self.k_scales, self.v_scales)
        self._c = [_ArenaC(self.k_codes[i].data_ptr(), self.v_codes[i].data_ptr(),
                           self.k_scales[i].data_ptr(), self.v_scales[i].data_ptr(), pages,
                           kv_heads, page_tokens, head_dim) for i in range(layers)]
        self._refs = [ctypes.byref(c) for c in self._c]
        lib = _lib.load()
        self._index = self.device.index
        self._append, self._attend = lib.grm_b200_paged_append, lib.grm_b200_paged_attend
        self._read = lib.grm_b200_paged_read
        self._scale = 1.0 / math.sqrt(head_dim)

    def _rows(self, name, x, shape):
        """Checks rows of `shape`; returns (type, pointer, row and head strides)."""
        kind = _TYPES.get(x.dtype)
        if kind is None:
            raise ValueError(f"{name} must be float16 or bfloat16, got {x.dtype}")
        if x.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {list(x.shape)}")
        if x.get_device() != self._index:
            raise ValueError(f"{name} is on {x.device}, the arena on {self.device}")
        row, head, inner = x.stride()
        ptr = x.data_ptr()
        if (row | head) & 7:  # the stride of a dimension of one entry says nothing
            row, head = row if shape[0] > 1 else 0, head if shape[1] > 1 else 0
        if inner != 1 or (row | head) & 7 or ptr & 15:
            raise ValueError(f"{name}: a head's values must be contiguous, rows and heads at "
                             f"multiples of 8 elements and 16-byte aligned (strides {x.stride()})")
        return kind, ptr, row, head

    def _ready(self, plan, layer):
        """The layer's buffers, for a plan that is good for a call."""
        if not plan.planned:
            raise ValueError("the plan has not been planned yet (PageTables.plan)")
        if plan._index != self._index:
            raise ValueError(f"the plan is on {plan.device}, the arena on {self.device}")
        if plan._turn is not None:
            plan._in_turn()
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        return self._refs[layer]

    def _result(self, name, t, pattern, stream):
        if t is None:
            return _result(pattern, stream)
        if (t.shape != pattern.shape or t.dtype is not pattern.dtype or
                t.get_device() != self._index or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous {pattern.dtype} {list(pattern.shape)} on "
                             f"{self.device}")
        return t

    def append(self, plan: PagePlan, k, v, *, layer: int = 0, stream=None) -> None:
        """Quantise the step's rows ``k`` and ``v`` [tokens, kv_heads, head_dim]
        into the pages of `layer`, before those of any later step."""
        ref = self._ready(plan, layer)
        kind, k_ptr, k_row, k_head = self._rows("k", k, plan.kv_shape)
        v_kind, v_ptr, v_row, v_head = self._rows("v", v, plan.kv_shape)
        if kind != v_kind:
            raise ValueError(f"k and v differ in type: {k.dtype}, {v.dtype}")
        if not plan.grow:
            raise ValueError("the plan's rows do not join the arena (planned with grow=False)")
        _call(self._append, self._index, plan._ref, ref, k_ptr, v_ptr, kind, k_row, k_head, v_row,
              v_head, _handle(stream, self._index, (self, plan), k, v))

    def attend(self, plan: PagePlan, q, *, layer: int = 0, causal: bool = True,
               scale: float | None = None, out=None, lse=None, stream=None):
        """Attention of the step's query rows ``q`` [tokens, query_heads,
        head_dim]: over everything the row's request holds, or with `causal` over
        the positions up to the row's own.  `scale` (positive; default
        head_dim ** -0.5) multiplies the scores.  Returns (out like q, lse fp32
        [tokens, query_heads]); rows that see nothing are 0 with lse -inf."""
        ref = self._ready(plan, layer)
        kind, ptr, row, head = self._rows("q", q, plan.query_shape)
        if causal and not plan.grow:
            raise ValueError("rows that do not join the arena (planned with grow=False) have no "
                             "position in it; attend with causal=False")
        out = self._result("out", out, plan._out_like[q.dtype], stream)
        lse = self._result("lse", lse, plan._lse_like, stream)
        _call(self._attend, self._index, plan._ref, ref, ptr, kind, row, head,
              self._scale if scale is None else float(scale), 1 if causal else 0, out.data_ptr(),
              lse.data_ptr(), _handle(stream, self._index, (self, plan), q, out, lse))
        return out, lse

    def read(self, slots, *, layer: int = 0, dtype=None, stream=None):
        """Rows of values (k, v) [n, kv_heads, head_dim] of type `dtype`
        (default bfloat16; float16 and float32 too) at ``slots`` int64 [n]; a
        negative slot gives zeros."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        if (not isinstance(slots, torch.Tensor) or slots.dtype is not torch.int64 or
                slots.dim() != 1 or slots.get_device() != self._index or
                not slots.is_contiguous()):
            raise ValueError(f"slots must be int64 [n] on {self.device}")
        dtype = torch.bfloat16 if dtype is None else dtype
        kind = _READ_TYPES.get(dtype)
        if kind is None:
            raise ValueError(f"read gives float32, float16 or bfloat16, not {dtype}")
        n = slots.numel()
        k = _empty(slots, (n, self.kv_heads, self.head_dim), dtype, stream)
        v = _result(k, stream)
        if n:
            _call(self._read, self._index, self._refs[layer], slots.data_ptr(), n, kind,
                  k.data_ptr(), v.data_ptr(), _handle(stream, self._index, (self,), slots))
        return k, v
