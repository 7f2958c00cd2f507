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

Nothing here synchronises but ``PagePlan.check``; every call runs on ``stream``
(a torch stream or a raw handle; default: the tensors' device's current torch
stream) and can be captured in a CUDA graph.  Results do not depend on the
order in which blocks run.
"""

from __future__ import annotations

import ctypes
import math

from . import _lib

__all__ = ["PAGE_TOKENS", "HEAD_DIMS", "PageTables", "PagePlan", "PagedArena"]

PAGE_TOKENS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)

PLAN_BAD_LENGTH, PLAN_ROWS, PLAN_TABLE, PLAN_PAGES, PLAN_WAIT = 1, 2, 4, 8, 16
_REASONS = {
    PLAN_BAD_LENGTH: "a negative length, or one past 2^31 - 1",
    PLAN_ROWS: "more new rows than the plan has room for (tokens, max_fresh)",
    PLAN_TABLE: "a request needs more pages than its block table row has entries",
    PLAN_PAGES: "not enough free pages",
    PLAN_WAIT: "a wait inside attention gave up and rows are missing",
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


def _stream(stream, device, *tensors):
    """(torch stream, handle) of a call; the caching allocator is told of
    `tensors` where the stream is not the current one."""
    import torch

    current = torch.cuda.current_stream(device)
    if stream is None:
        return current, current.cuda_stream
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream), device=device)
    if stream.cuda_stream != current.cuda_stream:
        for t in tensors:
            t.record_stream(stream)
    return stream, stream.cuda_stream


def _empty(shape, dtype, device, stream):
    """A result that belongs to the stream that writes it."""
    import torch

    if stream == torch.cuda.current_stream(device):
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _device(device):
    import torch

    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"the paged arena lives on a CUDA device, not {device!r}")
    return d if d.index is not None else torch.device("cuda", torch.cuda.current_device())


def _call(name: str, device, *args) -> None:
    """One library call with `device` current."""
    import torch

    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    if rc:
        _lib.check(rc, _lib.thread_error)


def _check_page(page_tokens: int) -> int:
    if page_tokens not in PAGE_TOKENS:
        raise ValueError(f"page_tokens must be one of {PAGE_TOKENS}, got {page_tokens}")
    return int(page_tokens)


class PagePlan:
    """The buffers of one step (``PageTables.make_plan``), filled by
    ``PageTables.plan``: ``lens`` int32 [requests], ``starts`` int32
    [requests + 1], ``positions`` and ``rows`` int32 [tokens], ``slots`` int64
    [tokens] (-1 past the last row), ``cursor`` int64 [2], ``status`` int32 [1]."""

    def __init__(self, tables: "PageTables", tokens: int, kv_heads: int, query_heads: int,
                 head_dim: int, max_fresh: int | None):
        import torch

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
        self.device = tables.device

        def ints(n, dtype=torch.int32):
            return torch.zeros(n, dtype=dtype, device=self.device)

        self.lens, self.starts = ints(tables.requests), ints(tables.requests + 1)
        self.positions, self.rows = ints(self.tokens), ints(self.tokens)
        self.slots, self.cursor = ints(self.tokens, torch.int64), ints(2, torch.int64)
        self.status = ints(1)
        self.c = _PlanC(tables.requests, self.tokens, self.max_fresh, tables.width, tables.pages,
                        tables.page_tokens, kv_heads, query_heads, head_dim, 1)
        need = ctypes.c_int64(0)
        _call("grm_b200_paged_scratch_bytes", self.device, ctypes.byref(self.c),
              ctypes.byref(need))
        self.scratch = torch.zeros(need.value, dtype=torch.uint8, device=self.device)
        c = self.c
        c.cached, c.cursor_in = tables.lens.data_ptr(), tables.cursor.data_ptr()
        c.ring, c.table = tables.ring.data_ptr(), tables.table.data_ptr()
        c.lens, c.starts = self.lens.data_ptr(), self.starts.data_ptr()
        c.positions, c.rows = self.positions.data_ptr(), self.rows.data_ptr()
        c.slots, c.cursor = self.slots.data_ptr(), self.cursor.data_ptr()
        c.status = self.status.data_ptr()
        c.scratch, c.scratch_bytes = self.scratch.data_ptr(), need.value
        self.planned = False
        self._ref = ctypes.byref(c)

    @property
    def grow(self) -> bool:
        return bool(self.c.grow)

    def check(self) -> None:
        """Wait for the plan (and calls that used it) and raise if the step
        could not be planned: it then took no pages and has no rows."""
        bits = int(self.status.item())
        if bits:
            why = "; ".join(text for bit, text in _REASONS.items() if bits & bit)
            raise _lib.GrmB200Error(bits, f"the step failed: {why}")


class PageTables:
    """Block table ``table`` int32 [requests, width], lengths ``lens`` int32
    [requests], free pages ``ring`` int32 [pages] and ``cursor`` int64 [2]
    (pages ever taken, pages ever returned).  All pages are free at first."""

    def __init__(self, requests: int, pages: int, width: int, *, page_tokens: int = 64,
                 device="cuda"):
        import torch

        if requests < 1 or pages < 1 or width < 1:
            raise ValueError(f"requests, pages and width must be positive, got "
                             f"{requests}, {pages}, {width}")
        self.requests, self.pages, self.width = int(requests), int(pages), int(width)
        self.page_tokens = _check_page(page_tokens)
        self.device = _device(device)
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=self.device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=self.device)
        self.ring = torch.arange(pages, dtype=torch.int32, device=self.device)
        self.cursor = torch.tensor([0, pages], dtype=torch.int64, device=self.device)

    def make_plan(self, tokens: int, *, kv_heads: int, query_heads: int, head_dim: int,
                  max_fresh: int | None = None) -> PagePlan:
        """Buffers for steps of up to `tokens` new rows, at most `max_fresh` of
        one request (default: `tokens`; a step that keeps it small, such as
        max_fresh = 1 for decoding, is served by the kernel made for that).  A
        plan's steps may not overlap on the GPU; make one plan for each stream."""
        return PagePlan(self, tokens, kv_heads, query_heads, head_dim, max_fresh)

    def plan(self, plan: PagePlan, fresh, *, grow: bool = True, stream=None) -> PagePlan:
        """Lay out a step: request r brings ``fresh[r]`` new rows (int32 on the
        device).  `grow`: the rows are tokens that join the requests; without
        it they are query rows that only read what is cached."""
        import torch

        if plan.tables is not self:
            raise ValueError("the plan was made for other tables")
        if (not isinstance(fresh, torch.Tensor) or fresh.dtype != torch.int32 or
                fresh.device != self.device or fresh.shape != (self.requests,) or
                not fresh.is_contiguous()):
            raise ValueError(f"fresh must be int32 [{self.requests}] on {self.device}")
        plan.c.grow = 1 if grow else 0
        _, handle = _stream(stream, self.device, fresh)
        _call("grm_b200_paged_plan_step", self.device, plan._ref, fresh.data_ptr(), handle)
        plan.planned = True
        return plan

    def commit(self, plan: PagePlan, *, stream=None) -> None:
        """Take up the lengths of a planned step: requests hold `plan.lens`
        tokens from here on.  The plan stays good for append and attend."""
        import torch

        if plan.tables is not self or not plan.planned:
            raise ValueError("commit takes a plan of these tables that has been planned")
        if not plan.grow:
            return
        stream, _ = _stream(stream, self.device)
        with torch.cuda.stream(stream):
            self.lens.copy_(plan.lens)
            self.cursor.copy_(plan.cursor)

    def release(self, rows, *, stream=None) -> None:
        """Return the pages of the requests ``rows`` (int32 on the device) to
        the ring and empty them."""
        import torch

        if (not isinstance(rows, torch.Tensor) or rows.dtype != torch.int32 or rows.dim() != 1 or
                rows.device != self.device or not rows.is_contiguous()):
            raise ValueError(f"rows must be int32 [n] on {self.device}")
        if rows.numel() == 0:
            return
        _, handle = _stream(stream, self.device, rows)
        _call("grm_b200_paged_release", self.device, rows.data_ptr(), rows.numel(), self.requests,
              self.width, self.pages, self.page_tokens, self.table.data_ptr(),
              self.lens.data_ptr(), self.ring.data_ptr(), self.cursor.data_ptr(), handle)


class PagedArena:
    """Codes int8 [layers, pages, kv_heads, page_tokens, head_dim] and scales
    fp32 [layers, pages, kv_heads] of the keys and of the values."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *,
                 page_tokens: int = 64, device="cuda"):
        import torch

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
        self._c = [_ArenaC(self.k_codes[i].data_ptr(), self.v_codes[i].data_ptr(),
                           self.k_scales[i].data_ptr(), self.v_scales[i].data_ptr(), pages,
                           kv_heads, page_tokens, head_dim) for i in range(layers)]
        self._refs = [ctypes.byref(c) for c in self._c]
        self._types = {torch.float16: _lib.GRM_B200_F16, torch.bfloat16: _lib.GRM_B200_BF16}

    def _rows(self, plan, name, x, heads):
        """Checks rows [tokens, heads, head_dim]; returns (type, row and head strides)."""
        kind = self._types.get(x.dtype)
        if kind is None:
            raise ValueError(f"{name} must be float16 or bfloat16, got {x.dtype}")
        if x.shape != (plan.tokens, heads, self.head_dim):
            raise ValueError(f"{name} must be [{plan.tokens}, {heads}, {self.head_dim}], got "
                             f"{tuple(x.shape)}")
        if x.device != self.device:
            raise ValueError(f"{name} is on {x.device}, the arena on {self.device}")
        row, head, inner = x.stride()
        if inner != 1 or row % 8 or head % 8 or x.data_ptr() % 16:
            raise ValueError(f"{name}: a head's values must be contiguous, rows and heads at "
                             f"multiples of 8 elements and 16-byte aligned (strides {x.stride()})")
        return kind, row, head

    def _plan(self, plan, layer):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        if not plan.planned:
            raise ValueError("the plan has not been planned yet (PageTables.plan)")

    def append(self, plan: PagePlan, k, v, *, layer: int = 0, stream=None) -> None:
        """Quantise the step's rows ``k`` and ``v`` [tokens, kv_heads, head_dim]
        into the pages of `layer`."""
        self._plan(plan, layer)
        kind, k_row, k_head = self._rows(plan, "k", k, self.kv_heads)
        v_kind, v_row, v_head = self._rows(plan, "v", v, self.kv_heads)
        if kind != v_kind:
            raise ValueError(f"k and v differ in type: {k.dtype}, {v.dtype}")
        if not plan.c.grow:
            raise ValueError("the plan's rows do not join the arena (planned with grow=False)")
        _, handle = _stream(stream, self.device, k, v)
        _call("grm_b200_paged_append", self.device, plan._ref, self._refs[layer], k.data_ptr(),
              v.data_ptr(), kind, k_row, k_head, v_row, v_head, handle)

    def attend(self, plan: PagePlan, q, *, layer: int = 0, causal: bool = True,
               scale: float | None = None, out=None, lse=None, stream=None):
        """Attention of the step's query rows ``q`` [tokens, query_heads,
        head_dim]: over everything the row's request holds, or with `causal` over
        the positions up to the row's own.  `scale` defaults to
        head_dim ** -0.5.  Returns (out like q, lse fp32 [tokens, query_heads]);
        rows that see nothing are 0 with lse -inf."""
        import torch

        self._plan(plan, layer)
        kind, row, head = self._rows(plan, "q", q, plan.query_heads)
        if causal and not plan.c.grow:
            raise ValueError("rows that do not join the arena (planned with grow=False) have no "
                             "position in it; attend with causal=False")
        stream, handle = _stream(stream, self.device, q)
        shape = (plan.tokens, plan.query_heads, self.head_dim)
        if out is None:
            out = _empty(shape, q.dtype, self.device, stream)
        elif (out.shape != shape or out.dtype != q.dtype or out.device != self.device or
              not out.is_contiguous()):
            raise ValueError(f"out must be contiguous {q.dtype} {list(shape)} on {self.device}")
        if lse is None:
            lse = _empty(shape[:2], torch.float32, self.device, stream)
        elif (lse.shape != shape[:2] or lse.dtype != torch.float32 or
              lse.device != self.device or not lse.is_contiguous()):
            raise ValueError(f"lse must be contiguous float32 {list(shape[:2])} on {self.device}")
        _call("grm_b200_paged_attend", self.device, plan._ref, self._refs[layer], q.data_ptr(),
              kind, row, head, 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale),
              1 if causal else 0, out.data_ptr(), lse.data_ptr(), handle)
        return out, lse

    def read(self, slots, *, layer: int = 0, dtype=None, stream=None):
        """Rows of values (k, v) [n, kv_heads, head_dim] of type `dtype`
        (default bfloat16; float16 and float32 too) at ``slots`` int64 [n]; a
        negative slot gives zeros."""
        import torch

        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        if (not isinstance(slots, torch.Tensor) or slots.dtype != torch.int64 or
                slots.dim() != 1 or slots.device != self.device or not slots.is_contiguous()):
            raise ValueError(f"slots must be int64 [n] on {self.device}")
        dtype = torch.bfloat16 if dtype is None else dtype
        kind = _lib.GRM_B200_F32 if dtype == torch.float32 else self._types.get(dtype)
        if kind is None:
            raise ValueError(f"read gives float32, float16 or bfloat16, not {dtype}")
        shape = (slots.numel(), self.kv_heads, self.head_dim)
        stream, handle = _stream(stream, self.device, slots)
        k = _empty(shape, dtype, self.device, stream)
        v = _empty(shape, dtype, self.device, stream)
        if slots.numel():
            _call("grm_b200_paged_read", self.device, self._refs[layer], slots.data_ptr(),
                  slots.numel(), kind, k.data_ptr(), v.data_ptr(), handle)
        return k, v
