"""Pages of latent rows, and latent attention over them.

Models with latent attention keep one row a token for all heads: ``latent``
values c that every head's keys and values are made from, and ``rope`` values r
that hold the position.  ``graft_mount`` writes such rows, 256 + 32 values wide,
for one request; ``LatentArena`` holds them for many, in 16 bits, in pages of the
same ``PageTables`` as the 8-bit arena's:

* ``make_plan``        -- the buffers of one step, planned by ``PageTables.plan``;
* ``append``           -- the step's rows into their pages, the positional part
                          rotated on the way if a ``Rotary`` is given;
* ``attend``           -- the absorbed form: queries that a head's weights have taken
                          into the latent space attend to the rows themselves, and
                          results are latent, too.  For decoding, where a row of
                          the cache serves all heads;
* ``attend_expanded``  -- the expanded form: each head's keys and values are made
                          from the rows first.  About a third of the operations a
                          (row, token), so for prompts.

A step::

    plan = arena.make_plan(tables, tokens, heads=40)
    tables.plan(plan, fresh)
    for layer in range(layers):
        arena.append(plan, c, r, layer=layer, rotary=rotary)
        q_latent = torch.einsum("thn,hnc->thc", q_nope, weights[layer][:, :64])
        q_rope = rotary.rotate(q_pe, plan.positions)
        out, lse = arena.attend(plan, q_latent, q_rope, scale=96 ** -0.5, layer=layer)
        out = torch.einsum("thc,hvc->thv", out, weights[layer][:, 64:])
    tables.commit(plan)

``arena.rows[layer]`` is a plain tensor [pages, page_tokens, latent + rope]; a
harvest indexes it by slots.  Streams, graphs, turns and ``plan.check()`` are as in
``paged_arena``.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .paged_arena import (_Buffers, _TYPES, PagePlan, PageTables, _PlanC, _call, _check_page,
                          _device, _handle, _result)
from .rotary import _first, _last

__all__ = ["LATENTS", "ROPES", "EXPANDED", "LatentPlan", "LatentArena"]

LATENTS = (128, 256, 512)
ROPES = (32, 64)
EXPANDED = (64, 128)  # nope and value of the expanded form


class _LatentArenaC(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_void_p), ("pages", ctypes.c_int64),
                ("page_tokens", ctypes.c_int32), ("latent", ctypes.c_int32),
                ("rope", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class _LatentPlanC(ctypes.Structure):
    _fields_ = [("step", _PlanC), ("heads", ctypes.c_int32), ("latent", ctypes.c_int32),
                ("rope", ctypes.c_int32), ("nope", ctypes.c_int32), ("value", ctypes.c_int32),
                ("expand_tokens", ctypes.c_int64), ("work", ctypes.c_void_p),
                ("work_bytes", ctypes.c_int64)]


class LatentPlan(PagePlan):
    """The buffers of one step over latent rows (``LatentArena.make_plan``): those
    of a ``PagePlan``, the lists of attention and room for its partial results and
    for what the expanded form expands."""

    def __init__(self, tables: PageTables, tokens: int, heads: int, latent: int, rope: int,
                 dtype, max_fresh: int | None, nope: int, value: int, expand_tokens: int):
        if not 1 <= heads <= 1024:
            raise ValueError(f"heads must be 1 to 1024, got {heads}")
        if (nope, value, expand_tokens) != (0, 0, 0) and (
                nope not in EXPANDED or value != nope or not 1 <= expand_tokens <= 1 << 28 or
                expand_tokens * heads >= 1 << 31):
            raise ValueError(f"the expanded form takes nope = value of {EXPANDED} and "
                             f"expand_tokens from 1 to 2^28 and below 2^31 / heads, got {nope}, "
                             f"{value}, {expand_tokens}")
        super().__init__(tables, tokens, 1, 1, 64, max_fresh)
        self.heads, self.latent, self.rope, self.dtype = int(heads), latent, rope, dtype
        self.nope, self.value, self.expand_tokens = int(nope), int(value), int(expand_tokens)
        t = self.tokens
        self.latent_shape, self.rope_shape = torch.Size((t, latent)), torch.Size((t, rope))
        self.query_shapes = torch.Size((t, heads, latent)), torch.Size((t, heads, rope))
        self.query_shape = torch.Size((t, heads, nope + rope))
        self.weight_shape = torch.Size((heads, nope + value, latent))
        one = torch.empty(1, dtype=dtype, device=self.device)
        self._out_like = one.expand(t, heads, latent)
        self._expanded_like = one.expand(t, heads, max(value, 1))
        self._lse_like = torch.empty(1, device=self.device).expand(t, heads)
        self.latent_c = _LatentPlanC(self.c, heads, latent, rope, nope, value, expand_tokens)
        need = ctypes.c_int64(0)
        lib = _lib.load()
        _call(lib.grm_b200_latent_work_bytes, self._index, ctypes.byref(self.latent_c),
              ctypes.byref(need))
        self.work = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        self._made(*self._tensors, self.work)
        self.latent_c.work, self.latent_c.work_bytes = self.work.data_ptr(), need.value
        self.c = self.latent_c.step  # `grow` is set in place
        self._ref = ctypes.byref(self.c)
        self._step, self._step_ref = lib.grm_b200_latent_plan_step, ctypes.byref(self.latent_c)


class LatentArena(_Buffers):
    """Rows ``rows`` [layers, pages, page_tokens, latent + rope] of float16 or
    bfloat16."""

    def __init__(self, layers: int, pages: int, latent: int, rope: int, *, page_tokens: int = 64,
                 dtype=torch.bfloat16, device="cuda"):
        if layers < 1 or pages < 1:
            raise ValueError(f"layers and pages must be positive, got {layers}, {pages}")
        if latent not in LATENTS or rope not in ROPES:
            raise ValueError(f"latent must be one of {LATENTS} and rope one of {ROPES}, got "
                             f"{latent}, {rope}")
        if dtype not in _TYPES:
            raise ValueError(f"latent rows are float16 or bfloat16, got {dtype}")
        self.layers, self.pages, self.latent, self.rope = int(layers), int(pages), latent, rope
        self.page_tokens, self.dtype = _check_page(page_tokens), dtype
        self.device = _device(device)
        self._index = self.device.index
        self.rows = torch.zeros((layers, pages, page_tokens, latent + rope), dtype=dtype,
                                device=self.device)
        self._made(self.rows)
        self._c = [_LatentArenaC(self.rows[i].data_ptr(), pages, page_tokens, latent, rope,
                                 _TYPES[dtype]) for i in range(layers)]
        self._refs = [ctypes.byref(c) for c in self._c]
        lib = _lib.load()
        self._append, self._attend = lib.grm_b200_latent_append, lib.grm_b200_latent_attend
        self._attend_expanded = lib.grm_b200_latent_attend_expanded

    def make_plan(self, tables: PageTables, tokens: int, *, heads: int,
                  max_fresh: int | None = None, nope: int = 0, value: int = 0,
                  expand_tokens: int = 0) -> LatentPlan:
        """Buffers for steps of up to `tokens` new rows, at most `max_fresh` of one
        request, and `heads` query heads.  For ``attend_expanded`` also what a row
        becomes for each head (`nope` values of its keys, as many of its values, 64
        or 128) and room for `expand_tokens` tokens: the lengths of the requests
        with rows in a step, each rounded up to 64.  That room is expand_tokens *
        heads * (2 * nope + value) * 2 bytes.  A plan's steps may not overlap on the
        GPU."""
        if tables.pages != self.pages or tables.page_tokens != self.page_tokens:
            raise ValueError(f"the tables have {tables.pages} pages of {tables.page_tokens} "
                             f"tokens, the arena {self.pages} of {self.page_tokens}")
        if tables._index != self._index:
            raise ValueError(f"the tables are on {tables.device}, the arena on {self.device}")
        return LatentPlan(tables, tokens, heads, self.latent, self.rope, self.dtype, max_fresh,
                          nope, value, expand_tokens)

    def _rows(self, name, x, shape):
        """Checks rows of `shape`, 2 or 3 dimensions; returns (pointer, strides but the
        last)."""
        if x.dtype is not self.dtype:
            raise ValueError(f"{name} must be {self.dtype} as the arena, got {x.dtype}")
        if x.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {list(x.shape)}")
        if x.get_device() != self._index:
            raise ValueError(f"{name} is on {x.device}, the arena on {self.device}")
        *steps, inner = x.stride()
        # the stride of a dimension of one entry says nothing
        steps = [s if n > 1 else 0 for s, n in zip(steps, shape)]
        ptr = x.data_ptr()
        if inner != 1 or any(s & 7 for s in steps) or ptr & 15:
            raise ValueError(f"{name}: the last dimension must be contiguous, the others at "
                             f"multiples of 8 elements and 16-byte aligned (strides {x.stride()})")
        return ptr, *steps

    def _ready(self, plan, layer):
        """The layer's buffers, for a plan that is good for a call."""
        if plan.latent != self.latent or plan.rope != self.rope or plan.dtype is not self.dtype:
            raise ValueError("the plan was not made for such rows (LatentArena.make_plan)")
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

    def _apart(self, out, lse, **read):
        """Refuses results over what the call reads (other blocks may still read the queries
        of rows whose result is there), and over each other."""
        for name, t in (("out", out), ("lse", lse)):
            for what, x in read.items():
                if _first(t) < _last(x) and _first(x) < _last(t):
                    raise ValueError(f"{name} overlaps {what}")
        if _first(out) < _last(lse) and _first(lse) < _last(out):
            raise ValueError("out overlaps lse")

    def append(self, plan: LatentPlan, latent, rope, *, layer: int = 0, rotary=None,
               stream=None) -> None:
        """Write the step's rows ``latent`` [tokens, latent] and ``rope`` [tokens, rope]
        into the pages of `layer`.  With a ``rotary.Rotary`` (dim = rope, offset 0) the
        positional part is rotated by ``plan.positions`` on the way."""
        ref = self._ready(plan, layer)
        c_ptr, c_row = self._rows("latent", latent, plan.latent_shape)
        r_ptr, r_row = self._rows("rope", rope, plan.rope_shape)
        if not plan.grow:
            raise ValueError("the plan's rows do not join the arena (planned with grow=False)")
        owners = (self, plan)
        if rotary is not None:
            rotary._on(self._index)
            if rotary.dim != self.rope or rotary.offset:
                raise ValueError(f"the rotary's dim {rotary.dim} and offset {rotary.offset} must "
                                 f"be {self.rope} and 0")
            owners = (self, plan, rotary)
        _call(self._append, self._index, plan._step_ref, ref,
              None if rotary is None else rotary._ref, c_ptr, c_row, r_ptr, r_row,
              _handle(stream, self._index, owners, latent, rope))

    def _causal(self, plan, causal):
        if causal and not plan.grow:
            raise ValueError("rows that do not join the arena (planned with grow=False) have no "
                             "position in it; attend with causal=False")
        return 1 if causal else 0

    def attend(self, plan: LatentPlan, q_latent, q_rope, *, scale: float, layer: int = 0,
               causal: bool = True, out=None, lse=None, stream=None):
        """Absorbed form: queries ``q_latent`` [tokens, heads, latent] and ``q_rope``
        [tokens, heads, rope] over everything the row's request holds, or with
        `causal` over the positions up to the row's own.  `scale` (positive)
        multiplies the scores: for heads of nope + rope values usually (nope + rope)
        ** -0.5.  Returns (out [tokens, heads, latent], lse fp32 [tokens, heads]), new
        ones or those given, which may not overlap what the call reads (or lie among its
        rows) nor each other; rows that see nothing are 0 with lse -inf.  A
        visible score of NaN or +inf makes its row NaN; one of -inf weighs nothing, and a
        row that has no other is NaN with lse -inf."""
        ref = self._ready(plan, layer)
        wide, narrow = plan.query_shapes
        c_ptr, c_row, c_head = self._rows("q_latent", q_latent, wide)
        r_ptr, r_row, r_head = self._rows("q_rope", q_rope, narrow)
        causal = self._causal(plan, causal)
        given = out is not None or lse is not None
        out = self._result("out", out, plan._out_like, stream)
        lse = self._result("lse", lse, plan._lse_like, stream)
        if given:
            self._apart(out, lse, q_latent=q_latent, q_rope=q_rope, rows=self.rows)
        _call(self._attend, self._index, plan._step_ref, ref, c_ptr, c_row, c_head, r_ptr, r_row,
              r_head, float(scale), causal, out.data_ptr(), lse.data_ptr(),
              _handle(stream, self._index, (self, plan), q_latent, q_rope, out, lse))
        return out, lse

    def attend_expanded(self, plan: LatentPlan, q, weights, *, scale: float, layer: int = 0,
                        causal: bool = True, out=None, lse=None, stream=None):
        """Expanded form: queries ``q`` [tokens, heads, nope + rope]; ``weights`` [heads,
        nope + value, latent] make each head's keys (the first nope, beside the
        row's positional part) and values from a row.  Values are rounded to the
        arena's type, keys held as two numbers of it; a token of which one of these is
        beyond the type's range makes the rows that see it NaN.  Returns (out
        [tokens, heads, value], lse); otherwise as ``attend``.  Where the step has
        more tokens to expand than ``plan.expand_tokens`` (``plan.check`` says so)
        rows are NaN."""
        ref = self._ready(plan, layer)
        if not plan.nope:
            raise ValueError("the plan has no room for the expanded form (make_plan with nope, "
                             "value and expand_tokens)")
        q_ptr, q_row, q_head = self._rows("q", q, plan.query_shape)
        w_ptr, w_head, w_row = self._rows("weights", weights, plan.weight_shape)
        causal = self._causal(plan, causal)
        given = out is not None or lse is not None
        out = self._result("out", out, plan._expanded_like, stream)
        lse = self._result("lse", lse, plan._lse_like, stream)
        if given:
            self._apart(out, lse, q=q, weights=weights, rows=self.rows)
        _call(self._attend_expanded, self._index, plan._step_ref, ref, q_ptr, q_row, q_head,
              w_ptr, w_head, w_row, float(scale), causal, out.data_ptr(), lse.data_ptr(),
              _handle(stream, self._index, (self, plan), q, weights, out, lse))
        return out, lse
