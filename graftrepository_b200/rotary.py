"""Rotary positions of queries and keys, put on and taken off.

``graft_mount.RopeSpec`` re-RoPEs mounted rows by tables that the caller has.  A
``Rotary`` holds the frequencies themselves, as 64-bit fractions of a turn, so
that no position is too far for a table or for 32-bit angles, and serves

* ``rotate`` -- rows of several heads, a step's queries for instance, or keys
  whose position a harvest takes off (``inverse=True``);
* ``PagedArena.append(..., rotary=)`` and ``LatentArena.append(..., rotary=)``,
  which rotate a step's keys on the way into their pages.

    rotary = Rotary(128, base=10000.0, scaling=dict(kind="yarn", factor=16.0, original=4096))
    q = rotary.rotate(q, plan.positions)            # [tokens, heads, head_dim]
    arena.append(plan, k, v, layer=layer, rotary=rotary)

Layouts of a pair's two members: ``"half"`` (i and i + dim / 2),
``"interleaved"`` (2 i and 2 i + 1) and ``"pair_swap"`` (taken from 2 i and
2 i + 1, put to i and i + dim / 2, as ``RopeSpec(pair_swap=True)`` does).
Scalings for long contexts are in ``rotary_frequencies``.
"""

from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import torch

from . import _lib
from .paged_arena import _Buffers, _call, _device, _handle, _torch_stream

__all__ = ["LAYOUTS", "Rotary", "rotary_frequencies"]

LAYOUTS = {"half": 0, "interleaved": 1, "pair_swap": 2}
MOST_DIM = 4096
_TYPES = {torch.float32: _lib.GRM_B200_F32, torch.float16: _lib.GRM_B200_F16,
          torch.bfloat16: _lib.GRM_B200_BF16}
_TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937511")


class _RotaryC(ctypes.Structure):
    _fields_ = [("turns", ctypes.c_void_p), ("dim", ctypes.c_int32), ("offset", ctypes.c_int32),
                ("layout", ctypes.c_int32), ("amplitude", ctypes.c_float)]


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: dict | None = None):
    """(radians a position of each of the dim / 2 pairs, amplitude).  Pair i turns by
    base^(-2i / dim) a position.  `scaling`, by its ``kind``:

    * ``linear``: every frequency divided by ``factor``;
    * ``ntk``: the base multiplied by factor^(dim / (dim - 2)), which leaves the first
      pair alone and divides the last one's frequency by ``factor``;
    * ``yarn``: pairs that turn more than ``beta_fast`` (32) times over the
      ``original`` context keep their frequency, those that turn less than
      ``beta_slow`` (1) times have it divided by ``factor``, with a ramp over the
      pairs between; amplitude 0.1 ln(factor) + 1, or as given;
    * ``factors``: pair i's frequency divided by ``factors[i]``, with an
      ``amplitude`` (1)."""
    if dim < 2 or dim % 2 or dim > MOST_DIM:
        raise ValueError(f"a rotary dim is even, from 2 to {MOST_DIM}, got {dim}")
    if not 0 < base < math.inf:
        raise ValueError(f"the rotary base must be positive, got {base}")
    opts = dict(scaling or {})
    kind = opts.pop("kind", None)
    known = {None: (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original", "beta_fast", "beta_slow", "amplitude"),
             "factors": ("factors", "amplitude")}
    if kind not in known:
        raise ValueError(f"unknown rotary scaling {kind!r}; one of linear, ntk, yarn, factors")
    needed = {"linear": ("factor",), "ntk": ("factor",), "yarn": ("factor", "original"),
              "factors": ("factors",)}.get(kind, ())
    if set(opts) - set(known[kind]) or set(needed) - set(opts):
        raise ValueError(f"rotary scaling {kind!r} takes {known[kind]} and needs {needed}, got "
                         f"{tuple(opts)}")
    pairs = range(dim // 2)
    factor = float(opts.get("factor", 1.0))
    if not 0 < factor < math.inf:
        raise ValueError(f"a rotary factor must be positive, got {factor}")
    amplitude = opts.get("amplitude")
    if kind == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs a dim above 2")
        base = base * factor ** (dim / (dim - 2))
    f = [base ** (-2.0 * i / dim) for i in pairs]
    if kind == "linear":
        f = [x / factor for x in f]
    elif kind == "factors":
        by = [float(x) for x in opts["factors"]]
        if len(by) != dim // 2 or not all(0 < x < math.inf for x in by):
            raise ValueError(f"factors must be {dim // 2} positive numbers")
        f = [x / y for x, y in zip(f, by)]
    elif kind == "yarn":
        original = float(opts["original"])
        fast, slow = float(opts.get("beta_fast", 32.0)), float(opts.get("beta_slow", 1.0))
        if not (0 < original < math.inf and 0 < slow < fast < math.inf and base > 1):
            raise ValueError("yarn scaling needs a positive original, beta_fast above beta_slow "
                             "above 0 and a base above 1")

        def pair(turns):  # that turns so many times over the original context
            return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in pairs]
        f = [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)]
        if amplitude is None:
            amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    amplitude = 1.0 if amplitude is None else float(amplitude)
    if not 0 < amplitude < math.inf:
        raise ValueError(f"the rotary amplitude must be positive, got {amplitude}")
    return f, amplitude


class Rotary(_Buffers):
    """Rotary positions of `dim` values of a head, from `offset` on.  Lives on one
    device and follows the streams that it is used on."""

    def __init__(self, dim: int, *, offset: int = 0, base: float = 10000.0, layout: str = "half",
                 scaling: dict | None = None, device="cuda"):
        if layout not in LAYOUTS:
            raise ValueError(f"layout must be one of {tuple(LAYOUTS)}, got {layout!r}")
        if offset < 0:
            raise ValueError(f"offset must not be negative, got {offset}")
        self.frequencies, self.amplitude = rotary_frequencies(dim, base, scaling)
        self.dim, self.offset, self.layout = int(dim), int(offset), layout
        self.device = _device(device)
        self._index = self.device.index
        whole = 1 << 64
        turns = [round(Fraction(f) / _TWO_PI * whole) % whole for f in self.frequencies]
        self.turns = torch.tensor([t - whole if t >= whole // 2 else t for t in turns],
                                  dtype=torch.int64, device=self.device)
        self._made(self.turns)
        self.c = _RotaryC(self.turns.data_ptr(), self.dim, self.offset, LAYOUTS[layout],
                          self.amplitude)
        self._ref = ctypes.byref(self.c)
        self._rotate = _lib.load().grm_b200_rotate

    def _on(self, index) -> None:
        if index != self._index:
            raise ValueError(f"the rotary is on {self.device}, the rows on cuda:{index}")

    def rotate(self, x, positions, *, inverse: bool = False, out=None, stream=None):
        """Rows ``x`` [tokens, heads, head_dim] (float32, float16 or bfloat16, a head's
        values contiguous) rotated by ``positions`` int32 [tokens]; `inverse` takes
        the rotation off.  Returns `out` (default: a new tensor), where the other
        values of a head are copied, as are rows with a negative position.  With
        ``out=x`` (not for layout pair_swap) those are left alone."""
        kind = _TYPES.get(x.dtype)
        if kind is None:
            raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
        if x.dim() != 3:
            raise ValueError(f"x must be [tokens, heads, head_dim], got {list(x.shape)}")
        tokens, heads, head_dim = x.shape
        if x.get_device() != self._index:
            raise ValueError(f"x is on {x.device}, the rotary on {self.device}")
        if (not isinstance(positions, torch.Tensor) or positions.dtype is not torch.int32 or
                positions.get_device() != self._index or positions.shape != x.shape[:1] or
                not positions.is_contiguous()):
            raise ValueError(f"positions must be int32 [{tokens}] on {self.device}")
        if heads < 1 or self.offset + self.dim > head_dim:
            raise ValueError(f"dims {self.offset} to {self.offset + self.dim} are rotated, a head "
                             f"of x has {head_dim} ({heads} heads)")
        if x.stride(2) != 1:
            raise ValueError(f"a head's values must be contiguous (strides {x.stride()})")
        if out is None:
            if stream is None:
                out = x.new_empty(x.shape)
            else:
                with torch.cuda.stream(_torch_stream(stream, self._index)):
                    out = x.new_empty(x.shape)
        else:
            self._check_out(x, out)
        if tokens:
            _call(self._rotate, self._index, self._ref, x.data_ptr(), kind, tokens, heads,
                  head_dim, x.stride(0), x.stride(1), positions.data_ptr(), 1 if inverse else 0,
                  out.data_ptr(), out.stride(0), out.stride(1),
                  _handle(stream, self._index, (self,), x, positions, out))
        return out

    def _check_out(self, x, out) -> None:
        if (out.shape != x.shape or out.dtype is not x.dtype or
                out.get_device() != self._index or out.stride(2) != 1):
            raise ValueError(f"out must be {x.dtype} {list(x.shape)} on {self.device}, a head's "
                             f"values contiguous")
        if _rows_overlap(out):
            raise ValueError(f"rows of out overlap (strides {out.stride()})")
        if out.data_ptr() == x.data_ptr():
            if out.stride() != x.stride() or self.layout == "pair_swap":
                raise ValueError("in place takes the same strides, and no pair swap")
            return
        if x.numel() and _first(x) < _last(out) and _first(out) < _last(x) and not _apart(x, out):
            raise ValueError("out overlaps x")


def _first(t) -> int:
    return t.data_ptr()


def _last(t) -> int:
    return t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * \
        t.element_size()


def _steps(t):
    """(stride, entries) of the dimensions of rows [tokens, heads, head_dim] but the last,
    the larger stride first; those of one entry say nothing."""
    return sorted(((s, n) for s, n in zip(t.stride()[:2], t.shape[:2]) if n > 1), reverse=True)


def _rows_overlap(t) -> bool:
    """Whether one row may lie on another: each stride has to pass what lies within it."""
    span = t.shape[2]
    for s, n in reversed(_steps(t)):
        if s < span:
            return True
        span += (n - 1) * s
    return False


def _apart(x, out) -> bool:
    """Whether two views of one buffer share no value, where both lie the same way and rows of
    neither overlap, as the query and key parts of a projection's rows do.  (Views that lie
    in different ways are not looked into.)"""
    steps = _steps(x)
    step, odd = divmod(out.data_ptr() - x.data_ptr(), x.element_size())
    if steps != _steps(out) or odd or _rows_overlap(x):
        return False

    def meet(step, i):  # whether a row of x and one of out do, so many values apart
        if i == len(steps):
            return abs(step) < x.shape[2]
        s, n = steps[i]  # what lies within a stride is shorter, so one of two multiples
        return any(abs(k) < n and meet(step - k * s, i + 1) for k in (step // s, step // s + 1))

    return not meet(step, 0)
