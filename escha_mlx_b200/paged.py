"""Paged key-value cache of a decode step: page plans, stores and attention of one new token.

No counterpart in the reference, which leaves caches and attention to mlx-lm.  A step over a
batch of requests is

    plan = plan_pages(table, lengths, added, free_pages, head, ...)   # once per step
    cache.append(k, v, plan.slots)                                    # per layer
    y = cache.attend(q, table, plan.ends)                             # per layer

Everything stays on the device: nothing synchronises, so a step can be captured in a CUDA
graph (``graphs.GraphedCall``) and replayed while lengths and tables change.
"""
from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from ._lib import check, lib

# element types of the C boundary (include/escha_b200.h)
_F16, _BF16, _I8 = 0, 1, 3
_TYPES = {torch.float16: _F16, torch.bfloat16: _BF16, torch.int8: _I8}
HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)
PLAN_MAX_BATCH = 4096


_raw_stream = torch._C._cuda_getCurrentRawStream     # (device index) -> current stream's handle
_current_device = torch.cuda.current_device


def call_on(index: int, fn, *args) -> None:
    """``fn(*args, stream)`` on the current stream of device ``index``, whichever device is
    current."""
    if _current_device() == index:
        check(fn(*args, _raw_stream(index)))
    else:
        with torch.cuda.device(index):
            check(fn(*args, _raw_stream(index)))


def _is_int32(t, index: int, shape: tuple) -> bool:
    """A dense int32 tensor of that shape on device ``index`` (the checks of every call, in
    short; ``_check`` says what is wrong with one that fails)."""
    return (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.shape == shape
            and t.get_device() == index and t.is_contiguous())


def _check(name: str, t: torch.Tensor, shape: tuple, dtype, device: torch.device | None) -> None:
    """``t`` is a dense CUDA tensor of that type and shape (None: any extent)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path in this package)")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != len(shape) or any(w is not None and w != n for w, n in zip(shape, t.shape)):
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{name} must have shape [{want}], got {list(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


@functools.lru_cache(maxsize=4096)
def _attend_workspace(index: int, *shape: int) -> int:
    """Bytes of scratch for an attention call of that shape on that device."""
    with torch.cuda.device(index):
        return lib.escha_paged_attend_workspace_bytes(*shape)


class PagePlan(NamedTuple):
    """What ``plan_pages`` gives (all int32, on the device)."""
    slots: torch.Tensor      # [rows] slot of each row's token in the cache, -1: none
    positions: torch.Tensor  # [rows] the token's place in its request (0 where there is none)
    starts: torch.Tensor     # [B + 1] first row of each request; last: rows asked for
    ends: torch.Tensor       # [B] tokens of each request after the step
    head: torch.Tensor       # [1] position in the free list after the step
    refused: torch.Tensor    # [1] requests that could not be served


def plan_pages(table: torch.Tensor, lengths: torch.Tensor, added: torch.Tensor,
               free_pages: torch.Tensor, head: torch.Tensor, *, page_size: int, n_pages: int,
               rows: int) -> PagePlan:
    """Give each request the pages that its new tokens need, and each new token its slot.

    ``table`` [B, W] int32 holds the requests' page ids and is updated in place; ``lengths``
    [B] are the tokens they hold, ``added`` [B] those of this step, whose rows are packed by
    request (``rows`` of them at most; the batch's number of rows under a CUDA graph).  Pages
    are taken from ``free_pages[head:]`` in request order.  A request that cannot be served
    (negative numbers, more tokens than W pages hold, rows past ``rows``, free pages used up by
    it and those before it) gets nothing: its rows have slot -1, ``ends`` keeps its length and
    ``refused`` counts it.  One launch, for up to 4096 requests."""
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        _check("table", table, (None, None), torch.int32, None)
    (b, w), index = table.shape, table.get_device()
    if not (index >= 0 and _is_int32(table, index, (b, w)) and _is_int32(lengths, index, (b,))
            and _is_int32(added, index, (b,)) and _is_int32(head, index, (1,))
            and _is_int32(free_pages, index, free_pages.shape[:1])):
        _check("table", table, (None, None), torch.int32, None)
        _check("lengths", lengths, (b,), torch.int32, table.device)
        _check("added", added, (b,), torch.int32, table.device)
        _check("free_pages", free_pages, (None,), torch.int32, table.device)
        _check("head", head, (1,), torch.int32, table.device)
    rows = int(rows)
    if not 1 <= b <= PLAN_MAX_BATCH:
        raise ValueError(f"plan_pages takes 1..{PLAN_MAX_BATCH} requests, got {b}")
    if not 0 <= rows <= 1 << 30:
        raise ValueError(f"rows must be in [0, 2^30], got {rows}")
    if page_size not in PAGE_SIZES or not 1 <= n_pages < 1 << 31:
        raise ValueError(f"page_size must be one of {PAGE_SIZES} and n_pages in [1, 2^31), got "
                         f"{page_size} and {n_pages}")
    buf = table.new_empty(2 * rows + 2 * b + 3)
    at = buf.data_ptr()
    ends = at + 4 * (2 * rows + b + 1)
    call_on(index, lib.escha_page_plan, table.data_ptr(), lengths.data_ptr(), added.data_ptr(),
            free_pages.data_ptr(), free_pages.shape[0], head.data_ptr(), b, w, page_size, n_pages, rows,
            at, at + 4 * rows, at + 8 * rows, ends, ends + 4 * b, ends + 4 * b + 4)
    return PagePlan(*buf.split_with_sizes((rows, rows, b + 1, b, 1, 1)))


def _rows(name: str, x: torch.Tensor, shape: tuple, index: int) -> tuple:
    """``x`` [rows, heads, channels] as the kernels can read it (dense channels, other strides
    multiples of 8 elements, 16-byte aligned; a dense copy if it is not so), with its row and
    head strides."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path in this package)")
    if x.get_device() != index:
        raise ValueError(f"{name} is on {x.device}, the cache on cuda:{index}")
    if x.dim() != 3 or any(w is not None and w != n for w, n in zip(shape, x.shape)):
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{name} must have shape [{want}], got {list(x.shape)}")
    s0, s1, s2 = x.stride()
    if s2 != 1 or (s0 | s1) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        s0, s1, s2 = x.stride()
    return x, s0, s1


class PagedCache:
    """Keys and values of one layer in pages of ``page_size`` tokens.

    ``k``, ``v``: [n_pages, kv_heads, page_size, head_dim] in float16, bfloat16, or int8 with
    ``k_scale``, ``v_scale`` [n_pages, kv_heads, page_size] float32 (one scale per token and
    head).  A slot is ``page * page_size + offset``."""

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device=None) -> None:
        shape = (n_pages, kv_heads, page_size, head_dim)
        dev = torch.device(device or "cuda")
        self._adopt(torch.zeros(shape, dtype=dtype, device=dev),
                    torch.zeros(shape, dtype=dtype, device=dev),
                    *([torch.zeros(shape[:3], dtype=torch.float32, device=dev) for _ in range(2)]
                      if dtype == torch.int8 else [None, None]))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedCache":
        """A cache over tensors that the caller owns (nothing is copied)."""
        self = cls.__new__(cls)
        self._adopt(k, v, k_scale, v_scale)
        return self

    def _adopt(self, k, v, k_scale, v_scale) -> None:
        if not isinstance(k, torch.Tensor) or k.dtype not in _TYPES:
            raise ValueError("a paged cache is float16, bfloat16 or int8, got "
                             f"{getattr(k, 'dtype', type(k))}")
        _check("k", k, (None, None, None, None), k.dtype, None)
        _check("v", v, tuple(k.shape), k.dtype, k.device)
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        if self.head_dim not in HEAD_DIMS:
            raise ValueError(f"head size {self.head_dim}; the paged cache takes {HEAD_DIMS}")
        if self.page_size not in PAGE_SIZES:
            raise ValueError(f"page size {self.page_size}; the paged cache takes {PAGE_SIZES}")
        if self.n_pages < 1 or self.kv_heads < 1:
            raise ValueError("a paged cache needs at least one page and one head")
        if k.data_ptr() % 16 or v.data_ptr() % 16:
            raise ValueError("a paged cache's tensors must be 16-byte aligned")
        if (k.dtype == torch.int8) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise ValueError("an int8 cache has scales for keys and values, the others have none")
        if k_scale is not None:
            _check("k_scale", k_scale, tuple(k.shape[:3]), torch.float32, k.device)
            _check("v_scale", v_scale, tuple(k.shape[:3]), torch.float32, k.device)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.dtype, self.device = k.dtype, k.device
        self._index = k.get_device()
        # what every call passes on
        self._tensors = (k.data_ptr(), v.data_ptr(), _TYPES[k.dtype],
                         *((None, None) if k_scale is None else (k_scale.data_ptr(), v_scale.data_ptr())))

    def arrays(self) -> list[torch.Tensor]:
        return [t for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None]

    def _row_type(self, name: str, x: torch.Tensor) -> int:
        ok = (torch.float16, torch.bfloat16) if self.dtype == torch.int8 else (self.dtype,)
        if x.dtype not in ok:
            raise ValueError(f"{name} must be {' or '.join(str(d) for d in ok)} for a {self.dtype} "
                             f"cache, got {x.dtype}")
        return _TYPES[x.dtype]

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Store rows ``k``, ``v`` [T, kv_heads, head_dim] at ``slots`` [T] int32.  Rows with a
        negative slot (or one past the cache) are skipped; the slots of one call must differ.
        Rows may be views into a merged projection (any row and head stride).  In an int8 cache
        a row becomes ``scale = max|x| / 127`` and its nearest codes, per head."""
        k, k_row, k_head = _rows("k", k, (None, self.kv_heads, self.head_dim), self._index)
        t = k.shape[0]
        v, v_row, v_head = _rows("v", v, (t, self.kv_heads, self.head_dim), self._index)
        if k.dtype is not v.dtype:
            raise ValueError(f"k is {k.dtype}, v is {v.dtype}")
        kind = self._row_type("k", k)
        if not _is_int32(slots, self._index, (t,)):
            _check("slots", slots, (t,), torch.int32, self.device)
        if t == 0:
            return
        k_cache, v_cache, cache_type, k_scale, v_scale = self._tensors
        call_on(self._index, lib.escha_paged_append, k.data_ptr(), k_row, k_head, v.data_ptr(), v_row,
                v_head, kind, slots.data_ptr(), t, self.kv_heads, self.head_dim, self.page_size,
                self.n_pages, k_cache, v_cache, cache_type, k_scale, v_scale)

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               scale: float | None = None) -> torch.Tensor:
        """Attention of one new token per request: ``q`` [B, heads, head_dim] over the first
        ``lengths[b]`` tokens in pages ``table[b]`` [B, W], query head i reading key/value head
        ``i // (heads // kv_heads)``.  ``scale`` defaults to ``head_dim ** -0.5``.  Returns
        [B, heads, head_dim] in q's type.  A request of length 0 gives zeros; tokens on pages
        outside the cache are left out; lengths past the table are cut to it."""
        q, q_row, q_head = _rows("q", q, (None, None, self.head_dim), self._index)
        kind = self._row_type("q", q)
        b, heads, d = q.shape
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads do not share {self.kv_heads} key/value heads evenly")
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            _check("table", table, (b, None), torch.int32, self.device)
        group, w, index = heads // self.kv_heads, table.shape[1], self._index
        if not (_is_int32(table, index, (b, w)) and _is_int32(lengths, index, (b,))):
            _check("table", table, (b, None), torch.int32, self.device)
            _check("lengths", lengths, (b,), torch.int32, self.device)
        if w < 1:
            raise ValueError("table needs at least one page per request")
        out = q.new_empty((b, heads, d))
        if b == 0:
            return out
        need = _attend_workspace(index, b, self.kv_heads, group, d, w, self.page_size)
        work = q.new_empty(need, dtype=torch.uint8) if need else None
        call_on(index, lib.escha_paged_attend, q.data_ptr(), q_row, q_head, kind, *self._tensors,
                table.data_ptr(), lengths.data_ptr(), b, self.kv_heads, group, d, w, self.page_size,
                self.n_pages, d ** -0.5 if scale is None else scale, work.data_ptr() if need else None,
                need, out.data_ptr())
        return out
