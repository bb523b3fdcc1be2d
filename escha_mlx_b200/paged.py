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

from typing import NamedTuple

import torch

from ._lib import load_decode

decode = load_decode()

_DTYPES = (torch.float16, torch.bfloat16, torch.int8)
HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)


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
    return PagePlan._make(decode.plan(table, lengths, added, free_pages, head, page_size, n_pages, rows))


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
        if not isinstance(k, torch.Tensor) or k.dtype not in _DTYPES:
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
        self._tensors = (k, v, k_scale, v_scale)

    def arrays(self) -> list[torch.Tensor]:
        return [t for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None]

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Store rows ``k``, ``v`` [T, kv_heads, head_dim] at ``slots`` [T] int32.  Rows with a
        negative slot (or one past the cache) are skipped; the slots of one call must differ.
        Rows may be views into a merged projection (any row and head stride).  In an int8 cache
        a row becomes ``scale = max|x| / 127`` and its nearest codes, per head."""
        decode.append(*self._tensors, k, v, slots)

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               scale: float | None = None) -> torch.Tensor:
        """Attention of one new token per request: ``q`` [B, heads, head_dim] over the first
        ``lengths[b]`` tokens in pages ``table[b]`` [B, W], query head i reading key/value head
        ``i // (heads // kv_heads)``.  ``scale`` defaults to ``head_dim ** -0.5``.  Returns
        [B, heads, head_dim] in q's type.  A request of length 0 gives zeros; tokens on pages
        outside the cache are left out; lengths past the table are cut to it."""
        return decode.attend(*self._tensors, q, table, lengths,
                             self.head_dim ** -0.5 if scale is None else scale)
