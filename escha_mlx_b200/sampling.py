"""A token per row of logits: temperature, top-k, top-p and min-p, from given uniform numbers.

No counterpart in the reference, which samples through mlx-lm.  Takes what the int8 vocabulary
head (``quant.EschaQ8Head``) gives and gives what ``quant.EschaQ8Embedding`` takes; one launch,
no host synchronisation, so it can end a captured decode step.
"""
from __future__ import annotations

import torch

from ._lib import lib
from .paged import call_on

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def max_vocab(dtype: torch.dtype) -> int:
    """The longest row of logits of that type that ``sample`` takes."""
    if dtype not in _TYPES:
        raise ValueError(f"logits must be one of {list(_TYPES)}, got {dtype}")
    return lib.escha_sample_max_vocab(_TYPES[dtype])


def _setting(name: str, value, rows: int, dtype, index: int) -> tuple:
    """(pointer or None, number) of a setting: one number, or a tensor with one per row."""
    if not isinstance(value, torch.Tensor):
        # any top_k past the vocabulary says the same
        return None, (max(-1, min(int(value), 0x7fffffff)) if dtype is torch.int32 else float(value))
    if value.dtype is not dtype or value.numel() != rows or not value.is_contiguous():
        raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of {rows} values, "
                         f"got {value.dtype} {list(value.shape)}")
    if value.get_device() != index:
        raise ValueError(f"{name} is on {value.device}, the logits on cuda:{index}")
    return value.data_ptr(), 0


def sample(logits: torch.Tensor, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0) -> torch.Tensor:
    """``logits`` [..., V] float16, bfloat16 or float32; ``uniforms`` [...] float32 in [0, 1);
    the settings are numbers or tensors [...] (float32; ``top_k`` int32).  Returns int64 [...].

    With ``d = (x - max x) / temperature`` and weights ``exp(d)``, 0 where ``d < -30``: of the
    tokens ordered by (x descending, index ascending) the first ``top_k`` are kept, of those
    the shortest prefix that has at least ``top_p`` of their weight, of those the ones with at
    least ``min_p`` of the largest weight.  The token is the first, in index order, whose
    cumulative kept weight exceeds ``uniform * total``.  A temperature that is not above 0 takes
    the first largest logit; ``top_k`` outside [1, V), ``top_p >= 1`` and ``min_p <= 0`` cut
    nothing.  NaN logits count as -inf; a row without any logit above -inf gives -1."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor (there is no CPU path in this package)")
    if logits.dtype not in _TYPES:
        raise ValueError(f"logits must be one of {list(_TYPES)}, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape [..., V], got {list(logits.shape)}")
    lead, v, index = logits.shape[:-1], logits.shape[-1], logits.get_device()
    x = logits if len(lead) == 1 else logits.reshape(-1, v)
    if v > 0x7fffffff:
        raise ValueError(f"V={v} logits per row; sample takes {max_vocab(x.dtype)} at most")
    if x.stride(1) != 1:
        x = x.contiguous()
    b = x.shape[0]
    if not isinstance(uniforms, torch.Tensor) or uniforms.dtype is not torch.float32 \
            or uniforms.shape != lead or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be a contiguous float32 tensor of shape {list(lead)}")
    if uniforms.get_device() != index:
        raise ValueError(f"uniforms is on {uniforms.device}, the logits on {logits.device}")
    t, t1 = _setting("temperature", temperature, b, torch.float32, index)
    k, k1 = _setting("top_k", top_k, b, torch.int32, index)
    p, p1 = _setting("top_p", top_p, b, torch.float32, index)
    m, m1 = _setting("min_p", min_p, b, torch.float32, index)
    tokens = uniforms.new_empty(lead, dtype=torch.int64)
    if b:
        call_on(index, lib.escha_sample, x.data_ptr(), _TYPES[x.dtype], x.stride(0), b, v,
                uniforms.data_ptr(), t, t1, k, k1, p, p1, m, m1, tokens.data_ptr())
    return tokens
