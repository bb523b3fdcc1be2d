"""A token per row of logits: temperature, top-k, top-p and min-p, from given uniform numbers.

No counterpart in the reference, which samples through mlx-lm.  Takes what the int8 vocabulary
head (``quant.EschaQ8Head``) gives and gives what ``quant.EschaQ8Embedding`` takes; one launch,
no host synchronisation, so it can end a captured decode step.
"""
from __future__ import annotations

import torch

from ._lib import lib, load_decode

decode = load_decode()

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def max_vocab(dtype: torch.dtype) -> int:
    """The longest row of logits of that type that ``sample`` takes."""
    if dtype not in _TYPES:
        raise ValueError(f"logits must be one of {list(_TYPES)}, got {dtype}")
    return lib.escha_sample_max_vocab(_TYPES[dtype])


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
    return decode.sample(logits, uniforms, temperature, top_k, top_p, min_p)
