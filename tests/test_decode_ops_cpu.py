"""CPU: the decode step's entry points refuse what they do not take before any launch."""
from __future__ import annotations

import ctypes

import pytest
import torch

from escha_mlx_b200 import paged
from escha_mlx_b200._lib import check, lib

P = ctypes.c_void_p(0x1000)      # aligned, never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x1002)


def refused(rc, text):
    with pytest.raises(ValueError, match=text):
        check(rc)


def plan(B=1, W=4, F=1, page=16, n_pages=8, rows=1, table=P, free=P, slots=P):
    return lib.escha_page_plan(table, P, P, free, F, P, B, W, page, n_pages, rows, slots, P, P, P, P,
                               P, None)


def test_page_plan_refusals():
    refused(plan(B=0), "B=0")
    refused(plan(B=4097), "B=4097")
    refused(plan(page=24), "page_size=24")
    refused(plan(page=8), "page_size=8")
    refused(plan(W=0), "W=0")
    refused(plan(W=1 << 27), "W=")
    refused(plan(n_pages=0), "n_pages=0")
    refused(plan(n_pages=1 << 27, page=16), "n_pages=")
    refused(plan(F=-1), "F=-1")
    refused(plan(rows=-1), "rows=-1")
    refused(plan(table=None), "table is NULL")
    refused(plan(table=ODD), "4-byte")
    refused(plan(free=None), "free_pages is NULL")
    refused(plan(slots=None), "slots is NULL")


def append(k=P, stride=128, kind=0, T=1, H=2, D=64, page=16, n_pages=8, cache=0, scale=None):
    return lib.escha_paged_append(k, stride, 64, P, stride, 64, kind, P, T, H, D, page, n_pages, P, P,
                                  cache, scale, scale, None)


def test_paged_append_refusals():
    refused(append(D=96), "head size 96")
    refused(append(H=0), "H=0")
    refused(append(page=20), "page_size=20")
    refused(append(n_pages=0), "n_pages=0")
    refused(append(kind=2), "element type 2")
    refused(append(kind=0, cache=1), "cache of type 1")
    refused(append(cache=3), "needs k_scale")
    refused(append(T=0), "at least one row")
    refused(append(stride=129), "multiples of 8")
    refused(append(stride=-8), "multiples of 8")
    refused(append(k=None), "k is NULL")
    refused(append(k=ctypes.c_void_p(0x1008)), "16-byte")


def attend(q=P, stride=128, kind=0, cache=0, B=1, H=1, group=2, D=64, W=1024, page=16, n_pages=8,
           work=P, nbytes=1 << 30):
    return lib.escha_paged_attend(q, stride, 64, kind, P, P, cache, None, None, P, P, B, H, group, D, W,
                                  page, n_pages, 1.0, work, nbytes, P, None)


def test_paged_attend_refusals():
    refused(attend(D=32), "head size 32")
    refused(attend(B=0), "B=0")
    refused(attend(group=0), "group=0")
    refused(attend(W=0), "W=0")
    refused(attend(W=1 << 28), "W=")
    refused(attend(stride=4), "multiples of 8")
    refused(attend(kind=3), "element type 3")
    refused(attend(cache=3), "needs k_scale")
    refused(attend(q=ODD), "16-byte")
    refused(attend(work=None), "workspace")
    refused(attend(nbytes=16), "workspace")
    refused(attend(B=1024, H=1024, W=1 << 20), "more than one launch")


def test_workspace_is_asked_for_only_when_a_second_launch_joins():
    size = lib.escha_paged_attend_workspace_bytes
    assert size(1000, 2, 8, 256, 4, 16) == 0         # 64 tokens: one block, never cut
    assert size(8, 2, 8, 256, 128, 16) == 0          # short rows, few enough: clusters
    assert size(4, 2, 8, 256, 512, 16) == 0          # 8192 tokens: a few rows, wide clusters
    # 9600 tokens are 150 blocks of both heads: two CTAs for each of 148 SMs, two pieces of 8
    # heads per CTA, each with its maximum, sum and channels
    ctas = 296
    assert size(1, 2, 8, 256, 600, 16) == ctas * 8 + 2 * ctas * 8 * (8 + 4 * 256)
    assert size(0, 2, 8, 256, 600, 16) == size(1, 2, 8, 256, 600, 20) == 0


def test_python_level_refusals_without_a_gpu():
    x = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.PagedCache.from_tensors(x, x)
    with pytest.raises(ValueError, match="float16"):
        paged.PagedCache.from_tensors(x.float(), x.float())
    i = torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.plan_pages(i, i[0], i[0], i[0], i[0], page_size=16, n_pages=4, rows=1)


def sample(logits=P, kind=0, stride=8, B=1, V=8, u=P, tokens=P):
    return lib.escha_sample(logits, kind, stride, B, V, u, None, 1.0, None, 0, None, 1.0, None, 0.0,
                            tokens, None)


def test_sample_refusals():
    refused(sample(kind=3), "type 3")
    refused(sample(B=0), "B=0")
    refused(sample(V=0), "V=0")
    refused(sample(V=lib.escha_sample_max_vocab(0) + 1), "V=")
    refused(sample(kind=2, V=lib.escha_sample_max_vocab(0)), "V=")
    refused(sample(stride=-1), "stride=-1")
    refused(sample(logits=None), "logits is NULL")
    refused(sample(logits=ctypes.c_void_p(0x1001)), "aligned")
    refused(sample(u=None), "uniforms is NULL")
    refused(sample(tokens=None), "tokens is NULL")
    refused(sample(tokens=ctypes.c_void_p(0x1004)), "8-byte")
    assert lib.escha_sample_max_vocab(0) >= 2 * lib.escha_sample_max_vocab(2) - 64 >= 300000
    assert lib.escha_sample_max_vocab(7) == 0
    from escha_mlx_b200 import sampling
    with pytest.raises(ValueError, match="CUDA"):
        sampling.sample(torch.zeros((1, 8)), torch.zeros(1))
    with pytest.raises(ValueError, match="logits"):
        sampling.max_vocab(torch.float64)
