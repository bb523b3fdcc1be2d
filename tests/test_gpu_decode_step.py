"""A decode step end to end: embedding, layers with paged attention, head, sampling; eagerly
and replayed from one CUDA graph."""
from __future__ import annotations

import pytest
import torch

from escha_mlx_b200 import paged, quant, workloads

pytestmark = pytest.mark.gpu

CFG = dict(hidden=256, inter=128, experts=8, top_k=2, K_gate_up=2, K_down=2, q_heads=4, kv_heads=2,
           head_dim=64)
VOCAB, B, PAGE, PAGES, STEPS = 1000, 3, 16, 24, 40


def stack(device, dtype, pages=PAGES):
    layers = workloads.moe_stack(2, device, seed=5, attention=True, cfg=CFG)
    gen = torch.Generator(device=device).manual_seed(11)
    lin = workloads._q8(VOCAB, CFG["hidden"], device, gen)
    emb = workloads._q8(VOCAB, CFG["hidden"], device, gen)   # untied: a tied one repeats its token
    d = workloads.DecodeStack(layers, quant.EschaQ8Embedding(emb._w8, (emb._scale.float() * 16).half()),
                              quant.EschaQ8Head(lin._w8, lin._scale), B, pages, PAGE, 6 * PAGE, dtype)
    d.free_pages.copy_(torch.randperm(pages, device=device, generator=gen))
    d.tokens.copy_(torch.tensor([1, 2, 3], device=device))
    return d


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_replayed_steps_equal_eager_ones(cuda, dtype):
    gen = torch.Generator(device=cuda).manual_seed(3)
    us = torch.rand((STEPS, B), device=cuda, generator=gen)
    settings = (0.9, 50, 0.95)
    eager, runs = stack(cuda, dtype), []
    for u in us:
        runs.append(eager.step(u, *settings).clone())
        assert eager.refused.item() == 0
    assert eager.lengths.tolist() == [STEPS] * B and eager.taken.item() == B * -(-STEPS // PAGE)
    assert len({tuple(t.tolist()) for t in runs}) > STEPS // 2      # it does not stand still

    graphed = stack(cuda, dtype)
    saved = [t.clone() for t in graphed.state()]
    u = torch.zeros(B, device=cuda)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graphed.step(u, *settings)                                  # sizes workspaces
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        graphed.step(u, *settings)
    for t, s in zip(graphed.state(), saved):
        t.copy_(s)
    for c in graphed.caches:
        for a in c.arrays():
            a.zero_()
    for now, want in zip(us, runs):
        u.copy_(now)
        graph.replay()
        assert torch.equal(graphed.tokens, want)
    for a, b in zip(eager.caches, graphed.caches):
        assert all(torch.equal(x, y) for x, y in zip(a.arrays(), b.arrays()))


def test_requests_without_a_page_keep_their_length(cuda):
    """Five pages for three requests: when all have filled one, only two more are served."""
    d = stack(cuda, torch.float16, pages=5)
    u = torch.full((B,), 0.5, device=cuda)
    for step in range(20):
        d.step(u, 0.9)
    # 16 tokens each in the first three pages, then two pages more: requests 0 and 1
    assert d.lengths.tolist() == [20, 20, 16] and d.refused.item() == 1 and d.taken.item() == 5


def test_layer_attends_to_its_history(cuda):
    """The layer's attention against a plain one over the projections of every earlier input."""
    d = stack(cuda, torch.float16)
    one = torch.ones(B, dtype=torch.int32, device=cuda)
    layer, cache = d.layers[0], d.caches[0]
    gen = torch.Generator(device=cuda).manual_seed(9)
    ks, vs = [], []
    for step in range(20):
        x = torch.randn((B, CFG["hidden"]), device=cuda, generator=gen).half()
        plan = paged.plan_pages(d.table, d.lengths, one, d.free_pages, d.taken, page_size=PAGE, n_pages=PAGES,
                                rows=B)
        got = layer.attend(x, cache, d.table, plan)
        q, k, v = (lin(x).double().view(B, -1, 64) for lin in (layer.q, layer.k, layer.v))
        ks.append(k)
        vs.append(v)
        k, v = (torch.stack(y, 2).repeat_interleave(2, 1) for y in (ks, vs))     # [B, 4, n, 64]
        s = (k @ q[..., None])[..., 0] / 8
        p = torch.softmax(s, -1)
        want = (p[..., None, :] @ v)[..., 0, :]
        # half a step of the output, 64 products per score in 32 bits (2^-23 a step, the
        # magnitudes' sum as bound), exp2 good to 2^-21, 16-bit weight pairs to 2^-17
        mag = (k.abs() @ q.abs()[..., None]).amax() / 8
        tol = 2.0**-11 * want.abs() + (2 * (70 * 2.0**-23 * mag + 2.0**-20) + 2.0**-16) * \
            (p[..., None, :] @ v.abs())[..., 0, :] + 2.0**-24
        assert bool(((got.double().view_as(want) - want).abs() <= tol).all())
        out = layer.decode(x, cache, d.table, plan)      # stores the same rows again
        assert torch.equal(out, layer.block(torch.add(x, layer.o(got), alpha=0.01)))
        d.lengths, d.taken = plan.ends, plan.head
