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


class Decoder:
    def __init__(self, device, dtype):
        self.layers = workloads.moe_stack(2, device, seed=5, attention=True, cfg=CFG)
        gen = torch.Generator(device=device).manual_seed(11)
        lin = workloads._q8(VOCAB, CFG["hidden"], device, gen)
        self.head = quant.EschaQ8Head(lin._w8, lin._scale)
        self.embed = quant.EschaQ8Embedding(lin._w8, (lin._scale.float() * 16).half())
        self.caches = [x.new_cache(PAGES, PAGE, dtype) for x in self.layers]
        i32 = dict(dtype=torch.int32, device=device)
        self.table = torch.full((B, 6), -1, **i32)
        self.free = torch.randperm(PAGES, device=device, generator=gen).to(torch.int32)
        self.lens, self.pos = torch.zeros(B, **i32), torch.zeros(1, **i32)
        self.one = torch.ones(B, **i32)
        self.tokens = torch.tensor([1, 2, 3], device=device)
        self.u = torch.zeros(B, device=device)

    def step(self):
        plan = paged.plan_pages(self.table, self.lens, self.one, self.free, self.pos, page_size=PAGE,
                                n_pages=PAGES, rows=B)
        x = self.embed(self.tokens)
        for layer, cache in zip(self.layers, self.caches):
            x = torch.nn.functional.rms_norm(layer.decode(x, cache, self.table, plan),
                                             (CFG["hidden"],), eps=1e-6)
        self.tokens.copy_(self.head.sample(x, self.u, 0.9, 50, 0.95))
        self.lens.copy_(plan.ends)
        self.pos.copy_(plan.head)
        return plan


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_replayed_steps_equal_eager_ones(cuda, dtype):
    gen = torch.Generator(device=cuda).manual_seed(3)
    us = torch.rand((STEPS, B), device=cuda, generator=gen)
    eager, runs = Decoder(cuda, dtype), []
    for u in us:
        eager.u.copy_(u)
        plan = eager.step()
        assert plan.refused.item() == 0
        runs.append(eager.tokens.clone())
    assert eager.lens.tolist() == [STEPS] * B and eager.pos.item() == B * -(-STEPS // PAGE)
    assert len({tuple(t.tolist()) for t in runs}) > STEPS // 2      # it does not stand still

    graphed = Decoder(cuda, dtype)
    saved = [t.clone() for t in (graphed.table, graphed.lens, graphed.pos, graphed.tokens)]
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graphed.step()                                              # sizes workspaces
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        graphed.step()
    for t, s in zip((graphed.table, graphed.lens, graphed.pos, graphed.tokens), saved):
        t.copy_(s)
    for c in graphed.caches:
        for a in c.arrays():
            a.zero_()
    for u, want in zip(us, runs):
        graphed.u.copy_(u)
        graph.replay()
        assert torch.equal(graphed.tokens, want)
    for a, b in zip(eager.caches, graphed.caches):
        assert all(torch.equal(x, y) for x, y in zip(a.arrays(), b.arrays()))


def test_layer_attends_to_its_history(cuda):
    """The layer's attention against a plain one over the projections of every earlier input."""
    d = Decoder(cuda, torch.float16)
    layer, cache = d.layers[0], d.caches[0]
    gen = torch.Generator(device=cuda).manual_seed(9)
    ks, vs = [], []
    for step in range(20):
        x = torch.randn((B, CFG["hidden"]), device=cuda, generator=gen).half()
        plan = paged.plan_pages(d.table, d.lens, d.one, d.free, d.pos, page_size=PAGE, n_pages=PAGES,
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
        d.lens, d.pos = plan.ends, plan.head
