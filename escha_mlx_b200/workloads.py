"""Synthetic, device-resident layer stacks with the shapes of the published
benchmark configurations (random code bits, |N(0, 0.02)| + 1e-3 scales with random
signs, random int8 weights): there are no checkpoints here, and a random code
stream decodes with exactly the same instruction and byte counts as a trained one.

* ``MoeLayer`` -- one 35B-A3B-class MoE decode layer: 256 routed 2-bit experts
  (gate_up 2048 -> 1024, down 512 -> 2048), top-8 softmax routing, one int8 shared
  expert, optionally preceded by the int8 attention projections of the full
  decode step (16 query heads, 2 key/value heads, head size 256).
* ``moe_stack`` -- several such layers with distinct weights, so that a pass over
  the stack never finds a layer's bytes in L2.
* ``DecodeStack`` -- the stack's decode step end to end, with paged attention,
  vocabulary head and sampling.
"""
from __future__ import annotations

from typing import TYPE_CHECKING

import numpy as np
import torch

from . import moe, quant
from .models.qwen3_5_moe import EschaSparseMoeBlock

if TYPE_CHECKING:
    from . import paged

MOE_35B = dict(hidden=2048, inter=512, experts=256, top_k=8, K_gate_up=2, K_down=2,
               q_heads=16, kv_heads=2, head_dim=256)


def _signed_scale(shape, device, gen) -> torch.Tensor:
    scale = torch.randn(shape, device=device, generator=gen).abs() * 0.02 + 1e-3
    sign = torch.randint(0, 2, shape, device=device, generator=gen).float() * 2 - 1
    return (scale * sign).half().float()      # f16-representable, held as f32


def _experts(E, ic, oc, k, device, gen) -> moe.EschaExperts:
    code = torch.randint(-2**31, 2**31 - 1, (E, ic // 16, oc // 16, 8 * k), dtype=torch.int32,
                         device=device, generator=gen)
    return moe.EschaExperts(code, _signed_scale((E, ic), device, gen),
                            _signed_scale((E, oc), device, gen))


def _q8(n, kd, device, gen) -> quant.EschaQ8Linear:
    w8 = torch.randint(-127, 128, (n, kd), dtype=torch.int8, device=device, generator=gen)
    # uniform int8 has rms ~73: scales near 1 / (73 sqrt(kd)) keep the output at the
    # input's magnitude, so activations stay in range through a stack of layers
    scale = ((torch.rand((n,), device=device, generator=gen) + 0.5) / (73.0 * kd ** 0.5)).half()
    return quant.EschaQ8Linear(w8, scale)


class MoeLayer(torch.nn.Module):
    """One decode layer's projections on this path: [int8 q/k/v/o] + the MoE block.

    ``forward`` leaves attention itself out: the o projection consumes the q projection's
    output so that the four int8 linears run with their real shapes and dependencies.
    ``decode`` is the same layer with its attention, over a paged cache.
    """

    def __init__(self, device, gen, cfg=MOE_35B, attention: bool = False,
                 expert_range: tuple[int, int] | None = None, gen_experts=None,
                 peer_group=None) -> None:
        """``gen`` draws everything every rank replicates (router, shared expert, int8
        projections) and must be seeded alike on all ranks; ``gen_experts`` draws this
        rank's expert shard."""
        super().__init__()
        H, I, E = cfg["hidden"], cfg["inter"], cfg["experts"]
        lo, hi = expert_range or (0, E)
        self._e_lo, self._e_hi = lo, hi
        ge = gen_experts or gen
        gu = _experts(hi - lo, H, 2 * I, cfg["K_gate_up"], device, ge)
        dn = _experts(hi - lo, I, H, cfg["K_down"], device, ge)
        cpu = np.random.default_rng(int(torch.randint(0, 2**31 - 1, (1,), device=device,
                                                      generator=gen).item()))
        gate_w = (cpu.standard_normal((E, H)) * 0.5).astype(np.float16)
        shg_w = (cpu.standard_normal((H,)) * 0.05).astype(np.float16)
        shared = {}
        for name, (n, kd) in (("gate", (I, H)), ("up", (I, H)), ("down", (H, I))):
            lin = _q8(n, kd, device, gen)
            shared[f"{name}_w8"], shared[f"{name}_scale"] = lin._w8, lin._scale
        self.block = EschaSparseMoeBlock(H, E, cfg["top_k"], gu, dn, gate_w, shg_w, shared,
                                         expert_range=expert_range, peer_group=peer_group)
        self.attention = attention
        if attention:
            qd, kvd = cfg["q_heads"] * cfg["head_dim"], cfg["kv_heads"] * cfg["head_dim"]
            self.q, self.k, self.v = _q8(qd, H, device, gen), _q8(kvd, H, device, gen), \
                _q8(kvd, H, device, gen)
            self.o = _q8(H, qd, device, gen)
            self._kv_heads, self._head_dim = cfg["kv_heads"], cfg["head_dim"]
        self.expert_bytes = (H * 2 * I * cfg["K_gate_up"] + I * H * cfg["K_down"]) // 8
        self.int8_bytes = 3 * H * I + (2 * H * (qd + kvd) if attention else 0)
        self.router_bytes = 2 * E * H

    def _attention_projections(self, x: torch.Tensor) -> torch.Tensor:
        if not self.attention:
            return x
        q, _, _ = quant.project_many_q8([self.q, self.k, self.v], x)   # one launch, as one input
        return torch.add(x, self.o(q), alpha=0.01)   # residual keeps the scale bounded

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.block(self._attention_projections(x))

    def new_cache(self, n_pages: int, page_size: int, dtype=torch.float16) -> paged.PagedCache:
        """An empty paged cache of this layer's key/value heads."""
        from . import paged
        return paged.PagedCache(n_pages, page_size, self._kv_heads, self._head_dim, dtype,
                                self.k._w8.device)

    def attend(self, x: torch.Tensor, cache: paged.PagedCache, table: torch.Tensor,
               plan: paged.PagePlan) -> torch.Tensor:
        """Attention of one new token per request: int8 q/k/v projections of ``x`` [B, hidden]
        in one launch, the new keys and values stored in ``cache``, attention over it.  Returns
        the heads side by side, [B, q_heads * head_dim]."""
        q, k, v = quant.project_many_q8([self.q, self.k, self.v], x)
        heads = (lambda y: y.unflatten(1, (-1, self._head_dim)))
        cache.append(heads(k), heads(v), plan.slots)
        return cache.attend(heads(q), table, plan.ends).flatten(1)

    def decode(self, x: torch.Tensor, cache: paged.PagedCache, table: torch.Tensor,
               plan: paged.PagePlan) -> torch.Tensor:
        """The layer with its attention, for one new token per request (``plan``: the step's
        ``paged.plan_pages`` with ``rows`` = B); otherwise as ``forward``."""
        y = self.o(self.attend(x, cache, table, plan))
        return self.block(torch.add(x, y, alpha=0.01))

    def routed_experts(self, x: torch.Tensor) -> int:
        """Distinct experts of this rank's shard that the rows of ``x`` are routed to
        (host count, for byte accounting)."""
        xb = self._attention_projections(x)
        ids, _ = self.block.route(xb.reshape(-1, xb.shape[-1]).half())
        u = torch.unique(ids)
        return int(((u >= self._e_lo) & (u < self._e_hi)).sum().item())


def moe_stack(n_layers: int, device, seed: int = 1234, attention: bool = False,
              expert_range: tuple[int, int] | None = None, rank: int = 0,
              cfg=MOE_35B, peer_group=None) -> list[MoeLayer]:
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    gen_experts = torch.Generator(device=device)
    gen_experts.manual_seed(seed + 1 + rank)
    return [MoeLayer(device, gen, cfg, attention, expert_range, gen_experts, peer_group)
            for _ in range(n_layers)]


class DecodeStack:
    """The decode step of a layer stack end to end, one new token per request and call: page plan,
    int8 embedding, the layers with attention over their paged caches (``MoeLayer.decode``) and a
    residual and RMS norm after each as in the benchmark's step, vocabulary head, sampling.

    Everything a step changes (page table, lengths, position in the free list, tokens, caches) is
    device state of this object, updated in place and in stream order, so a step can be captured
    in a CUDA graph and replayed.  Requests that find no free page are refused by the plan and
    keep their length; ``refused`` holds their number after a step.
    """

    def __init__(self, layers: list[MoeLayer], embed: quant.EschaQ8Embedding, head: quant.EschaQ8Head,
                 batch: int, n_pages: int, page_size: int, max_tokens: int,
                 cache_dtype=torch.float16) -> None:
        self.layers, self.embed, self.head = layers, embed, head
        dev = head._w8.device
        self.page_size, self.n_pages = page_size, n_pages
        self.caches = [layer.new_cache(n_pages, page_size, cache_dtype) for layer in layers]
        i32 = dict(dtype=torch.int32, device=dev)
        self.table = torch.full((batch, -(-max_tokens // page_size)), -1, **i32)
        self.free_pages = torch.arange(n_pages, **i32)
        self.taken = torch.zeros(1, **i32)
        self.lengths = torch.zeros(batch, **i32)
        self.refused = torch.zeros(1, **i32)
        self.tokens = torch.zeros(batch, dtype=torch.int64, device=dev)
        self._one = torch.ones(batch, **i32)

    def state(self) -> list[torch.Tensor]:
        """What a step changes apart from the caches."""
        return [self.table, self.taken, self.lengths, self.refused, self.tokens]

    def step(self, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
        """One token per request from ``uniforms`` [batch]; the settings as in
        ``sampling.sample``.  Returns (and keeps) the tokens [batch]."""
        from . import paged
        plan = paged.plan_pages(self.table, self.lengths, self._one, self.free_pages, self.taken,
                                page_size=self.page_size, n_pages=self.n_pages,
                                rows=self.tokens.shape[0])
        x = self.embed(self.tokens)
        for layer, cache in zip(self.layers, self.caches):
            x = x + layer.decode(x, cache, self.table, plan)
            x = torch.nn.functional.rms_norm(x, (x.shape[-1],), eps=1e-6)
        self.tokens.copy_(self.head.sample(x, uniforms, temperature, top_k, top_p, min_p))
        self.lengths.copy_(plan.ends)
        self.taken.copy_(plan.head)
        self.refused.copy_(plan.refused)
        return self.tokens
