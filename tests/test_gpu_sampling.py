"""Sampling against the definition in 64 bits, row by row."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from escha_mlx_b200 import graphs, quant, sampling

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def kept_weights(x, t, k, p, m):
    """Kept weight of each token (numpy, 64 bits), by the definition; None: nothing to choose."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return None
    if not t > 0:
        w = np.zeros_like(x)
        w[int(np.argmax(x == top))] = 1.0
        return w
    d = np.where(x == top, 0.0, (np.where(x == top, 0.0, x) - (0.0 if np.isinf(top) else top)) / t)
    if np.isinf(top):
        d = np.where(x == top, 0.0, -np.inf)
    w = np.where(d < -30.0, 0.0, np.exp(d))
    order = np.lexsort((np.arange(len(x)), -x))
    ws = w[order]
    if 0 < k < len(x):
        ws[k:] = 0.0
    if p < 1:
        before = np.cumsum(ws) - ws
        cut = before >= max(p, 0.0) * ws.sum()
        cut[0] = False
        ws = np.where(cut, 0.0, ws)
    if m > 0:
        ws = np.where(ws >= min(m, 1.0), ws, 0.0)
    out = np.zeros_like(w)
    out[order] = ws
    return out


def check(tokens, logits, uniforms, t, k, p, m):
    """Each token is the definition's.  The cumulative weights here are sums of rounded
    64-bit numbers; where the target is within 2^-40 of a border either side is right."""
    x = logits.float().cpu().numpy()
    b, v = x.shape
    full = lambda a: np.broadcast_to(a.cpu().numpy() if isinstance(a, torch.Tensor) else a, (b,))
    t, k, p, m = (full(np.float32(a) if isinstance(a, float) else a) for a in (t, k, p, m))
    u, got = uniforms.cpu().numpy().astype(np.float64), tokens.cpu().numpy()
    for i in range(b):
        w = kept_weights(x[i], np.float64(t[i]), int(k[i]), np.float64(p[i]), np.float64(m[i]))
        if w is None:
            assert got[i] == -1
            continue
        cum = np.cumsum(w)
        target = u[i] * cum[-1]
        want = int(np.searchsorted(cum, target, side="right"))
        want = min(want, int(np.nonzero(w)[0][-1]))
        if got[i] != want:
            g = int(got[i])
            assert 0 <= g < v and w[g] > 0, (i, g, want)
            lo, hi = min(g, want), max(g, want)
            assert abs(cum[hi - 1] - target) <= 2.0**-40 * cum[-1] and w[lo + 1:hi].sum() <= 2.0**-40, \
                (i, g, want)


def logits_of(cuda, b, v, kind, seed=0, spread=2.0):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    x = spread * torch.randn((b, v), device=cuda, generator=gen)
    up = torch.randint(0, v, (b, min(v, 40)), device=cuda, generator=gen)
    x.scatter_add_(1, up, 6 + 4 * torch.rand(up.shape, device=cuda, generator=gen))
    return x.to(DT[kind]), torch.rand((b,), device=cuda, generator=gen)


SETTINGS = [
    (1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05),
    (0.8, 40, 0.95, 0.02), (1.3, 1, 0.5, 0.5), (0.0, 5, 0.5, 0.1), (1.5, 1000, 0.99, 0.0),
    (2.0, 3000, 0.999, 0.0), (3.0, 0, 0.97, 0.0), (3.0, 5000, 1.0, 0.0), (1.0, 0, 0.0, 0.0),
    (1.0, 0, 0.3, 1.0), (0.05, 10, 0.9, 0.0), (20.0, 0, 0.9, 0.0), (100.0, 20000, 0.6, 0.001),
    (1.0, 0, 0.9, 0.05), (3.0, 0, 0.95, 0.3), (20.0, 0, 0.8, 0.5), (float("nan"), 3, 0.5, 0.1), (1e-30, 0, 0.9, 0.0), (1e30, 0, 0.9, 0.0), (1.0, -3, 2.0, -1.0),
]


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("v", [1, 2, 31, 1000, 4096, 4097, 50257, 151936])
@pytest.mark.parametrize("setting", SETTINGS, ids=str)
def test_sample_matches_the_definition(cuda, kind, v, setting):
    x, u = logits_of(cuda, 3, v, kind, seed=v)
    got = sampling.sample(x, u, *setting)
    assert got.dtype == torch.int64
    check(got, x, u, *setting)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("setting", [(1.0, 0, 1.0, 0.0), (1.0, 7000, 1.0, 0.0), (1.0, 0, 0.4, 0.0),
                                     (1.0, 9000, 0.5, 0.0), (1.0, 9000, 0.99999, 0.0),
                                     (0.5, 3, 0.9, 0.0), (1.0, 0, 1.0, 1.0)], ids=str)
@pytest.mark.parametrize("levels", [1, 2, 3, 40])
def test_ties_go_to_the_lowest_index(cuda, kind, setting, levels):
    """Rows of few distinct values: cuts fall among thousands of equal tokens."""
    gen = torch.Generator(device=cuda).manual_seed(levels)
    x = torch.randint(0, levels, (4, 20000), device=cuda, generator=gen).to(DT[kind]) / 64
    u = torch.tensor([0.0, 0.25, 0.6180339, 0.99999994], device=cuda)
    check(sampling.sample(x, u, *setting), x, u, *setting)


@pytest.mark.parametrize("v", [200, 30000])
def test_masked_and_unusual_logits(cuda, v):
    x, u = logits_of(cuda, 9, v, "f32", seed=1)
    x[0] = float("-inf")                                  # nothing to choose from
    x[1, :] = float("-inf"); x[1, v - 2] = -3.0           # one token left
    x[2, ::2] = float("-inf")
    x[3, 5:] = float("nan")
    x[4, 7] = x[4, 11] = float("inf")
    x[5] = float("nan")
    x[6] = torch.finfo(torch.float32).min                 # all at the type's lowest value
    x[7, 1:] = torch.finfo(torch.float32).min
    x[8] = 0.0; x[8, ::3] = -0.0                          # signed zeros tie
    for s in SETTINGS[:8]:
        check(sampling.sample(x, u, *s), x, u, *s)
    h = x.half()                                          # the lowest value becomes -inf
    for s in SETTINGS[:8]:
        check(sampling.sample(h, u, *s), h, u, *s)


def test_logits_at_the_ends_of_their_type(cuda):
    """Differences past the type's largest value, at temperatures that bring them back."""
    gen = torch.Generator(device=cuda).manual_seed(0)
    x = 6.6e38 * (torch.rand((4, 30000), device=cuda, generator=gen, dtype=torch.float64) - 0.5)
    x = x.float()
    u = torch.rand((4,), device=cuda, generator=gen)
    for s in ((1e38, 0, 1.0, 0.0), (1e38, 0, 0.7, 0.0), (5e37, 300, 1.0, 0.0), (1e37, 0, 0.9, 0.05),
              (3e38, 9000, 0.9, 0.0), (1.0, 0, 0.9, 0.0)):
        check(sampling.sample(x, u, *s), x, u, *s)


def test_settings_by_row(cuda):
    b, v = 40, 33000
    x, u = logits_of(cuda, b, v, "f16", seed=2)
    rng = np.random.default_rng(0)
    t = torch.tensor(rng.choice([0.0, 0.5, 1.0, 1.7], b)).float().to(cuda)
    k = torch.tensor(rng.choice([0, 1, 40, 900, v + 1, v, v - 1], b)).int().to(cuda)
    p = torch.tensor(rng.choice([1.0, 0.3, 0.9, 0.999], b)).float().to(cuda)
    m = torch.tensor(rng.choice([0.0, 0.05], b)).float().to(cuda)
    check(sampling.sample(x, u, t, k, p, m), x, u, t, k, p, m)
    got = sampling.sample(x.view(8, 5, v), u.view(8, 5), t, k, 0.9, m)
    assert got.shape == (8, 5)
    check(got.view(-1), x, u, t, k, 0.9, m)


def test_one_row_without_a_batch(cuda):
    x, u = logits_of(cuda, 2, 3001, "f16", seed=9)
    got = sampling.sample(x[1], u[1], 0.8, 50, 0.9)
    assert got.shape == () and got.item() == sampling.sample(x, u, 0.8, 50, 0.9)[1].item()


@pytest.mark.parametrize("b", [38, 511, 512, 513])
def test_long_rows_first(cuda, b):
    """More rows than the GPU holds at once, with settings of their own: every row's token is its
    own whatever order they run in."""
    v = 33000
    x, u = logits_of(cuda, 4, v, "f16", seed=b)
    x, u = x.repeat(-(-b // 4), 1)[:b], u.repeat(-(-b // 4))[:b]
    pick = torch.randint(0, 4, (b,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(b))
    t = torch.tensor([0.0, 0.7, 1.0, 1.5], device=cuda)[pick]
    k = torch.tensor([0, 40, 0, 2000], dtype=torch.int32, device=cuda)[pick]
    got = sampling.sample(x, u, t, k, 0.95, 0.0)
    for i in range(4):
        one = sampling.sample(x[:4], u[:4], [0.0, 0.7, 1.0, 1.5][i], [0, 40, 0, 2000][i], 0.95, 0.0)
        check(one, x[:4], u[:4], [0.0, 0.7, 1.0, 1.5][i], [0, 40, 0, 2000][i], 0.95, 0.0)
        mine = (pick == i).nonzero()[:, 0]
        assert torch.equal(got[mine], one[mine % 4])


def test_uniforms_at_their_ends(cuda):
    x, _ = logits_of(cuda, 4, 9000, "f32", seed=3)
    u = torch.tensor([0.0, 2.0**-24, 1 - 2.0**-24, 0.5], device=cuda)
    for s in SETTINGS[:6]:
        check(sampling.sample(x, u, *s), x, u, *s)


def test_rows_of_a_wider_matrix(cuda):
    x, u = logits_of(cuda, 6, 5003, "f16", seed=4)
    want = sampling.sample(x, u, 0.8, 50, 0.9, 0.0)
    wide = torch.full((6, 6001), 30.0, device=cuda).half()
    wide[:, 7:5010] = x
    assert torch.equal(sampling.sample(wide[:, 7:5010], u, 0.8, 50, 0.9, 0.0), want)
    assert torch.equal(sampling.sample(x.t().contiguous().t(), u, 0.8, 50, 0.9, 0.0), want)
    assert torch.equal(sampling.sample(x[:1].expand(6, -1), u, 0.8, 50, 0.9, 0.0),
                       sampling.sample(x[:1].repeat(6, 1), u, 0.8, 50, 0.9, 0.0))


def test_longest_rows(cuda):
    for kind in ("f16", "f32"):
        v = sampling.max_vocab(DT[kind])
        x, u = logits_of(cuda, 2, v, kind, seed=5)
        # at the last temperatures every token weighs as much as the largest
        for s in ((0.7, 50, 0.9, 0.0), (2.0, 0, 0.999, 0.0), (1.0, 0, 1.0, 0.0), (1e30, 0, 1.0, 0.0),
                  (1e30, 0, 0.97, 0.0), (1e30, v - 7, 1.0, 0.0)):
            check(sampling.sample(x, u, *s), x, u, *s)
        with pytest.raises(ValueError, match="V="):
            sampling.sample(torch.zeros((1, v + 1), dtype=DT[kind], device=cuda), u[:1])


def test_reproducible_on_streams_and_in_graphs(cuda):
    x, u = logits_of(cuda, 64, 151936, "f16", seed=6)
    want = sampling.sample(x, u, 1.2, 0, 0.98, 0.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [sampling.sample(x, u, 1.2, 0, 0.98, 0.0) for _ in range(4)]
    outs += [sampling.sample(x, u, 1.2, 0, 0.98, 0.0) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    call = graphs.GraphedCall(lambda a, b: sampling.sample(a, b, 1.2, 0, 0.98, 0.0), [x, u])
    for seed in (7, 8):
        x, u = logits_of(cuda, 64, 151936, "f16", seed=seed)
        got = call(x, u).clone()
        assert torch.equal(got, sampling.sample(x, u, 1.2, 0, 0.98, 0.0))


def test_frequencies(cuda):
    """Evenly spread uniforms draw each token as often as its weight says."""
    n, v = 4096, 50
    x = torch.linspace(-2, 2, v, device=cuda)[torch.randperm(v, device=cuda)]
    u = (torch.arange(n, device=cuda).float() + 0.5) / n
    got = torch.bincount(sampling.sample(x.expand(n, v), u), minlength=v).double() / n
    # the count of an interval's points on an even grid is off by one at most
    assert float((got - torch.softmax(x.double(), 0)).abs().max()) <= 1.0 / n + 1e-9


def test_head_to_token(cuda):
    rng = np.random.default_rng(0)
    head = quant.make_head(rng.integers(-127, 128, (1000, 128), dtype=np.int8),
                           (rng.random(1000) * 0.01).astype(np.float32), device=cuda)
    h = torch.randn((5, 128), device=cuda).half()
    u = torch.rand(5, device=cuda)
    logits = head(h)
    got = head.sample(h, u, 0.9, 20, 0.9)
    assert torch.equal(got, sampling.sample(logits, u, 0.9, 20, 0.9))
    check(got, logits, u, 0.9, 20, 0.9, 0.0)


def test_refusals(cuda):
    x = torch.zeros((2, 8), device=cuda)
    u = torch.zeros(2, device=cuda)
    for bad, text in (((x.cpu(), u), "CUDA"), ((x.double(), u), "logits"), ((x, u[:1]), "uniforms"),
                      ((x, u.double()), "uniforms"), ((x, u.cpu()), "uniforms"),
                      ((x, u, u.double()), "temperature"), ((x, u, 1.0, u), "top_k"),
                      ((x, u, 1.0, 0, u[:1]), "top_p"), ((x, u, 1.0, 0, 1.0, u.cpu()), "min_p"),
                      ((x[:, :0], u), "shape")):
        with pytest.raises(ValueError, match=text):
            sampling.sample(*bad)
    assert sampling.sample(x[:0], u[:0]).shape == (0,)


def test_a_nucleus_that_the_counts_misplace(cuda):
    """Three quarters of the weight in tokens equal to the largest (at the top of their bin), the
    rest thinly spread at the bottom of the others: the bins' counts put a cut behind the first
    several bins from where it is, and the exact weights of all bins have to find it."""
    per_nat = 1023 / 30.25                     # bins of (max x - x) / T per unit
    spread = np.concatenate([np.full(round(1500 / 190 * np.exp((b + 0.995) / per_nat)), b)
                             for b in range(30, 220)])
    x = np.concatenate([np.zeros(4500), -(spread + 0.995) / per_nat])
    x = np.random.default_rng(0).permutation(x)
    x = torch.from_numpy(x).float().to(cuda).repeat(3, 1)
    u = torch.tensor([0.1, 0.7, 0.999], device=cuda)
    for p in (0.76, 0.77, 0.8, 0.9):
        for m in (0.0, 0.01):
            check(sampling.sample(x, u, 1.0, 0, p, m), x, u, 1.0, 0, p, m)
            check(sampling.sample(x, u, 1.0, 150000, p, m), x, u, 1.0, 150000, p, m)
