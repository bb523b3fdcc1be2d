"""Page plans, stores into the paged cache and attention over it, against plain
implementations in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from escha_mlx_b200 import graphs, paged

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}


def ints(a, dev):
    return torch.from_numpy(np.asarray(a, dtype=np.int32).copy()).to(dev)


# ---------------------------------------------------------------------------------------------
# plans

def plan_reference(table, lengths, added, free, head, page, n_pages, rows):
    """The definition, request by request."""
    table = table.copy()
    b, w = table.shape
    avail = len(free) - head if 0 <= head <= len(free) else 0
    slots, pos = np.full(rows, -1, np.int64), np.zeros(rows, np.int64)
    starts, ends = [0], []
    first = before = took = refused = 0
    for i in range(b):
        ln, ad = int(lengths[i]), int(added[i])
        valid = ln >= 0 and ad >= 0 and ln + ad <= w * page and first + max(ad, 0) <= rows
        have, need = -(-ln // page), 0
        if valid:
            need = -(-(ln + ad) // page) - have
        fine = valid and (need == 0 or before + need <= avail)
        if fine:
            for j in range(need):
                table[i, have + j] = free[head + before + j]
            took += need
            for r in range(ad):
                p = ln + r
                pg = int(table[i, p // page])
                pos[first + r] = p
                slots[first + r] = pg * page + p % page if 0 <= pg < n_pages else -1
        else:
            refused += 1
        ends.append(ln + ad if fine else min(max(ln, 0), w * page))
        before += need
        first += max(ad, 0)
        starts.append(min(first, 2**31 - 1))
    return dict(table=table, slots=slots, positions=pos, starts=np.array(starts),
                ends=np.array(ends), head=np.array([head + took]), refused=np.array([refused]))


def check_plan(cuda, table, lengths, added, free, head, page, n_pages, rows):
    t = ints(table, cuda)
    got = paged.plan_pages(t, ints(lengths, cuda), ints(added, cuda), ints(free, cuda),
                           ints([head], cuda), page_size=page, n_pages=n_pages, rows=rows)
    want = plan_reference(np.asarray(table), lengths, added, free, head, page, n_pages, rows)
    assert np.array_equal(t.cpu().numpy(), want["table"])
    for name in paged.PagePlan._fields:
        assert np.array_equal(getattr(got, name).cpu().numpy(), want[name]), name
    return want


def make_plan(rng, b, page, most_len, most_new, spare=3):
    lengths = rng.integers(0, most_len + 1, b)
    added = rng.integers(0, most_new + 1, b)
    w = int((-(-(lengths + added) // page)).max()) + spare
    used = -(-lengths // page)
    n_pages = int(used.sum()) + int((added // page + 2).sum())
    ids = rng.permutation(n_pages)
    table, at = np.full((b, w), -1, np.int32), 0
    for i in range(b):
        table[i, :used[i]] = ids[at:at + used[i]]
        at += used[i]
    return table, lengths, added, ids[at:], n_pages


@pytest.mark.parametrize("b,page,most_len,most_new", [
    (1, 16, 0, 1), (1, 16, 40, 1), (3, 256, 700, 5), (32, 16, 500, 1), (257, 32, 300, 40),
    (1000, 64, 2000, 3), (4096, 16, 64, 2)])
def test_plan_matches_the_definition(cuda, b, page, most_len, most_new):
    rng = np.random.default_rng(b)
    table, lengths, added, free, n_pages = make_plan(rng, b, page, most_len, most_new)
    want = check_plan(cuda, table, lengths, added, free, 0, page, n_pages, int(added.sum()) + 5)
    assert want["refused"][0] == 0


@pytest.mark.parametrize("left", [0, 1, 7, 20])
def test_plan_refuses_what_the_free_list_cannot_serve(cuda, left):
    rng = np.random.default_rng(left)
    table, lengths, added, free, n_pages = make_plan(rng, 40, 16, 100, 30)
    head = len(free) - left
    want = check_plan(cuda, table, lengths, added, free, head, 16, n_pages, int(added.sum()))
    assert want["refused"][0] > 0


def test_plan_refuses_bad_requests_one_by_one(cuda):
    rng = np.random.default_rng(5)
    table, lengths, added, free, n_pages = make_plan(rng, 24, 32, 200, 20)
    lengths[3], added[5], lengths[7] = -4, -1, 32 * table.shape[1] + 1
    added[9] = 2**31 - 1
    lengths[11] = added[13] = -2**31
    table[2, 0] = n_pages                     # a page that does not exist
    rows = int(np.clip(added, 0, 100).sum())
    check_plan(cuda, table, lengths, added, free, 0, 32, n_pages, rows)
    check_plan(cuda, table, np.zeros_like(lengths), np.minimum(added, 20), free, 0, 32, n_pages, 9)
    for head in (-1, len(free) + 1):
        check_plan(cuda, table, lengths, added, free, head, 32, n_pages, rows)
    check_plan(cuda, table, lengths, added, np.zeros(0, np.int32), 0, 32, n_pages, rows)
    check_plan(cuda, table, np.abs(lengths % 50), np.zeros_like(added), free, 0, 32, n_pages, 0)


# ---------------------------------------------------------------------------------------------
# stores

def quantised(x):
    """Codes and 32-bit scales by the definition; x float64 [..., D]."""
    top = np.abs(x).max(-1)
    scale = (top / 127.0).astype(np.float32)
    by = np.where(scale > 0, scale, 1.0).astype(np.float64)
    return np.clip(np.rint(x / by[..., None]), -127, 127).astype(np.int8), scale


@pytest.mark.parametrize("cache,kind", [("f16", "f16"), ("bf16", "bf16"), ("int8", "f16"),
                                        ("int8", "bf16")])
@pytest.mark.parametrize("t,h,d,page", [(1, 1, 64, 16), (7, 2, 256, 16), (33, 3, 128, 64),
                                        (130, 5, 64, 256), (700, 2, 128, 32)])
def test_append_stores_rows_at_their_slots(cuda, cache, kind, t, h, d, page):
    gen = torch.Generator(device=cuda).manual_seed(t)
    n_pages = -(-t // page) + 2
    pc = paged.PagedCache(n_pages, page, h, d, DT[cache], cuda)
    for a in pc.arrays():
        a.fill_(3)
    merged = torch.randn((t, 2 * h * d + 8), device=cuda, generator=gen).to(DT[kind])
    k = merged[:, :h * d].unflatten(1, (h, d))
    v = merged[:, h * d:2 * h * d].unflatten(1, (h, d))
    v[0, 0] = 0.0                                     # a row without a scale
    slots = torch.randperm(n_pages * page, device=cuda, generator=gen)[:t].to(torch.int32)
    if t > 5:
        slots[2], slots[4] = -1, n_pages * page       # skipped
    pc.append(k, v, slots)
    s = slots.cpu().numpy()
    keep = (s >= 0) & (s < n_pages * page)
    for name, rows in (("k", k), ("v", v)):
        x = rows.double().cpu().numpy()
        want = np.full((n_pages * page, h, d), 3.0)
        got = getattr(pc, name).cpu().double().numpy().transpose(0, 2, 1, 3).reshape(want.shape)
        if cache == "int8":
            codes, scale = quantised(x)
            want_scale = np.full((n_pages * page, h), 3.0)
            want[s[keep]], want_scale[s[keep]] = codes[keep], scale[keep]
            got_scale = getattr(pc, name + "_scale").cpu().numpy().transpose(0, 2, 1)
            assert np.array_equal(got_scale.reshape(want_scale.shape), want_scale)
        else:
            want[s[keep]] = x[keep]
        assert np.array_equal(got, want)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_append_codes_at_every_magnitude(cuda, kind):
    """Codes and scales equal the definition's from the smallest denormals to the largest values,
    ties between codes among them."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    low, high = (-24, 15) if kind == "f16" else (-133, 127)
    x = torch.randn((64 * 16, 2, 64), device=cuda, generator=gen, dtype=torch.float64)
    x[::3] = torch.randint(-254, 255, x[::3].shape, device=cuda, generator=gen).double() / 2
    x[::3, :, 0] = 127.0                                       # scale 1: halves are ties
    by = torch.randint(low, high, (x.shape[0], 2, 1), device=cuda, generator=gen)
    top = x.abs().amax(-1, keepdim=True)
    x = torch.where(torch.arange(x.shape[0], device=cuda)[:, None, None] % 3 == 0,
                    x * torch.exp2((by.clamp(max=high - 8)).double()), x / top * 1.98 * torch.exp2(by.double()))
    x = x.to(DT[kind])
    pc = paged.PagedCache(64, 16, 2, 64, torch.int8, cuda)
    pc.append(x, x.flip(0), torch.arange(64 * 16, device=cuda, dtype=torch.int32))
    for name, rows in (("k", x), ("v", x.flip(0))):
        codes, scale = quantised(rows.double().cpu().numpy())
        got = getattr(pc, name).cpu().numpy().transpose(0, 2, 1, 3).reshape(codes.shape)
        got_scale = getattr(pc, name + "_scale").cpu().numpy().transpose(0, 2, 1).reshape(scale.shape)
        assert np.array_equal(got_scale, scale)
        assert np.array_equal(got, codes)


def test_append_takes_any_stride_and_alignment(cuda):
    h, d, t = 2, 64, 9
    gen = torch.Generator(device=cuda).manual_seed(0)
    base = torch.randn((t * h * d * 2 + 3), device=cuda, generator=gen).half()
    odd = base[1:1 + t * h * d].view(t, h, d)                      # 2-byte aligned
    turned = base[:t * h * d].view(h, t, d).transpose(0, 1)        # heads outermost
    flipped = base[:t * h * d].view(t, d, h).transpose(1, 2)       # channels not dense
    slots = torch.arange(t, device=cuda, dtype=torch.int32)
    for k, v in ((odd, turned), (turned, flipped), (flipped, odd)):
        pc = paged.PagedCache(1, 16, h, d, torch.float16, cuda)
        pc.append(k, v, slots)
        assert torch.equal(pc.k[0, :, :t].transpose(0, 1), k)
        assert torch.equal(pc.v[0, :, :t].transpose(0, 1), v)
        assert not pc.k[0, :, t:].any()
    pc.append(odd[:0], odd[:0], slots[:0])                         # nothing


def test_append_more_rows_than_one_launch_numbers(cuda):
    """70000 rows of 1024 heads of 256 (one row, repeated): three launches; almost all skipped."""
    t, h, d = 70000, 1024, 256
    x = torch.randn((1, h, d), device=cuda).half()
    pc = paged.PagedCache(1, 16, h, d, torch.float16, cuda)
    slots = torch.full((t,), -1, dtype=torch.int32, device=cuda)
    at = [0, 32510, 32511, 32512, 32513, 65023, 65024, 69999]
    slots[torch.tensor(at, device=cuda)] = torch.arange(8, dtype=torch.int32, device=cuda)
    pc.append(x.expand(t, h, d), x.expand(t, h, d), slots)
    for c in (pc.k, pc.v):
        assert torch.equal(c[0, :, :8], x[0][:, None].expand(h, 8, d)) and not c[0, :, 8:].any()


def test_rows_that_are_not_finite_are_stored_as_nan(cuda):
    for kind in (torch.float16, torch.bfloat16):
        x = torch.ones((4, 1, 64), device=cuda, dtype=kind)
        x[1, 0, 5], x[2, 0, 7] = float("nan"), float("-inf")
        pc = paged.PagedCache(1, 16, 1, 64, torch.int8, cuda)
        pc.append(x, x, torch.arange(4, device=cuda, dtype=torch.int32))
        back = (pc.k.float() * pc.k_scale[..., None])[0, 0, :4]
        assert torch.isnan(back[1:3]).all() and torch.equal(back[[0, 3]], x.float()[[0, 3], 0])


# ---------------------------------------------------------------------------------------------
# attention

class Case:
    """Requests over a shuffled cache; unused slots hold NaN (codes: with NaN scales)."""

    def __init__(self, cuda, lens, kv_heads, group, d, page, cache, kind, seed=0, spare=1, mult=1.0):
        gen = torch.Generator(device=cuda).manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.lens, self.group, self.page, self.kind = list(lens), group, page, kind
        b = len(self.lens)
        each = [-(-n // page) for n in self.lens]
        w = max(max(each), 1) + spare
        n_pages = sum(each) + 2
        ids, at = rng.permutation(n_pages), 0
        self.table = np.full((b, w), -1, np.int32)
        there = torch.zeros((n_pages, page), dtype=torch.bool, device=cuda)
        for i, n in enumerate(each):
            self.table[i, :n] = ids[at:at + n]
            for j in range(n):
                there[ids[at + j], :min(page, self.lens[i] - j * page)] = True
            at += n
        shape = (n_pages, kv_heads, page, d)
        x = [torch.randn(shape, device=cuda, generator=gen).to(DT[kind]) for _ in range(2)]
        gone = ~there[:, None, :]
        self.values = []
        if cache == "int8":
            made = []
            for y in x:
                codes, scale = quantised(y.double().cpu().numpy())
                codes, scale = torch.from_numpy(codes).to(cuda), torch.from_numpy(scale).to(cuda)
                self.values.append(codes.double() * scale.double()[..., None])
                scale[gone.expand_as(scale)] = float("nan")
                made.append((codes, scale))
            self.cache = paged.PagedCache.from_tensors(made[0][0], made[1][0], made[0][1], made[1][1])
        else:
            for y in x:
                self.values.append(y.double())
                y[gone[..., None].expand_as(y)] = float("nan")
            self.cache = paged.PagedCache.from_tensors(*x)
        self.q = (mult * torch.randn((b, kv_heads * group, d), device=cuda, generator=gen)).to(DT[kind])
        self.t, self.l = ints(self.table, cuda), ints(self.lens, cuda)
        self.scale = d ** -0.5

    def want(self, lens=None, table=None):
        """Output in 64 bits and the bound of the kernel's error, by request."""
        out, tol = [], []
        table = self.table if table is None else table
        n_pages, h, page, d = self.cache.k.shape
        half = torch.finfo(DT[self.kind]).eps / 2
        for i, n in enumerate(self.lens if lens is None else lens):
            used = [int(j) for j in table[i, :-(-n // page)]]
            idx = torch.tensor([j if 0 <= j < n_pages else 0 for j in used], device=self.q.device,
                               dtype=torch.long)
            ok = torch.tensor([0 <= j < n_pages for j in used], device=self.q.device, dtype=torch.bool)
            ok = ok.repeat_interleave(page)[:n]
            k, v = (x[idx].transpose(0, 1).reshape(h, -1, d)[:, :n][:, ok] for x in self.values)
            q = self.q[i].double().view(h, self.group, d)
            if k.shape[1] == 0:
                out.append(torch.zeros_like(q).view(-1, d))
                tol.append(torch.zeros_like(q).view(-1, d))
                continue
            s = q @ k.transpose(1, 2) * self.scale
            p = torch.softmax(s, -1)
            o = p @ v
            # a score: D products summed in 32 bits (the tensor core may truncate: 2^-23 a
            # step), scaled by rounded factors; a weight: exp2 of it (2^-22 and its
            # argument's rounding); both enter numerator and denominator.  The weights' own
            # 16-bit pairs are good to 2^-17 (bfloat16) or better; sums over n tokens.
            mag = (q.abs() @ k.abs().transpose(1, 2) * abs(self.scale)).amax(-1, keepdim=True)
            rel = 2 * ((d + 6) * 2.0**-23 * mag + 2.0**-20) + 2.0**-17 + n * 2.0**-23
            out.append(o.view(-1, d))
            tol.append((half * o.abs() + rel * (p @ v.abs())).view(-1, d) + 2.0**-24)
        return torch.stack(out), torch.stack(tol)

    def run(self):
        return self.cache.attend(self.q, self.t, self.l)

    def check(self, got=None, **kw):
        got = self.run() if got is None else got
        want, tol = self.want(**kw)
        assert got.dtype == DT[self.kind] and got.shape == want.shape
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-30)).max())


TYPES = [("f16", "f16"), ("bf16", "bf16"), ("int8", "f16"), ("int8", "bf16")]
EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 250, 257]


@pytest.mark.parametrize("cache,kind", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group,page", [(1, 1, 16), (2, 8, 16), (3, 5, 64), (1, 16, 256),
                                                 (2, 20, 32)])
def test_attend_at_the_edges_of_lengths(cuda, cache, kind, d, kv_heads, group, page):
    Case(cuda, EDGES, kv_heads, group, d, page, cache, kind).check()


@pytest.mark.parametrize("cache,kind", TYPES)
@pytest.mark.parametrize("lens", [[1], [700], [5000], [20011], [0, 0, 0], [0, 4097, 0, 1, 0],
                                  [3000, 17, 9000, 0, 64, 64, 64, 2049]])
def test_attend_long_and_ragged(cuda, cache, kind, lens):
    Case(cuda, lens, 2, 8, 256, 16, cache, kind).check()
    Case(cuda, lens, 8, 4, 128, 64, cache, kind, seed=1).check()


@pytest.mark.parametrize("cache,kind", TYPES)
def test_attend_sharp_scores(cuda, cache, kind):
    Case(cuda, [1000, 33, 4096], 2, 4, 128, 32, cache, kind, mult=12.0).check()


@pytest.mark.parametrize("b", [300, 1024, 1025, 2500])
def test_attend_large_batches(cuda, b):
    rng = np.random.default_rng(b)
    Case(cuda, rng.integers(0, 90, b), 1, 2, 64, 16, "f16", "f16").check()


@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 1, 5], [64, 0, 65, 0, 0, 3]])
def test_attend_short_rows_of_wide_tables(cuda, lens):
    """Fewer blocks of tokens than CTAs, or none, where rows may be cut."""
    Case(cuda, lens, 2, 8, 128, 16, "f16", "f16", spare=400).check()


@pytest.mark.parametrize("cache,kind", TYPES)
@pytest.mark.parametrize("b,h", [(400, 1), (37, 2), (100, 1), (20, 8), (3, 99), (4, 2), (1, 8)])
def test_attend_every_way_of_sharing_rows(cuda, cache, kind, b, h):
    rng = np.random.default_rng(b)
    Case(cuda, rng.integers(0, 65, b), h, 2, 64, 16, cache, kind, spare=0).check()     # one block
    Case(cuda, rng.integers(0, 600, b), h, 2, 64, 16, cache, kind, spare=0).check()
    Case(cuda, rng.integers(0, 600, b), h, 2, 64, 16, cache, kind, spare=100).check()


def test_attend_requests_that_share_pages(cuda):
    c = Case(cuda, [200, 200, 64], 2, 4, 64, 16, "f16", "f16")
    c.table[1] = c.table[0]
    c.t = ints(c.table, cuda)
    c.check()


def test_attend_queries_of_one_large_channel(cuda):
    """bfloat16 queries whose largest channel dwarfs the others and meets zeros in the cache:
    the others decide the scores."""
    c = Case(cuda, [300, 20], 2, 4, 64, 16, "int8", "bf16")
    c.q[:, :, 5] = 2.0**18
    c.cache.k[..., 5] = 0
    c.values[0][..., 5] = 0
    c.check()


def test_attend_leaves_out_pages_that_do_not_exist(cuda):
    c = Case(cuda, [100, 40, 300, 16], 2, 4, 128, 16, "f16", "f16")
    c.table[0, 2], c.table[2, 0], c.table[2, 18] = -1, 10**6, -2**31
    c.table[3, 0] = -7                                   # nothing is left of this one
    c.t = ints(c.table, cuda)
    c.check()
    assert not c.run()[3].any()


def test_attend_cuts_lengths_to_the_table(cuda):
    c = Case(cuda, [64, 32, 64, 48], 1, 2, 64, 16, "bf16", "bf16", spare=0)
    c.l = ints([2**31 - 1, -5, 64, -2**31], cuda)
    c.check(lens=[64, 0, 64, 0])


def test_attend_weights_of_every_size(cuda):
    """8-bit values whose scales differ by many powers of two, and a zero one."""
    c = Case(cuda, [500, 77], 2, 4, 64, 16, "int8", "f16")
    by = torch.exp2(torch.randint(-18, 8, c.cache.v_scale.shape, device=cuda).double())
    by[torch.rand(by.shape, device=cuda) < 0.1] = 0.0
    c.cache.v_scale.mul_(by.float())
    c.values[1] = c.values[1] * by[..., None]
    c.check()


def test_attend_reads_strided_queries(cuda):
    c = Case(cuda, [100, 3, 40], 2, 4, 64, 16, "f16", "f16")
    wide = torch.randn((3, 3, 8, 64), device=cuda).half()
    wide[:, 1] = c.q
    flat = torch.zeros(3 * 8 * 64 + 1, device=cuda).half()
    flat[1:] = c.q.reshape(-1)
    want = c.run()
    for q in (wide[:, 1], flat[1:].view(3, 8, 64), c.q.transpose(0, 1).contiguous().transpose(0, 1),
              c.q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(c.cache.attend(q, c.t, c.l), want)


def test_attend_past_32_bit_offsets(cuda):
    """Pages whose first element is past 2^31 (keys and values share one tensor here)."""
    n_pages, h, page, d = 1100, 32, 256, 256                       # 2.3 G values, 4.6 GB
    kv = torch.empty((n_pages, h, page, d), dtype=torch.float16, device=cuda)
    pc = paged.PagedCache.from_tensors(kv, kv)
    x = torch.randn((300, h, d), device=cuda).half()
    table = torch.tensor([[1099, 1098]], dtype=torch.int32, device=cuda)
    pos = torch.arange(300, device=cuda)
    pc.append(x, x, (table[0, pos // 256].long() * 256 + pos % 256).to(torch.int32))
    assert torch.equal(kv[1099].transpose(0, 1), x[:256])
    q = torch.randn((1, h, d), device=cuda).half()
    got = pc.attend(q, table, torch.tensor([300], dtype=torch.int32, device=cuda)).double()
    xd = x.double().transpose(0, 1)
    want = torch.softmax(q[0].double()[:, None] @ xd.transpose(1, 2) / 16, -1) @ xd
    # outputs of a mean of values near 1: half a step and the sums' bound, as above
    assert float((got[0] - want[:, 0]).abs().max()) <= 2.0**-11 * float(want.abs().max()) + 2.0**-12


def test_attend_is_reproducible_and_follows_its_stream(cuda):
    c = Case(cuda, [9000, 17, 4000, 333], 2, 8, 256, 16, "f16", "f16")
    want = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    with torch.cuda.stream(side):
        outs += [c.run() for _ in range(8)]
    outs += [c.run() for _ in range(8)]                            # both streams at once
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_captured_steps_replayed_together(cuda):
    """Two graphs of the same cache on two streams share nothing; lengths change between
    replays."""
    c = Case(cuda, [2000, 50, 700], 2, 8, 128, 16, "f16", "f16")
    e = Case(cuda, [1, 3000, 64], 2, 8, 128, 16, "f16", "f16", seed=3)
    calls = [graphs.GraphedCall(x.cache.attend, [x.q, x.t, x.l]) for x in (c, e)]
    streams = [torch.cuda.Stream() for _ in calls]
    for lens in ([2000, 50, 700], [3, 0, 65], [1999, 50, 1]):
        torch.cuda.synchronize()
        for x, n in ((c, lens), (e, [min(a, b) for a, b in zip(lens, e.lens)])):
            x.l.copy_(ints(n, cuda))
            x.now = n
        torch.cuda.synchronize()
        for _ in range(3):
            for g, st, x in zip(calls, streams, (c, e)):
                with torch.cuda.stream(st):
                    g(x.q, x.t, x.l)
        torch.cuda.synchronize()
        for g, x in zip(calls, (c, e)):
            x.check(got=g.outputs, lens=x.now)


# ---------------------------------------------------------------------------------------------
# together

@pytest.mark.parametrize("cache", ["f16", "int8"])
def test_a_run_of_steps(cuda, cache):
    """Prompts, then single tokens: plan, store and attend step by step against attention over
    the plain history."""
    h, group, d, page, b = 2, 4, 128, 16, 5
    gen = torch.Generator(device=cuda).manual_seed(7)
    pc = paged.PagedCache(64, page, h, d, DT[cache], cuda)
    table = torch.full((b, 12), -1, dtype=torch.int32, device=cuda)
    free = torch.randperm(64, device=cuda, generator=gen).to(torch.int32)
    head = torch.zeros(1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(b, dtype=torch.int32, device=cuda)
    history = [[] for _ in range(b)]
    steps = [[31, 1, 0, 77, 16]] + [[1, 1, 1, 1, 1]] * 20 + [[0, 1, 4, 0, 1]] + [[1] * 5] * 3
    for added in steps:
        rows = sum(added) + 2
        kv = torch.randn((rows, 2, h, d), device=cuda, generator=gen).half()
        plan = paged.plan_pages(table, lens, ints(added, cuda), free, head, page_size=page,
                                n_pages=64, rows=rows)
        pc.append(kv[:, 0], kv[:, 1], plan.slots)
        q = torch.randn((b, h * group, d), device=cuda, generator=gen).half()
        got = pc.attend(q, table, plan.ends)
        at = 0
        for i, n in enumerate(added):
            history[i] += [kv[at + r] for r in range(n)]
            at += n
        assert plan.refused.item() == 0 and plan.ends.tolist() == [len(x) for x in history]
        for i, x in enumerate(history):
            if not x:
                assert not got[i].any()
                continue
            k, v = (torch.stack(x)[:, j].transpose(0, 1).double() for j in range(2))
            if cache == "int8":
                k, v = (torch.from_numpy(c * s.astype(np.float64)[..., None]).to(cuda)
                        for c, s in (quantised(y.cpu().numpy()) for y in (k, v)))
            qi = q[i].double().view(h, group, d)
            p = torch.softmax(qi @ k.transpose(1, 2) * d ** -0.5, -1)
            want = (p @ v).view(-1, d)
            # at most 101 tokens, |q.k| / sqrt(d) sums below 40: see Case.want
            tol = 2.0**-11 * want.abs() + (2 * (134 * 2.0**-23 * 40 + 2.0**-20) + 2.0**-15) * \
                (p @ v.abs()).view(-1, d) + 2.0**-24
            assert bool(((got[i].double() - want).abs() <= tol).all())
        head, lens = plan.head, plan.ends
    assert head.item() == sum(-(-len(x) // page) for x in history)


def test_refusals(cuda):
    pc = paged.PagedCache(4, 16, 2, 64, torch.float16, cuda)
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device=cuda)
    t = torch.zeros((2, 3), dtype=torch.int32, device=cuda)
    n = torch.zeros((2,), dtype=torch.int32, device=cuda)
    pc.attend(q, t, n)
    for bad, text in (((q[:, :3], t, n), "evenly"), ((q.bfloat16(), t, n), "float16"),
                      ((q[..., :32], t, n), "shape"), ((q, t[:1], n), "shape"),
                      ((q, t.long(), n), "int32"), ((q, t, n.cpu()), "CUDA"),
                      ((q, t[:, :0], n), "page"), ((q, t.t().contiguous().t(), n), "contiguous"),
                      ((q.cpu(), t, n), "CUDA")):
        with pytest.raises(ValueError, match=text):
            pc.attend(*bad)
    k = torch.zeros((3, 2, 64), dtype=torch.float16, device=cuda)
    s = torch.zeros((3,), dtype=torch.int32, device=cuda)
    for bad, text in (((k, k[:2], s), "shape"), ((k, k.bfloat16(), s), "bfloat16"),
                      ((k.float(), k.float(), s), "float16"), ((k, k, s[:2]), "shape"),
                      ((k, k, s.long()), "int32"), ((k[:, :1], k[:, :1], s), "shape")):
        with pytest.raises(ValueError, match=text):
            pc.append(*bad)
    for make, text in ((lambda: paged.PagedCache(4, 24, 2, 64), "page size"),
                       (lambda: paged.PagedCache(4, 16, 2, 96), "head size"),
                       (lambda: paged.PagedCache(4, 16, 2, 64, torch.float32), "float16"),
                       (lambda: paged.PagedCache.from_tensors(pc.k, pc.v.bfloat16()), "float16"),
                       (lambda: paged.PagedCache.from_tensors(pc.k, pc.v, n, n), "int8")):
        with pytest.raises(ValueError, match=text):
            make()
