"""Cases of the operators around a decode step's cache and its vocabulary head: page plans,
stores into a paged key-value cache, attention of one new token per request over it, and
sampling.  ``run`` computes an operator either in its plain form (elementary torch operations)
or, where ``own`` is true, through the package's own entry points."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "int8": torch.int8}
# weights under e^-30 of the largest count as nothing when sampling
SAMPLE_CUTOFF = -30.0


# ---------------------------------------------------------------------------------------------
# cases

def listed():
    return [
        # one decode step of a few requests: the smallest plan there is
        dict(name="plan_decode_8", op="plan", batch=8, max_len=4000, max_new=1, page=16),
        # continuous batching: ragged prompts beside running requests
        dict(name="plan_mixed_512", op="plan", batch=512, max_len=6000, max_new=300, page=64),
        # keys and values of one decode step at batch 32, 2 heads of 256 (the 40-layer step)
        dict(name="append_step_32", op="append", rows=32, kv_heads=2, dim=256, page=16,
             cache="f16", q="f16", pages=4096),
        # a chunk of prompts, 8 heads of 128, pages of 64
        dict(name="append_chunk_bf16", op="append", rows=16001, kv_heads=8, dim=128, page=64,
             cache="bf16", q="bf16", pages=300),
        # the same into the 8-bit cache, 2 heads of 256
        dict(name="append_chunk_int8", op="append", rows=8190, kv_heads=2, dim=256, page=32,
             cache="int8", q="f16", pages=300),
        # one user, a short conversation: latency
        dict(name="attend_one_short", op="attend", batch=1, max_len=700, even=True, kv_heads=2,
             group=8, dim=256, page=16, cache="f16", q="f16"),
        # the 40-layer step's attention at batch 32, ragged lengths
        dict(name="attend_step_32", op="attend", batch=32, max_len=8191, even=False, kv_heads=2,
             group=8, dim=256, page=16, cache="f16", q="f16"),
        # few requests with very long contexts
        dict(name="attend_long_bf16", op="attend", batch=2, max_len=131000, even=True, kv_heads=8,
             group=4, dim=128, page=64, cache="bf16", q="bf16"),
        # many requests over the 8-bit cache
        dict(name="attend_int8_64", op="attend", batch=64, max_len=12000, even=False, kv_heads=2,
             group=8, dim=256, page=32, cache="int8", q="f16"),
        # one user's next token from the vocabulary head
        dict(name="sample_one", op="sample", batch=1, vocab=151936, dtype="f16", mode="all"),
        # a batch with every request's own settings
        dict(name="sample_64", op="sample", batch=64, vocab=151936, dtype="f16", mode="mixed"),
        # 32-bit logits, an odd vocabulary, nucleus alone
        dict(name="sample_f32_odd", op="sample", batch=16, vocab=50257, dtype="f32", mode="top_p"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "sample"])
    if op == "plan":
        batch = _log_int(rng, 1, 512)
        return dict(op=op, batch=batch, max_len=_log_int(rng, 1, 6000),
                    max_new=_log_int(rng, 1, 300), page=rng.choice([16, 32, 64, 128, 256]))
    if op == "append":
        cache = rng.choice(["f16", "bf16", "int8"])
        q = rng.choice(["f16", "bf16"]) if cache == "int8" else cache
        dim, page = rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        rows = _log_int(rng, 1, min(16000, 16384 * 1024 // (dim * kv_heads)))
        return dict(op=op, rows=rows, kv_heads=kv_heads, dim=dim, page=page, cache=cache, q=q,
                    pages=-(-rows // page) + rng.randrange(1, 40))
    if op == "attend":
        cache = rng.choice(["f16", "bf16", "int8"])
        q = rng.choice(["f16", "bf16"]) if cache == "int8" else cache
        batch, kv_heads = _log_int(rng, 1, 64), rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 128, 256])
        # keys and values together at most a gigabyte of 16-bit values
        most = min(131000, (1 << 29) // (2 * batch * kv_heads * dim))
        return dict(op=op, batch=batch, max_len=_log_int(rng, 1, most), even=rng.random() < 0.3,
                    kv_heads=kv_heads, group=rng.choice([1, 2, 4, 5, 8, 16]), dim=dim,
                    page=rng.choice([16, 32, 64, 128, 256]), cache=cache, q=q)
    return dict(op=op, batch=_log_int(rng, 1, 64), vocab=_log_int(rng, 1000, 151936),
                dtype=rng.choice(["f16", "bf16", "f32"]),
                mode=rng.choice(["all", "mixed", "top_k", "top_p", "min_p", "plain"]))


# ---------------------------------------------------------------------------------------------
# what a case fixes apart from the seed: lengths (the seed only orders them)

def _lens(case):
    b, m = case["batch"], case["max_len"]
    if case.get("even"):
        return [max(1, m - 3 * (i % 7)) for i in range(b)]
    return [1 + (m - 1) * ((i * 37 + 11) % (b + 2)) // (b + 1) for i in range(b - 1)] + [m]


def _news(case):
    # two of three requests decode one token, the others bring a chunk; one brings nothing
    n = [1 if i % 3 else 1 + (case["max_new"] - 1) * ((i * 53 + 7) % 64) // 63
         for i in range(case["batch"])]
    if case["batch"] > 4:
        n[4] = 0
    return n


def _need(case):
    p = case["page"]
    return sum(-(-(a + n) // p) - -(-a // p) for a, n in zip(_lens_plan(case), _news(case)))


def _lens_plan(case):
    return [n - 1 for n in _lens(case)]      # a request may have nothing cached yet


def work(case):
    es = {"f16": 2, "bf16": 2, "f32": 4, "int8": 1}
    if case["op"] == "plan":
        b, rows, need = case["batch"], sum(_news(case)), _need(case)
        # lengths, new, starts, ends; the last open page of each; pages taken and entered; rows
        return {"bytes": 4 * (5 * b + 2 * need + 2 * rows), "flops": 0}
    if case["op"] == "append":
        n = 2 * case["rows"] * case["kv_heads"]
        size = n * case["dim"] * (es[case["q"]] + es[case["cache"]]) + 4 * case["rows"]
        return {"bytes": size + (4 * n if case["cache"] == "int8" else 0), "flops": 0}
    if case["op"] == "attend":
        tokens = sum(_lens(case))
        row = case["dim"] * es[case["cache"]] + (4 if case["cache"] == "int8" else 0)
        heads = case["kv_heads"] * case["group"]
        pages = sum(-(-n // case["page"]) for n in _lens(case))
        return {"bytes": 2 * tokens * case["kv_heads"] * row
                + 2 * case["batch"] * heads * case["dim"] * es[case["q"]] + 4 * pages,
                "flops": 4 * tokens * heads * case["dim"]}
    return {"bytes": case["batch"] * case["vocab"] * es[case["dtype"]] + 28 * case["batch"],
            "flops": 0}


# ---------------------------------------------------------------------------------------------
# inputs

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _quantised(x):
    """Rows of x as 8-bit codes and one 32-bit scale each: scale = max|x| / 127, and the code
    nearest to x / scale.  16-bit values fall next to the middle between two codes often enough
    that the quotient is taken in 64 bits."""
    scale = (x.double().abs().amax(-1) / 127.0).float()
    by = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    return torch.round(x.double() / by[..., None]).clamp(-127, 127).to(torch.int8), scale


def _filled(shape, kind, gen, q):
    if kind != "int8":
        return torch.randn(shape, device="cuda", generator=gen, dtype=DTYPES[kind]), None
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    scales = torch.empty(shape[:-1], dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (shape[1] * shape[2] * shape[3]))
    for i in range(0, shape[0], step):
        part = torch.randn((min(step, shape[0] - i), *shape[1:]), device="cuda", generator=gen,
                           dtype=DTYPES[q])
        codes[i:i + step], scales[i:i + step] = _quantised(part)
    return codes, scales


def prepare(case, seed):
    gen, order = _generator(seed), np.random.default_rng(seed)
    s = {"case": case}
    if case["op"] == "plan":
        b, page = case["batch"], case["page"]
        lens, news = np.array(_lens_plan(case)), np.array(_news(case))
        perm = order.permutation(b)
        lens, news = lens[perm], news[perm]
        used, need = int((-(-lens // page)).sum()), _need(case)
        width = int((-(-(lens + news) // page)).max()) + 3
        pages = order.permutation(used + need + 64)
        table = np.full((b, width), -1, np.int32)
        at = 0
        for i in range(b):
            n = -(-int(lens[i]) // page)
            table[i, :n] = pages[at:at + n]
            at += n
        # a few of the listed free pages were taken by earlier steps
        free = np.concatenate([order.integers(0, len(pages), 5), pages[at:]])
        s.update(table=_ints(table), lengths=_ints(lens), new=_ints(news), free=_ints(free),
                 head=_ints([5]), page=page, n_pages=len(pages),
                 rows=-(-int(news.sum() + 1) // 32) * 32)
    elif case["op"] == "append":
        shape = (case["pages"], case["kv_heads"], case["page"], case["dim"])
        t = case["rows"]
        heads = case["kv_heads"] * case["dim"]
        # keys and values as they leave a merged projection: rows of one wider matrix
        kv = torch.randn((t, 2 * heads), device="cuda", generator=gen, dtype=DTYPES[case["q"]])
        s["k_new"] = kv[:, :heads].unflatten(1, (case["kv_heads"], case["dim"]))
        s["v_new"] = kv[:, heads:].unflatten(1, (case["kv_heads"], case["dim"]))
        slots = torch.randperm(case["pages"] * case["page"], device="cuda", generator=gen)[:t]
        if t > 2:
            slots[t - 1] = -1        # a padded row
        s["slots"] = slots.to(torch.int32)
        zero = (lambda sh, ty: torch.zeros(sh, dtype=ty, device="cuda"))
        s["k"], s["v"] = zero(shape, DTYPES[case["cache"]]), zero(shape, DTYPES[case["cache"]])
        scaled = case["cache"] == "int8"
        s["k_scale"] = zero(shape[:3], torch.float32) if scaled else None
        s["v_scale"] = zero(shape[:3], torch.float32) if scaled else None
    elif case["op"] == "attend":
        b, page = case["batch"], case["page"]
        lens = np.array(_lens(case))[order.permutation(b)]
        each = -(-lens // page)
        n_pages, width = int(each.sum()) + 3, int(each.max())
        pages = order.permutation(n_pages)
        table = np.full((b, width), -1, np.int32)
        at = 0
        for i in range(b):
            table[i, :each[i]] = pages[at:at + each[i]]
            at += each[i]
        shape = (n_pages, case["kv_heads"], page, case["dim"])
        s["k"], s["k_scale"] = _filled(shape, case["cache"], gen, case["q"])
        s["v"], s["v_scale"] = _filled(shape, case["cache"], gen, case["q"])
        s["q"] = torch.randn((b, case["kv_heads"] * case["group"], case["dim"]), device="cuda",
                             generator=gen, dtype=DTYPES[case["q"]])
        s["table"], s["lengths"] = _ints(table), _ints(lens)
        s["scale"] = case["dim"] ** -0.5
    else:
        b, v = case["batch"], case["vocab"]
        # a broad floor and some tokens that stand out, as a language model's logits have
        x = 2.0 * torch.randn((b, v), device="cuda", generator=gen)
        up = torch.randint(0, v, (b, 40), device="cuda", generator=gen)
        x.scatter_add_(1, up, 6.0 + 4.0 * torch.rand((b, 40), device="cuda", generator=gen))
        if case["mode"] == "mixed":     # every fourth request may only use a part of the vocabulary
            masked = torch.rand((b, v), device="cuda", generator=gen) < 0.5
            x[3::4] = torch.where(masked[3::4], float("-inf"), x[3::4])
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["uniforms"] = torch.rand((b,), device="cuda", generator=gen)
        m = case["mode"]
        pick = (lambda values: torch.tensor(order.choice(values, b)).cuda())
        t = pick([0.6, 0.7, 0.8, 1.0, 1.3])
        k, p, mp = pick([0]), pick([1.0]), pick([0.0])
        if m in ("all", "top_k"):
            k = pick([20, 40, 50])
        if m in ("all", "top_p"):
            p = pick([0.8, 0.9, 0.95])
        if m in ("all", "min_p"):
            mp = pick([0.02, 0.05, 0.1])
        if m == "mixed":
            t, k = pick([0.0, 0.5, 0.8, 1.0, 1.5]), pick([0, 1, 40, 1000, v + 5])
            p, mp = pick([1.0, 0.5, 0.9, 0.99]), pick([0.0, 0.0, 0.05])
        s["temperature"], s["top_k"] = t.float(), k.to(torch.int32)
        s["top_p"], s["min_p"] = p.float(), mp.float()
    return s


def _cache(s):
    """The cache object that a user's program keeps: made on the first pass."""
    if "cache" not in s:
        from escha_mlx_b200 import paged
        s["cache"] = paged.PagedCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s["cache"]


# ---------------------------------------------------------------------------------------------
# one pass

def run(s):
    return {"plan": _run_plan, "append": _run_append, "attend": _run_attend,
            "sample": _run_sample}[s["case"]["op"]](s)


def _run_plan(s):
    if own:
        from escha_mlx_b200 import paged
        plan = paged.plan_pages(s["table"], s["lengths"], s["new"], s["free"], s["head"],
                                page_size=s["page"], n_pages=s["n_pages"], rows=s["rows"])
        return {"table": s["table"], "slots": plan.slots, "positions": plan.positions,
                "starts": plan.starts, "ends": plan.ends, "head": plan.head,
                "refused": plan.refused}
    page, rows, table = s["page"], s["rows"], s["table"].long()
    b, width = table.shape
    dev = table.device
    lens, new, free = s["lengths"].long(), s["new"].long(), s["free"].long()
    head = s["head"].long()
    wanted = new.clamp(min=0)
    first = torch.cumsum(wanted, 0) - wanted
    valid = (lens >= 0) & (new >= 0) & (lens + new <= width * page) & (first + wanted <= rows)
    have, then = (lens + page - 1) // page, (lens + new + page - 1) // page
    need = torch.where(valid, then - have, 0)
    before = torch.cumsum(need, 0) - need
    fine = valid & ((need == 0) | (before + need <= free.numel() - head))
    took = torch.where(fine, need, 0)
    # entries of the table that this step adds
    j = torch.arange(width, device=dev)[None] - have[:, None]
    taken = (j >= 0) & (j < took[:, None])
    at = (head + before[:, None] + j).clamp(0, free.numel() - 1)
    table = torch.where(taken, free[at], table)
    # rows, packed by request
    starts = torch.cat([first, first[-1:] + wanted[-1:]]).clamp(max=2**31 - 1)
    r = torch.arange(rows, device=dev)
    owner = (torch.searchsorted(starts, r, right=True) - 1).clamp(max=b - 1)
    inside = (r < starts[-1]) & fine[owner]
    pos = torch.where(inside, lens[owner] + r - starts[owner], 0)
    got = table[owner, pos // page]
    inside_page = inside & (got >= 0) & (got < s["n_pages"])
    slots = torch.where(inside_page, got * page + pos % page, -1)
    ends = torch.where(fine, lens + new, lens.clamp(0, width * page))
    i32 = torch.int32
    return {"table": table.to(i32), "slots": slots.to(i32), "positions": pos.to(i32),
            "starts": starts.to(i32), "ends": ends.to(i32),
            "head": head.to(i32) + took.sum().to(i32), "refused": (~fine).sum().to(i32)[None]}


def _run_append(s):
    if own:
        _cache(s).append(s["k_new"], s["v_new"], s["slots"])
    else:
        page = s["case"]["page"]
        rows = torch.nonzero(s["slots"] >= 0)[:, 0]
        at = s["slots"][rows].long()
        page_of, row_of = at // page, at % page
        for name in ("k", "v"):
            new = s[name + "_new"][rows]
            if s[name + "_scale"] is not None:
                new, s[name + "_scale"][page_of, :, row_of] = _quantised(new)
            s[name][page_of, :, row_of] = new.to(s[name].dtype)
    if s["k_scale"] is not None:
        return {"k": s["k"].float() * s["k_scale"][..., None],
                "v": s["v"].float() * s["v_scale"][..., None]}
    return {"k": s["k"], "v": s["v"]}


def _run_attend(s):
    if own:
        return {"out": _cache(s).attend(s["q"], s["table"], s["lengths"], scale=s["scale"])}
    c = s["case"]
    b, width = s["table"].shape
    table = s["table"].long().clamp(min=0)

    def gathered(name):
        x = s[name][table].float()                              # [B, W, H, P, D]
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][table][..., None]
        return x.transpose(1, 2).reshape(b, c["kv_heads"], width * c["page"], c["dim"])

    there = torch.arange(width * c["page"], device=table.device)[None] < s["lengths"][:, None]
    there = there[:, None, None]
    q = s["q"].float().reshape(b, c["kv_heads"], c["group"], c["dim"])
    scores = (q @ gathered("k").transpose(2, 3)) * s["scale"]
    scores = torch.where(there, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(there[:, :, 0, :, None], gathered("v"), 0.0)
    out = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return {"out": out.reshape(b, -1, c["dim"]).to(s["q"].dtype)}


def _run_sample(s):
    if own:
        from escha_mlx_b200 import sampling
        return {"tokens": sampling.sample(s["logits"], s["uniforms"], s["temperature"],
                                          s["top_k"], s["top_p"], s["min_p"])}
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), float("-inf"), x)
    b, v = x.shape
    t = s["temperature"].double()[:, None]
    top = x.amax(-1, keepdim=True)
    d = torch.where(x == top, 0.0, (x - top) / torch.where(t > 0, t, torch.ones_like(t)))
    w = torch.where(d < SAMPLE_CUTOFF, 0.0, torch.exp(d))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = torch.gather(w, 1, order)
    rank = torch.arange(v, device=x.device)[None]
    k = s["top_k"].long()[:, None]
    keep = (k <= 0) | (rank < k)
    ws = torch.where(keep, ws, 0.0)
    total = ws.sum(-1, keepdim=True)
    before = torch.cumsum(ws, -1) - ws
    p, mp = s["top_p"].double()[:, None], s["min_p"].double()[:, None].clamp(max=1.0)
    keep &= (p >= 1) | (rank == 0) | (before < p * total)
    keep &= ~(mp > 0) | (ws >= mp)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0))
    total = torch.cumsum(w, -1)
    target = s["uniforms"].double()[:, None] * total[:, -1:]
    token = torch.searchsorted(total, target, right=True)
    last = torch.searchsorted(total, total[:, -1:].contiguous())
    token = torch.minimum(token, last)
    token = torch.where(t > 0, token, torch.argmax((x == top).to(torch.int8), -1, keepdim=True))
    return {"tokens": torch.where(torch.isinf(top) & (top < 0), -1, token)[:, 0]}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits

def exact(case, seed):
    if case["op"] == "plan":
        return None          # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        out = {}
        slots = s["slots"].cpu().numpy().astype(np.int64)
        for name in ("k", "v"):
            new = s[name + "_new"].double().cpu().numpy()
            if case["cache"] == "int8":
                # the scale is a 32-bit number by definition
                scale = (np.abs(new).max(-1, keepdims=True) / 127.0).astype(np.float32)
                scale = scale.astype(np.float64)
                new = np.rint(new / np.where(scale > 0, scale, 1.0)) * scale
            cache = np.zeros((case["pages"] * case["page"], case["kv_heads"], case["dim"]))
            cache[slots[slots >= 0]] = new[slots >= 0]
            cache = cache.reshape(case["pages"], case["page"], case["kv_heads"], case["dim"])
            out[name] = torch.from_numpy(np.ascontiguousarray(cache.transpose(0, 2, 1, 3)))
        return out
    if case["op"] == "attend":
        tables, lens = s["table"].cpu().tolist(), s["lengths"].cpu().tolist()
        outs = []
        for i, n in enumerate(lens):
            per_head = []
            for h in range(case["kv_heads"]):
                used = tables[i][:-(-n // case["page"])]
                k = torch.cat([s["k"][j, h] for j in used])[:n].double()
                v = torch.cat([s["v"][j, h] for j in used])[:n].double()
                if case["cache"] == "int8":
                    k = k * torch.cat([s["k_scale"][j, h] for j in used])[:n, None].double()
                    v = v * torch.cat([s["v_scale"][j, h] for j in used])[:n, None].double()
                q = s["q"][i, h * case["group"]:(h + 1) * case["group"]].double()
                per_head.append(torch.softmax(torch.mm(q, k.T) * s["scale"], -1) @ v)
            outs.append(torch.cat(per_head))
        return {"out": torch.stack(outs)}
    return None              # whole numbers


if __name__ == "__main__":
    for _case in listed():
        print(_case["name"], work(_case))
