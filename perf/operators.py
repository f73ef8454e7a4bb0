"""Cases of the paged KV cache: block tables and slot maps from request lengths, the write of new
tokens into the pages, and attention of new tokens over the pages.

A serving step runs them in this order: `release` gives the pages of finished requests back, `plan`
takes pages for the step's new tokens and maps each token to its slot, `append` normalises and rotates
q and k and stores k and v, and `attention` lets every new token see its sequence's cached positions.

Layouts: a cache is [pages, kv heads, page, head dim]; a block table row lists a sequence's pages in
order; a slot is page id * page + offset; the new tokens of a batch are rows one after the other,
sequence i's at cu[i] .. cu[i + 1].

Lengths are a function of the case (its `tag`), values of the seed.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}
EPS = 1e-5


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a few users, one token each: the smallest step, bound by launches
        dict(name="tables, 7 decoding sequences", op="tables", seqs=7, new=1, mix=0.0, cached=500, page=16, done=1,
             tag=11),
        # 64 sequences around context 2048 (the batched decode workload), some of them finished
        dict(name="tables, 64 sequences at 2048", op="tables", seqs=64, new=1, mix=0.0, cached=2048, page=64, done=5,
             tag=12),
        # a full server: chunks of prompts beside decoding sequences, small pages
        dict(name="tables, 1000 sequences with chunks", op="tables", seqs=1000, new=1100, mix=0.03, cached=8000,
             page=16, done=41, tag=13),
        # one decode step of the batched decode workload: f32 projections into a bf16 cache
        dict(name="append, 64 decoded tokens", op="append", tokens=64, heads=16, kv_heads=16, head_dim=128, page=64,
             source="f32", dtype="bf16", norm=True, pad=0, positions=2048, tag=21),
        # prompt chunks of a grouped-query model in bf16
        dict(name="append, 4096 prompt tokens", op="append", tokens=4096, heads=32, kv_heads=8, head_dim=128, page=16,
             source="bf16", dtype="bf16", norm=False, pad=0, positions=8192, tag=22),
        # a padded batch (a captured step of fixed size) into an f32 cache, head dim 64
        dict(name="append, 1535 rows with padding, f32", op="append", tokens=1535, heads=12, kv_heads=6, head_dim=64,
             page=32, source="f32", dtype="f32", norm=True, pad=211, positions=4096, tag=23),
        # one user, one token: latency
        dict(name="attend, 1 token at 4095", op="attend", dtype="bf16", heads=16, kv_heads=16, head_dim=128, page=64,
             seqs=1, new=1, mix=0.0, cached=4095, spread=False, window=0, lse=False, tag=31),
        # the batched decode workload with the f32 cache that parity asks for
        dict(name="attend, 64 tokens at 2048, f32", op="attend", dtype="f32", heads=16, kv_heads=16, head_dim=128,
             page=64, seqs=64, new=1, mix=0.0, cached=2047, spread=False, window=0, lse=False, tag=32),
        # grouped-query decode over ragged long contexts with small pages
        dict(name="attend, 96 ragged tokens to 16384", op="attend", dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             page=16, seqs=96, new=1, mix=0.0, cached=16383, spread=True, window=0, lse=False, tag=33),
        # whole prompts of 4096 tokens (the prompt workload's length): the largest call
        dict(name="attend, 4 prompts of 4096", op="attend", dtype="bf16", heads=16, kv_heads=16, head_dim=128, page=64,
             seqs=4, new=4096, mix=1.0, cached=0, spread=False, window=0, lse=False, tag=34),
        # chunks of prompts beside decoding sequences, a sliding window, head dim 64
        dict(name="attend, chunks and tokens, window", op="attend", dtype="bf16", heads=32, kv_heads=8, head_dim=64,
             page=32, seqs=24, new=700, mix=0.3, cached=5000, spread=True, window=1024, lse=True, tag=35),
        # chunks of an f32 model (head dim 64) on cached prefixes
        dict(name="attend, 5 chunks to 333, f32", op="attend", dtype="f32", heads=12, kv_heads=6, head_dim=64, page=16,
             seqs=5, new=333, mix=1.0, cached=1500, spread=True, window=0, lse=True, tag=36),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend"])
    page = rng.choice([8, 16, 32, 64, 128])
    tag = rng.randrange(1, 1 << 30)
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    if op == "tables":
        seqs = _log(rng, 1, 1500)
        return dict(op=op, seqs=seqs, new=_log(rng, 1, 1200), mix=rng.choice([0.0, 0.02, 0.2]),
                    cached=_log(rng, 1, 9000), page=page, done=rng.randint(0, seqs // 2), tag=tag)
    if op == "append":
        tokens = _log(rng, 1, 4096)
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                    source=rng.choice(["bf16", "f32"]), dtype=rng.choice(["bf16", "f32"]),
                    norm=rng.random() < 0.5, pad=rng.choice([0, 0, tokens // 7]), positions=_log(rng, 64, 8192),
                    tag=tag)
    decode = rng.random() < 0.5
    return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                page=page, seqs=_log(rng, 1, 128 if decode else 24), new=1 if decode else _log(rng, 2, 4096),
                mix=0.0 if decode else rng.choice([0.2, 0.5, 1.0]), cached=_log(rng, 1, 16384) - 1,
                spread=rng.random() < 0.7, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                lse=rng.random() < 0.5, tag=tag)


def draw(rng):
    most = [work(c) for c in listed()]
    flops, nbytes = max(w["flops"] for w in most), max(w["bytes"] for w in most)
    while True:
        c = _draw(rng)
        w = work(c)
        if w["flops"] > flops or w["bytes"] > nbytes:
            continue
        if c["op"] == "attend":
            cached, new = lengths(c)
            kv = -(-(max(a + b for a, b in zip(cached, new))) // c["page"]) * c["page"]
            # what the plain form holds: scores over the padded batch, and the gathered cache
            if c["seqs"] * c["heads"] * max(new) * kv > 1.2e9 or c["seqs"] * c["kv_heads"] * c["head_dim"] * kv > 2.5e9:
                continue
            if c["dtype"] == "f32" and w["flops"] > 6e10:
                continue
        return c


def lengths(case):
    """(cached positions, new tokens) of every sequence."""
    r = random.Random(case["tag"])
    n, top, most = case["seqs"], case["cached"], case["new"]
    ragged = case.get("spread", True)
    cached = [top if i == 0 or not ragged else r.randint(0, top) for i in range(n)]
    new = []
    for i in range(n):
        chunk = i == 0 or r.random() < case["mix"]
        new.append((most if i == 0 or not ragged else r.randint(1, most)) if chunk else 1)
    return cached, new


def _finished(case):
    """Which sequences of a tables case end (never the first), and the new tokens without theirs."""
    cached, new = lengths(case)
    picks = random.Random(case["tag"] + 1).sample(range(1, case["seqs"]), min(case["done"], case["seqs"] - 1))
    done = [0] * case["seqs"]
    for i in picks:
        done[i], new[i] = 1, 0
    return cached, new, done


def _visible(case):
    """(query, key) pairs that a head computes, and cached positions that some query of it reads."""
    pairs = keys = 0
    w = case["window"]
    for c, n in zip(*lengths(case)):
        if w:
            for p in range(c, min(c + n, w)):  # the rows whose window is not full yet
                pairs += p + 1
            pairs += w * max(0, c + n - max(c, w))
            keys += min(c + n, n + w - 1)
        else:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
    return pairs, keys


def work(case):
    if case["op"] == "tables":
        cached, new, done = _finished(case)
        p, n = case["page"], case["seqs"]
        fresh = sum(-(-(c + m) // p) - -(-c // p) for c, m, d in zip(cached, new, done) if not d)
        freed = sum(-(-c // p) for c, d in zip(cached, done) if d)
        # lengths, flags and counts in and out; slots and positions; each page id moved once
        return {"bytes": n * (4 * 6) + 12 * sum(new) + 8 * (fresh + freed) + 16, "flops": 0}
    if case["op"] == "append":
        t = case["tokens"] - case["pad"]
        nq, nkv = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
        angles = min(t, case["positions"]) * case["head_dim"] * 4
        return {"bytes": t * (nq + 2 * nkv) * (BYTES[case["source"]] + BYTES[case["dtype"]]) + 12 * case["tokens"] + angles,
                "flops": t * (nq + nkv) * (7 if case["norm"] else 3)}
    pairs, keys = _visible(case)
    t = sum(lengths(case)[1])
    e, d = BYTES[case["dtype"]], case["head_dim"]
    nbytes = 2 * keys * case["kv_heads"] * d * e + 2 * t * case["heads"] * d * e
    return {"bytes": nbytes + (4 * t * case["heads"] if case["lse"] else 0), "flops": 4 * d * pairs * case["heads"]}


# ---------------------------------------------------------------- inputs
def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 17)
    s = {"case": case}
    page = case["page"]

    def randn(*shape, dtype=torch.float32, by=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(by).to(dtype)

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device="cuda")

    def pages(n):
        return torch.randperm(n, generator=g, device="cuda").to(torch.int32)

    if case["op"] == "tables":
        cached, new, done = _finished(case)
        held = [-(-c // page) for c in cached]
        fresh = sum(-(-(c + m) // page) for c, m in zip(cached, new)) - sum(held)
        n, total = case["seqs"], sum(held)
        ids = pages(total + fresh + 64)
        width = max(-(-(c + m) // page) for c, m in zip(cached, new)) + 1
        table = np.zeros((n, width), np.int64)
        at = 0
        for i, h in enumerate(held):
            table[i, :h] = np.arange(at, at + h)
            at += h
        s["table"] = ids[torch.from_numpy(table).cuda()].contiguous()
        s["free"] = torch.zeros(ids.numel(), dtype=torch.int32, device="cuda")
        s["free"][: ids.numel() - total] = ids[total:]
        s["n_free"] = ints([ids.numel() - total])
        s["length"], s["new"], s["done"] = ints(cached), ints(new), ints(done)
        # the buffers that a step writes; a few rows more than tokens, as in a step of fixed size
        rows = sum(new) + 13
        s["held"], s["n_mid"] = torch.zeros_like(s["length"]), torch.zeros_like(s["n_free"])
        s["after"], s["n_left"] = torch.zeros_like(s["length"]), torch.zeros_like(s["n_free"])
        s["cu"] = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        s["slot"] = torch.zeros(rows, dtype=torch.int64, device="cuda")
        s["pos"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        return s

    h, kvh, d, dt = case["heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    if case["op"] == "append":
        t, src = case["tokens"], DTYPES[case["source"]]
        n_pages = -(-t // page) + 5
        s["k_cache"] = randn(n_pages, kvh, page, d, dtype=dt)
        s["v_cache"] = randn(n_pages, kvh, page, d, dtype=dt)
        qkv = randn(t, (h + 2 * kvh) * d, dtype=src, by=1.3)  # one projection's rows
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([h * d, kvh * d, kvh * d], 1))
        slot = torch.randperm(n_pages * page, generator=g, device="cuda")[:t]
        if case["pad"]:
            slot[t - case["pad"]:] = -1
        s["slot"] = slot
        s["pos"] = torch.randint(0, case["positions"], (t,), generator=g, device="cuda", dtype=torch.int32)
        if case["norm"]:
            s["q_norm"], s["k_norm"] = 1 + randn(h * d, by=0.1), 1 + randn(kvh * d, by=0.1)
        angle = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            torch.tensor(10000.0, device="cuda", dtype=torch.float64),
            torch.arange(d // 2, device="cuda", dtype=torch.float64) * (-2.0 / d))
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_out"] = torch.zeros(t, h, d, dtype=dt, device="cuda")
        return s

    cached, new = lengths(case)
    total = [a + b for a, b in zip(cached, new)]
    blocks = [-(-x // page) for x in total]
    n_pages = sum(blocks) + 3
    s["k_cache"] = randn(n_pages, kvh, page, d, dtype=dt)
    s["v_cache"] = randn(n_pages, kvh, page, d, dtype=dt)
    ids, at = pages(n_pages), 0
    table = torch.zeros(case["seqs"], max(blocks), dtype=torch.int32, device="cuda")
    for i, b in enumerate(blocks):
        table[i, :b] = ids[at:at + b]
        at += b
    s["table"], s["length"] = table, ints(total)
    s["cu"] = ints([0] + list(np.cumsum(new)))
    s["q"] = randn(sum(new), h, d, dtype=dt, by=1.5)
    s["out"] = torch.zeros(sum(new), h, d, dtype=dt, device="cuda")
    s["lse"] = torch.zeros(sum(new), h, device="cuda") if case["lse"] else None
    s["max_new"] = max(new)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the handle that a program keeps beside its cache
        from rabbit2_b200 import paged

        if case["op"] == "tables":
            s["kv"] = paged.PagedTables(case["page"], s["free"].numel())
        else:
            s["kv"] = paged.PagedKv(s["k_cache"], s["v_cache"], n_heads=case["heads"])
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _own[op](s)
    return _plain[op](s)


def _own_tables(s):
    kv = s["kv"]
    kv.release(s["length"], s["done"], s["table"], s["free"], s["n_free"], s["held"], s["n_mid"])
    kv.plan(s["held"], s["new"], s["table"], s["free"], s["n_mid"], s["after"], s["n_left"], s["cu"], s["slot"], s["pos"])
    return _tables_out(s)


def _own_append(s):
    s["kv"].append(s["q"], s["k"], s["v"], s["slot"], s["pos"], s["q_out"], cos=s["cos"], sin=s["sin"],
                   q_norm=s.get("q_norm"), k_norm=s.get("k_norm"), eps=EPS)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attend(s):
    s["kv"].attention(s["q"], s["out"], s["cu"], s["length"], s["table"], s["max_new"], lse=s["lse"],
                      window=s["case"]["window"])
    return {"out": s["out"], "lse": s["lse"]}


def _tables_out(s):
    return {k: s[k] for k in ("held", "n_mid", "after", "n_left", "free", "table", "cu", "slot", "pos")}


def _plain_tables(s):
    page, table, free = s["case"]["page"], s["table"], s["free"]
    block = torch.arange(table.shape[1], device="cuda")
    # release: the pages of finished sequences go to the end of the free list, in order
    ended = s["done"] != 0
    gone = ended[:, None] & (block < ((s["length"] + page - 1) // page)[:, None])
    free[s["n_free"] + torch.arange(gone.sum(), device="cuda")] = table[gone]
    s["n_mid"].copy_(s["n_free"] + gone.sum())
    s["held"].copy_(torch.where(ended, 0, s["length"]))
    # plan: pages from the end of the free list, sequence by sequence, block by block
    old = (s["held"] + page - 1) // page
    s["after"].copy_(s["held"] + s["new"])
    fresh = (s["after"] + page - 1) // page - old
    first = torch.cumsum(fresh, 0) - fresh
    nth = first[:, None] + block - old[:, None]
    taken = (block >= old[:, None]) & (block < (old + fresh)[:, None])
    table.copy_(torch.where(taken, free[torch.where(taken, s["n_mid"] - 1 - nth, 0)], table))
    s["n_left"].copy_(s["n_mid"] - fresh.sum())
    s["cu"][1:] = torch.cumsum(s["new"], 0)
    row = torch.arange(s["slot"].numel(), device="cuda")
    seq = torch.searchsorted(s["cu"][1:].contiguous(), row, right=True)
    real = seq < table.shape[0]
    seq = torch.where(real, seq, 0)
    pos = torch.where(real, s["held"][seq] + row - s["cu"][seq], 0)
    s["pos"].copy_(pos)
    s["slot"].copy_(torch.where(real, table[seq, pos // page].long() * page + pos % page, -1))
    return _tables_out(s)


def _turn(x, cos, sin):
    """Rotation of (i, i + half) pairs by the row's angles."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    page, dt = s["case"]["page"], s["k_cache"].dtype
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if "q_norm" in s:
        q = q * torch.rsqrt(q.square().mean((1, 2), keepdim=True) + EPS) * s["q_norm"].view(q.shape[1:])
        k = k * torch.rsqrt(k.square().mean((1, 2), keepdim=True) + EPS) * s["k_norm"].view(k.shape[1:])
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    q, k = _turn(q, cos, sin), _turn(k, cos, sin)
    real = (s["slot"] >= 0).nonzero()[:, 0]
    slot = s["slot"][real]
    s["q_out"][real] = q[real].to(dt)
    s["k_cache"][slot // page, :, slot % page] = k[real].to(dt)
    s["v_cache"][slot // page, :, slot % page] = v[real].to(dt)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    c = s["case"]
    h, kvh, d, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    table, cu, length = s["table"].long(), s["cu"].long(), s["length"].long()
    n, most, group = table.shape[0], s["max_new"], h // kvh
    # the batch padded to its longest: pages gathered per sequence, rows per sequence
    k = s["k_cache"][table].float().transpose(1, 2).reshape(n, kvh, -1, d)
    v = s["v_cache"][table].float().transpose(1, 2).reshape(n, kvh, -1, d)
    new = cu[1:] - cu[:-1]
    step = torch.arange(most, device="cuda")
    real = step < new[:, None]
    row = torch.where(real, cu[:-1, None] + step, 0)
    q = s["q"][row].float().view(n, most, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * most, d)
    at = (length - new)[:, None] + step  # each row's position
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= at[..., None]) & real[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    score = torch.matmul(q, k.transpose(2, 3)).view(n, kvh, group, most, -1).mul_(1 / math.sqrt(d))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kvh, group * most, -1), v).view(n, kvh, group, most, d) / total
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, most, h, d)[real])
    if s["lse"] is not None:
        s["lse"].copy_((top + total.log()).permute(0, 3, 1, 2, 4).reshape(n, most, h)[real])
    return {"out": s["out"], "lse": s["lse"]}


_plain = {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}
_own = {"tables": _own_tables, "append": _own_append, "attend": _own_attend}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    if case["op"] == "tables":
        return None  # whole numbers
    s = _inputs(case, seed)
    page, d = case["page"], case["head_dim"]
    if case["op"] == "append":
        out = {"q": s["q_out"].double(), "k_cache": s["k_cache"].double(), "v_cache": s["v_cache"].double()}
        at = torch.nonzero(s["slot"] >= 0).flatten()
        rot = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"][at].long()][:, None, :]
        to = {"q": None, "k": "k_cache", "v": "v_cache"}
        for name, cache in to.items():
            x = s[name][at].double()
            if name != "v":
                if case["norm"]:
                    flat = x.flatten(1)
                    flat = flat / (flat.pow(2).sum(1, keepdim=True) / flat.shape[1] + EPS).sqrt()
                    x = (flat * s[name + "_norm"].double()).view_as(x)
                z = torch.complex(x[..., : d // 2], x[..., d // 2:]) * rot
                x = torch.cat((z.real, z.imag), 2)
            if cache is None:
                out["q"][at] = x
            else:
                slot = s["slot"][at]
                out[cache][torch.div(slot, page, rounding_mode="floor"), :, torch.remainder(slot, page)] = x
        return out
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    cached, new = lengths(case)
    start = 0
    for i, (c, t) in enumerate(zip(cached, new)):
        ids = s["table"][i, : -(-(c + t) // page)].long()
        for j in range(case["kv_heads"]):
            k = s["k_cache"][ids, j].reshape(-1, d)[: c + t].double()
            v = s["v_cache"][ids, j].reshape(-1, d)[: c + t].double()
            for a in range(0, t, 2048):  # rows at a time
                b = min(t, a + 2048)
                q = s["q"][start + a:start + b, j * group:(j + 1) * group].double()
                x = torch.einsum("tgd,kd->tgk", q, k) / math.sqrt(d)
                pos = torch.arange(c + a, c + b, device="cuda")[:, None, None]
                key = torch.arange(c + t, device="cuda")
                hidden = key > pos
                if case["window"]:
                    hidden = hidden | (key <= pos - case["window"])
                x = x.masked_fill(hidden, -math.inf)
                out[start + a:start + b, j * group:(j + 1) * group] = torch.einsum("tgk,kd->tgd", torch.softmax(x, -1), v)
                lse[start + a:start + b, j * group:(j + 1) * group] = torch.logsumexp(x, -1)
        start += t
    return {"out": out, "lse": lse if case["lse"] else None}
