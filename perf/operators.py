"""The operators of a paged key-value cache and of beam search, as cases that can be timed and compared.

A case is a dict of plain values with an "op":

  token   attention of one new token per row over the row's pages (``attend_token``)
  chunk   causal attention of several new tokens per row over the row's pages, with or without a sliding window and
          first tokens that stay visible (``attend_chunk``)
  fork    a beam step's page work: rows take their parents' pages, the page that is written next becomes the row's
          own by a copy where it is shared, new pages are given out (``advance_pages``)
  tidy    pages that fell out of the window and those of finished rows are given back, the rest move together
          (``free_pages``, ``compact_pages``)
  beam    the best continuations over beams and vocabulary, and the states that follow them (``beam_select``,
          ``reorder_states``)

With ``own`` false the operators run in elementary torch operations, with ``own`` true as this package's calls.
Lengths, page numbers and parents follow from the case alone, the values from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # batch-1 decode after a short prompt: what one layer of the largest configured decoder asks for, all latency
        dict(name="token_1x577", op="token", rows=1, longest=577, heads=64, kv_heads=8, dim=128, page=64, window=0,
             sinks=0, dtype="bf16"),
        # a few conversations of different lengths
        dict(name="token_8x4100", op="token", rows=8, longest=4100, heads=64, kv_heads=8, dim=128, page=64, window=0,
             sinks=0, dtype="bf16"),
        # a full server with long contexts
        dict(name="token_48x16384", op="token", rows=48, longest=16384, heads=32, kv_heads=8, dim=128, page=64,
             window=0, sinks=0, dtype="fp16"),
        # streaming over far more tokens than are kept visible, small pages, heads that do not fill a tile
        dict(name="token_32x31000_window", op="token", rows=32, longest=31000, heads=28, kv_heads=4, dim=128, page=16,
             window=4096, sinks=4, dtype="bf16"),
        # a prompt of the greedy benchmark's length into an empty cache
        dict(name="chunk_512", op="chunk", rows=1, new=512, cached=0, heads=64, kv_heads=8, dim=128, page=64, window=0,
             sinks=0, dtype="bf16"),
        # a long document under a sliding window
        dict(name="chunk_8192_window", op="chunk", rows=1, new=8192, cached=0, heads=32, kv_heads=8, dim=128, page=64,
             window=1024, sinks=4, dtype="bf16"),
        # second turns of several conversations: new tokens behind what the cache holds, every row of another length
        dict(name="chunk_6x1500_cached", op="chunk", rows=6, new=1500, cached=4000, heads=28, kv_heads=4, dim=128,
             page=32, window=0, sinks=0, dtype="fp16"),
        # one request with four beams on a small model
        dict(name="fork_1x4", op="fork", groups=1, beams=4, layers=4, length=597, prompt=512, pages=64, kv_heads=2,
             dim=128, page=64, dtype="bf16"),
        # eight requests with four beams each
        dict(name="fork_8x4", op="fork", groups=8, beams=4, layers=16, length=2039, prompt=1500, pages=640, kv_heads=8,
             dim=128, page=64, dtype="bf16"),
        # a streaming server that hands memory back
        dict(name="tidy_24", op="tidy", rows=24, layers=8, longest=6000, pages=2048, kv_heads=4, dim=128, page=32,
             window=2048, sinks=4, dtype="bf16"),
        # one request's selection over the largest configured vocabulary
        dict(name="beam_1x4", op="beam", batch=1, beams=4, vocab=151936, keep=4, history=640, dtype="bf16"),
        # many requests, fp32 logits, some beams finished
        dict(name="beam_32x8", op="beam", batch=32, beams=8, vocab=151936, keep=8, history=1000, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["token", "chunk", "fork", "tidy", "beam"])
    while True:
        if op == "token":
            c = dict(op=op, rows=_log(rng, 1, 64), longest=_log(rng, 1, 32000), kv_heads=rng.choice([1, 2, 3, 4, 8]),
                     dim=rng.choice([64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]),
                     window=rng.choice([0, 0, _log(rng, 1, 8192)]), dtype=rng.choice(["bf16", "fp16"]))
            c["heads"] = c["kv_heads"] * rng.choice([1, 3, 4, 7, 8, 16])
            c["sinks"] = rng.choice([0, 1, 4, 20]) if c["window"] else 0
            seen = min(c["longest"], c["window"] + c["sinks"] or c["longest"])
            if c["rows"] * seen * c["kv_heads"] * c["dim"] <= 48 * 16384 * 8 * 128 \
                    and c["rows"] * c["longest"] * c["kv_heads"] * c["dim"] <= 1 << 31:
                return c
        elif op == "chunk":
            c = dict(op=op, rows=_log(rng, 1, 12), new=_log(rng, 1, 6000), cached=rng.choice([0, _log(rng, 1, 6000)]),
                     kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64, 128]),
                     window=rng.choice([0, 0, _log(rng, 1, 4096)]), dtype=rng.choice(["bf16", "fp16"]))
            c["heads"] = c["kv_heads"] * rng.choice([1, 4, 7, 8])
            c["sinks"] = rng.choice([0, 1, 4, 20]) if c["window"] else 0
            if c["rows"] * c["heads"] * c["new"] * (c["new"] + c["cached"]) <= 1.5e9:
                return c
        elif op == "fork":
            c = dict(op=op, groups=_log(rng, 1, 16), beams=rng.randint(2, 8), layers=rng.randint(1, 16),
                     length=_log(rng, 2, 4096), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                     page=rng.choice([16, 32, 64]), dtype=rng.choice(["bf16", "fp16"]))
            c["prompt"] = rng.randint(1, c["length"] - 1)
            c["pages"] = c["groups"] * (c["prompt"] // c["page"] + 1 + c["beams"]
                                        * ((c["length"] - c["prompt"]) // c["page"] + 4)) + rng.randint(0, 200)
            if c["pages"] * c["layers"] * 2 * c["kv_heads"] * c["page"] * c["dim"] <= 640 * 16 * 2 * 8 * 64 * 128:
                return c
        elif op == "tidy":
            c = dict(op=op, rows=_log(rng, 1, 48), layers=rng.randint(1, 8), longest=_log(rng, 20, 8000),
                     kv_heads=rng.choice([1, 2, 4]), dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64]),
                     window=_log(rng, 8, 4096), sinks=rng.choice([0, 1, 4, 20]), dtype=rng.choice(["bf16", "fp16"]))
            c["pages"] = c["rows"] * (min(c["longest"], 2 * c["window"]) // c["page"] + 4) + rng.randint(1, 300)
            if c["pages"] * c["layers"] * 2 * c["kv_heads"] * c["page"] * c["dim"] <= 2048 * 8 * 2 * 4 * 32 * 128:
                return c
        else:
            c = dict(op=op, batch=_log(rng, 1, 64), beams=rng.randint(1, 16), vocab=_log(rng, 50, 151936),
                     history=_log(rng, 1, 2000), dtype=rng.choice(["bf16", "fp16", "fp32"]))
            c["keep"] = rng.choice([c["beams"], 2 * c["beams"]])
            if c["batch"] * c["beams"] * c["vocab"] <= 32 * 8 * 151936:
                return c


# ---------------------------------------------------------------------------
# what follows from the case: lengths, tables, parents
# ---------------------------------------------------------------------------

def _rng(c):
    return random.Random(" ".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))


def _ragged(c):
    """token: length per row.  chunk: (new tokens, cached tokens) per row.  The first row has the most."""
    r = _rng(c)
    if c["op"] == "token":
        return [c["longest"]] + [r.randint(1, c["longest"]) for _ in range(c["rows"] - 1)]
    new = [c["new"]] + [r.randint(1, c["new"]) for _ in range(c["rows"] - 1)]
    return new, [c["cached"]] + [r.randint(0, c["cached"]) for _ in range(c["rows"] - 1)]


def _scattered(lengths, page, r, spare=3):
    """A table whose rows hold pages in no order, and the number of pages."""
    need = [-(-n // page) for n in lengths]
    pages = list(range(sum(need) + spare))
    r.shuffle(pages)
    table = np.full((len(lengths), max(need) + 1), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = pages[at:at + n]
        at += n
    return table, len(pages)


def _fork_books(c):
    """Table, lengths, reference counts and parents of a beam step: the beams of a request share the prompt's full
    pages and go on with their own; some beams are dropped, others continue twice."""
    r, page, K = _rng(c), c["page"], c["beams"]
    free = list(range(c["pages"]))
    r.shuffle(free)
    rows = c["groups"] * K
    table = np.full((rows, (c["length"] + 64) // page + 2), -1, np.int32)
    lengths = np.zeros(rows, np.int32)
    parents = np.zeros(rows, np.int32)
    for g in range(c["groups"]):
        n = c["length"] if g == 0 else r.randint(c["prompt"] + 1, c["length"])
        held = -(-n // page)
        shared = c["prompt"] // page
        common = [free.pop() for _ in range(shared)]
        for b in range(K):
            i = g * K + b
            table[i, :held] = common[:held] + [free.pop() for _ in range(held - shared)]
            lengths[i] = n
            parents[i] = g * K + r.choice([0, b, r.randrange(K)])
    refs = np.bincount(table[table >= 0], minlength=c["pages"]).astype(np.int32)
    return table, lengths, refs, parents


def _tidy_books(c):
    """Table, lengths, reference counts and the rows that go on: every row still holds up to a window of pages that
    it no longer sees."""
    r, page = _rng(c), c["page"]
    free = list(range(c["pages"]))
    r.shuffle(free)
    lengths = [c["longest"]] + [r.randint(1, c["longest"]) for _ in range(c["rows"] - 1)]
    table = np.full((c["rows"], -(-c["longest"] // page) + 1), -1, np.int32)
    for i, n in enumerate(lengths):
        for p in range(-(-n // page)):
            if p * page < c["sinks"] or (p + 1) * page > n - c["window"] - r.randint(0, c["window"]):
                if free:
                    table[i, p] = free.pop()
    refs = np.bincount(table[table >= 0], minlength=c["pages"]).astype(np.int32)
    keep = np.array([r.random() < 0.85 for _ in range(c["rows"])])
    keep[0] = True
    return table, np.array(lengths, np.int32), refs, keep


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _values(shape, gen, dtype, scale=1.0):
    """Normal values, made in pieces so that a large pool needs no fp32 copy of its own."""
    x = torch.empty(shape, dtype=dtype, device=DEV)
    flat = x.view(-1)
    for part in flat.split(1 << 28):
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV).mul_(scale))
    return x


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c, "op": c["op"]}
    if c["op"] in ("token", "chunk"):
        if c["op"] == "token":
            lengths = _ragged(c)
            tokens = c["rows"]
        else:
            new, cached = _ragged(c)
            lengths = [a + b for a, b in zip(new, cached)]
            tokens = sum(new)
            s["starts"] = _gpu(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
            s["most"] = max(new)
        table, pages = _scattered(lengths, c["page"], _rng(c))
        shape = (pages, c["kv_heads"], c["page"], c["dim"])
        # keys with a few strong channels, so that some positions get most of a query's weight
        s["k"] = _values(shape, gen, dt)
        s["k"][..., ::17] *= 2.5
        s["v"] = _values(shape, gen, dt)
        s["q"] = _values((tokens, c["heads"], c["dim"]), gen, dt)
        s["table"], s["lengths"] = _gpu(table), _gpu(np.array(lengths, np.int32))
        s["scale"] = c["dim"] ** -0.5
    elif c["op"] in ("fork", "tidy"):
        s["kv"] = _values((c["layers"], 2, c["pages"], c["kv_heads"], c["page"], c["dim"]), gen, dt)
        books = _fork_books(c) if c["op"] == "fork" else _tidy_books(c)
        s["table"], s["lengths"], s["refs"], s["rows"] = (_gpu(b) for b in books)
    else:
        n = c["batch"] * c["beams"]
        x = torch.randn(n, c["vocab"], generator=gen, device=DEV).mul_(2.0)
        # a handful of likely tokens per row
        hot = torch.randint(0, c["vocab"], (n, 12), generator=gen, device=DEV)
        x.scatter_(1, hot, torch.rand(n, 12, generator=gen, device=DEV) * 4 + 9)
        s["logits"] = x.to(dt)
        s["scores"] = -30 * torch.rand(c["batch"], c["beams"], generator=gen, device=DEV).sort(dim=1)[0]
        s["finished"] = torch.rand(c["batch"], c["beams"], generator=gen, device=DEV) < 0.1
        s["eos"] = c["vocab"] // 3
        s["history"] = torch.randint(0, c["vocab"], (n, c["history"]), generator=gen, device=DEV)
        s["marks"] = torch.randint(0, 1 << 20, (n,), generator=gen, device=DEV, dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _own(s) if own else PLAIN[s["op"]](s)


def _own(s):
    from quipsharp_amd import beam, pages

    c = s["case"]
    if s["op"] == "token":
        return pages.attend_token(s["q"], s["k"], s["v"], s["table"], s["lengths"], scale=s["scale"],
                                  window=c["window"], sinks=c["sinks"])
    if s["op"] == "chunk":
        return pages.attend_chunk(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["starts"], scale=s["scale"],
                                  window=c["window"], sinks=c["sinks"])
    if s["op"] == "fork":
        table, lengths, refs, _ = pages.advance_pages(s["kv"], s["table"], s["lengths"], s["refs"], tokens=1,
                                                      parents=s["rows"])
        return s["kv"], table, lengths, refs
    if s["op"] == "tidy":
        table, lengths, refs = pages.free_pages(s["table"], s["lengths"], s["refs"], page=c["page"], keep=s["rows"],
                                                window=c["window"], sinks=c["sinks"])
        table, refs = pages.compact_pages(s["kv"], table, refs)
        return s["kv"], table, lengths, refs
    scores, parents, tokens = beam.beam_select(s["logits"], s["scores"], keep=c["keep"], finished=s["finished"],
                                               eos=s["eos"])
    history, marks = beam.reorder_states([s["history"], s["marks"]], parents)
    return scores, parents, tokens, history, marks


def _attend(q, k, v, where, scale):
    """q (R, H, n, d), k and v (R, Hk, L, d) of any type, where (R, n, L): softmax over the positions that it allows."""
    R, H, n, d = q.shape
    Hk, L = k.shape[1:3]
    q = q.float().reshape(R, Hk, (H // Hk) * n, d)
    x = torch.matmul(q, k.float().transpose(2, 3).contiguous()).mul_(scale)
    x = x.view(R, Hk, H // Hk, n, L).masked_fill_(~where[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(R, Hk, (H // Hk) * n, L), v.float()).view(R, Hk, H // Hk, n, d)
    return (o / torch.where(total == 0, 1.0, total)).reshape(R, H, n, d)


def _gathered(pool, table):
    """(rows, kv heads, positions, dim) of every row's pages."""
    g = pool[table.clamp(min=0).long()]
    return g.transpose(1, 2).reshape(g.shape[0], g.shape[2], -1, g.shape[4])


def _visible(c, where, last):
    """Whether positions `where` are seen by a query at position `last`."""
    seen = where <= last
    return seen & ((where > last - c["window"]) | (where < c["sinks"])) if c["window"] else seen


def _plain_token(s):
    c = s["case"]
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    where = torch.arange(k.shape[2], device=DEV)
    ok = _visible(c, where[None, None, :], (s["lengths"] - 1)[:, None, None])
    return _attend(s["q"][:, :, None], k, v, ok, s["scale"])[:, :, 0].to(s["q"].dtype)


def _plain_chunk(s):
    c = s["case"]
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    starts = s["starts"].long()
    count = starts[1:] - starts[:-1]
    j = torch.arange(s["most"], device=DEV)
    inside = j[None, :] < count[:, None]
    token = torch.where(inside, starts[:-1, None] + j, 0)
    last = (s["lengths"].long() - count)[:, None] + j
    ok = _visible(c, torch.arange(k.shape[2], device=DEV)[None, None, :], last[:, :, None]) & inside[:, :, None]
    o = _attend(s["q"][token].transpose(1, 2), k, v, ok, s["scale"])
    return o.transpose(1, 2)[inside].to(s["q"].dtype)


def _plain_fork(s):
    kv, refs = s["kv"], s["refs"]
    page, P = kv.shape[4], kv.shape[2]
    table, length = s["table"][s["rows"].long()], s["lengths"][s["rows"].long()].long()
    rows, cols = table.shape
    i, col = torch.arange(rows, device=DEV), torch.arange(cols, device=DEV)
    # who else holds the page that the row writes next: the longest of them keeps it, the first where they are alike
    c0, used = length // page, length % page
    mine = table.gather(1, c0[:, None])
    held = (table.t()[c0] == mine) & (used > 0)[:, None] & (mine >= 0)
    ahead = (length[None, :] > length[:, None]) | ((length[None, :] == length[:, None]) & (i[None, :] < i[:, None]))
    copy = (held & ahead).any(1)
    count = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    count.scatter_add_(0, torch.where(table < 0, P, table).view(-1).long(), torch.ones_like(table).view(-1))
    free = torch.argsort((count[:P] > 0).int(), stable=True)
    # one page for a copy, one where the next token begins a page; free pages in their order
    want = (col == c0[:, None]) & (copy | (used == 0))[:, None]
    nth = want.view(-1).long().cumsum(0).view(rows, cols) - 1
    given = torch.where(nth < (count[:P] == 0).sum(), free[nth.clamp(0, P - 1)].int(), -1)
    src, dst, n = mine[copy, 0].long(), given.gather(1, c0[:, None])[copy, 0].long(), used[copy]
    inside = torch.arange(page, device=DEV)[None, :] < n[:, None]
    kv[:, :, dst] = torch.where(inside[None, None, :, None, :, None], kv[:, :, src], kv[:, :, dst])
    table = torch.where(want, given, table)
    refs = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    refs.scatter_add_(0, torch.where(table < 0, P, table).view(-1).long(), torch.ones_like(table).view(-1))
    return kv, table, (length + 1).int(), refs[:P]


def _plain_tidy(s):
    c, kv = s["case"], s["kv"]
    table, lengths, P = s["table"], s["lengths"], kv.shape[2]
    at = torch.arange(table.shape[1], device=DEV) * c["page"]
    gone = (at >= c["sinks"])[None, :] & ((at + c["page"])[None, :] <= (lengths - c["window"] + 1)[:, None])
    table = torch.where(gone | ~s["rows"][:, None], -1, table)
    lengths = torch.where(s["rows"], lengths, 0)
    refs = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
    refs.scatter_add_(0, torch.where(table < 0, P, table).view(-1).long(), torch.ones_like(table).view(-1))
    refs = refs[:P]
    live, page = refs > 0, torch.arange(P, device=DEV)
    n = live.sum()
    src, dst = page[live & (page >= n)], page[~live & (page < n)]
    kv[:, :, dst] = kv[:, :, src]
    to = page.clone()
    to[src] = dst
    out = refs.clone()
    out[dst] = refs[src]
    out[src] = 0
    return kv, torch.where(table >= 0, to[table.clamp(min=0).long()].int(), -1), lengths, out


def _plain_beam(s):
    c = s["case"]
    B, K, V = c["batch"], c["beams"], c["vocab"]
    x = s["logits"].view(B, K, V).double()
    x = x - x.amax(-1, keepdim=True)
    x = x - x.exp().sum(-1, keepdim=True).log()
    only = torch.where(torch.arange(V, device=DEV) == s["eos"], 0.0, -math.inf).double()
    x = torch.where(s["finished"][:, :, None], only, x) + s["scores"][:, :, None]
    top, at = torch.sort(x.view(B, K * V), dim=1, descending=True, stable=True)
    top, at = top[:, :c["keep"]], at[:, :c["keep"]]
    parents = at // V + torch.arange(B, device=DEV)[:, None] * K
    rows = parents.view(-1)
    return top.float(), parents.int(), (at % V).int(), s["history"][rows], s["marks"][rows]


PLAIN = {"token": _plain_token, "chunk": _plain_chunk, "fork": _plain_fork, "tidy": _plain_tidy, "beam": _plain_beam}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _tail(first, last, c):
    """Positions that queries at positions first .. last - 1 see, together, and the number of (query, position) pairs."""
    w, sinks = c["window"], c["sinks"]
    if not w:
        return last, (last * (last + 1) - first * (first + 1)) // 2
    low = max(0, first - w + 1)
    pairs = sum(min(p + 1, w) + min(sinks, max(0, p - w + 1)) for p in range(first, last))
    return last - low + min(sinks, low), pairs


def work(case):
    c, size = case, torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if c["op"] in ("token", "chunk"):
        if c["op"] == "token":
            spans = [(n - 1, n) for n in _ragged(c)]
        else:
            spans = [(b, a + b) for a, b in zip(*_ragged(c))]
        seen = [_tail(*t, c) for t in spans]
        tokens = sum(b - a for a, b in spans)
        return {"bytes": size * c["dim"] * (2 * c["kv_heads"] * sum(n for n, _ in seen) + 2 * c["heads"] * tokens),
                "flops": 4 * c["dim"] * c["heads"] * sum(p for _, p in seen)}
    row = c["layers"] * 2 * c["kv_heads"] * c["dim"] * size if c["op"] != "beam" else 0
    if c["op"] == "fork":
        table, lengths, refs, parents = _fork_books(c)
        # every further row of a partly filled page copies what the page holds
        copies = sum(int(lengths[p]) % c["page"] for i, p in enumerate(parents) if p in parents[:i])
        return {"bytes": 2 * copies * row + 8 * table.size + 8 * refs.size + 12 * lengths.size, "flops": 0}
    if c["op"] == "tidy":
        table, lengths, refs, keep = _tidy_books(c)
        at = np.arange(table.shape[1]) * c["page"]
        gone = (at >= c["sinks"])[None] & (at[None] + c["page"] <= lengths[:, None] - c["window"] + 1)
        left = table[(table >= 0) & ~gone & keep[:, None]]
        moves = int((left >= left.size).sum())
        return {"bytes": 2 * moves * c["page"] * row + 8 * table.size + 8 * refs.size + 8 * lengths.size, "flops": 0}
    n, keep = c["batch"] * c["beams"], c["batch"] * c["keep"]
    return {"bytes": n * c["vocab"] * size + 5 * n + keep * (12 + 2 * (8 * c["history"] + 4)),
            "flops": 3 * n * c["vocab"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"token": _exact_attention, "chunk": _exact_attention, "fork": _exact_fork, "tidy": _exact_tidy,
            "beam": _exact_beam}[case["op"]](case, s)


def _exact_attention(c, s):
    if c["op"] == "token":
        spans = [(n - 1, n) for n in _ragged(c)]
    else:
        spans = [(b, a + b) for a, b in zip(*_ragged(c))]
    out, t, group = [], 0, c["heads"] // c["kv_heads"]
    table = s["table"].cpu()
    for r, (first, last) in enumerate(spans):
        ids = table[r, :-(-last // c["page"])].long().to(DEV)
        query = torch.arange(first, last, device=DEV)[:, None]
        key = torch.arange(last, device=DEV)[None, :]
        ok = key <= query
        if c["window"]:
            ok = ok & ((query - key < c["window"]) | (key < c["sinks"]))
        heads = []
        for h in range(c["kv_heads"]):
            k = s["k"][ids, h].reshape(-1, c["dim"])[:last].double()
            v = s["v"][ids, h].reshape(-1, c["dim"])[:last].double()
            kt = k.t().contiguous()
            for g in range(group):
                x = (s["q"][t:t + last - first, h * group + g].double() @ kt) / math.sqrt(c["dim"])
                heads.append(torch.softmax(torch.where(ok, x, -math.inf), 1) @ v)
        out.append(torch.stack(heads, 1))
        t += last - first
    return torch.cat(out)


def _exact_fork(c, s):
    table, lengths, refs, parents = _fork_books(c)
    page, kv = c["page"], s["kv"].double()
    now = [[p for p in table[q].tolist() if p >= 0] for q in parents.tolist()]
    length = [int(lengths[q]) for q in parents.tolist()]
    taken = {p for row in now for p in row}
    free = [p for p in range(c["pages"]) if p not in taken]
    writer = {}  # the row that goes on in a page which several rows hold
    for i, row in enumerate(now):
        if length[i] % page and (row[-1] not in writer or length[writer[row[-1]]] < length[i]):
            writer[row[-1]] = i
    for i, row in enumerate(now):
        if length[i] % page == 0:
            row.append(free.pop(0))
        elif writer[row[-1]] != i:
            new = free.pop(0)
            kv[:, :, new, :, :length[i] % page] = kv[:, :, row[-1], :, :length[i] % page]
            row[-1] = new
    after, held = np.full(table.shape, -1, np.int32), np.zeros(c["pages"], np.int32)
    for i, row in enumerate(now):
        after[i, :len(row)] = row
        for p in row:
            held[p] += 1
    return kv, after, np.array(length, np.int32) + 1, held


def _exact_tidy(c, s):
    table, lengths, _, keep = _tidy_books(c)
    kv, page = s["kv"].double(), c["page"]
    for i in range(len(lengths)):
        for p in range(table.shape[1]):
            # no later token sees any position of the page
            unseen = all(j >= c["sinks"] and j <= int(lengths[i]) - c["window"] for j in (p * page, p * page + page - 1))
            if not keep[i] or unseen:
                table[i, p] = -1
        if not keep[i]:
            lengths[i] = 0
    held = sorted(set(table[table >= 0].tolist()))
    n = len(held)
    low = set(held)
    to = dict(zip([p for p in held if p >= n], [p for p in range(n) if p not in low]))
    if to:
        kv[:, :, list(to.values())] = kv[:, :, list(to.keys())]
    refs = np.zeros(c["pages"], np.int32)
    for i in range(table.shape[0]):
        for p in range(table.shape[1]):
            if table[i, p] >= 0:
                table[i, p] = to.get(int(table[i, p]), int(table[i, p]))
                refs[table[i, p]] += 1
    return kv, table, lengths, refs


def _exact_beam(c, s):
    B, K, V, keep = c["batch"], c["beams"], c["vocab"], c["keep"]
    best = []
    for b in range(B):
        total = torch.log_softmax(s["logits"][b * K:(b + 1) * K].double(), 1) + s["scores"][b].double()[:, None]
        for j in range(K):
            if bool(s["finished"][b, j]):
                total[j] = -math.inf
                total[j, s["eos"]] = s["scores"][b, j].double()
        edge = torch.topk(total.view(-1), keep)[0][-1]
        at = torch.nonzero(total.view(-1) >= edge)[:, 0].tolist()
        value = total.view(-1)[at].tolist() if len(at) < 1 << 20 else None
        if value is None:
            return None
        best.append(sorted(zip([-x for x in value], at))[:keep])
    scores = torch.tensor([[-x for x, _ in row] for row in best], dtype=torch.float64)
    parents = torch.tensor([[b * K + i // V for _, i in row] for b, row in enumerate(best)], dtype=torch.int32)
    tokens = torch.tensor([[i % V for _, i in row] for row in best], dtype=torch.int32)
    rows = parents.view(-1).long().to(DEV)
    return scores, parents, tokens, s["history"][rows], s["marks"][rows]
