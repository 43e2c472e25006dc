"""The operators of a served decoder's step around its quantized linears, as cases that can be timed and compared.

A case is a dict of plain values with an "op":

  adapt  low-rank adapters of many requests beside up to four projections of one input (``add_adapters``): single
         tokens, each with an adapter of its own, or prompts
  rope   rotary positions of new tokens: queries turned, keys turned and stored with their values in the pages
         (``append_rotated``); pairs of half a head apart or side by side, all or part of a head, scaled frequencies
  score  log probabilities of given tokens with entropy, rank and the best alternatives (``token_logprobs``)

With ``own`` false the operators run in elementary torch operations, with ``own`` true as this package's calls.
Lengths, page numbers and the requests' adapters follow from the case alone, the values from the seed.
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
        # one request's token beside the q, k and v projections of an 8B decoder: all latency
        dict(name="adapt_1_qkv", op="adapt", rows=1, new=1, prompt=False, count=8, rank=16, n=4096, m="4096,1024,1024",
             dtype="bf16"),
        # a full server, most requests with an adapter of their own, beside the widest configured gate and up
        dict(name="adapt_48_gate_up", op="adapt", rows=48, new=1, prompt=False, count=24, rank=64, n=5120,
             m="25600,25600", dtype="bf16"),
        # several prompts of different lengths, each with its adapter, widths with odd factors
        dict(name="adapt_prompts_6x900", op="adapt", rows=6, new=900, prompt=True, count=6, rank=24, n=3584,
             m="3584,512,512", dtype="fp16"),
        # long documents beside the widest down projection
        dict(name="adapt_prompts_3x4096_down", op="adapt", rows=3, new=4096, prompt=True, count=4, rank=64, n=25600,
             m="5120", dtype="bf16"),
        # one token of the largest configured decoder, far into a stretched context: all latency
        dict(name="rope_1", op="rope", rows=1, new=1, cached=120000, heads=64, kv_heads=8, dim=128, rotary=128, page=64,
             layout="half", scaling="yarn", fused=False, dtype="bf16"),
        # a full server's step, q, k and v in one tensor, half of each head turned, pairs side by side
        dict(name="rope_48_part", op="rope", rows=48, new=1, cached=30000, heads=28, kv_heads=4, dim=128, rotary=64,
             page=16, layout="interleaved", scaling="none", fused=True, dtype="fp16"),
        # second turns of several conversations
        dict(name="rope_6x1500", op="rope", rows=6, new=1500, cached=4000, heads=28, kv_heads=4, dim=128, rotary=128,
             page=32, layout="half", scaling="linear", fused=False, dtype="fp16"),
        # a long document's prompt
        dict(name="rope_8192", op="rope", rows=1, new=8192, cached=0, heads=32, kv_heads=8, dim=128, rotary=128,
             page=64, layout="half", scaling="llama3", fused=False, dtype="bf16"),
        # the token that a request just took, over the largest configured vocabulary
        dict(name="score_1", op="score", rows=1, vocab=151936, top=5, masked=False, dtype="bf16"),
        # a full server, fp32 logits, some of the rows limited to a few tokens
        dict(name="score_48_masked", op="score", rows=48, vocab=151936, top=20, masked=True, dtype="fp32"),
        # one evaluation window of a 7B decoder
        dict(name="score_2047", op="score", rows=2047, vocab=32000, top=0, masked=False, dtype="fp32"),
        # a prompt's log probabilities with alternatives
        dict(name="score_1500", op="score", rows=1500, vocab=151936, top=10, masked=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["adapt", "rope", "score"])
    while True:
        if op == "adapt":
            c = dict(op=op, rows=_log(rng, 1, 64), new=1, prompt=rng.random() < 0.5, count=_log(rng, 1, 32),
                     rank=8 * _log(rng, 1, 16), n=8 * _log(rng, 8, 3200), dtype=rng.choice(["bf16", "fp16"]))
            c["m"] = ",".join(str(_log(rng, 30, 25600)) for _ in range(rng.randint(1, 4)))
            if c["prompt"]:
                c["rows"], c["new"] = min(c["rows"], 8), _log(rng, 2, 4096)
            out = sum(_widths(c))
            if c["count"] * c["rank"] * (c["n"] + out) <= 24 * 64 * (2 * 5120 + 51200) \
                    and c["rows"] * c["new"] * (c["n"] + 2 * out) <= 3 * 4096 * (25600 + 2 * 5120):
                return c
        elif op == "rope":
            c = dict(op=op, rows=_log(rng, 1, 64), new=rng.choice([1, _log(rng, 1, 8192)]), cached=_log(rng, 1, 200000),
                     kv_heads=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([64, 96, 128, 128, 256]),
                     page=rng.choice([16, 32, 64, 128]), layout=rng.choice(["half", "interleaved"]),
                     scaling=rng.choice(["none", "linear", "llama3", "yarn"]), fused=rng.random() < 0.3,
                     dtype=rng.choice(["bf16", "fp16"]))
            c["cached"] -= 1
            c["heads"] = c["kv_heads"] * rng.choice([1, 3, 4, 7, 8])
            c["rotary"] = c["dim"] // rng.choice([1, 1, 2, 4])
            if c["rows"] * c["new"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] <= 8192 * 48 * 128:
                return c
        else:
            c = dict(op=op, rows=_log(rng, 1, 4096), vocab=_log(rng, 50, 151936), top=rng.choice([0, 1, 5, 20, 64]),
                     masked=rng.random() < 0.3, dtype=rng.choice(["bf16", "fp16", "fp32"]))
            c["top"] = min(c["top"], c["vocab"] // 2)
            if c["rows"] * c["vocab"] <= 1500 * 151936 // (2 if c["dtype"] == "fp32" else 1):
                return c


# ---------------------------------------------------------------------------
# what follows from the case: lengths, tables, adapters, frequencies
# ---------------------------------------------------------------------------

def _rng(c):
    return random.Random(" ".join("%s=%s" % (k, c[k]) for k in sorted(c) if k != "name"))


def _widths(c):
    return [int(w) for w in c["m"].split(",")]


def _requests(c):
    """adapt: (first token, end, adapter) of every request, adapter -1 for none.  The first has the most tokens."""
    r, at, out = _rng(c), 0, []
    for i in range(c["rows"]):
        n = c["new"] if i == 0 else r.randint(max(1, c["new"] // 3), c["new"])
        out.append((at, at + n, r.randrange(c["count"]) if i == 0 or r.random() < 0.9 else -1))
        at += n
    return out


def _turns(c):
    """rope: (new tokens, cached tokens) of every row.  The first row has the most."""
    r = _rng(c)
    new = [c["new"]] + [r.randint(1, c["new"]) for _ in range(c["rows"] - 1)]
    return new, [c["cached"]] + [r.randint(0, c["cached"]) for _ in range(c["rows"] - 1)]


def _pages(c, spare=3):
    """A table that has pages for the new tokens alone (those before fell out of a window, say), and the number of pages."""
    r, page = _rng(c), c["page"]
    spans = [(b // page, -(-(a + b) // page)) for a, b in zip(*_turns(c))]
    pages = list(range(sum(last - first for first, last in spans) + spare))
    r.shuffle(pages)
    table = np.full((c["rows"], max(last for _, last in spans) + 1), -1, np.int32)
    at = 0
    for i, (first, last) in enumerate(spans):
        table[i, first:last] = pages[at:at + last - first]
        at += last - first
    return table, len(pages)


def _frequencies(c):
    """Radians a position of every pair, and what queries and keys are multiplied with."""
    half = c["rotary"] // 2
    w = [500000.0 ** (-i / half) for i in range(half)]
    if c["scaling"] == "linear":
        return [x / 4 for x in w], 1.0
    if c["scaling"] == "llama3":  # factor 8, from 8192 positions, slow ones divided, those between blended
        out = []
        for x in w:
            turns = 8192 * x / (2 * math.pi)
            s = min(1.0, max(0.0, (turns - 1) / (4 - 1)))
            out.append(s * x + (1 - s) * x / 8)
        return out, 1.0
    if c["scaling"] == "yarn":  # factor 4, from 32768 positions, a ramp over the pairs
        def pair(turns):
            return half * math.log(32768 / (turns * 2 * math.pi)) / math.log(500000.0)
        low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), 2 * half - 1)
        out = []
        for i, x in enumerate(w):
            s = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            out.append(x / 4 * s + x * (1 - s))
        return out, 0.1 * math.log(4) + 1
    return w, 1.0


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def prepare(case, seed):
    c, dt = case, DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": c, "op": c["op"]}

    def values(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device=DEV).mul_(scale).to(dt)

    if c["op"] == "adapt":
        s["requests"] = _requests(c)
        tokens = s["requests"][-1][1]
        s["which"] = _gpu(np.concatenate([np.full(b - a, i, np.int32) for a, b, i in s["requests"]]))
        s["x"] = values(tokens, c["n"])
        s["y"] = [values(tokens, m) for m in _widths(c)]
        s["down"] = [values(c["count"], c["rank"], c["n"], scale=c["n"] ** -0.5) for _ in s["y"]]
        s["up"] = [values(c["count"], m, c["rank"], scale=0.05) for m in _widths(c)]
        s["scale"] = [torch.rand(c["count"], generator=gen, device=DEV) + 1 for _ in s["y"]]
    elif c["op"] == "rope":
        new, cached = _turns(c)
        tokens, dim = sum(new), c["dim"]
        parts = [c["heads"] * dim, c["kv_heads"] * dim, c["kv_heads"] * dim]
        qkv = values(tokens, sum(parts)).split(parts, 1) if c["fused"] else [values(tokens, p) for p in parts]
        s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, dim)) for t in qkv)
        table, pages = _pages(c)
        s["k_pages"], s["v_pages"] = (values(pages, c["kv_heads"], c["page"], dim) for _ in range(2))
        s["table"], s["lengths"] = _gpu(table), _gpu(np.array([a + b for a, b in zip(new, cached)], np.int32))
        s["starts"] = _gpu(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)) if c["new"] > 1 else None
        w, s["factor"] = _frequencies(c)
        s["frequencies"] = _gpu(np.array(w, np.float64))
    else:
        R, V = c["rows"], c["vocab"]
        x = torch.randn(R, V, generator=gen, device=DEV).mul_(2.0)
        # a handful of likely tokens per row
        hot = torch.randint(0, V, (R, 12), generator=gen, device=DEV)
        x.scatter_(1, hot, torch.rand(R, 12, generator=gen, device=DEV) * 4 + 9)
        s["tokens"] = hot[:, 0].clone()
        if c["masked"]:
            # a third of the rows may take a few tokens only, another third has the vocabulary's end closed by the
            # type's lowest value; tokens beyond the vocabulary are not scored
            few = x[1::3].gather(1, hot[1::3, :7])
            x[1::3] = -math.inf
            x[1::3] = x[1::3].scatter(1, hot[1::3, :7], few)
            x[2::3, V - V // 3:] = torch.finfo(dt).min
            s["tokens"][2::3] %= V - V // 3
            s["tokens"][4::5] = -100
        s["logits"] = x.to(dt)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _own(s) if own else PLAIN[s["op"]](s)


def _own(s):
    from quipsharp_amd import adapters, logprobs, rope

    c = s["case"]
    if s["op"] == "adapt":
        return adapters.add_adapters(s["y"], s["x"], s["which"], s["down"], s["up"], s["scale"])
    if s["op"] == "rope":
        q = rope.append_rotated(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                s["frequencies"], starts=s["starts"], layout=c["layout"], factor=s["factor"])
        return q, s["k_pages"], s["v_pages"]
    return logprobs.token_logprobs(s["logits"], s["tokens"], c["top"])


def _plain_adapt(s):
    x, which = s["x"].float(), s["which"]
    out = []
    for y, down, up, scale in zip(s["y"], s["down"], s["up"], s["scale"]):
        if s["case"]["prompt"]:
            o = y.float()
            for first, end, a in s["requests"]:
                if a >= 0:
                    v = torch.matmul(x[first:end], down[a].float().t())
                    o[first:end] += scale[a] * torch.matmul(v, up[a].float().t())
        else:
            a = which.clamp(min=0).long()
            v = torch.matmul(down[a].float(), x[:, :, None])
            delta = scale[a][:, None] * torch.matmul(up[a].float(), v)[:, :, 0]
            o = y.float() + torch.where(which[:, None] >= 0, delta, 0.0)
        out.append(o.to(y.dtype))
    return out


def _turned(x, cos, sin, layout):
    """x (tokens, heads, dim): the first 2 * cos.shape[1] elements of every head turned."""
    n = cos.shape[1]
    x = x.float()
    part = x[:, :, :2 * n]
    a, b = (part[:, :, :n], part[:, :, n:]) if layout == "half" else (part[:, :, 0::2], part[:, :, 1::2])
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.cat([a, b], 2) if layout == "half" else torch.stack([a, b], 3).flatten(2)
    return torch.cat([part, x[:, :, 2 * n:]], 2)


def _plain_rope(s):
    c, q = s["case"], s["q"]
    t = torch.arange(q.shape[0], device=DEV)
    if s["starts"] is None:
        row, pos = t, s["lengths"].long() - 1
    else:
        row = (s["starts"][None, 1:] <= t[:, None]).sum(1)
        pos = s["lengths"][row].long() - s["starts"][row + 1] + t
    angle = pos[:, None].double() * s["frequencies"]
    cos, sin = (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()
    page, at = s["table"][row, pos // c["page"]].long(), pos % c["page"]
    s["k_pages"][page, :, at] = _turned(s["k"], cos, sin, c["layout"]).to(q.dtype)
    s["v_pages"][page, :, at] = s["v"]
    return _turned(q, cos, sin, c["layout"]).to(q.dtype), s["k_pages"], s["v_pages"]


def _plain_score(s):
    x, V, top = s["logits"].float(), s["case"]["vocab"], s["case"]["top"]
    m = x.amax(1, keepdim=True)
    below = x - m
    e = below.exp()
    S = e.sum(1, dtype=torch.float64)
    # 0 log 0 is 0
    H = S.log() - torch.where(e > 0, e * below, 0.0).sum(1, dtype=torch.float64) / S
    scored = (s["tokens"] >= 0) & (s["tokens"] < V)
    t = torch.where(scored, s["tokens"], 0)[:, None]
    xt = x.gather(1, t)
    at = torch.arange(V, device=DEV)
    rank = ((x > xt) | ((x == xt) & (at < t))).sum(1)
    logp = (xt - m)[:, 0].double() - S.log()
    # in order of the logit, then of the token, as one whole number
    bits = (x + 0.0).view(torch.int32)
    key = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) + (V - 1 - at)
    best = V - 1 - (torch.topk(key, top, dim=1)[0] & 0xFFFFFFFF)
    xb = x.gather(1, best)
    return (torch.where(scored, logp, 0.0).float(), H.float(), torch.where(scored, rank, -1).int(),
            ((xb - m).double() - S.log()[:, None]).float(), torch.where(xb > -math.inf, best, -1).int())


PLAIN = {"adapt": _plain_adapt, "rope": _plain_rope, "score": _plain_score}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    c, size = case, torch.empty(0, dtype=DTYPES[case["dtype"]]).element_size()
    if c["op"] == "adapt":
        requests = _requests(c)
        used = {a for _, _, a in requests if a >= 0}
        adapted = sum(b - a for a, b, i in requests if i >= 0)
        wide = [c["n"] + m for m in _widths(c)]
        return {"bytes": size * (requests[-1][1] * (c["n"] + 2 * sum(_widths(c))) + len(used) * c["rank"] * sum(wide)),
                "flops": 2 * adapted * c["rank"] * sum(wide)}
    if c["op"] == "rope":
        tokens = sum(_turns(c)[0])
        return {"bytes": 2 * size * tokens * c["dim"] * (c["heads"] + 2 * c["kv_heads"]),
                "flops": 3 * tokens * c["rotary"] * (c["heads"] + c["kv_heads"])}
    return {"bytes": c["rows"] * (c["vocab"] * size + 20 + 8 * c["top"]), "flops": 5 * c["rows"] * c["vocab"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"adapt": _exact_adapt, "rope": _exact_rope, "score": _exact_score}[case["op"]](case, s)


def _exact_adapt(c, s):
    out = []
    for g, y in enumerate(s["y"]):
        o = y.double()
        for a in range(c["count"]):
            mine = torch.nonzero(s["which"] == a)[:, 0]
            if len(mine):
                v = s["down"][g][a].double() @ s["x"][mine].double().t().contiguous()
                o[mine] += s["scale"][g][a].double() * (s["up"][g][a].double() @ v).t()
        out.append(o)
    return out


def _exact_rope(c, s):
    table, _ = _pages(c)
    w, factor = _frequencies(c)
    w = torch.tensor(w, dtype=torch.float64, device=DEV)
    k, v, q, t, n = s["k_pages"].double(), s["v_pages"].double(), [], 0, len(w)
    for r, (new, cached) in enumerate(zip(*_turns(c))):
        pos = torch.arange(cached, cached + new, device=DEV)
        # a pair as one complex number
        turn = torch.polar(torch.full((1, 1), factor, dtype=torch.float64, device=DEV), pos[:, None] * w)[:, None]
        ids = torch.from_numpy(table[r]).long().to(DEV)[pos // c["page"]]
        for name in ("q", "k"):
            x = s[name][t:t + new].double()
            part = x[:, :, :2 * n]
            pairs = part.unflatten(2, (2, n)).transpose(2, 3) if c["layout"] == "half" else part.unflatten(2, (n, 2))
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            x[:, :, :2 * n] = (z.transpose(2, 3) if c["layout"] == "half" else z).flatten(2)
            if name == "q":
                q.append(x)
            else:
                k[ids, :, pos % c["page"]] = x
        v[ids, :, pos % c["page"]] = s["v"][t:t + new].double()
        t += new
    return torch.cat(q), k, v


def _exact_score(c, s):
    out = []
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        logp = torch.log_softmax(x, 1)
        p = logp.exp()
        entropy = -torch.where(p > 0, p * logp, 0.0).sum(1)
        value, order = torch.sort(x, dim=1, descending=True, stable=True)
        fine = (t >= 0) & (t < c["vocab"])
        # a token's rank is where the sort puts it
        rank = torch.argmax((order == t[:, None]).byte(), 1)
        mine = logp.gather(1, t.clamp(0, c["vocab"] - 1)[:, None])[:, 0]
        best = order[:, :c["top"]]
        out.append((torch.where(fine, mine, 0.0), entropy, torch.where(fine, rank, -1).int(), logp.gather(1, best),
                    torch.where(value[:, :c["top"]] > -math.inf, best, -1).int()))
    return tuple(torch.cat(t) for t in zip(*out))
