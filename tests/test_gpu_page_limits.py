"""Rows at the limits of their table and of the pool (csrc/qs_pages.hip,
csrc/qs_attend_token.hip, csrc/qs_attend_chunk.hip): what is cached stays as it
is, tokens without a place are left out, and they are counted.  Pools are
compared bit by bit, attention to the tolerance of test_gpu_attend.py."""
import random

import pytest
import torch

from test_gpu_attend import want_and_tolerance

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
PAGE, COLS = 16, 3
ROOM = PAGE * COLS


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def filled(lengths, dev, pages=12, heads=2, dim=64, parents=None):
    """A cache whose rows hold these lengths (or their parents'), every place of the pool a number of its own."""
    from quipsharp_amd.pages import PagedCache
    cache = PagedCache(1, pages, heads, dim, len(lengths), COLS, page=PAGE, device=dev)
    cache.kv.copy_(torch.randn(cache.kv.shape, generator=torch.Generator().manual_seed(11)))
    cache.advance(ints(lengths, dev))
    if parents:
        cache.advance(0, ints(parents, dev))
    return cache


def held(pool, table, row):
    """(positions, heads, dim) of a row's pages in order, on the CPU."""
    pages = [p for p in table[row].tolist() if p >= 0]
    return pool[pages].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3]).cpu()


def near(got, q, k, v, see, dim):
    group = q.shape[0] // k.shape[1]
    for g in range(k.shape[1]):
        want, tol = want_and_tolerance(q[g * group:(g + 1) * group], k[see, g], v[see, g], dim ** -0.5)
        assert ((got[g * group:(g + 1) * group].double() - want).abs() <= tol).all()


def tokens_of(n, heads, dim, seed, dev):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, h, dim, generator=g).to(BF).to(dev) for h in (heads, heads, 2 * heads)]


@pytest.mark.parametrize("calls", ["cache", "functions"])
def test_more_tokens_than_the_table_has_room_for(dev, calls):
    """Row 0 goes on from 40 by 20 where 8 have room: those 8 are stored, nothing else changes, row 1, which shares
    the first pages, least of all; each query sees the positions up to its own that there are."""
    from quipsharp_amd.pages import advance_pages, append_pages, attend_chunk
    cache = filled([40, 0], dev, parents=[0, 0])
    before = cache.kv.clone()
    k, v, q = tokens_of(20, 2, 64, 1, dev)
    starts = ints([0, 20, 20], dev)
    if calls == "cache":
        cache.advance(ints([20, 0], dev))
        table = cache.table
        cache.append(0, k, v, starts)
        got = cache.attend_chunk(0, q, starts)
        lead = cache.attend_chunk(0, q, starts, window=12, sinks=2)
    else:
        table, lengths, _, short = advance_pages(cache.kv, cache.table, cache.lengths, cache.refs, ints([20, 0], dev))
        assert short.item() == 1
        append_pages(cache.keys(0), cache.values(0), k, v, table, lengths, starts)
        pools = (cache.keys(0), cache.values(0), table, lengths, starts)
        got, lead = attend_chunk(q, *pools), attend_chunk(q, *pools, window=12, sinks=2)
    want = before.clone()
    last = table[0, 2].item()
    if last != table[1, 2].item():  # copied before it is written
        want[0, :, last, :, :8] = before[0, :, table[1, 2].item(), :, :8]
    want[0, 0, last, :, 8:] = k[:8].transpose(0, 1)
    want[0, 1, last, :, 8:] = v[:8].transpose(0, 1)
    assert torch.equal(cache.kv, want)
    rk, rv = held(want[0, 0], table, 0), held(want[0, 1], table, 0)
    for i in range(20):
        near(got[i].cpu(), q[i].cpu(), rk, rv, list(range(min(41 + i, ROOM))), 64)
        near(lead[i].cpu(), q[i].cpu(), rk, rv, [p for p in range(min(41 + i, ROOM)) if p > 28 + i or p < 2], 64)


@pytest.mark.parametrize("calls", ["cache", "functions"])
def test_steps_of_a_full_row(dev, calls):
    """Single tokens of a row without room, several of them: nothing is stored, and the row attends to what it has."""
    from quipsharp_amd.pages import advance_pages, append_pages, attend_token
    cache = filled([ROOM, 5], dev)
    table, lengths, refs = cache.table, cache.lengths, cache.refs
    for step in range(3):
        k, v, q = tokens_of(2, 2, 64, 2 + step, dev)
        before = cache.kv.clone()
        if calls == "cache":
            cache.advance(1)
            short = cache.short
            cache.append(0, k, v)
            got, lead = cache.attend_token(0, q), cache.attend_token(0, q, window=10)
            n = ROOM
        else:
            table, lengths, refs, short = advance_pages(cache.kv, table, lengths, refs, 1)
            append_pages(cache.keys(0), cache.values(0), k, v, table, lengths)
            pools = (cache.keys(0), cache.values(0), table, lengths)
            got, lead = attend_token(q, *pools), attend_token(q, *pools, window=10)
            n = ROOM + step
        assert short.item() == 1
        at = table[1, 0].item()
        before[0, 0, at, :, 5 + step], before[0, 1, at, :, 5 + step] = k[1], v[1]
        assert torch.equal(cache.kv, before)
        rk, rv = held(cache.keys(0), table, 0), held(cache.values(0), table, 0)
        near(got[0].cpu(), q[0].cpu(), rk, rv, list(range(ROOM)), 64)
        near(lead[0].cpu(), q[0].cpu(), rk, rv, list(range(n - 9, ROOM)), 64)


def test_full_rows_that_share_their_pages(dev):
    """Rows forked from a full one write nothing, together or one after the other."""
    cache = filled([ROOM, 0, 0], dev, parents=[0, 0, 0])
    before = cache.kv.clone()
    k, v, q = tokens_of(3, 2, 64, 6, dev)
    for parents in (None, [2, 0, 1]):
        cache.advance(1, None if parents is None else ints(parents, dev))
        cache.append(0, k, v)
        assert torch.equal(cache.kv, before) and cache.short.item() == 3
        got = cache.attend_token(0, q)
        rk, rv = held(cache.keys(0), cache.table, 0), held(cache.values(0), cache.table, 0)
        for r in range(3):
            near(got[r].cpu(), q[r].cpu(), rk, rv, list(range(ROOM)), 64)


@pytest.mark.parametrize("far", [1, 100, 2 ** 31 - 1 - ROOM])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 0), (30, 5), (2 ** 31 - 1, 7), (200, 100), (1, 1000)])
@pytest.mark.parametrize("dim,cols", [(128, 3), (64, 60), (256, 3)])
def test_lengths_beyond_the_table(dev, dim, cols, window, sinks, far):
    """The newest token of a row lies where the length says, whatever the table's room: the window goes with it."""
    from quipsharp_amd.pages import attend_chunk, attend_token
    g = torch.Generator().manual_seed(dim)
    room, new = cols * PAGE, 9
    pools = [torch.randn(cols + 2, 2, PAGE, dim, generator=g).to(BF) for _ in range(2)]
    table = torch.randperm(cols + 2, generator=g)[:cols].to(torch.int32)[None]
    q = torch.randn(new, 4, dim, generator=g).to(BF)
    n = min(room + far, 2 ** 31 - 1)
    rk, rv = held(pools[0], table, 0), held(pools[1], table, 0)

    def seen(last):
        return [p for p in range(min(last + 1, room)) if not window or p > last - window or p < sinks]

    args = [t.to(dev) for t in pools] + [table.to(dev), ints([n], dev)]
    got = attend_token(q[:1].to(dev), *args, window=window, sinks=sinks).cpu()
    near(got[0], q[0], rk, rv, seen(n - 1), dim)
    got = attend_chunk(q.to(dev), *args, ints([0, new], dev), window=window, sinks=sinks).cpu()
    for i in range(new):
        near(got[i], q[i], rk, rv, seen(n - new + i), dim)


def test_pages_that_are_missing_are_counted_in_every_step(dev):
    """A token that goes to a page which its row did not get is counted as the one that should have opened it."""
    cache = filled([16, 16], dev, pages=2)
    for step in range(3):
        cache.advance(1)
        assert cache.short.item() == 2, step
    assert cache.table.tolist() == [[0, -1, -1], [1, -1, -1]]
    cache.free(torch.tensor([True, False], device=dev))
    cache.advance(ints([1, 0], dev))  # positions before it in its page are lost: a page now would not bring them back
    assert cache.short.item() == 1 and cache.table[0].tolist() == [0, -1, -1]
    cache.advance(ints([0, 0], dev))
    assert cache.short.item() == 0
    cache.advance(ints([12, 0], dev))
    assert cache.short.item() == 1 and cache.lengths.tolist() == [32, 0]
    cache.advance(ints([1, 0], dev))
    assert cache.short.item() == 0 and cache.table[0].tolist() == [0, -1, 1]


def test_a_copy_that_gets_no_page_is_counted_in_every_step(dev):
    """So is the page that a row lost because there was none for its copy."""
    cache = filled([20, 0], dev, pages=2, parents=[0, 0])
    for step in range(2):
        cache.advance(1)
        assert cache.short.item() == 1, step
        assert cache.table.tolist() == [[0, 1, -1], [0, -1, -1]]


def test_append_rope_stores_no_half_of_a_position(dev):
    """A row without tokens and a position beyond the rotary tables: zero queries, and the pools as they were."""
    from quipsharp_amd import _lib
    from quipsharp_amd.pages import _pool
    L = _lib.lib()
    rows, nh, nkv = 3, 4, 2
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(rows, h * 128, generator=g).to(BF).to(dev) for h in (nh, nkv, nkv))
    qw, kw = (torch.ones(128, dtype=BF, device=dev) for _ in range(2))
    cos, sin = (torch.randn(20, 128, generator=g).to(BF).to(dev) for _ in range(2))
    pools = [torch.randn(9, nkv, PAGE, 128, generator=g).to(BF).to(dev) for _ in range(2)]
    before = [p.clone() for p in pools]
    table = ints([[4, 1, 2], [0, 3, 5], [6, 7, 8]], dev)
    lengths = ints([0, 21, 20], dev)
    qo = torch.full_like(q, 7)
    _lib.check(L.qs_page_append_rope(*(t.data_ptr() for t in (q, k, v, qw, kw, cos, sin)), 20, qo.data_ptr(), rows, nh,
                                     nkv, 128, _pool(*pools, table, lengths), 1e-6, _lib.stream_of(q)))
    assert (qo[:2] == 0).all() and (qo[2] != 7).any()
    assert not torch.equal(pools[0][7, :, 3], before[0][7, :, 3])
    assert torch.equal(pools[1][7, :, 3], v[2].view(nkv, 128))
    for pool, old in zip(pools, before):
        pool[7, :, 3] = old[7, :, 3]
        assert torch.equal(pool, old)


@pytest.mark.parametrize("rows", [4, 64])
def test_the_sum_of_missing_pages(dev, rows):
    """It adds up over the steps, also over replayed ones, and stays at the largest int32."""
    from quipsharp_amd.pages import PagedCache
    cache = PagedCache(1, 4, 1, 64, rows, 2, page=16, device=dev)
    want = 0
    for tokens in (1, 16, 0, 40, 1):
        cache.advance(tokens)
        want += cache.short.item()
        assert cache.missing.item() == want
    assert want > 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.advance(1)
    for _ in range(3):
        graph.replay()
        want += cache.short.item()
        assert cache.short.item() == rows and cache.missing.item() == want
    cache.advance(1 << 30)
    cache.advance(1 << 30)
    assert cache.missing.item() == min(want + 2 * rows * 2 ** 26, 2 ** 31 - 1)
    with pytest.raises(RuntimeError, match="left out"):
        cache.check()
    cache.missing.zero_()
    cache.check()


@pytest.mark.parametrize("rows,cols,pages", [(5, 4, 14), (12, 3, 60), (3, 6, 9), (20, 5, 9000)])
def test_what_rows_hold_is_their_own(dev, rows, cols, pages):
    """A long run of forks, prompts, waiting rows, frees, windows and compactions over tables and pools that run out:
    wherever a row has a page, it holds that row's tokens, those of the rows it came from among them."""
    from quipsharp_amd.pages import PagedCache
    cache = PagedCache(1, pages, 1, 8, rows, cols, page=PAGE, device=dev)
    r = random.Random(rows)
    told, room, own = 0, cols * PAGE, [{} for _ in range(rows)]  # position -> number of the token stored there
    missing = lost = 0
    for step in range(70):
        op = r.choice(["step", "step", "fork", "counts", "counts", "free", "window", "compact"])
        if op in ("step", "fork", "counts"):
            parents = [r.choice([i, r.randrange(rows), r.randrange(-1, rows)]) for i in range(rows)] if op == "fork" else None
            counts = [r.choice([0, 1, 3, 2 * PAGE + 1]) if op == "counts" else 1 for _ in range(rows)]
            old = cache.lengths.tolist()
            cache.advance(ints(counts, dev) if op == "counts" else 1, None if parents is None else ints(parents, dev))
            start = old if parents is None else [old[p] if p >= 0 else 0 for p in parents]
            if parents is not None:
                own = [dict(own[p]) if p >= 0 else {} for p in parents]
            table, left = cache.table.tolist(), 0
            x = []
            for i in range(rows):
                for p in range(start[i], start[i] + counts[i]):
                    told += 1
                    x.append(told)
                    if p < room and table[i][p // PAGE] >= 0:
                        own[i][p] = told
                    else:
                        left += 1
            assert cache.lengths.tolist() == [min(s + n, room) for s, n in zip(start, counts)]
            assert cache.over.tolist() == [max(s + n - room, 0) for s, n in zip(start, counts)]
            assert (cache.short.item() > 0) == (left > 0)
            missing += cache.short.item()
            lost += left
            # a number in three elements, exact in bf16
            if x:
                k = torch.tensor([[[n % 128, n // 128 % 128, n // 16384] + [0] * 5] for n in x]).to(BF).to(dev)
                cache.append(0, k, -k, ints([sum(counts[:i]) for i in range(rows + 1)], dev))
        elif op == "free":
            keep = [r.random() < 0.8 for _ in range(rows)]
            cache.free(torch.tensor(keep, device=dev))
            own = [o if k else {} for o, k in zip(own, keep)]
        elif op == "window":
            cache.free(window=r.randint(1, room), sinks=r.choice([0, 3, PAGE]))
        else:
            cache.compact()
        assert cache.missing.item() == missing
        kv, table, lengths = cache.kv[0, :, :, 0].float().cpu(), cache.table.tolist(), cache.lengths.tolist()
        refs = [0] * pages
        for i in range(rows):
            for c, page in enumerate(table[i]):
                if page < 0:
                    continue
                refs[page] += 1
                for p in range(c * PAGE, min((c + 1) * PAGE, lengths[i])):
                    n = own[i][p]
                    want = torch.tensor([n % 128, n // 128 % 128, n // 16384], dtype=torch.float32)
                    assert torch.equal(kv[0, page, p % PAGE, :3], want) and torch.equal(kv[1, page, p % PAGE, :3], -want)
        assert cache.refs.tolist() == refs
    assert (lost > 0) == (missing > 0) and lost > 0
