"""The work on a paged cache's pages (csrc/qs_pages.hip) against lists in
Python: forking, copying before a shared page is written, giving pages out and
back, moving pages together, and storing tokens.  All of it is exact."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Books:
    """What the cache should hold: per row a list of (page or None) and a length, and every page's contents."""

    def __init__(self, kv, rows, cols, page):
        self.kv = kv.clone().cpu()
        self.table = [[None] * cols for _ in range(rows)]
        self.length = [0] * rows
        self.page, self.cols, self.pages = page, cols, kv.shape[-4]

    def refs(self):
        n = [0] * self.pages
        for row in self.table:
            for p in row:
                if p is not None:
                    n[p] += 1
        return n

    def advance(self, tokens, parents):
        rows, page, room = len(self.table), self.page, self.cols * self.page
        old = [list(r) for r in self.table], list(self.length)
        for i in range(rows):
            p = i if parents is None else parents[i]
            if 0 <= p < rows:
                self.length[i] = old[1][p]
                self.table[i] = [x if c * page < self.length[i] else None for c, x in enumerate(old[0][p])]
            else:
                self.length[i], self.table[i] = 0, [None] * self.cols
        if tokens == 0:
            return 0
        want = []
        for i in range(rows):
            n, c0 = self.length[i], self.length[i] // page
            if n % page and self.table[i][c0] is not None:
                others = [j for j in range(rows) if j != i and self.table[j][c0] == self.table[i][c0]]
                if any(self.length[j] > n or (self.length[j] == n and j < i) for j in others):
                    want.append((i, c0, True))
            for c in range(-(-n // page), (n + tokens - 1) // page + 1):
                want.append((i, c, False))
        refs = self.refs()
        free = [p for p in range(self.pages) if refs[p] == 0]
        short = sum(c >= self.cols for _, c, _ in want)
        copies = []
        for i, c, copy in want:
            if c >= self.cols:
                continue
            new = free.pop(0) if free else None
            short += new is None
            if copy and new is not None:
                copies.append((self.table[i][c], new, self.length[i] % page))
            self.table[i][c] = new
        for s, d, n in copies:
            self.kv[..., d, :, :n, :] = self.kv[..., s, :, :n, :]
        self.length = [min(n + tokens, room) for n in self.length]
        return short

    def free(self, keep, window, sinks):
        for i, row in enumerate(self.table):
            for c in range(self.cols):
                positions = range(c * self.page, (c + 1) * self.page)
                if keep is not None and not keep[i] or window and all(
                        p >= sinks and p <= self.length[i] - window for p in (positions[0], positions[-1])):
                    row[c] = None
            if keep is not None and not keep[i]:
                self.length[i] = 0

    def compact(self):
        used = [n > 0 for n in self.refs()]
        n = sum(used)
        moves = dict(zip([p for p in range(n, self.pages) if used[p]], [p for p in range(n) if not used[p]]))
        for s, d in moves.items():
            self.kv[..., d, :, :, :] = self.kv[..., s, :, :, :]
        self.table = [[moves.get(p, p) for p in row] for row in self.table]

    def same(self, cache):
        table = [[-1 if p is None else p for p in row] for row in self.table]
        assert cache.table.tolist() == table
        assert cache.lengths.tolist() == self.length
        assert cache.refs.tolist() == self.refs()
        assert torch.equal(cache.kv.cpu(), self.kv)


def filled(rows, cols, pages, page, dev, dtype=torch.bfloat16, layers=2, heads=2, dim=64, seed=0):
    from quipsharp_amd.pages import PagedCache
    cache = PagedCache(layers, pages, heads, dim, rows, cols, page=page, dtype=dtype, device=dev)
    cache.kv.copy_(torch.randn(cache.kv.shape, generator=torch.Generator().manual_seed(seed)))
    return cache, Books(cache.kv, rows, cols, page)


@pytest.mark.parametrize("rows,cols,pages,page,dtype", [
    (1, 3, 5, 16, torch.bfloat16), (4, 9, 40, 16, torch.float16), (7, 33, 90, 32, torch.bfloat16),
    (16, 20, 1500, 16, torch.bfloat16), (33, 5, 170, 64, torch.float16), (8, 6, 60, 16, torch.float32)])
def test_a_long_run_of_steps(dev, rows, cols, pages, page, dtype):
    """Forks, prompts, single tokens, rows that end, windows and compactions in a random order, some of them short
    of pages or of columns."""
    cache, books = filled(rows, cols, pages, page, dev, dtype)
    r = random.Random(rows * cols)
    for step in range(60):
        op = r.choice(["token", "token", "fork", "fork", "prompt", "free", "window", "compact", "none"])
        if op in ("token", "fork", "prompt", "none"):
            tokens = {"prompt": r.randint(1, 2 * page + 3), "none": 0}.get(op, 1)
            parents = [r.choice([i, r.randrange(rows), r.randrange(rows), -1 if step % 7 == 0 else i])
                       for i in range(rows)] if op in ("fork", "none") else None
            cache.advance(tokens, None if parents is None else torch.tensor(parents, dtype=torch.int32, device=dev))
            assert cache.short.item() == books.advance(tokens, parents), (step, op)
        elif op == "free":
            keep = [r.random() < 0.7 for _ in range(rows)]
            cache.free(torch.tensor(keep, device=dev))
            books.free(keep, 0, 0)
        elif op == "window":
            window, sinks = r.randint(1, 3 * page), r.choice([0, 1, page, page + 1])
            cache.free(window=window, sinks=sinks)
            books.free(None, window, sinks)
        else:
            cache.compact()
            books.compact()
        books.same(cache)


def test_outputs_apart_leave_the_inputs(dev):
    from quipsharp_amd.pages import advance_pages, compact_pages, free_pages
    cache, books = filled(6, 8, 60, 16, dev)
    cache.advance(40)
    books.advance(40, None)
    parents = [0, 0, 5, 3, 3, 1]
    before = [t.clone() for t in (cache.table, cache.lengths, cache.refs)]
    t, n, f, short = advance_pages(cache.kv, cache.table, cache.lengths, cache.refs, 1,
                                   torch.tensor(parents, dtype=torch.int32, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.table, cache.lengths, cache.refs)))
    books.advance(1, parents)
    assert short.item() == 0
    cache.table, cache.lengths, cache.refs = t, n, f
    books.same(cache)
    keep = [True, False, True, True, False, True]
    cache.table, cache.lengths, cache.refs = free_pages(t, n, f, page=16, keep=torch.tensor(keep, device=dev), window=20)
    books.free(keep, 20, 0)
    books.same(cache)
    cache.table, cache.refs = compact_pages(cache.kv, cache.table, cache.refs)
    books.compact()
    books.same(cache)


def test_a_longer_holder_keeps_the_page(dev):
    """A page that a longer row still reads is not written by a shorter one, whatever their order."""
    cache, books = filled(3, 4, 12, 16, dev)
    cache.advance(5)
    books.advance(5, None)
    for parents in ([2, 2, 2], [0, 1, 0]):
        cache.advance(1, torch.tensor(parents, dtype=torch.int32, device=dev))
        books.advance(1, parents)
        books.same(cache)
    cache.lengths.copy_(torch.tensor([3, 7, 4], dtype=torch.int32))  # rows that went back
    books.length = [3, 7, 4]
    parents = [1, 1, 0]
    cache.advance(1, torch.tensor(parents, dtype=torch.int32, device=dev))
    books.advance(1, parents)
    books.same(cache)


def test_entries_that_name_no_page(dev):
    """Entries outside the pool count as none: nothing outside it is read, written or counted."""
    cache, _ = filled(2, 3, 6, 16, dev)
    cache.advance(20)
    cache.table[0, 1] = 99
    cache.table[1, 2] = -5
    cache.advance(0)
    assert cache.table.tolist()[0][1] == -1 and cache.table.tolist()[1][2] == -1
    cache.table[0, 1] = 1 << 30
    kv = cache.kv.clone()
    cache.free(window=1)
    cache.compact()
    assert cache.refs.sum().item() == (cache.table >= 0).sum().item() + 1  # the page that row 0 lost its hold of
    assert cache.kv.shape == kv.shape


def test_a_number_of_tokens_for_every_row(dev):
    """Rows that begin, go on and wait in one call give what one call after the other gives where no page is shared,
    and the rows that wait keep what they share."""
    from quipsharp_amd.pages import PagedCache
    cache, books = filled(5, 9, 60, 16, dev)
    r = random.Random(2)
    for step in range(12):
        each = [r.choice([0, 0, 1, 5, 17, 33]) for _ in range(5)]
        cache.advance(torch.tensor(each, dtype=torch.int32, device=dev))
        taken = sum(-(-n // 16) - -(-m // 16) for n, m in zip(cache.lengths.tolist(), books.length))
        free = [p for p in range(60) if books.refs()[p] == 0][:taken]
        for i, n in enumerate(each):
            n0, n1 = books.length[i], min(books.length[i] + n, 9 * 16)
            for c in range(-(-n0 // 16), -(-n1 // 16)):
                books.table[i][c] = free.pop(0)
            books.length[i] = n1
        books.same(cache)
    # two rows of one parent: the one that writes copies the page, the one that waits keeps it
    cache = PagedCache(1, 20, 1, 64, 2, 4, page=16, device=dev)
    cache.advance(torch.tensor([20, 0], dtype=torch.int32, device=dev))
    cache.kv.copy_(torch.randn(cache.kv.shape, generator=torch.Generator().manual_seed(1)))
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    cache.advance(0, zero)
    kept = cache.table[0].tolist()
    cache.advance(torch.tensor([0, 3], dtype=torch.int32, device=dev))
    assert cache.table[0].tolist() == kept and cache.lengths.tolist() == [20, 23]
    assert cache.table[1, 0] == kept[0] and cache.table[1, 1] != kept[1]
    assert torch.equal(cache.kv[:, :, cache.table[1, 1].item(), :, :4], cache.kv[:, :, kept[1], :, :4])
    cache.advance(torch.tensor([-7, 0], dtype=torch.int32, device=dev))
    assert cache.lengths.tolist() == [20, 23]


def test_many_rows_and_pages(dev):
    """The largest number of rows, and a pool that takes many rounds to look through."""
    from quipsharp_amd.pages import PagedCache
    rows, cols = 1024, 7
    cache = PagedCache(1, 9000, 1, 64, rows, cols, page=16, device=dev)
    books = Books(cache.kv, rows, cols, 16)
    r = random.Random(4)
    cache.advance(37)
    books.advance(37, None)
    books.same(cache)
    for _ in range(3):
        parents = [r.randrange(rows) for _ in range(rows)]
        cache.advance(1, torch.tensor(parents, dtype=torch.int32, device=dev))
        books.advance(1, parents)
        books.same(cache)
    keep = [r.random() < 0.5 for _ in range(rows)]
    cache.free(torch.tensor(keep, device=dev))
    cache.compact()
    books.free(keep, 0, 0)
    books.compact()
    books.same(cache)


@pytest.mark.parametrize("dtype,heads,dim,page", [(torch.bfloat16, 3, 128, 16), (torch.float16, 1, 64, 64),
                                                  (torch.float32, 2, 96, 8), (torch.uint8, 2, 80, 128)])
def test_copy_pages(dev, dtype, heads, dim, page):
    from quipsharp_amd.pages import copy_pages
    kv = (torch.randn(3, 2, 20, heads, page, dim, generator=torch.Generator().manual_seed(1)) * 50).to(dtype).to(dev)
    want = kv.clone()
    src, dst = [3, 0, 19, 7, -1, 20, 4], [1, 2, 5, 18, 9, 10, 33]
    for s, d in list(zip(src, dst))[:4]:
        want[:, :, d] = want[:, :, s]
    copy_pages(kv, torch.tensor(src, dtype=torch.int32, device=dev), torch.tensor(dst, dtype=torch.int32, device=dev))
    assert torch.equal(kv, want)


@pytest.mark.parametrize("dtype,layout", [(torch.bfloat16, "heads"), (torch.float16, "positions")])
def test_append(dev, dtype, layout):
    from quipsharp_amd.pages import append_pages
    pages, heads, page, dim = 12, 3, 16, 64
    g = torch.Generator().manual_seed(2)
    shape = (pages, heads, page, dim) if layout == "heads" else (pages, page, heads, dim)
    k, v = (torch.randn(shape, generator=g).to(dtype).to(dev) for _ in range(2))
    if layout != "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    table = torch.tensor([[4, 0, -1], [7, 2, 50], [1, 3, 5], [6, 8, 9]], dtype=torch.int32)
    lengths, new = [30, 40, 0, 48], [21, 12, 0, 48]
    starts = [0, 21, 33, 33, 81]
    wide = torch.randn(81, 2 * heads, dim, generator=g).to(dtype).to(dev)
    nk, nv = wide[:, :heads], wide[:, heads:]
    wk, wv = k.clone(), v.clone()
    for r in range(4):
        for i in range(new[r]):
            p = lengths[r] - new[r] + i
            id = int(table[r, p // page])
            if 0 <= id < pages:
                wk[id, :, p % page], wv[id, :, p % page] = nk[starts[r] + i], nv[starts[r] + i]
    append_pages(k, v, nk, nv, table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev),
                 torch.tensor(starts, dtype=torch.int32, device=dev))
    assert torch.equal(k, wk) and torch.equal(v, wv)
    # one token per row; the row of length 0 and one beyond the table store nothing
    lengths = [17, 33, 0, 49]
    for r, n in enumerate(lengths):
        p = n - 1
        id = int(table[r, p // page]) if 0 <= p < 48 else -1
        if 0 <= id < pages:
            wk[id, :, p % page], wv[id, :, p % page] = nk[r], nv[r]
    append_pages(k, v, nk[:4], nv[:4], table.to(dev), torch.tensor(lengths, dtype=torch.int32, device=dev))
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_append_rope_equals_the_static_cache(dev):
    """q / k norm, rotary embedding and the store into pages give the static cache's bits, each row at its own
    position."""
    from quipsharp_amd import _lib
    from quipsharp_amd.pages import _pool
    L = _lib.lib()
    rows, nh, nkv, page = 3, 8, 2, 16
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(rows, h * 128, generator=g).bfloat16().to(dev) for h in (nh, nkv, nkv))
    qw, kw = ((1 + 0.1 * torch.randn(128, generator=g)).bfloat16().to(dev) for _ in range(2))
    cos, sin = (torch.randn(64, 128, generator=g).bfloat16().to(dev) for _ in range(2))
    pools = [torch.zeros(9, nkv, page, 128, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    table = torch.tensor([[4, 1, 2], [0, 3, 5], [6, 7, 8]], dtype=torch.int32, device=dev)
    lengths = torch.tensor([20, 1, 48], dtype=torch.int32, device=dev)
    qo = torch.empty_like(q)
    _lib.check(L.qs_page_append_rope(*(t.data_ptr() for t in (q, k, v, qw, kw, cos, sin)), 64, qo.data_ptr(), rows, nh,
                                     nkv, 128, _pool(*pools, table, lengths), 1e-6, _lib.stream_of(q)))
    for r, n in enumerate(lengths.tolist()):
        kc, vc = (torch.zeros(1, nkv, 64, 128, dtype=torch.bfloat16, device=dev) for _ in range(2))
        one, pos = torch.empty(1, nh * 128, dtype=torch.bfloat16, device=dev), torch.tensor([n - 1], device=dev)
        args = [t.data_ptr() for t in (q[r], k[r], v[r], qw, kw, cos, sin, pos, one, kc, vc)]
        _lib.check(L.qs_dec_qk_norm_rope(*args, 1, nh, nkv, 128, 64, 1e-6, _lib.stream_of(q)))
        id = int(table[r, (n - 1) // page])
        assert torch.equal(qo[r], one[0])
        assert torch.equal(pools[0][id, :, (n - 1) % page], kc[0, :, n - 1])
        assert torch.equal(pools[1][id, :, (n - 1) % page], vc[0, :, n - 1])
    assert (pools[0] != 0).any(-1).sum().item() == rows * nkv


def test_captured_steps(dev):
    """A beam step's page work, append and attention as one graph: every replay equals the eager step, with other
    work and synchronizations between."""
    from quipsharp_amd.pages import PagedCache
    rows, heads, dim = 4, 4, 64
    caches = [PagedCache(2, 60, 2, dim, rows, 12, page=16, device=dev) for _ in range(2)]
    parents = torch.zeros(rows, dtype=torch.int32, device=dev)
    k, v = (torch.zeros(rows, 2, dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
    q = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device=dev)

    def step(c):
        c.advance(1, parents)
        for layer in range(2):
            c.append(layer, k, v)
        out = c.attend_token(1, q, window=40, sinks=2)
        c.free(window=40, sinks=2)
        return out

    g = torch.Generator().manual_seed(9)
    r = random.Random(1)
    graph, out = torch.cuda.CUDAGraph(), None
    for i in range(70):
        parents.copy_(torch.tensor([r.randrange(rows) for _ in range(rows)], dtype=torch.int32))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        want = step(caches[0])
        if i == 0:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got = step(caches[1])
            torch.cuda.current_stream().wait_stream(s)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                out = step(caches[1])
        else:
            graph.replay()
            if i % 3 == 0:
                torch.cuda.synchronize()
            got = out
        a, b = caches
        assert torch.equal(got, want), i
        assert torch.equal(a.table, b.table) and torch.equal(a.lengths, b.lengths) and torch.equal(a.refs, b.refs)
        assert torch.equal(a.kv, b.kv) and a.short.item() == 0


@pytest.mark.parametrize("rows", [8, 64])
def test_far_more_tokens_than_columns(dev, rows):
    """The pages that are missing are counted up to the largest int32."""
    cache, _ = filled(rows, 2, 4, 16, dev, layers=1, heads=1)
    cache.advance(1 << 30)
    assert cache.short.item() == min(rows * 2 ** 26 - 4, 2 ** 31 - 1)
    assert cache.lengths.tolist() == [32] * rows
    assert cache.table.view(-1).tolist() == [0, 1, 2, 3] + [-1] * (2 * rows - 4)
