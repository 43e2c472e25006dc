"""Attention over a paged cache (csrc/qs_attend_token.hip, qs_attend_chunk.hip)
against its definition in 64 bits on the CPU, element by element.

Tolerance of an element, with A = sum_p w_p |v_p|, w the softmax's weights and
e the type's eps (a rounding is off by e / 2 at most):
  A e / 2         each weight is rounded once to the cache's type;
  |out| e / 2     the result is rounded once;
  2 s A           a score is off by s at most, a weight then by 2 s relative
                  (numerator and sum): s = scale (dim + 2) 2^-24 max_p sum_d
                  |q_d k_pd| for fp32 sums of exact products, and 2^-22 max |score|
                  for the product with scale and log2(e) and the exponential's argument;
  16 2^-24 A      the exponential (2 units), the sums and the rescaling;
  fp16: weights below 2^-14 of the running maximum are off by 2^-25 absolutely:
                  2^-25 sum_p |v_p|, divided by a sum of at least 1.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def seen_by(last, window, sinks):
    p = torch.arange(last + 1)
    return p[(p > last - window) | (p < sinks)] if window else p


def want_and_tolerance(q, k, v, scale):
    """q (heads, d), k and v (n, d) in 64 bits."""
    dt = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    if not len(k):
        return torch.zeros_like(q), torch.zeros_like(q)
    x = q @ k.T * scale
    w = torch.softmax(x, 1)
    out = w @ v
    A = w @ v.abs()
    size = (q.abs() @ k.abs().T).amax(1, keepdim=True) * abs(scale)
    s = size * (q.shape[1] + 2) * 2.0 ** -24 + x.abs().amax(1, keepdim=True) * 2.0 ** -22
    half = torch.finfo(dt).eps / 2
    tol = A * (half + 2 * s + 16 * 2.0 ** -24) + out.abs() * half
    if dt == torch.float16:
        tol = tol + 2.0 ** -25 * v.abs().sum(0)
    return out, tol


class Cache:
    """Rows of given lengths on scattered pages; every place that no row fills holds NaN."""

    def __init__(self, lengths, kv_heads, dim, page, dtype, seed, layout="heads", cols=None):
        g = torch.Generator().manual_seed(seed)
        self.page, self.lengths = page, lengths
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g)
        cols = cols or max(1, max(need))
        self.table = torch.full((len(lengths), cols), -1, dtype=torch.int32)
        # positions of a head together, or heads of a position together
        shape = (pages, kv_heads, page, dim) if layout == "heads" else (pages, page, kv_heads, dim)
        k, v = torch.full(shape, math.nan, dtype=dtype), torch.full(shape, math.nan, dtype=dtype)
        self.k, self.v = (k, v) if layout == "heads" else (k.transpose(1, 2), v.transpose(1, 2))
        self.rows, at = [], 0
        for r, n in enumerate(lengths):
            rk = (torch.randn(n, kv_heads, dim, generator=g) * 1.5).to(dtype)
            rv = torch.randn(n, kv_heads, dim, generator=g).to(dtype)
            self.rows.append((rk, rv))
            for c in range(need[r]):
                self.table[r, c] = order[at]
                m = min(page, n - c * page)
                self.k[order[at], :, :m] = rk[c * page:c * page + m].transpose(0, 1)
                self.v[order[at], :, :m] = rv[c * page:c * page + m].transpose(0, 1)
                at += 1

    def to(self, dev):
        return (self.k.to(dev), self.v.to(dev), self.table.to(dev),
                torch.tensor(self.lengths, dtype=torch.int32, device=dev))


def check(got, q, cache, where, scale, window, sinks):
    """got, q (tokens, heads, d); where: (row, position) of each token."""
    heads, group = q.shape[1], q.shape[1] // cache.k.shape[1]
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    for t, (r, p) in enumerate(where):
        rk, rv = cache.rows[r]
        see = seen_by(p, window, sinks) if p >= 0 else torch.zeros(0, dtype=torch.long)
        for g in range(heads // group):
            want, tol = want_and_tolerance(q[t, g * group:(g + 1) * group].cpu(), rk[see, g], rv[see, g], scale)
            over = ((got[t, g * group:(g + 1) * group] - want).abs() - tol).max().item()
            assert over <= 0, (r, p, g, over)


TOKEN = [
    # lengths, heads, kv heads, dim, page, window, sinks
    ([1], 8, 8, 128, 16, 0, 0),
    ([0, 5, 0], 8, 2, 128, 16, 0, 0),
    ([15, 16, 17, 31, 32, 33], 4, 4, 64, 16, 0, 0),
    ([63, 64, 65, 127, 128, 129], 28, 4, 128, 32, 0, 0),
    ([577], 64, 8, 128, 64, 0, 0),
    ([1000, 3, 0, 411], 32, 2, 128, 128, 0, 0),
    ([700, 90], 40, 2, 64, 32, 0, 0),
    ([300, 1, 77], 6, 2, 256, 16, 0, 0),
    ([2100], 16, 1, 256, 64, 0, 0),
    ([400, 50, 4], 8, 2, 128, 16, 1, 0),
    ([400, 50, 4], 8, 2, 128, 16, 33, 0),
    ([400, 50, 4, 0], 8, 2, 128, 16, 40, 4),
    ([900, 130], 28, 4, 128, 64, 100, 20),
    ([900, 130], 7, 1, 64, 32, 64, 64),
    ([4000], 8, 2, 128, 16, 5000, 3),
    ([6000, 17], 8, 1, 128, 256, 0, 0),
]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page,window,sinks", TOKEN)
def test_token(dev, lengths, heads, kv_heads, dim, page, window, sinks, dtype):
    from quipsharp_amd.pages import attend_token
    dt = TYPES[dtype]
    c = Cache(lengths, kv_heads, dim, page, dt, sum(lengths) + heads)
    q = torch.randn(len(lengths), heads, dim, generator=torch.Generator().manual_seed(dim)).to(dt).to(dev)
    got = attend_token(q, *c.to(dev), window=window, sinks=sinks)
    check(got, q, c, [(r, n - 1) for r, n in enumerate(lengths)], dim ** -0.5, window, sinks)


CHUNK = [
    # (new, cached) per row, heads, kv heads, dim, page, window, sinks
    ([(1, 0)], 8, 8, 128, 16, 0, 0),
    ([(5, 0), (0, 9), (1, 30)], 8, 2, 128, 16, 0, 0),
    ([(33, 0)], 4, 4, 64, 16, 0, 0),
    ([(64, 64), (65, 63), (31, 1)], 28, 4, 128, 32, 0, 0),
    ([(200, 0)], 16, 2, 128, 64, 0, 0),
    ([(130, 300), (7, 0), (257, 40)], 7, 1, 128, 32, 0, 0),
    ([(90, 33)], 40, 2, 64, 32, 0, 0),
    ([(40, 100), (3, 0)], 6, 2, 256, 16, 0, 0),
    ([(150, 0)], 8, 2, 128, 16, 1, 0),
    ([(150, 100), (20, 0)], 8, 2, 128, 16, 33, 4),
    ([(300, 0)], 8, 1, 128, 64, 64, 1),
    ([(300, 500), (129, 0)], 7, 1, 64, 16, 100, 20),
    ([(300, 100)], 8, 8, 128, 128, 4000, 7),
    ([(513, 0), (1, 700)], 4, 1, 128, 64, 256, 64),
]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,window,sinks", CHUNK)
def test_chunk(dev, rows, heads, kv_heads, dim, page, window, sinks, dtype):
    from quipsharp_amd.pages import attend_chunk
    dt = TYPES[dtype]
    lengths = [a + b for a, b in rows]
    c = Cache(lengths, kv_heads, dim, page, dt, sum(lengths) + heads)
    starts = [0]
    for a, _ in rows:
        starts.append(starts[-1] + a)
    q = torch.randn(starts[-1], heads, dim, generator=torch.Generator().manual_seed(dim)).to(dt).to(dev)
    got = attend_chunk(q, *c.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), window=window, sinks=sinks)
    check(got, q, c, [(r, b + i) for r, (a, b) in enumerate(rows) for i in range(a)], dim ** -0.5, window, sinks)


def test_chunk_with_more_tokens_than_the_row_holds(dev):
    """Tokens at positions below 0 see nothing and get zeros."""
    from quipsharp_amd.pages import attend_chunk
    c = Cache([20], 2, 128, 16, torch.bfloat16, 3)
    q = torch.randn(50, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    got = attend_chunk(q, *c.to(dev), torch.tensor([0, 50], dtype=torch.int32, device=dev))
    check(got, q, c, [(0, i - 30) for i in range(50)], 128 ** -0.5, 0, 0)


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 1, 128), (3, 3, 64), (4, 2, 256)])
def test_token_in_a_wide_table(dev, heads, kv_heads, dim, window, sinks):
    """Short and long rows in a table with columns for far longer ones: most shares of a row have nothing to do."""
    from quipsharp_amd.pages import attend_token
    lengths = [1, 0, 577, 130, 3000, 33]
    c = Cache(lengths, kv_heads, dim, 16, torch.bfloat16, 31, cols=2500)
    q = torch.randn(len(lengths), heads, dim, generator=torch.Generator().manual_seed(dim)).bfloat16().to(dev)
    got = attend_token(q, *c.to(dev), window=window, sinks=sinks)
    check(got, q, c, [(r, n - 1) for r, n in enumerate(lengths)], dim ** -0.5, window, sinks)


@pytest.mark.parametrize("kind", ["token", "chunk"])
def test_layouts_and_strides(dev, kind):
    """Heads of a position together in the pool, queries as a slice of a wider projection, output into a view."""
    from quipsharp_amd.pages import attend_chunk, attend_token
    lengths, heads = [70, 33, 128], 8
    c = Cache(lengths, 2, 128, 32, torch.bfloat16, 5, layout="positions", cols=9)
    k, v, table, n = c.to(dev)
    assert not k.is_contiguous()
    tokens = 3 if kind == "token" else 60
    wide = torch.randn(tokens, 2 * heads + 3, 128, generator=torch.Generator().manual_seed(2)).bfloat16().to(dev)
    q = wide[:, 3:3 + 2 * heads:2]
    room = torch.zeros(tokens, 2048, dtype=torch.bfloat16, device=dev)
    out = room[:, 512:512 + heads * 128].view(tokens, heads, 128)
    if kind == "token":
        attend_token(q, k, v, table, n, scale=0.2, out=out)
        where = [(r, m - 1) for r, m in enumerate(lengths)]
    else:
        attend_chunk(q, k, v, table, n, torch.tensor([0, 20, 30, 60], dtype=torch.int32, device=dev), scale=0.2, out=out)
        where = [(0, 50 + i) for i in range(20)] + [(1, 23 + i) for i in range(10)] + [(2, 98 + i) for i in range(30)]
    check(out, q, c, where, 0.2, 0, 0)
    assert not room[:, :512].any() and not room[:, 512 + heads * 128:].any()


@pytest.mark.parametrize("dim,pad_k,pad_v", [(64, 8, 24), (128, 8, 40), (256, 72, 8)])
def test_padded_positions(dev, dim, pad_k, pad_v):
    """Positions that lie further apart than their elements need, keys and values each in their own way."""
    from quipsharp_amd.pages import attend_chunk, attend_token
    c = Cache([150, 37], 2, dim, 16, torch.bfloat16, 13)
    k = torch.full(tuple(c.k.shape[:3]) + (dim + pad_k,), math.nan, dtype=torch.bfloat16, device=dev)[..., :dim]
    v = torch.full(tuple(c.v.shape[:3]) + (dim + pad_v,), math.nan, dtype=torch.bfloat16, device=dev)[..., pad_v:]
    k.copy_(c.k)
    v.copy_(c.v)
    _, _, table, n = c.to(dev)
    q = torch.randn(70, 6, dim, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    check(attend_token(q[:2], k, v, table, n), q[:2], c, [(0, 149), (1, 36)], dim ** -0.5, 0, 0)
    got = attend_chunk(q, k, v, table, n, torch.tensor([0, 60, 70], dtype=torch.int32, device=dev))
    check(got, q, c, [(0, 90 + i) for i in range(60)] + [(1, 27 + i) for i in range(10)], dim ** -0.5, 0, 0)


@pytest.mark.parametrize("kind", ["token", "chunk"])
def test_pages_out_of_the_window_may_be_gone(dev, kind):
    """Entries that no query of the call looks at may be -1 or name no page."""
    from quipsharp_amd.pages import attend_chunk, attend_token
    c = Cache([500], 2, 128, 16, torch.bfloat16, 6)
    k, v, table, n = c.to(dev)
    tokens = 1 if kind == "token" else 10
    last_free = 500 - tokens + 1 - 64  # a page that ends here or before is seen by nobody
    for p in range(1, last_free // 16):
        table[0, p] = -1 if p % 2 else 10 ** 6
    q = torch.randn(tokens, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    if kind == "token":
        got = attend_token(q, k, v, table, n, window=64, sinks=4)
    else:
        got = attend_chunk(q, k, v, table, n, torch.tensor([0, 10], dtype=torch.int32, device=dev), window=64, sinks=4)
    check(got, q, c, [(0, 500 - tokens + i) for i in range(tokens)], 128 ** -0.5, 64, 4)


@pytest.mark.parametrize("kind", ["token", "chunk"])
def test_positions_without_a_page_are_left_out(dev, kind):
    from quipsharp_amd.pages import attend_chunk, attend_token
    c = Cache([100], 1, 64, 16, torch.float16, 7)
    k, v, table, n = c.to(dev)
    table[0, 2] = -1
    table[0, 4] = k.shape[0]
    rk, rv = c.rows[0]
    left = [p for p in range(100) if p // 16 not in (2, 4)]
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1)).half().to(dev)
    if kind == "token":
        got = attend_token(q, k, v, table, n)
    else:
        got = attend_chunk(q, k, v, table, n, torch.tensor([0, 1], dtype=torch.int32, device=dev))
    want, tol = want_and_tolerance(q[0].cpu(), rk[left, 0], rv[left, 0], 0.125)
    assert ((got[0].cpu().double() - want).abs() <= tol).all()


def test_infinite_keys_outside_the_window(dev):
    """Infinities and NaN in places that the token does not see, in tiles that it reads."""
    from quipsharp_amd.pages import attend_token
    c = Cache([200], 1, 128, 64, torch.bfloat16, 8)
    for p, bad in ((150, math.inf), (151, math.nan), (10, -math.inf), (40, math.nan)):
        page = c.table[0, p // 64]
        c.k[page, :, p % 64] = bad
        c.v[page, :, p % 64] = bad
    q = torch.randn(1, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    got = attend_token(q, *c.to(dev), window=48, sinks=10)
    check(got, q, c, [(0, 199)], 128 ** -0.5, 48, 10)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim,window,sinks", [(4, 1, 128, 0, 0), (4, 2, 64, 40, 3), (8, 8, 128, 90, 0),
                                                             (2, 1, 256, 33, 20), (136, 136, 64, 70, 3)])
def test_values_that_are_no_numbers(dev, heads, kv_heads, dim, window, sinks, dtype):
    """Infinities and NaN reach the tokens that see their position, and no other."""
    from quipsharp_amd.pages import attend_chunk
    dt, n, new = TYPES[dtype], 300, 200
    c = Cache([n], kv_heads, dim, 32, dt, 21)
    k, v, table, length = c.to(dev)
    bad = {290: math.nan, 150: math.inf, 130: -math.inf, 199: math.nan, 64: math.inf, 1: math.nan if window else 0.5}
    for p, x in bad.items():
        v[int(c.table[0, p // 32]), kv_heads - 1, p % 32, 5::7] = x
        c.rows[0][1][p, kv_heads - 1, 5::7] = x
    q = torch.randn(new, heads, dim, generator=torch.Generator().manual_seed(1)).to(dt).to(dev)
    got = attend_chunk(q, k, v, table, length, torch.tensor([0, new], dtype=torch.int32, device=dev), window=window,
                       sinks=sinks).cpu().double()
    group = heads // kv_heads
    for t in range(new):
        see = seen_by(n - new + t, window, sinks)
        for g in range(kv_heads):
            rv = c.rows[0][1][see, g]
            out, tol = want_and_tolerance(q[t, g * group:(g + 1) * group].cpu(), c.rows[0][0][see, g],
                                          torch.nan_to_num(rv, 0, 0, 0), dim ** -0.5)
            fine = torch.isfinite(rv).all(0)  # dimensions without such a value
            mine = got[t, g * group:(g + 1) * group]
            assert torch.equal(torch.isfinite(mine), fine.expand(group, -1)), (t, g)
            assert ((mine - out).abs() <= tol)[:, fine].all(), (t, g)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,heads,kv_heads,dim,page,window,sinks", [
    ([(1, 6000)], 8, 1, 128, 64, 0, 0), ([(5, 4096), (0, 300), (3, 20), (2, 2500)], 4, 2, 64, 32, 0, 0),
    ([(7, 5000)], 6, 2, 256, 16, 0, 0), ([(9, 7000), (4, 5)], 7, 1, 128, 128, 3000, 20)])
def test_few_tokens_behind_a_long_cache(dev, rows, heads, kv_heads, dim, page, window, sinks, dtype):
    """Positions shared by several work-groups, some of whose shares hold nothing that a row sees; without a
    workspace one takes them all."""
    from quipsharp_amd import _lib
    from quipsharp_amd.pages import _pool, attend_chunk, chunk_workspace_bytes
    dt = TYPES[dtype]
    lengths = [a + b for a, b in rows]
    c = Cache(lengths, kv_heads, dim, page, dt, sum(lengths))
    starts = [0]
    for a, _ in rows:
        starts.append(starts[-1] + a)
    k, v, table, n = c.to(dev)
    q = torch.randn(starts[-1], heads, dim, generator=torch.Generator().manual_seed(dim)).to(dt).to(dev)
    begin = torch.tensor(starts, dtype=torch.int32, device=dev)
    assert chunk_workspace_bytes(starts[-1], heads, k, table, window, sinks) > 0
    where = [(r, b + i) for r, (a, b) in enumerate(rows) for i in range(a)]
    check(attend_chunk(q, k, v, table, n, begin, window=window, sinks=sinks), q, c, where, dim ** -0.5, window, sinks)
    whole = torch.empty_like(q)
    _lib.check(_lib.lib().qs_attend_chunk(q.data_ptr(), _lib.dtype_code(dt), starts[-1], len(rows), heads, kv_heads, dim,
                                          heads * dim, dim, begin.data_ptr(), _pool(k, v, table, n), dim ** -0.5, window,
                                          sinks, whole.data_ptr(), heads * dim, _lib.stream_of(q)))
    check(whole, q, c, where, dim ** -0.5, window, sinks)


@pytest.mark.parametrize("rows", [64, 65, 70, 200, 4200])
def test_many_rows_of_several_tokens(dev, rows):
    """More rows than a wave has lanes, of mixed lengths, some without new tokens."""
    from quipsharp_amd.pages import attend_chunk
    new = [(7 * r) % 5 for r in range(rows)]
    cached = [(13 * r) % 60 for r in range(rows)]
    c = Cache([a + b for a, b in zip(new, cached)], 1, 64, 16, torch.bfloat16, rows)
    starts = [0]
    for a in new:
        starts.append(starts[-1] + a)
    q = torch.randn(starts[-1], 3, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    got = attend_chunk(q, *c.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev))
    check(got, q, c, [(r, cached[r] + i) for r in range(rows) for i in range(new[r])], 0.125, 0, 0)


def test_lowest_and_equal_scores(dev):
    """Scores that are all the type's lowest, and all the same."""
    from quipsharp_amd.pages import attend_chunk, attend_token
    c = Cache([90], 1, 128, 16, torch.bfloat16, 9)
    k, v, table, n = c.to(dev)
    k[...] = 0
    k[..., 0] = torch.finfo(torch.bfloat16).min
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=dev)
    q[:, :, 0] = 1
    mean = c.rows[0][1].double().mean(0)
    bound = c.rows[0][1].double().abs().mean(0) * 2 ** -8 * 1.01 + mean.abs() * 2 ** -8
    one = torch.tensor([0, 1], dtype=torch.int32, device=dev)
    for got in (attend_token(q, k, v, table, n, scale=1.0), attend_chunk(q, k, v, table, n, one, scale=1.0)):
        assert ((got[0].cpu().double() - mean).abs() <= bound).all()


@pytest.mark.parametrize("scale", [-0.3, 1e-4, 2.0])
def test_other_scales(dev, scale):
    from quipsharp_amd.pages import attend_chunk, attend_token
    c = Cache([150], 2, 128, 32, torch.float16, 10)
    q = torch.randn(70, 4, 128, generator=torch.Generator().manual_seed(1)).half().to(dev)
    k, v, table, n = c.to(dev)
    check(attend_token(q[:1], k, v, table, n, scale=scale), q, c, [(0, 149)], scale, 0, 0)
    got = attend_chunk(q, k, v, table, n, torch.tensor([0, 70], dtype=torch.int32, device=dev), scale=scale)
    check(got, q, c, [(0, 80 + i) for i in range(70)], scale, 0, 0)


def test_long_cache_beyond_32_bits(dev):
    """Pages whose elements lie beyond 2^31 of the pool's start."""
    from quipsharp_amd.pages import append_pages, attend_chunk, attend_token
    kv_heads, page, dim = 8, 64, 128
    pages = (1 << 31) // (kv_heads * page * dim) + 40
    pool = torch.empty(pages, kv_heads, page, dim, dtype=torch.bfloat16, device=dev)
    lengths = torch.tensor([130], dtype=torch.int32, device=dev)
    table = torch.tensor([[pages - 1, pages - 7, pages - 3]], dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(130, kv_heads, dim, generator=g).bfloat16()
    append_pages(pool, pool, x.to(dev), x.to(dev), table, lengths, torch.tensor([0, 130], dtype=torch.int32, device=dev))
    q = torch.randn(2, 16, dim, generator=g).bfloat16()
    got = attend_token(q[1:].to(dev), pool, pool, table, lengths)
    both = attend_chunk(q.to(dev), pool, pool, table, lengths, torch.tensor([0, 2], dtype=torch.int32, device=dev))
    for h in range(kv_heads):
        for t, out, n in ((1, got[0], 130), (0, both[0], 129), (1, both[1], 130)):
            want, tol = want_and_tolerance(q[t, 2 * h:2 * h + 2], x[:n, h], x[:n, h], dim ** -0.5)
            assert ((out[2 * h:2 * h + 2].cpu().double() - want).abs() <= tol).all()


def test_on_another_stream(dev):
    from quipsharp_amd.pages import attend_token
    c = Cache([333, 80], 2, 128, 32, torch.float16, 11)
    k, v, table, n = c.to(dev)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(1)).half().to(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = attend_token(q, k, v, table, n)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, attend_token(q, k, v, table, n))


def test_same_call_gives_the_same_bits(dev):
    from quipsharp_amd.pages import attend_chunk, attend_token
    c = Cache([3000, 100, 777], 2, 128, 32, torch.bfloat16, 12)
    k, v, table, n = c.to(dev)
    q = torch.randn(60, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    starts = torch.tensor([0, 20, 40, 60], dtype=torch.int32, device=dev)
    first = attend_token(q[:3], k, v, table, n), attend_chunk(q, k, v, table, n, starts)
    for _ in range(5):
        assert torch.equal(first[0], attend_token(q[:3], k, v, table, n))
        assert torch.equal(first[1], attend_chunk(q, k, v, table, n, starts))


@pytest.mark.parametrize("cols", [4, 200])
def test_lengths_below_zero(dev, cols):
    """A row whose length is below zero, down to the type's lowest, sees nothing."""
    from quipsharp_amd import pages
    cache = Cache([40, 40, 40], 2, 64, 16, torch.bfloat16, 29, cols=cols)
    k, v, table, _ = cache.to(dev)
    lengths = torch.tensor([-1, -2 ** 31, 40], dtype=torch.int32, device=dev)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(30)).to(torch.bfloat16)
    where = [(0, -1), (1, -1), (2, 39)]
    for window, sinks in [(0, 0), (20, 3)]:
        got = pages.attend_token(q.to(dev), k, v, table, lengths, window=window, sinks=sinks)
        check(got, q, cache, where, 64 ** -0.5, window, sinks)
        starts = torch.arange(4, dtype=torch.int32, device=dev)
        got = pages.attend_chunk(q.to(dev), k, v, table, lengths, starts, window=window, sinks=sinks)
        check(got, q, cache, where, 64 ** -0.5, window, sinks)


@pytest.mark.parametrize("rows,new,cached,heads,kv_heads,dim", [(16, 3, 2500, 8, 2, 128), (40, 2, 300, 16, 8, 64),
                                                              (5, 20, 1100, 7, 1, 256)])
def test_rows_of_few_tokens(dev, rows, new, cached, heads, kv_heads, dim):
    """Blocks that are mostly empty, with and without shares of the positions; some rows have no token."""
    from quipsharp_amd.pages import attend_chunk
    g = torch.Generator().manual_seed(rows)
    news = torch.randint(0, new + 1, (rows,), generator=g).tolist()
    lengths = [n + m for n, m in zip(news, torch.randint(0, cached, (rows,), generator=g).tolist())]
    c = Cache(lengths, kv_heads, dim, 16, torch.bfloat16, rows + 1)
    starts = torch.tensor([0] + news).cumsum(0).to(torch.int32)
    q = torch.randn(sum(news), heads, dim, generator=g).bfloat16()
    got = attend_chunk(q.to(dev), *c.to(dev), starts.to(dev))
    check(got, q, c, [(r, lengths[r] - news[r] + i) for r in range(rows) for i in range(news[r])], dim ** -0.5, 0, 0)
