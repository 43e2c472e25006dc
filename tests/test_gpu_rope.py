"""Rotary positions with the cache write (csrc/qs_rope.hip) against the
definition in 64 bits, a pair as one complex number.  What is allowed per
element: half a step of its type for the one rounding (2^-8 of a bf16 value,
2^-11 of an fp16 value, 2^-25 below fp16's normal ones), and of the sizes of
its pair 2^-21 for the sine and cosine (a fraction of a turn in 32 bits, 2 steps
of the functions, products) and 2^-50 of the angle for the 64-bit product."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, I32 = torch.bfloat16, torch.float16, torch.int32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def turned(x, pos, w, layout, factor):
    """x (tokens, heads, dim) on the CPU: the result in 64 bits, and the sizes of every element's pair."""
    n = len(w)
    x = x.double()
    z = x[:, :, :2 * n]
    z = z.unflatten(2, (2, n)).transpose(2, 3) if layout == "half" else z.unflatten(2, (n, 2))
    turn = torch.polar(torch.full((1, 1), factor, dtype=torch.float64), pos[:, None].double() * w)[:, None]
    o = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    size = z.abs().sum(-1, keepdim=True).expand_as(z) * abs(factor)
    back = (lambda t: t.transpose(2, 3).flatten(2)) if layout == "half" else (lambda t: t.flatten(2))
    angle = (pos[:, None].abs().double() * w)[:, None, :, None].expand_as(z)
    out, err = x.clone(), torch.zeros_like(x)
    out[:, :, :2 * n] = back(o)
    err[:, :, :2 * n] = back(size * (2.0 ** -21 + angle * 2.0 ** -50))
    return out, err


def near(got, want, err, dtype):
    step = torch.finfo(dtype).eps / 2 * (want.abs() + err) + (2.0 ** -25 if dtype is HF else 0.0)
    over = (got.double() - want).abs() - (step + err)
    assert over.max().item() <= 0 if over.numel() else True


def run(dev, new, cached, heads=4, kv_heads=2, dim=128, pairs=64, page=16, layout="half", dtype=BF, factor=1.0, base=1e4,
        starts=None, tokens=None, spare_cols=1, over=None, fused=False, inplace=False, seed=0):
    """new, cached: per row.  Compares queries, keys and values with the definition, and that nothing else changed."""
    from quipsharp_amd.rope import append_rotated
    g = gen(seed)
    rows = len(new)
    one = starts is None and tokens is None and all(n == 1 for n in new)
    at = [0] + list(itertools.accumulate(new))
    total = at[-1] if tokens is None else tokens
    cols = max(-(-(a + b) // page) for a, b in zip(new, cached)) + spare_cols
    pages = sum(-(-(a + b) // page) - b // page for a, b in zip(new, cached)) + 2
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((rows, cols), -1, dtype=I32)
    for r, (a, b) in enumerate(zip(new, cached)):
        for c in range(b // page, -(-(a + b) // page)):
            table[r, c] = order.pop()
    lengths = torch.tensor([a + b for a, b in zip(new, cached)], dtype=I32)
    parts = [heads * dim, kv_heads * dim, kv_heads * dim]
    make = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    flat = make(total, sum(parts)).to(dev).split(parts, 1) if fused else [make(total, p).to(dev) for p in parts]
    q, k, v = (t.unflatten(1, (-1, dim)) for t in flat)
    kp, vp = make(pages, kv_heads, page, dim), make(pages, kv_heads, page, dim)
    kd, vd = kp.to(dev), vp.to(dev)
    w = float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
    hq, hk, hv = q.cpu(), k.cpu(), v.cpu()
    out = q if inplace else torch.full((total, heads, dim), 7.0, dtype=dtype, device=dev)
    got = append_rotated(q, k, v, kd, vd, table.to(dev), lengths.to(dev), w.to(dev),
                         starts=None if one else torch.tensor(at, dtype=I32, device=dev), layout=layout, factor=factor,
                         over=None if over is None else torch.tensor(over, dtype=I32, device=dev), out=out)
    assert got is out
    row = torch.repeat_interleave(torch.arange(rows), torch.tensor(new))
    inside = torch.arange(at[-1])
    pos = lengths.long()[row] - torch.tensor(at)[row + 1] + inside
    want, err = turned(hq[:at[-1]], pos, w, layout, factor)
    near(got.cpu()[:at[-1]], want, err, dtype)
    rest = got.cpu()[at[-1]:]
    assert torch.equal(rest, hq[at[-1]:] if inplace else torch.full_like(rest, 7.0))
    wk, ek = turned(hk[:at[-1]], pos, w, layout, factor)
    ids = table[row, pos // page].long()
    near(kd.cpu()[ids, :, pos % page], wk, ek, dtype)
    vp[ids, :, pos % page] = hv[:at[-1]]
    assert torch.equal(vd.cpu(), vp)
    untouched = torch.ones(pages, page, dtype=torch.bool)
    untouched[ids, pos % page] = False
    assert torch.equal(kd.cpu().transpose(1, 2)[untouched], kp.transpose(1, 2)[untouched])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,pairs", [(128, 64), (64, 32), (256, 128), (128, 32), (96, 48), (96, 12), (8, 1), (24, 5),
                                       (64, 4), (40, 20), (512, 256)])
def test_heads_and_pairs(dev, dim, pairs, layout, dtype):
    run(dev, [5, 1, 17], [30, 0, 15], dim=dim, pairs=pairs, layout=layout, dtype=dtype)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (64, 8), (28, 4), (3, 2), (2, 5), (16, 1)])
def test_head_counts(dev, heads, kv_heads, layout):
    run(dev, [1] * 7, [0, 1, 15, 16, 17, 31, 100], heads=heads, kv_heads=kv_heads, layout=layout, factor=1.3)
    run(dev, [9, 2], [3, 40], heads=heads, kv_heads=kv_heads, layout=layout)


@pytest.mark.parametrize("rows", [1, 2, 48, 257])
def test_single_tokens(dev, rows):
    g = gen(rows)
    cached = torch.randint(0, 3000, (rows,), generator=g).tolist()
    run(dev, [1] * rows, cached, page=32, dtype=HF)


@pytest.mark.parametrize("new", [[700], [0, 300, 0, 1, 260, 0], [1] * 40 + [900], [0, 0, 3]])
def test_prompts(dev, new):
    """Rows without tokens among them; more tokens than a work-group takes."""
    run(dev, new, [(37 * i) % 90 for i in range(len(new))], page=64)


@pytest.mark.parametrize("cached", [100_000, 1_000_000, 16_000_000])
def test_far_positions(dev, cached):
    """Angles of millions of radians: the fastest pair turns once a position."""
    run(dev, [3, 1], [cached, cached - 5], page=4096, dtype=HF, base=5e5)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_in_place(dev, layout):
    run(dev, [5, 30], [3, 20], fused=True, layout=layout, pairs=32)
    run(dev, [5, 30], [3, 20], inplace=True, layout=layout)
    run(dev, [1, 1, 1], [3, 20, 16], fused=True, inplace=True, layout=layout, pairs=32)


def test_tokens_of_no_row(dev):
    run(dev, [5, 9], [3, 20], tokens=40)
    run(dev, [5, 9], [3, 20], tokens=15, inplace=True)


def test_pages_beyond_32_bits(dev):
    """Pages that lie 9 GB into a pool, and rows of q 2^28 elements apart."""
    from quipsharp_amd.rope import append_rotated
    g = gen(9)
    pages, page, dim = 1_150_000, 16, 128
    kv = torch.empty(2, pages, 2, page, dim, dtype=BF, device=dev)
    wide = torch.empty(9 * 2 ** 28, dtype=BF, device=dev)
    q = torch.as_strided(wide, (9, 4, dim), (2 ** 28, dim, 1))
    q.copy_(torch.randn(9, 4, dim, generator=g))
    k, v = torch.randn(2, 9, 2, dim, generator=g).to(BF)
    table = torch.arange(pages - 9, pages, dtype=I32)[:, None]
    lengths = torch.arange(1, 10, dtype=I32)
    w = 1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)
    got = append_rotated(q, k.to(dev), v.to(dev), kv[0], kv[1], table.to(dev), lengths.to(dev), w.to(dev))
    pos = lengths.long() - 1
    near(got.cpu(), *turned(q.cpu(), pos, w, "half", 1.0), BF)
    near(kv[0, pages - 9:].cpu()[torch.arange(9), :, pos], *turned(k, pos, w, "half", 1.0), BF)
    assert torch.equal(kv[1, pages - 9:].cpu()[torch.arange(9), :, pos], v)


def test_no_page_no_row_no_position(dev):
    """Tokens without a page, beyond the table, and before position 0."""
    from quipsharp_amd.rope import append_rotated
    page, dim = 16, 64
    g = gen(3)
    make = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)  # noqa: E731
    q, k, v = make(6, 2, dim), make(6, 1, dim), make(6, 1, dim)
    kp, vp = make(3, 1, page, dim), make(3, 1, page, dim)
    w = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    # a hole, an id beyond the pool, beyond the table, over the table's end, a row shorter than its tokens, one below 0
    table = torch.tensor([[-1, 2], [9, 1], [0, 1], [0, 1], [0, 1], [0, 1]], dtype=I32, device=dev)
    lengths = torch.tensor([5, 6, 40, 32, 0, -7], dtype=I32, device=dev)
    over = torch.tensor([0, 0, 0, 4, 0, 0], dtype=I32, device=dev)
    k0, v0 = kp.clone(), vp.clone()
    got = append_rotated(q, k, v, kp, vp, table, lengths, w.to(dev), over=over).cpu()
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    want, err = turned(q.cpu(), torch.tensor([4, 5, 39, 35, 0, 0]), w, "half", 1.0)
    near(got[:4], want[:4], err[:4], BF)
    assert (got[4:] == 0).all()


def test_scaled_frequencies_reach_the_kernel(dev):
    """The frequencies of a stretched context, as a model's config has them."""
    from quipsharp_amd.rope import append_rotated, rope_frequencies
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    w, factor = rope_frequencies(128, 1e6, scaling, dev)
    g = gen(4)
    q, k = torch.randn(1, 4, 128, generator=g).bfloat16(), torch.randn(1, 2, 128, generator=g).bfloat16()
    kp, vp = torch.zeros(1, 2, 64, 128, dtype=BF, device=dev), torch.zeros(1, 2, 64, 128, dtype=BF, device=dev)
    table = torch.full((1, 2000), -1, dtype=I32, device=dev)
    table[0, 100_000 // 64] = 0
    got = append_rotated(q.to(dev), k.to(dev), k.to(dev), kp, vp, table, torch.tensor([100_001], dtype=I32, device=dev), w,
                         factor=factor)
    want, err = turned(q, torch.tensor([100_000]), w.cpu(), "half", factor)
    near(got.cpu(), want, err, BF)
    want, err = turned(k, torch.tensor([100_000]), w.cpu(), "half", factor)
    near(kp.cpu()[:, :, 100_000 % 64], want, err, BF)


def test_replayed_and_on_another_stream(dev):
    """A captured call follows the lengths that lie in its tensors; on a stream of its own it waits for nothing else."""
    from quipsharp_amd.rope import append_rotated
    g = gen(5)
    rows, dim, page = 3, 128, 16
    make = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)  # noqa: E731
    q, k, v = make(rows, 4, dim), make(rows, 2, dim), make(rows, 2, dim)
    kp, vp = make(12, 2, page, dim), make(12, 2, page, dim)
    table = torch.arange(12, dtype=I32, device=dev).view(3, 4)
    lengths = torch.tensor([1, 17, 30], dtype=I32, device=dev)
    w = (1e4 ** (-torch.arange(64, dtype=torch.float64) / 64)).to(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        append_rotated(q, k, v, kp, vp, table, lengths, w)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = append_rotated(q, k, v, kp, vp, table, lengths, w)
    for step in range(4):
        lengths += 1
        graph.replay()
        torch.cuda.synchronize()
        ks, vs = kp.clone(), vp.clone()
        want = append_rotated(q, k, v, ks, vs, table, lengths, w)
        assert torch.equal(out, want) and torch.equal(kp, ks) and torch.equal(vp, vs)


def test_empty(dev):
    from quipsharp_amd.rope import append_rotated
    kp = torch.zeros(2, 1, 16, 64, dtype=BF, device=dev)
    w = torch.ones(32, dtype=torch.float64, device=dev)
    none = torch.zeros(0, 1, 64, dtype=BF, device=dev)
    starts = torch.zeros(3, dtype=I32, device=dev)
    out = append_rotated(none, none, none, kp, kp.clone(), torch.zeros(2, 1, dtype=I32, device=dev),
                         torch.zeros(2, dtype=I32, device=dev), w, starts=starts)
    assert out.shape == (0, 1, 64)
