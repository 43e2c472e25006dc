"""Low-rank adapters beside shared linears (csrc/qs_adapters.hip) against the
definition in 64 bits.  With u = 2^-24, what is allowed per output: half a step
of its type; u |y|; for the second product (2 rank + 8) u of its sum of sizes;
and of |scale| sum |up| what an inner product may be off: (n + 8) u of its sum of
sizes, and of the token's largest one 2^-16 (bf16: two numbers of 8 bits) or
2^-22 (fp16: two of 11 bits, the second down to 2^-25)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, I32 = torch.bfloat16, torch.float16, torch.int32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def expected(y, x, which, down, up, scale):
    """In 64 bits on the CPU: the sum, and how far an output may be off apart from the last rounding."""
    u = 2.0 ** -24
    out, err = y.double(), y.double().abs() * u
    dtype, n, rank = x.dtype, x.shape[1], down.shape[1]
    for a in range(down.shape[0]):
        t = (which == a).nonzero()[:, 0]
        if not len(t):
            continue
        d, w, s, xs = down[a].double(), up[a].double(), scale[a].double(), x[t].double()
        v = xs @ d.t()
        off = (n + 8) * u * (xs.abs() @ d.abs().t()) + v.abs().amax(1, keepdim=True) * 2.0 ** (-16 if dtype is BF else -22)
        out[t] += s * (v @ w.t())
        err[t] += s.abs() * (off @ w.abs().t() + (2 * rank + 8) * u * ((v.abs() + off) @ w.abs().t()))
    return out, err


def near(got, want, err, dtype):
    step = torch.finfo(dtype).eps / 2 * (want.abs() + err) + (2.0 ** -25 if dtype is HF else 0.0)
    assert ((got.cpu().double() - want).abs() <= step + err).all()


def run(dev, which, n, ms, rank, adapters=4, dtype=BF, inplace=False, seed=0, ranks=None, scale=1.0):
    from quipsharp_amd.adapters import add_adapters
    g = gen(seed)
    which = torch.as_tensor(which, dtype=I32)
    tokens = len(which)
    ranks = ranks or [rank] * len(ms)
    x = make(g, tokens, n, dtype=dtype)
    ys = [make(g, tokens, m, dtype=dtype) for m in ms]
    downs = [make(g, adapters, r, n, dtype=dtype, scale=n ** -0.5) for r in ranks]
    ups = [make(g, adapters, m, r, dtype=dtype, scale=0.2) for m, r in zip(ms, ranks)]
    scales = [scale * (torch.rand(adapters, generator=g) + 0.5) for _ in ms]
    to = lambda ts: [t.to(dev) for t in ts]  # noqa: E731
    dy = to(ys)
    got = add_adapters(dy, x.to(dev), which.to(dev), to(downs), to(ups), to(scales), outs=dy if inplace else None)
    for g_, o in enumerate(got):
        want, err = expected(ys[g_], x, which, downs[g_], ups[g_], scales[g_])
        near(o, want, err, dtype)
        none = (which < 0) | (which >= adapters)
        assert torch.equal(o.cpu()[none], ys[g_][none])
        assert inplace or torch.equal(dy[g_].cpu(), ys[g_])
    return got


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128])
def test_ranks(dev, rank, dtype):
    run(dev, [2], 512, [256], rank, dtype=dtype)
    run(dev, [0, 3, -1, 3, 2], 512, [256, 96], rank, dtype=dtype)


@pytest.mark.parametrize("n", [8, 16, 40, 256, 264, 1000, 4096, 18944])
@pytest.mark.parametrize("m", [1, 15, 16, 17, 64, 255, 1031])
def test_widths(dev, n, m):
    run(dev, [1, 0, 1], n, [m], 16, dtype=HF)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 63, 64, 65, 130, 500])
def test_tokens_in_any_order(dev, tokens, dtype):
    g = gen(tokens)
    which = torch.randint(-1, 7, (tokens,), generator=g)
    run(dev, which, 320, [160, 48], 16, adapters=7, dtype=dtype)
    run(dev, which, 320, [160, 48], 16, adapters=7, dtype=dtype, inplace=True)


@pytest.mark.parametrize("counts", [[100, 3, 64, 0, 200], [1, 63, 64, 65, 1], [700], [17, 16, 15, 14]])
def test_prompts_in_runs(dev, counts):
    which = [a % 5 - 1 for a, c in enumerate(counts) for _ in range(c)]
    run(dev, which, 512, [384, 128, 128], 32, dtype=BF)


def test_long_prompts(dev):
    which = [0] * 1500 + [-1] * 70 + [3] * 900
    run(dev, which, 1024, [640], 64, dtype=BF)
    run(dev, which, 1024, [640], 64, dtype=HF, inplace=True)


@pytest.mark.parametrize("ranks", [[8, 24, 8], [72], [88, 8], [96, 40, 104], [128, 128, 128, 128]])
@pytest.mark.parametrize("tokens", [100, 1100, 4200])
def test_ranks_that_differ_for_prompts(dev, tokens, ranks):
    """Blocks of ranks that belong to two linears, whole runs of them and the last one's end; groups of more and of
    fewer than 16 tokens; widths that end inside an access."""
    cuts = [tokens // 3 + 5, 9, tokens // 2, tokens]
    which = [a for a, c in zip((2, 1, -1, 0), cuts) for _ in range(c)][:tokens]
    run(dev, which, 200, [131, 64, 33, 7][:len(ranks)], 0, ranks=ranks, adapters=3, dtype=HF if tokens == 100 else BF)


def test_every_token_its_own_adapter(dev):
    run(dev, torch.randperm(64, generator=gen(1)), 256, [256], 16, adapters=64)
    run(dev, torch.randperm(300, generator=gen(1)), 256, [64], 8, adapters=300)


def test_ranks_that_differ(dev):
    run(dev, [0, 1, 1, 2, -1, 0], 512, [64, 32, 128, 16], 0, ranks=[8, 128, 16, 40])


def test_adapters_that_no_row_names(dev):
    """Rows that name none, and numbers beyond: out is y, bit for bit, and weights that are no numbers are not touched."""
    from quipsharp_amd.adapters import add_adapters
    g = gen(2)
    x, y = make(g, 5, 64), make(g, 5, 40)
    which = torch.tensor([-1, 3, 2 ** 31 - 1, -2 ** 31, 1], dtype=I32)
    down, up = make(g, 3, 8, 64), make(g, 3, 40, 8)
    down[0] = up[2] = float("nan")
    scale = torch.ones(3)
    got, = add_adapters([y.to(dev)], x.to(dev), which.to(dev), [down.to(dev)], [up.to(dev)], [scale.to(dev)])
    assert torch.equal(got.cpu()[:4], y[:4])
    want, err = expected(y, x, which, down, up, scale)
    near(got[4:], want[4:], err[4:], BF)


def test_products_beyond_the_range_of_fp16(dev):
    """Inner products of 10^5 and of 10^-6 in one call: neither is rounded to infinity or to nothing."""
    from quipsharp_amd.adapters import add_adapters
    g = gen(3)
    x = make(g, 2, 1024, dtype=HF)
    x[0] *= 100
    x[1] *= 1e-3
    down = make(g, 1, 16, 1024, dtype=HF, scale=100.0)
    up = make(g, 1, 64, 16, dtype=HF, scale=1e-3)
    y = torch.zeros(2, 64, dtype=HF)
    y[1] = 0
    which, scale = torch.zeros(2, dtype=I32), torch.tensor([0.05])
    got, = add_adapters([y.to(dev)], x.to(dev), which.to(dev), [down.to(dev)], [up.to(dev)], [scale.to(dev)])
    assert (x[0].double() @ down[0].double().t()).abs().max() > 1e5
    want, err = expected(y, x, which, down, up, scale)
    near(got, want, err, HF)


def test_rows_that_are_no_numbers_stay_alone(dev):
    """An infinite or undefined input spoils its own token's outputs and no other's, of the same adapter or not."""
    from quipsharp_amd.adapters import add_adapters
    g = gen(4)
    which = torch.tensor([0, 0, 1, 0, 1, 0], dtype=I32)
    x, y = make(g, 6, 128), make(g, 6, 80)
    down, up, scale = make(g, 2, 16, 128, scale=0.1), make(g, 2, 80, 16), torch.ones(2)
    want, err = expected(y, x, which, down, up, scale)
    x[1, 5], x[4, 100] = float("inf"), float("nan")
    got, = add_adapters([y.to(dev)], x.to(dev), which.to(dev), [down.to(dev)], [up.to(dev)], [scale.to(dev)])
    fine = torch.tensor([0, 2, 3, 5])
    near(got.cpu()[fine], want[fine], err[fine], BF)
    assert not torch.isfinite(got[1]).any() and torch.isnan(got[4]).all()


def test_strides(dev):
    """Rows of wider tensors, banks cut from larger ones, outputs at odd places."""
    from quipsharp_amd.adapters import add_adapters
    g = gen(5)
    tokens, n, m, rank = 70, 128, 75, 16
    which = torch.randint(-1, 3, (tokens,), generator=g).int()
    x, y = make(g, tokens, n + 24).to(dev)[:, 8:8 + n], make(g, tokens, m + 6).to(dev)[:, 3:3 + m]
    down = make(g, 3, rank + 8, n + 16, scale=0.1).to(dev)[:, :rank, 8:8 + n]
    up = make(g, 3, m + 2, rank + 8).to(dev)[:, :m, :rank]
    out = torch.zeros(tokens, m + 9, dtype=BF, device=dev)
    scale = torch.ones(3)
    got, = add_adapters([y], x, which.to(dev), [down], [up], [scale.to(dev)], outs=[out[:, 5:5 + m]])
    want, err = expected(y.cpu(), x.cpu(), which, down.cpu(), up.cpu(), scale)
    near(got, want, err, BF)
    assert (out[:, :5] == 0).all() and (out[:, 5 + m:] == 0).all()


@pytest.mark.parametrize("tokens", [9, 70, 300])
def test_rows_as_far_apart_as_they_may_be(dev, tokens):
    """x, y, out and weights with rows 2^24 elements apart: 2^32 bytes are in 128 of them, a tile's last token lies 2^31
    behind its first."""
    from quipsharp_amd.adapters import add_adapters
    g = gen(10)
    far, n, m, rank = 2 ** 24, 72, 75, 16
    space = torch.empty(tokens * far, dtype=BF, device=dev).view(tokens, far)
    x, y, out = space[:, :n], space[:, 1001:1001 + m], space[:, 2003:2003 + m]
    weights = torch.empty(2 * m * far, dtype=BF, device=dev).view(2, m, far)
    down, up = weights[:, :rank, 128:128 + n], weights[:, :, :rank]
    for t, scale in ((x, 1.0), (y, 1.0), (down, 0.1), (up, 1.0)):
        t.copy_(torch.randn(t.shape, generator=g) * scale)
    out.zero_()
    which = (torch.arange(tokens) // 40 % 3 - 1).int()
    got, = add_adapters([y], x, which.to(dev), [down], [up], [torch.ones(2, device=dev)], outs=[out])
    want, err = expected(y.cpu(), x.cpu(), which, down.cpu(), up.cpu(), torch.ones(2))
    near(got, want, err, BF)


def test_a_call_repeats_itself(dev):
    g = gen(6)
    which = torch.randint(-1, 5, (200,), generator=g)
    a = run(dev, which, 2048, [512], 64, adapters=5)
    b = run(dev, which, 2048, [512], 64, adapters=5)
    assert torch.equal(a[0], b[0])


def test_replayed_and_on_another_stream(dev):
    """A captured call follows the adapters that its rows name and the weights that are loaded; two graphs that are
    given one workspace replay in turn."""
    from quipsharp_amd.adapters import Adapters, add_adapters
    g = gen(7)
    tokens, n, m = 5, 256, 96
    bank = Adapters(3, 10, n, m, device=dev)
    x, y = make(g, tokens, n).to(dev), make(g, tokens, m).to(dev)
    which = torch.zeros(tokens, dtype=I32, device=dev)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    call = lambda xs: add_adapters([y], xs, which, [bank.down], [bank.up], [bank.scale], workspace=ws)[0]  # noqa: E731
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(x)
    torch.cuda.current_stream().wait_stream(s)
    x2 = make(g, tokens, n).to(dev)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, xs in zip(graphs, (x, x2)):
        with torch.cuda.graph(graph):
            outs.append(call(xs))
    for step in range(4):
        bank.load(step % 3, make(g, 10, n, scale=0.1).to(dev), make(g, m, 10).to(dev), 0.5 + step)
        which.copy_(torch.randint(-1, 3, (tokens,), generator=g).int())
        x.copy_(make(g, tokens, n))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], call(x)) and torch.equal(outs[1], call(x2))


def test_bank(dev):
    """Adapters of lower ranks than the bank's, replaced and taken out."""
    from quipsharp_amd.adapters import Adapters, add_adapters
    g = gen(8)
    bank = Adapters(2, 13, 64, 40, device=dev)
    assert bank.down.shape == (2, 16, 64)
    bank.load(1, make(g, 13, 64).to(dev), make(g, 40, 13).to(dev), 9.0)
    d, u = make(g, 5, 64), make(g, 40, 5)
    bank.load(1, d.to(dev), u.to(dev), 2.0)
    x, y = make(g, 3, 64), make(g, 3, 40)
    which = torch.tensor([1, 0, 1], dtype=I32)
    got, = add_adapters([y.to(dev)], x.to(dev), which.to(dev), [bank.down], [bank.up], [bank.scale])
    want, err = expected(y, x, torch.tensor([0, -1, 0]), d[None], u[None], torch.tensor([2.0]))
    near(got, want, err, BF)
    assert torch.equal(got.cpu()[1], y[1])
    bank.clear(1)
    got, = add_adapters([y.to(dev)], x.to(dev), which.to(dev), [bank.down], [bank.up], [bank.scale])
    assert torch.equal(got.cpu(), y)


def test_empty(dev):
    from quipsharp_amd.adapters import add_adapters
    z = lambda *s: torch.zeros(*s, dtype=BF, device=dev)  # noqa: E731
    got, = add_adapters([z(0, 16)], z(0, 32), torch.zeros(0, dtype=I32, device=dev), [z(2, 8, 32)], [z(2, 16, 8)],
                        [torch.zeros(2, device=dev)])
    assert got.shape == (0, 16)
