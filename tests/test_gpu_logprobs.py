"""Log probabilities of given tokens (csrc/qs_logprobs.hip) against the
definition in 64 bits on the CPU.  Ranks and alternatives are exact.  With u =
2^-24 a log sum may be off by (3 ln(vocab) + 20) u (derived at the kernel), a log
probability by that and its rounding, u of itself.  The entropy's second sum has
terms p D, each off by (2.25 D + 18) u of itself, so the entropy may be off by
((3 ln(vocab) + 20) (1 + E) + 18 E + 3 E2) u and its rounding, E and E2 the means
of D and D^2 over the distribution, D how far a logit lies below the largest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def expected(x, tokens, top):
    """x (rows, vocab) on the CPU."""
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    R, V = x.shape
    out = []
    for r in range(R):
        row, t = x[r], int(tokens[r])
        m = row.max()
        value, order = torch.sort(row, descending=True, stable=True)
        scored = 0 <= t < V
        rank = int((order == t).nonzero()[0, 0]) if scored else -1
        if not torch.isfinite(m):
            out.append((-math.inf if scored else 0.0, 0.0, rank, [-math.inf] * top, [-1] * top, 0.0, 0.0))
            continue
        logp = row - m - (row - m).exp().sum().log()
        p = logp.exp()
        D = torch.where(p > 0, m - row, 0.0)
        H = -(torch.where(p > 0, p * logp, 0.0)).sum()
        best = [(float(logp[i]), int(i)) if value[j] > -math.inf else (-math.inf, -1) for j, i in enumerate(order[:top])]
        out.append((float(logp[t]) if scored else 0.0, float(H), rank, [b[0] for b in best], [b[1] for b in best],
                    float((p * D).sum()), float((p * D * D).sum())))
    return out


def check(dev, x, tokens, top, on_gpu=None):
    from quipsharp_amd.logprobs import token_logprobs
    V = x.shape[1]
    got = [t.cpu() for t in token_logprobs((x.to(dev) if on_gpu is None else on_gpu), tokens.to(dev), top)]
    assert [t.dtype for t in got] == [torch.float32, torch.float32, torch.int32, torch.float32, torch.int32]
    unit = (3 * math.log(V) + 20) * U
    for r, (lp, H, rank, best, ids, E, E2) in enumerate(expected(x, tokens, top)):
        assert got[2][r] == rank and got[4][r].tolist() == ids
        for a, b in [(got[0][r].item(), lp)] + list(zip(got[3][r].tolist(), best)):
            if math.isinf(b):
                assert a == b
            elif abs(b) > 3.4028235e38:
                assert a == -math.inf
            else:
                assert abs(a - b) <= unit + U * abs(b)
        assert abs(got[1][r].item() - H) <= unit * (1 + E) + (18 * E + 3 * E2) * U + U * H
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 1, 0), (3, 7, 7), (1, 64, 64), (2, 50, 20), (1, 1000, 5), (5, 2048, 10), (4, 2049, 1), (3, 8191, 64),
    (2, 32000, 33), (7, 12289, 8), (2, 50257, 9), (1, 151936, 5), (70, 20000, 4), (600, 900, 3)])
def test_scores(dev, rows, vocab, top, dtype):
    g = torch.Generator().manual_seed(vocab + top)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    check(dev, x, tokens, top)
    check(dev, x, x.float().argmax(1).int(), top)


@pytest.mark.parametrize("rows", [1, 40, 700])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
@pytest.mark.parametrize("order", ["ascending", "descending", "equal", "two values", "steps", "rare", "few"])
def test_orders(dev, order, top, rows):
    """Every slice brings better ones, none does, and all are alike: the lower tokens win."""
    V = 20011
    x = {"ascending": torch.arange(V) / 997.0, "descending": -torch.arange(V) / 997.0, "equal": torch.full((V,), 1.5),
         "two values": (torch.arange(V) % 7 == 3).float(), "steps": (torch.arange(V) // 40).float() / 8,
         "rare": (torch.arange(V) % 61 == 60).float(), "few": torch.arange(V) % 500 // 499 + (torch.arange(V) % 33 == 7) / 2}[order]
    x = x.float()[None].repeat(rows, 1)
    tokens = torch.tensor([(7 * i + 3) % V for i in range(rows)])
    tokens[-1] = V - 1
    if rows > 40:  # the same rows over and over: a few against the definition, the others against them
        got = check(dev, x[:8].repeat(88, 1)[:rows], tokens[:8].repeat(88)[:rows], top)
        assert all(torch.equal(t[:8], t[8:16]) for t in got)
    else:
        check(dev, x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("top", [0, 5, 64])
def test_masked_rows(dev, dtype, top):
    """Rows that allow one token, a few, none; masks of the type's lowest value, whole rows of it; infinities and no
    numbers; tokens that are none."""
    V = 9000
    low, inf, nan = torch.finfo(dtype).min, math.inf, math.nan
    g = torch.Generator().manual_seed(top)
    x = (torch.randn(16, V, generator=g) * 2).to(dtype)
    tokens = torch.randint(0, V, (16,), generator=g)
    x[0] = -inf
    x[1] = -inf
    x[1, 4321] = 2.0
    tokens[1] = 4321
    x[2, :] = -inf
    x[2, [5, 8000, 8999]] = torch.tensor([1.0, 3.0, 1.0], dtype=dtype)
    tokens[2] = 7
    x[3] = low
    x[4, 100:] = low
    tokens[4] = 50
    x[5, 100:] = low
    tokens[5] = 5000
    x[6, 17] = inf
    x[7, ::2] = nan
    tokens[7] = 4
    x[8] = nan
    x[9, 3] = nan
    tokens[9] = 2
    tokens[10], tokens[11], tokens[12] = -100, V, 2 ** 40
    x[13, :] = -inf
    tokens[13] = -1
    x[14, 0], x[14, 1] = 0.0, -0.0
    tokens[14] = 1
    check(dev, x, tokens, top)


def test_rows_at_odd_places(dev):
    """Rows that begin anywhere within 16 bytes, and end there."""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for V, ld, first in ((1000, 1003, 0), (8193, 8195, 1), (501, 509, 7), (2047, 2049, 3)):
            g = torch.Generator().manual_seed(V)
            whole = torch.full((9 * ld + 16,), 1000.0, dtype=dtype)  # what lies beside the rows is larger than all in them
            rows = torch.as_strided(whole, (9, V), (ld, 1), first)
            rows.copy_((torch.randn(9, V, generator=g) * 3).to(dtype))
            tokens = torch.randint(0, V, (9,), generator=g)
            on_gpu = torch.as_strided(whole.to(dev), (9, V), (ld, 1), first)
            check(dev, rows, tokens, 6, on_gpu)


def test_rows_beyond_32_bits(dev):
    """Rows 2^24 elements apart, 300 of them: the last begins 10 GB behind the first."""
    g = torch.Generator().manual_seed(12)
    x = (torch.randn(300, 5000, generator=g) * 3).bfloat16()
    rows = torch.empty(300 << 24, dtype=torch.bfloat16, device=dev).view(300, -1)[:, 3:5003]
    rows.copy_(x)
    check(dev, x, torch.randint(0, 5000, (300,), generator=g), 4, rows)


def test_the_longest_vocabulary(dev):
    """Parts of as many slices as their threads have room to note, and a vocabulary one short of a part's more."""
    for V, rows in ((1 << 24, 1), (20 * 8192 - 1, 600), (20 * 8192 + 1, 2)):
        g = torch.Generator().manual_seed(V)
        x = (torch.randn(1, V, generator=g) * 2).bfloat16().repeat(rows, 1)
        tokens = torch.randint(0, V, (1,), generator=g).repeat(rows)
        got = check(dev, x[:1], tokens[:1], 64, None if rows < 3 else x.to(dev)[:1])
        from quipsharp_amd.logprobs import token_logprobs
        for a, b in zip(token_logprobs(x.to(dev), tokens.to(dev), 64), got):
            a = a.cpu()
            assert (a == a[:1]).all() and (torch.equal(a[:1], b) if b.dtype is torch.int32 else torch.allclose(a[:1], b, rtol=0, atol=2e-5))


def test_sharp_and_flat_distributions(dev):
    """One token has nearly all, and all have the same."""
    V = 40000
    x = torch.zeros(4, V)
    x[0, 77] = 30.0
    x[1, 77] = 90.0
    x[2] += 5000.0
    x[3] = torch.linspace(-1e5, 1e5, V)
    check(dev, x, torch.tensor([77, 5, 9, V - 1]), 3)


def test_many_rows(dev):
    """More rows than work-groups fit at once, and more tokens than 2^31 of them."""
    from quipsharp_amd.logprobs import token_logprobs
    V, R = 32000, 70000
    g = torch.Generator().manual_seed(1)
    few = (torch.randn(7, V, generator=g) * 2).bfloat16()
    tokens = torch.randint(0, V, (7,), generator=g)
    x = torch.empty(R, V, dtype=torch.bfloat16, device=dev)
    x.view(R // 7, 7, V).copy_(few.to(dev))
    got = token_logprobs(x, tokens.repeat(R // 7).to(dev), 4)
    want = check(dev, few, tokens, 4)
    for a, b in zip(got, want):
        a = a.cpu().view(R // 7, 7, *b.shape[1:])
        assert torch.equal(a[0], a[-1]) and (a == a[0]).all()
        assert torch.equal(a[0], b) if b.dtype is torch.int32 else torch.allclose(a[0], b, rtol=0, atol=2e-5)


def test_replayed_and_on_another_stream(dev):
    from quipsharp_amd.logprobs import token_logprobs
    g = torch.Generator().manual_seed(2)
    x, tokens = torch.randn(3, 30000, generator=g).to(dev), torch.tensor([1, 2, 3], device=dev)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        token_logprobs(x, tokens, 5, workspace=ws)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, tokens, 5, workspace=ws)
    for step in range(4):
        x.copy_(torch.randn(3, 30000, generator=g))
        tokens += 1000
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, token_logprobs(x, tokens, 5)):
            assert torch.equal(a, b)


def test_empty(dev):
    from quipsharp_amd.logprobs import token_logprobs
    got = token_logprobs(torch.zeros(0, 50, device=dev), torch.zeros(0, dtype=torch.long, device=dev), 5)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0,), (0, 5), (0, 5)]
