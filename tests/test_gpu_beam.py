"""Beam search's selection and its states (csrc/qs_beam.hip) against the
definition in 64 bits on the CPU.  Parents and tokens are exact; a score is
one rounding to fp32 (2^-24 relative) of a number whose log-sum is taken from
fp32 exponentials and slice sums: each term is off by 4 units relative (2^-22)
at most and the sums of up to 16 terms and 256 partial sums by 24 units more,
so the logarithm by 28 2^-24 absolutely."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def select(logits, scores, keep, finished, eos):
    B, K = scores.shape
    V = logits.shape[-1]
    x = logits.reshape(B, K, V).double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    out = []
    for b in range(B):
        total = torch.full((K, V), -math.inf, dtype=torch.float64)
        for j in range(K):
            s, top = scores[b, j].double(), x[b, j].max()
            if not torch.isfinite(s):
                continue
            if finished is not None and finished[b, j]:
                if 0 <= eos < V:
                    total[j, eos] = s
            elif torch.isfinite(top):
                total[j] = s + (x[b, j] - (top + (x[b, j] - top).exp().sum().log()))
        value, at = torch.sort(total.view(-1), descending=True, stable=True)
        out.append((value[:keep], at[:keep] // V + b * K, at[:keep] % V))
    return [torch.stack(t) for t in zip(*out)]


def check(dev, logits, scores, keep, finished=None, eos=-1):
    from quipsharp_amd.beam import beam_select
    want = select(logits, scores, keep, finished, eos)
    got = beam_select(logits.to(dev), scores.to(dev), keep, None if finished is None else finished.to(dev), eos)
    s, p, t = (x.cpu() for x in got)
    assert torch.equal(p.long(), want[1]) and torch.equal(t.long(), want[2])
    infinite = torch.isinf(want[0])
    assert torch.equal(torch.isinf(s), infinite) and (s[infinite] < 0).all()
    bound = want[0].abs() * 2.0 ** -24 + 28 * 2.0 ** -24
    assert ((s.double() - want[0]).abs()[~infinite] <= bound[~infinite]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 1, 50, 50), (2, 3, 7, 20), (1, 4, 1000, 4), (3, 5, 4096, 10), (2, 4, 4097, 8), (1, 2, 32000, 128),
    (5, 8, 12289, 16), (2, 16, 50257, 16), (1, 4, 151936, 8)])
def test_select(dev, batch, beams, vocab, keep, dtype):
    g = torch.Generator().manual_seed(vocab + keep)
    logits = (torch.randn(batch * beams, vocab, generator=g) * 3).to(dtype)
    scores = -20 * torch.rand(batch, beams, generator=g)
    check(dev, logits, scores, keep)


@pytest.mark.parametrize("order", ["ascending", "descending", "equal", "two values"])
def test_ties_and_orders(dev, order):
    """Everything equal, long runs of equal logits, and logits that lie in order (the best in few threads)."""
    V = 9000
    x = {"ascending": torch.arange(V) / 512.0, "descending": -torch.arange(V) / 512.0, "equal": torch.zeros(V),
         "two values": (torch.arange(V) % 3 == 0).float()}[order]
    logits = x.repeat(6, 1)
    check(dev, logits, torch.tensor([[-1.0, -1.0, -1.0], [-2.0, -1.0, -2.0]]), 64)
    check(dev, logits.half(), torch.zeros(2, 3), 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [3, 16, 40, 128])
@pytest.mark.parametrize("kind", ["equal", "few allowed", "periodic", "steps"])
def test_many_at_the_edge(dev, kind, keep, dtype):
    """Rows enough for the longest slices, and more candidates in one than it has room for: all equal, all but some
    banned, the large ones in few threads, and runs of equal values."""
    V, rows = 34000, 300
    t = torch.arange(V)
    x = {"equal": torch.zeros(V), "few allowed": torch.where(t % 4999 == 7, 1.0, -math.inf),
         "periodic": torch.where(t % 1024 < 12, (t % 997) / 997.0, -5.0), "steps": (t // 5000 % 2).float()}[kind]
    logits = x.repeat(rows, 1)
    logits[1::2, 100] = 3.0
    check(dev, logits.to(dtype), -(torch.arange(rows) % 5).float().view(100, 3), keep)


def test_zeros_of_both_signs_tie(dev):
    logits = torch.zeros(2, 100)
    logits[0, ::2] = -0.0
    check(dev, logits, torch.zeros(1, 2), 30)


def test_finished_and_dead_beams(dev):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(12, 300, generator=g)
    scores = -torch.rand(3, 4, generator=g) * 5
    finished = torch.tensor([[0, 1, 0, 1], [1, 1, 1, 1], [0, 0, 0, 1]], dtype=torch.bool)
    scores[2, 1] = -math.inf
    scores[2, 2] = math.nan
    for eos in (0, 2, 299, -1):
        check(dev, logits, scores, 6, finished, eos)
    first = torch.full((3, 4), -math.inf)
    first[:, 0] = 0  # the first step: one beam alive
    check(dev, logits, first, 4)
    check(dev, logits, torch.full((3, 4), -math.inf), 5)


def test_banned_tokens_nan_and_infinities(dev):
    logits = torch.full((4, 500), -math.inf)
    logits[0, 3] = 1.0  # one token allowed
    logits[1, 7], logits[1, 9] = math.nan, 0.5
    logits[2] = math.nan
    logits[3, :2] = torch.tensor([math.inf, 1.0])
    check(dev, logits, torch.tensor([[-1.0, -2.0], [-0.5, -0.1]]), 5)
    low = torch.full((2, 500), torch.finfo(torch.bfloat16).min).bfloat16()
    low[0, 77] = 0
    check(dev, low, torch.zeros(1, 2), 4)


def test_strided_logits(dev):
    from quipsharp_amd.beam import beam_select
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(8, 1003, generator=g).bfloat16()
    logits = wide[:, 3:1000]  # rows that no vector access fits
    check(dev, logits, -torch.rand(2, 4, generator=g), 4)
    # the last position of a prompt's logits
    seq = torch.randn(2, 4, 997, generator=g)
    s = -torch.rand(2, 4, generator=g)
    a = beam_select(seq.to(dev), s.to(dev))
    b = beam_select(seq.view(8, 997).to(dev), s.to(dev))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    check(dev, wide.to(dev)[:, :1000].cpu(), s, 4)


def test_reorder_states(dev):
    from quipsharp_amd.beam import reorder_states
    g = torch.Generator().manual_seed(3)
    states = [torch.randint(0, 1 << 40, (6, 37), generator=g), torch.randn(6, 3, 5, generator=g).half(),
              torch.randint(0, 255, (6, 7), generator=g, dtype=torch.uint8), torch.randn(6, generator=g),
              torch.randn(6, 4096, generator=g), torch.randn(6, 20, generator=g)[:, 4:12], torch.zeros(6, 0)]
    parents = torch.tensor([[5, 5, 0, 2], [1, -1, 6, 3]], dtype=torch.int32)
    got = reorder_states([s.to(dev) for s in states[:5]] + [torch.cat([states[5], states[5]], 1).to(dev)[:, :8], states[6].to(dev)],
                         parents.to(dev))
    flat = parents.view(-1).long()
    inside = (flat >= 0) & (flat < 6)
    for s, o in zip(states, got):
        want = s[flat.clamp(0, 5)].clone()
        want[~inside] = 0
        assert o.shape == want.shape and torch.equal(o.cpu(), want)


def test_states_without_rows(dev):
    """No parent names a row of an empty state."""
    from quipsharp_amd.beam import reorder_states
    torch.full((3, 9), 7.0, device=dev)  # what the output's place may hold
    got, = reorder_states([torch.zeros(0, 9, device=dev)], torch.tensor([0, -1, 2], dtype=torch.int32, device=dev))
    assert got.tolist() == [[0.0] * 9] * 3


def test_captured_select(dev):
    """A captured selection with its states: every replay equals the eager call."""
    from quipsharp_amd.beam import beam_select, reorder_states
    g = torch.Generator().manual_seed(4)
    logits = torch.zeros(8, 20000, dtype=torch.bfloat16, device=dev)
    scores = torch.zeros(2, 4, device=dev)
    history = torch.zeros(8, 50, dtype=torch.int64, device=dev)

    def step():
        s, p, t = beam_select(logits, scores)
        return [s, p, t] + reorder_states([history], p)

    def fill():
        logits.copy_(torch.randn(8, 20000, generator=g))
        scores.copy_(-torch.rand(2, 4, generator=g))
        history.copy_(torch.randint(0, 99, (8, 50), generator=g))

    fill()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(8):
        fill()
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i


@pytest.mark.parametrize("keep", [5, 64, 100, 128])
@pytest.mark.parametrize("kind", ["spread", "equal", "one ahead", "close"])
def test_many_beams(dev, kind, keep):
    """Hundreds of beams, whose slices' bests are far more than the join ranks at once.  Sums of different beams lie
    2^-15 apart at least, those of "close" agree in the upper half of an fp64."""
    K, V = 300, 9000
    g = torch.Generator().manual_seed(keep)
    x = torch.randint(0, 200, (V,), generator=g).float() / 64
    beam = torch.arange(K).float()
    scores = {"spread": -torch.randint(0, 500, (K,), generator=g).float() / 64 - beam / 2 ** 15, "equal": torch.zeros(K),
              "one ahead": torch.where(beam == 123, 50.0, -beam / 2 ** 15), "close": -1024.0 - beam / 2 ** 13}[kind]
    if kind in ("equal", "close"):
        x = torch.zeros(V)
    check(dev, x.repeat(K, 1), scores.view(1, K), keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [9, 17, 32])
@pytest.mark.parametrize("kind", ["lanes", "steps", "equal"])
def test_far_more_above_the_edge_than_room(dev, kind, keep, dtype):
    """"lanes": three of a slice's four waves have large logits, each in fewer threads than are kept, so that all of
    them lie above what the waves agree on."""
    V, rows = 34000, 300
    t, wide = torch.arange(V), 128 // torch.finfo(dtype).bits
    thread = t // wide % 256
    x = {"lanes": torch.where((thread < 192) & (thread % 64 < keep - 1), 1.0 + t % 7, (t % 5) / 8.0),
         "steps": (t // 5000 % 2).float(), "equal": torch.zeros(V)}[kind]
    logits = x.repeat(rows, 1)
    logits[1::2, 100] = 9.5
    check(dev, logits.to(dtype), -(torch.arange(rows) % 5).float().view(100, 3), keep)


def small_beside_one(at, vocab=12288, small=4096):
    """A logit of 0 at `at` and others whose exponentials are 0.95 of half an fp32 step of its, at the other tokens below
    `small`; the rest are nothing beside them."""
    x = torch.full((vocab,), -1e4)
    x[:small] = math.log(0.95 * 2.0 ** -24)
    x[at] = 0
    return x


def test_terms_below_half_a_step_of_the_largest_count(dev):
    """4095 of them make 3890 units (2^-24) of the sum.  A sum of 16 exponentials by pairs is off by 4 units at most
    (4 additions), the sums of those are 64-bit, and a relative error of 40 units in 4095 terms of 2^-24 is nothing:
    5 units for the logarithm and the rounding of a score near 0."""
    from quipsharp_amd.beam import beam_select
    for at in (0, 1, 700, 3075, 4095):
        logits = torch.stack([small_beside_one(at)] * 2)
        scores = torch.zeros(1, 2)
        want = select(logits, scores, 2, None, -1)
        got = beam_select(logits.to(dev), scores.to(dev), 2)
        assert torch.equal(got[1].cpu().long(), want[1]) and torch.equal(got[2].cpu().long(), want[2])
        assert ((got[0].cpu().double() - want[0]).abs() <= 5 * 2.0 ** -24).all(), at


def test_beams_with_the_same_logits_in_another_order(dev):
    """Two beams of one sum, the second 12 units ahead by its score: more than twice what a sum is off by, so it comes
    first, wherever the beams have their largest logit."""
    from quipsharp_amd.beam import beam_select
    for first, second in ((0, 3075), (3075, 0), (4095, 1), (1, 2048)):
        logits = torch.stack([small_beside_one(first), small_beside_one(second)]).to(dev)
        _, parents, tokens = beam_select(logits, torch.tensor([[0.0, 12 * 2.0 ** -24]], device=dev), 2)
        assert parents.tolist() == [[1, 0]] and tokens.tolist() == [[second, first]]
