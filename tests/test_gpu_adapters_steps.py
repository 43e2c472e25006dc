"""Adapters at the sizes whose loops go round more than once: several steps of
columns in each work-group, single tokens' second 256 columns, splits of inputs
whose last stage is partial beside wide blocks of ranks.  Against the definition in
64 bits with the tolerances of test_gpu_adapters.py; each case first says how the
call must be cut for that, so that it goes on to test what it is here for."""
import ctypes

import pytest
import torch

from test_gpu_adapters import BF, HF, I32, expected, gen, make, near

pytestmark = pytest.mark.gpu


def plan(tokens, n, adapters, ranks, ms):
    from quipsharp_amd import _lib
    out = (ctypes.c_int * 5)()
    _lib.check(_lib.lib().qs_adapters_plan(tokens, n, adapters, len(ranks), _lib.int_array(ranks), (ctypes.c_int64 * len(ms))(*ms), out))
    return dict(zip(("slots", "blocks", "runs", "splits", "columns"), out))


def run(dev, which, n, ms, ranks, adapters, dtype, inplace=False, seed=0, some=400):
    """Compared for `some` tokens, the first and the last tile among them."""
    from quipsharp_amd.adapters import add_adapters
    g = gen(seed)
    which = torch.as_tensor(which, dtype=I32)
    tokens = len(which)
    x, ys = make(g, tokens, n, dtype=dtype), [make(g, tokens, m, dtype=dtype) for m in ms]
    downs = [make(g, adapters, r, n, dtype=dtype, scale=n ** -0.5) for r in ranks]
    ups = [make(g, adapters, m, r, dtype=dtype, scale=0.2) for m, r in zip(ms, ranks)]
    scales = [torch.rand(adapters, generator=g) + 0.5 for _ in ms]
    to = lambda ts: [t.to(dev) for t in ts]  # noqa: E731
    dy = to(ys)
    got = add_adapters(dy, x.to(dev), which.to(dev), to(downs), to(ups), to(scales), outs=dy if inplace else None)
    t = torch.cat([torch.arange(min(64, tokens)), torch.arange(max(0, tokens - 64), tokens), torch.randperm(tokens, generator=g)[:some]]).unique()
    for o, y, down, up, scale in zip(got, ys, downs, ups, scales):
        want, err = expected(y[t], x[t], which[t], down, up, scale)
        near(o.cpu()[t], want, err, dtype)
        none = (which < 0) | (which >= adapters)
        assert torch.equal(o.cpu()[none], y[none])


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [16, 40, 72, 128])
@pytest.mark.parametrize("tokens,m", [(17, 320), (33, 331), (64, 331), (50, 257)])
def test_several_steps_of_one_tile(dev, tokens, m, rank, dtype, inplace):
    """One adapter's 17 to 64 tokens: four or five steps of 64 columns in a work-group of 256, the last ones partial."""
    assert plan(tokens, 264, 2, [rank], [m])["columns"] == 256
    run(dev, [1] * tokens, 264, [m], [rank], 2, dtype, inplace)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rank", [16, 40, 72, 128])
def test_several_steps_of_prompts(dev, rank, dtype):
    """11 tiles in 8 slots with 256 columns of a work-group, and 66 in one with 512, odd widths."""
    which = [a % 8 - 1 for a, c in enumerate((90, 3, 150, 64, 200, 17, 100, 76)) for _ in range(c)]
    assert plan(700, 200, 7, [rank] * 2, [1900, 131]) | dict(blocks=0, runs=0) == dict(slots=8, blocks=0, runs=0, splits=1, columns=256)
    run(dev, which, 200, [1900, 131], [rank] * 2, 7, dtype, inplace=dtype is HF)
    which = [0] * 1500 + [-1] * 70 + [2] * 2600 + [1] * 3
    assert plan(4173, 200, 3, [rank], [5003])["columns"] == 512
    run(dev, which, 200, [5003], [rank], 3, dtype, inplace=dtype is BF, some=200)


@pytest.mark.parametrize("rank,dtype", [(16, BF), (40, HF), (72, BF), (128, HF)])
def test_second_columns_of_single_tokens(dev, rank, dtype):
    """48 tokens of 24 adapters to so many columns that a wave takes 64 of them twice, and three times."""
    g = gen(rank)
    which = torch.randint(-1, 24, (48,), generator=g)
    assert plan(48, 72, 24, [rank] * 2, [8203, 8200])["columns"] == 512
    run(dev, which, 72, [8203, 8200], [rank] * 2, 24, dtype, inplace=dtype is HF)
    assert plan(16, 72, 24, [8], [65551])["columns"] == 1024
    run(dev, which[:16], 72, [65551], [8], 24, dtype, inplace=dtype is BF)


@pytest.mark.parametrize("n,splits", [(1000, 4), (2056, 3)])
@pytest.mark.parametrize("ranks,blocks", [([96], 6), ([128], 8), ([40, 56, 128], 8)])
def test_partial_stages_of_splits(dev, n, splits, ranks, blocks):
    """66 tiles, whose inputs are cut into splits that do not end with a stage of 64, beside 96 and 128 ranks together."""
    which = [0] * 1700 + [1] * 9 + [-1] * 100 + [2] * 2391
    p = plan(4200, n, 3, ranks, [64] * len(ranks))
    assert p["blocks"] == blocks and p["splits"] in ((splits,) if p["runs"] == 1 else (2,)) and n % 64
    run(dev, which, n, [64] * len(ranks), ranks, 3, BF if n == 1000 else HF)
