"""Rows at the limits of their table and of the pool (csrc/qs_pages.hip,
csrc/qs_attend_token.hip, csrc/qs_attend_chunk.hip): what is cached stays as it
is, tokens without a place are left out, and they are counted.  Pools are
compared bit by bit, attention to the tolerance of test_gpu_attend.py."""
import pytest
import torch

from test_gpu_attend import want_and_tolerance

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
PAGE, COLS = 16, 3
ROOM = PAGE * COLS


def ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def held(pool, table, row):
    """(positions, heads, dim) of a row's pages in order, on the CPU."""
    pages = [p for p in table[row].tolist() if p >= 0]
    return pool[pages].transpose(1, 2).reshape(-1, pool.shape[1], pool.shape[3]).cpu()


def near(got, q, k, v, see, dim):
    group = q.shape[0] // k.shape[1]
    for g in range(k.shape[1]):
        want, tol = want_and_tolerance(q[g * group:(g + 1) * group], k[see, g], v[see, g], dim ** -0.5)
        assert ((got[g * group:(g + 1) * group].double() - want).abs() <= tol).all()


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
