"""Adapters over the whole range of bf16: inner products near the ends of the
exponents, with scales that bring the result back.  Tolerances as in
test_gpu_adapters.py: half a step of the output, and of |scale| sum |up| what an
inner product may be off."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32
U = 2.0 ** -24


@pytest.mark.parametrize("tokens", [3, 40])
@pytest.mark.parametrize("x_size,down_size,up_size,scale", [
    (2.0 ** 60, 2.0 ** 60, 2.0 ** -20, 2.0 ** 6),     # products 2^122, the result 2^109
    (2.0 ** 60, 2.0 ** 60, 2.0 ** -90, 2.0 ** 40),
    (2.0 ** -60, 2.0 ** -60, 2.0 ** 60, 2.0 ** -29),  # 2^-118 and 2^-86
    (2.0 ** -60, 2.0 ** -60, 2.0 ** 100, 2.0 ** 20),
    (2.0 ** 40, 2.0 ** -60, 1.0, 1.0)])
def test_products_far_from_one(dev, tokens, x_size, down_size, up_size, scale):
    from quipsharp_amd.adapters import add_adapters
    g = torch.Generator().manual_seed(1)
    n, m, rank = 64, 80, 16
    x = (torch.randn(tokens, n, generator=g) * x_size).to(BF)
    down = (torch.randn(1, rank, n, generator=g) * down_size).to(BF)
    up = (torch.randn(1, m, rank, generator=g) * up_size).to(BF)
    up[0, 5], up[0, 70] = 0, 0  # what they add is nothing, however large the products are
    y = torch.randn(tokens, m, generator=g).to(BF)
    s = torch.tensor([scale])
    got, = add_adapters([y.to(dev)], x.to(dev), torch.zeros(tokens, dtype=I32, device=dev), [down.to(dev)], [up.to(dev)], [s.to(dev)])
    d, w, xs = down[0].double(), up[0].double(), x.double()
    v = xs @ d.t()
    off = (n + 8) * U * (xs.abs() @ d.abs().t()) + v.abs().amax(1, keepdim=True) * 2.0 ** -16
    want = y.double() + scale * (v @ w.t())
    err = y.double().abs() * U + scale * (off @ w.abs().t() + (2 * rank + 8) * U * ((v.abs() + off) @ w.abs().t()))
    got = got.cpu()
    assert ((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + err) + err).all()
    assert torch.equal(got[:, 5], y[:, 5]) and torch.equal(got[:, 70], y[:, 70])


@pytest.mark.parametrize("tokens", [3, 40])
def test_small_results_alone(dev, tokens):
    """Without y, whose size would hide them."""
    from quipsharp_amd.adapters import add_adapters
    g = torch.Generator().manual_seed(2)
    n, m, rank = 64, 80, 16
    x, down = ((torch.randn(*s, generator=g) * 2.0 ** -60).to(BF) for s in ((tokens, n), (1, rank, n)))
    up = (torch.randn(1, m, rank, generator=g) * 2.0 ** 60).to(BF)
    y, s = torch.zeros(tokens, m, dtype=BF), torch.tensor([1.375 * 2.0 ** -29])
    got, = add_adapters([y.to(dev)], x.to(dev), torch.zeros(tokens, dtype=I32, device=dev), [down.to(dev)], [up.to(dev)], [s.to(dev)])
    v, w = x.double() @ down[0].double().t(), up[0].double()
    off = (n + 8) * U * (x.double().abs() @ down[0].double().abs().t()) + v.abs().amax(1, keepdim=True) * 2.0 ** -16
    want = 1.375 * 2.0 ** -29 * (v @ w.t())
    err = 1.375 * 2.0 ** -29 * (off @ w.abs().t() + (2 * rank + 8) * U * ((v.abs() + off) @ w.abs().t()))
    assert ((got.cpu().double() - want).abs() <= 2.0 ** -8 * (want.abs() + err) + err).all()
