"""One workspace for calls of any size: what is computed with it is what a call's own gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, I32 = torch.bfloat16, torch.int32


def test_adapters_of_all_sizes_share_one(dev):
    from quipsharp_amd.adapters import add_adapters, workspace_bytes
    g = torch.Generator().manual_seed(1)
    most, n, m, rank, count = 600, 2048, 96, 24, 5
    make = lambda *s: torch.randn(*s, generator=g).bfloat16().to(dev)  # noqa: E731
    x, y, down, up = make(most, n), make(most, m), make(count, rank, n) * 0.02, make(count, m, rank)
    which, scale = torch.randint(-1, count, (most,), generator=g).to(I32).to(dev), torch.ones(count, device=dev)
    room = torch.empty(workspace_bytes(most, n, [rank]), dtype=torch.uint8, device=dev)
    for t in (600, 64, 1, 17, 65, 48, 130, 599):
        args = ([y[:t]], x[:t], which[:t], [down], [up], [scale])
        assert torch.equal(add_adapters(*args, workspace=room)[0], add_adapters(*args)[0])


def test_scores_of_all_sizes_share_one(dev):
    from quipsharp_amd.logprobs import token_logprobs, workspace_bytes
    g = torch.Generator().manual_seed(2)
    most, V = 1500, 20000
    x, t = torch.randn(most, V, generator=g).to(dev), torch.randint(0, V, (most,), generator=g).to(dev)
    room = torch.empty(workspace_bytes(most, V, torch.float32, 20), dtype=torch.uint8, device=dev)
    for rows in (1500, 1023, 1, 48, 600, 1024):
        for a, b in zip(token_logprobs(x[:rows], t[:rows], 20, workspace=room), token_logprobs(x[:rows], t[:rows], 20)):
            assert torch.equal(a, b)
