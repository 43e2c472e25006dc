"""Log probabilities of rows whose parts are as long as their threads have room
to note maxima for, and one logit longer.  Against the definition with the
tolerances of test_gpu_logprobs.py."""
import math

import pytest
import torch

from test_gpu_logprobs import U, expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,beside", [(torch.bfloat16, 7), (torch.float16, 7), (torch.float32, 3)])
@pytest.mark.parametrize("more", [0, 1])
@pytest.mark.parametrize("order", ["random", "last", "spread"])
def test_parts_as_long_as_there_is_room(dev, dtype, beside, more, order):
    """1024 rows are one part each if they have 20 slices of 8192 wherever they begin, and two with one logit more; the
    best lie anywhere, in the last slice, or one in every slice."""
    from quipsharp_amd import _lib
    from quipsharp_amd.logprobs import token_logprobs
    V, R, top = 20 * 8192 - beside + more, 1024, 64
    need = _lib.lib().qs_token_logprobs_workspace_bytes(R, V, _lib.dtype_code(dtype), top)
    assert need == 0 if not more else need >= R * 2 * (32 + 8 * top)
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(2, V, generator=g) * 2).to(dtype)
    if order == "last":
        x[:, V - 70:] = (torch.arange(70) % 50 / 8 + 20).to(dtype)
        x[1, V - 1] = 40
    elif order == "spread":
        x[:, 8191::8192] = (torch.arange(x[0, 8191::8192].numel()) / 4 + 20).to(dtype)
        x[:, 5000::8192] = 15
    tokens = torch.tensor([V - 1, V - 8192])
    got = [t.cpu() for t in token_logprobs(x.to(dev).repeat(R // 2, 1), tokens.repeat(R // 2).to(dev), top)]
    unit = (3 * math.log(V) + 20) * U
    # the same two rows over and over, at all places that a row may begin at
    for r, (lp, H, rank, best, ids, E, E2) in enumerate(expected(x, tokens, top)):
        logp, entropy, ranks, tops, top_ids = (t[r::2] for t in got)
        assert (ranks == rank).all() and (top_ids == torch.tensor(ids)).all()
        for a, b in ((logp, torch.tensor([lp], dtype=torch.float64)), (tops, torch.tensor(best, dtype=torch.float64))):
            assert ((a.double() - b).abs() <= unit + U * b.abs()).all()
        assert ((entropy.double() - H).abs() <= unit * (1 + E) + (18 * E + 3 * E2) * U + U * H).all()
