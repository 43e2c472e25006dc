"""Workspaces of the operators around a served step's linears: one of the size
for the largest call serves every smaller one, though few rows are cut into more
parts than many."""
import ctypes

import pytest
import torch

from quipsharp_amd import _lib, adapters, logprobs

P = ctypes.c_void_p(4096)


def needed(tokens, n, count, ranks):
    """The bytes that the entry point asks for when it is given none."""
    L = _lib.lib()
    jobs = (_lib.AdapterJob * 4)(*[_lib.AdapterJob(down=4096, up=4096, scale=4096, down_adapter=128 * n, down_row=n,
                                                   up_adapter=8 * 128, up_row=128, rank=r, m=8, y=1 << 44, ldy=8,
                                                   out=(2 + g) << 44, ldo=8) for g, r in enumerate(ranks)])
    assert L.qs_adapters_add(P, 2, n, tokens, n, P, count, len(ranks), jobs, P, 0, None) == 1
    message = L.qs_last_error().decode()
    assert "workspace of 0 bytes" in message
    return int(message.split(",")[1].split()[0])


@pytest.mark.parametrize("n,ranks", [(5120, [64, 64]), (64, [8]), (256, [128]), (4096, [16, 16, 16]), (25600, [64]),
                                     (3584, [24, 24, 24]), (18944, [128, 128, 128, 128]), (2048, [8, 40])])
def test_adapters_room_of_the_largest_call_serves_all(n, ranks):
    assert needed(64, 5120, 24, [64, 64]) > needed(65, 5120, 24, [64, 64])
    sizes = sorted({*range(1, 131), *(64 * i + d for i in range(3, 70) for d in (-1, 0, 1)), 8192, 20000, 1 << 17, 1 << 19})
    room = [adapters.workspace_bytes(t, n, ranks) for t in sizes]
    assert all(a <= b for a, b in zip(room, room[1:]))
    for t, r in zip(sizes, room):
        for count in (1, 2, 5, 24, 1000):
            assert needed(t, n, count, ranks) <= r
    assert _lib.lib().qs_adapters_workspace_bytes((1 << 19) + 1, n, 1, len(ranks), _lib.int_array(ranks)) == 0


@pytest.mark.parametrize("vocab", [1, 50, 2049, 32000, 151936, 163833, 163841, 1 << 24])
@pytest.mark.parametrize("top", [0, 1, 20, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_room_of_the_largest_call_serves_all(vocab, top, dtype):
    if top > vocab:
        return
    one = _lib.lib().qs_token_logprobs_workspace_bytes
    so_far = 0
    for rows in [*range(1, 1100), 1500, 2047, 4096, 5000, 1 << 20]:
        so_far = max(so_far, one(rows, vocab, _lib.dtype_code(dtype), top))
        if rows < 20 or rows % 97 == 0 or rows > 1020:
            assert logprobs.workspace_bytes(rows, vocab, dtype, top) == so_far
