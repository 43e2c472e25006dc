"""More of what the operators around a served step's linears refuse, on the host."""
import ctypes
import random

import pytest
import torch

from quipsharp_amd import _lib
from quipsharp_amd.adapters import add_adapters
from quipsharp_amd.rope import append_rotated

BF, I32 = torch.bfloat16, torch.int32


def test_outputs_and_frequencies_that_require_a_gradient_are_refused():
    """A tensor that the call writes would be overwritten behind autograd's back, and learned frequencies lose theirs."""
    grad = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, requires_grad=True)  # noqa: E731
    z = lambda *shape: torch.zeros(*shape, dtype=BF)  # noqa: E731
    added = lambda outs: add_adapters([z(3, 40)], z(3, 64), torch.zeros(3, dtype=I32), [z(2, 8, 64)], [z(2, 40, 8)],  # noqa: E731
                                      [torch.zeros(2)], outs=outs)
    turned = lambda w, out: append_rotated(z(2, 4, 64), z(2, 2, 64), z(2, 2, 64), z(3, 2, 16, 64), z(3, 2, 16, 64),  # noqa: E731
                                           torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32), w, out=out)
    ones = torch.ones(32, dtype=torch.float64)
    for call in (lambda: added([grad(3, 40)]), lambda: turned(ones, grad(2, 4, 64)), lambda: turned(grad(32, dtype=torch.float64), None)):
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="runs on the GPU"):
            call()


# ---------------------------------------------------------------------------
# outputs that share memory with what the call reads
# ---------------------------------------------------------------------------

P = ctypes.c_void_p(4096)


def elements(at, rows, apart, width):
    return {at // 2 + i * apart + e for i in range(rows) for e in range(width)}


def test_adapters_refuse_outputs_that_meet_what_is_read():
    """Against the elements themselves, for rows at random places of a small space: where nothing meets the call comes to
    its workspace, of which it is given none."""
    L, r = _lib.lib(), random.Random(1)
    met = clear = 0
    for _ in range(4000):
        tokens, n, m = r.randint(1, 4), 8 * r.randint(1, 2), r.randint(1, 6)
        ld = [r.choice([8, 16, 24, 32]) for _ in range(2)]
        strides = dict(ldx=max(n, 8 * r.randint(1, 4)), ldy=max(m, r.choice(ld + [11])), ldo=max(m, r.choice(ld)))
        place = lambda: 8192 + 2 * r.randrange(0, 160)  # noqa: E731
        x, y, out, other_y, other = (8192 + 16 * r.randrange(0, 20)), place(), place(), 1 << 40, 1 << 41
        where = r.random()
        if where < 0.3:
            y, strides["ldy"] = out, strides["ldo"]
        elif where < 0.5:
            other_y = place()
        down, up, scale, which = 1 << 42, 1 << 43, 1 << 44, 1 << 45
        if where > 0.8:
            down, up = r.choice([(8192 + 16 * r.randrange(0, 20), up), (down, 8192 + 16 * r.randrange(0, 20))])
        job = dict(down=down, up=up, scale=scale, down_adapter=8 * n + 8, down_row=n, up_adapter=8 * m, up_row=8, rank=8, m=m)
        jobs = (_lib.AdapterJob * 2)(_lib.AdapterJob(**job, y=y, ldy=strides["ldy"], out=out, ldo=strides["ldo"]),
                                     _lib.AdapterJob(**job, y=other_y, ldy=strides["ldy"], out=other, ldo=strides["ldo"]))
        rc = L.qs_adapters_add(x, 2, strides["ldx"], tokens, n, which, 2, 2, jobs, P, 0, None)
        one = tokens == 1
        mine = elements(out, tokens, strides["ldo"], m)
        in_place = y == out and (one or strides["ldy"] == strides["ldo"])
        reads = [elements(x, tokens, strides["ldx"], n), elements(other_y, tokens, strides["ldy"], m),
                 *(elements(down + 2 * a * (8 * n + 8), 8, n, n) for a in range(2)), *(elements(up + 16 * a * m, m, 8, 8) for a in range(2))]
        if not in_place:
            reads.append(elements(y, tokens, strides["ldy"], m))
        message = L.qs_last_error().decode()
        assert rc == 1
        if any(mine & s for s in reads):
            met += 1
            assert "shares memory" in message or "share memory" in message or "the output of linear 0 is" in message, message
        else:
            clear += 1
            assert "workspace of 0 bytes" in message, message
    assert met > 500 and clear > 500


def test_rotation_refuses_queries_that_meet_what_is_read():
    """The same, of the calls that must be refused alone: others would run."""
    L, r = _lib.lib(), random.Random(2)
    met = 0
    for _ in range(3000):
        tokens, heads, kv, dim = r.randint(1, 3), r.randint(1, 3), r.randint(1, 2), 8
        q_head, k_head, v_head = (8 * r.randint(1, 2) for _ in range(3))
        q_token, k_token, v_token, out_token = (8 * r.randint(0, 8) for _ in range(4))
        out_token = max(out_token, heads * dim)
        at = lambda: 8192 + 16 * r.randrange(0, 24)  # noqa: E731
        q, k, v, out = at(), at(), at(), at()
        if r.random() < 0.3:
            out = q
        head = lambda p, token, step, count: set().union(*(elements(p + 2 * h * step, tokens, token, dim) for h in range(count)))  # noqa: E731
        mine = elements(out, tokens, out_token, heads * dim)
        in_place = q == out and (tokens == 1 or q_token == out_token) and (heads == 1 or q_head == dim)
        reads = [head(k, k_token, k_head, kv), head(v, v_token, v_head, kv)] + ([] if in_place else [head(q, q_token, q_head, heads)])
        if not any(mine & s for s in reads):
            continue
        met += 1
        pool = _lib.PagePool(k=1 << 40, v=1 << 41, k_page=128, k_head=64, k_pos=8, v_page=128, v_head=64, v_pos=8, pages=3, page=8,
                             table=4096, table_ld=1, cols=1, lengths=4096)
        rc = L.qs_page_append_rotated(q, k, v, 2, tokens, tokens, heads, kv, dim, q_token, q_head, k_token, k_head, v_token, v_head,
                                      None, pool, None, P, 4, 0, 1.0, out, out_token, None)
        assert rc == 1 and "q_out shares memory" in L.qs_last_error().decode()
    assert met > 500


# ---------------------------------------------------------------------------
# launches that would have 2^32 threads or more
# ---------------------------------------------------------------------------

def test_more_rows_than_a_grid_has_are_refused():
    L = _lib.lib()
    scores = lambda rows: L.qs_token_logprobs(P, 0, 4, rows, 4, P, 8, 1, P, P, P, P, P, None, 0, None)  # noqa: E731
    assert scores(1 << 24) == 3 and "16777216 rows of 4 tokens" in L.qs_last_error().decode()
    assert L.qs_token_logprobs_workspace_bytes(1 << 24, 4, 0, 1) == L.qs_token_logprobs_workspace_most(1 << 24, 4, 0, 1) == 0
    pool = _lib.PagePool(k=1 << 40, v=1 << 41, k_page=4096, k_head=4096, k_pos=512, v_page=4096, v_head=4096, v_pos=512, pages=3,
                         page=8, table=4096, table_ld=1, cols=1, lengths=4096)
    turned = lambda tokens: L.qs_page_append_rotated(1 << 50, 1 << 51, 1 << 52, 2, tokens, 2, 1, 1, 512, 512, 512, 512, 512, 512, 512,  # noqa: E731
                                                     P, pool, None, P, 256, 0, 1.0, 1 << 50, 512, None)
    assert turned(1 << 26) == 3 and "67108864 tokens, 4 of a work-group" in L.qs_last_error().decode()
