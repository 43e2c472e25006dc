"""What the paged cache and the beam search refuse, on the host: tensors that
would send a kernel out of bounds, and sizes that the kernels do not cover."""
import ctypes
import math

import pytest
import torch

from quipsharp_amd import _lib
from quipsharp_amd.beam import beam_select, reorder_states
from quipsharp_amd.pages import (PagedCache, advance_pages, append_pages, attend_chunk, attend_token, compact_pages,
                                 copy_pages, free_pages)

BF = torch.bfloat16
I32 = torch.int32


def attention(**over):
    a = dict(q=torch.zeros(2, 8, 128, dtype=BF), k_pages=torch.zeros(5, 2, 32, 128, dtype=BF),
             v_pages=torch.zeros(5, 2, 32, 128, dtype=BF), table=torch.zeros(2, 3, dtype=I32),
             lengths=torch.zeros(2, dtype=I32))
    a.update(over)
    return a


ATTENTION = [
    (dict(k_pages=torch.zeros(5, 2, 32, 64, dtype=BF)), ValueError, "of one type"),
    (dict(k_pages=torch.zeros(5, 2, 32, 128), v_pages=torch.zeros(5, 2, 32, 128)), TypeError, "cache dtype"),
    (dict(v_pages=torch.zeros(5, 2, 32, 128, dtype=torch.float16)), ValueError, "of one type"),
    (dict(k_pages=torch.zeros(5, 2, 128, 32, dtype=BF).transpose(2, 3)), ValueError, "stride 1"),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), ValueError, "table must be"),
    (dict(table=torch.zeros(2, 6, dtype=I32)[:, ::2]), ValueError, "table must be"),
    (dict(table=torch.zeros(6, dtype=I32)), ValueError, "table must be"),
    (dict(lengths=torch.zeros(3, dtype=I32)), ValueError, "lengths must be"),
    (dict(lengths=torch.zeros(2, dtype=I32, device="meta")), ValueError, "lengths is on"),
    (dict(q=torch.zeros(2, 8, 64, dtype=BF)), ValueError, "q must be"),
    (dict(q=torch.zeros(2, 8, 128, dtype=torch.float16)), TypeError, "q is"),
    (dict(q=torch.zeros(2, 8, 256, dtype=BF)[:, :, ::2]), ValueError, "stride 1"),
    (dict(sinks=4), ValueError, "go with a window"),
    (dict(window=-1), ValueError, "0 or more"),
    (dict(out=torch.zeros(2, 8, 128)), ValueError, "out must be"),
    (dict(out=torch.zeros(2, 16, 128, dtype=BF)[:, ::2]), ValueError, "lie together"),
    (dict(), RuntimeError, "runs on the GPU"),
]


@pytest.mark.parametrize("over,error,message", ATTENTION)
def test_attention_refuses(over, error, message):
    a = attention(**over)
    with pytest.raises(error, match=message):
        attend_token(**a)
    with pytest.raises(error, match=message):
        attend_chunk(starts=torch.tensor([0, 1, 2], dtype=I32), **a)


def test_attention_refuses_rows_and_starts():
    with pytest.raises(ValueError, match="q must be"):
        attend_token(**attention(q=torch.zeros(3, 8, 128, dtype=BF)))
    with pytest.raises(ValueError, match="starts must be"):
        attend_chunk(starts=torch.tensor([0, 2], dtype=I32), **attention())


def test_append_refuses():
    a = attention()
    pools = (a["k_pages"], a["v_pages"])
    new = torch.zeros(2, 2, 128, dtype=BF)
    with pytest.raises(ValueError, match="heads for a cache"):
        append_pages(*pools, torch.zeros(2, 3, 128, dtype=BF), new, a["table"], a["lengths"])
    with pytest.raises(ValueError, match="k must be"):
        append_pages(*pools, torch.zeros(3, 2, 128, dtype=BF), new, a["table"], a["lengths"])
    with pytest.raises(ValueError, match="starts must be"):
        append_pages(*pools, new, new, a["table"], a["lengths"], torch.zeros(2, dtype=I32))
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        append_pages(*pools, new, new, a["table"], a["lengths"])


def books(rows=2, cols=3, pages=5):
    return torch.zeros(2, pages, 2, 16, 64, dtype=BF), torch.zeros(rows, cols, dtype=I32), torch.zeros(rows, dtype=I32), \
        torch.zeros(pages, dtype=I32)


def test_page_calls_refuse():
    kv, table, lengths, refs = books()
    with pytest.raises(ValueError, match="refs must be"):
        advance_pages(kv, table, lengths, refs[:4].clone())
    with pytest.raises(ValueError, match="parents must be"):
        advance_pages(kv, table, lengths, refs, parents=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="tokens"):
        advance_pages(kv, table, lengths, refs, tokens=-1)
    with pytest.raises(ValueError, match="contiguous"):
        advance_pages(kv.transpose(2, 3), table, lengths, refs)
    with pytest.raises(ValueError, match="keep must be"):
        free_pages(table, lengths, refs, page=16, keep=torch.zeros(3, dtype=torch.bool))
    with pytest.raises(ValueError, match="go with a window"):
        free_pages(table, lengths, refs, page=16, sinks=2)
    with pytest.raises(ValueError, match="table must be"):
        compact_pages(kv, table.long(), refs)
    with pytest.raises(ValueError, match="out"):
        compact_pages(kv, table, refs, out=(table[:1], refs))
    with pytest.raises(ValueError, match="dst must be"):
        copy_pages(kv, torch.zeros(2, dtype=I32), torch.zeros(3, dtype=I32))
    for call in (lambda: advance_pages(kv, table, lengths, refs), lambda: free_pages(table, lengths, refs, page=16),
                 lambda: compact_pages(kv, table, refs),
                 lambda: copy_pages(kv, torch.zeros(2, dtype=I32), torch.zeros(2, dtype=I32))):
        with pytest.raises(RuntimeError, match="runs on the GPU"):
            call()


def test_cache_on_the_cpu_refuses_work():
    cache = PagedCache(2, 8, 2, 64, 3, 4, page=16, device="cpu")
    assert cache.keys(1).shape == (8, 2, 16, 64) and cache.table.tolist() == [[-1] * 4] * 3
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        cache.advance()


@pytest.mark.parametrize("over,error,message", [
    (dict(scores=torch.zeros(2, 3, dtype=torch.float64)), ValueError, "scores must be"),
    (dict(scores=torch.zeros(2, 4)), ValueError, "do not fit"),
    (dict(logits=torch.zeros(6, 100)[:, ::2]), ValueError, "lie together"),
    (dict(logits=torch.zeros(2, 50, 3).transpose(1, 2)), ValueError, "lie together|one stride apart"),
    (dict(logits=torch.zeros(6, 50, dtype=torch.float64)), TypeError, "unsupported dtype"),
    (dict(finished=torch.zeros(2, 2, dtype=torch.bool)), ValueError, "finished must be"),
    (dict(finished=torch.zeros(2, 3)), ValueError, "finished must be"),
    (dict(keep=0), ValueError, "keep"),
    (dict(), RuntimeError, "runs on the GPU"),
])
def test_beam_select_refuses(over, error, message):
    a = dict(logits=torch.zeros(6, 50), scores=torch.zeros(2, 3))
    a.update(over)
    with pytest.raises(error, match=message):
        beam_select(**a)


def test_reorder_states_refuses():
    parents = torch.zeros(3, dtype=I32)
    with pytest.raises(ValueError, match="1 to 8"):
        reorder_states([], parents)
    with pytest.raises(ValueError, match="must have 4 rows"):
        reorder_states([torch.zeros(4, 2), torch.zeros(3, 2)], parents)
    with pytest.raises(ValueError, match="lie together"):
        reorder_states([torch.zeros(4, 6)[:, ::2]], parents)
    with pytest.raises(ValueError, match="parents must be"):
        reorder_states([torch.zeros(4, 6)], parents.long())
    with pytest.raises(RuntimeError, match="runs on the GPU"):
        reorder_states([torch.zeros(4, 6)], parents)


# the C entry points' own checks, which return before anything is launched

P = ctypes.c_void_p(64)


def pool(**over):
    a = dict(k=64, v=64, k_page=2 * 32 * 128, k_head=32 * 128, k_pos=128, v_page=2 * 32 * 128, v_head=32 * 128,
             v_pos=128, pages=5, page=32, table=64, table_ld=3, cols=3, lengths=64)
    a.update(over)
    return _lib.PagePool(**a)


def token(L, heads=8, kv_heads=2, dim=128, dtype=2, q_row=1024, q_head=128, window=0, sinks=0, out_row=1024, ws=1 << 20,
          q=P, scale=0.1, **over):
    return L.qs_attend_token(q, dtype, 2, heads, kv_heads, dim, q_row, q_head, pool(**over), scale, window, sinks, P,
                             out_row, P, ws, None)


@pytest.mark.parametrize("over,code,message", [
    (dict(dtype=0), 3, b"dtype"), (dict(dim=96), 3, b"head_dim"), (dict(heads=7), 1, b"heads"),
    (dict(page=24), 3, b"pages of 24"), (dict(page=8), 3, b"pages of 8"), (dict(page=8192), 3, b"pages of 8192"),
    (dict(pages=0), 1, b"0 pages"), (dict(cols=0), 1, b"0 columns"), (dict(table_ld=2), 1, b"stride 2"),
    (dict(cols=1 << 27, table_ld=1 << 27), 1, b"columns"), (dict(k_pos=100), 1, b"strides"),
    (dict(v_head=12), 1, b"strides"), (dict(k_pos=64), 1, b"position strides"), (dict(k=72), 1, b"aligned"),
    (dict(k=0), 1, b"null"), (dict(lengths=0), 1, b"null"), (dict(q=ctypes.c_void_p(66)), 1, b"aligned"),
    (dict(q_head=130), 1, b"aligned"), (dict(q_head=64), 1, b"aligned"), (dict(out_row=1000), 1, b"output rows"),
    (dict(scale=0.0), 1, b"scale 0"), (dict(scale=math.nan), 1, b"scale nan"), (dict(scale=math.inf), 1, b"scale inf"),
    (dict(sinks=2), 1, b"sinks"), (dict(window=-2), 1, b"window"),
])
def test_attend_token_c_refusals(over, code, message):
    L = _lib.lib()
    assert token(L, **over) == code and message in L.qs_last_error(), L.qs_last_error()


def test_workspace_c_refusals():
    L = _lib.lib()
    need = L.qs_attend_token_workspace_bytes(2, 8, 2, 128, 300, 32, 0, 0)
    assert need > 0
    assert token(L, cols=300, table_ld=300, ws=need - 1) == 1 and b"workspace" in L.qs_last_error()
    store = _lib.PageStore(64, 4, 16, 2, 16, 128)
    need = L.qs_page_advance_workspace_bytes(8)
    args = lambda n: (store, P, P, P, None, 8, 4, 1, P, P, P, P, P, n, None)  # noqa: E731
    assert L.qs_page_advance(*args(need - 1)) == 1 and b"workspace" in L.qs_last_error()
    need = L.qs_page_compact_workspace_bytes(16)
    assert L.qs_page_compact(store, P, P, 8, 4, P, P, P, need - 1, None) == 1 and b"workspace" in L.qs_last_error()
    need = L.qs_beam_select_workspace_bytes(2, 3, 1000, 3)
    assert L.qs_beam_select(P, 0, 1000, 2, 3, 1000, P, None, -1, 3, P, P, P, P, need - 1, None) == 1
    assert b"workspace" in L.qs_last_error()


def test_other_c_refusals():
    L = _lib.lib()
    ok = _lib.PageStore(64, 4, 16, 2, 16, 128)
    assert L.qs_page_advance(_lib.PageStore(64, 4, 16, 2, 16, 24), P, P, P, None, 8, 4, 1, P, P, P, P, P, 1 << 20, None) == 1
    assert b"multiple of 16" in L.qs_last_error()
    assert L.qs_page_advance(_lib.PageStore(72, 4, 16, 2, 16, 32), P, P, P, None, 8, 4, 1, P, P, P, P, P, 1 << 20, None) == 1
    assert b"aligned" in L.qs_last_error()
    assert L.qs_page_advance(ok, P, P, P, None, 1025, 4, 1, P, P, P, P, P, 1 << 20, None) == 3
    assert L.qs_page_advance(ok, P, None, P, None, 8, 4, 1, P, P, P, P, P, 1 << 20, None) == 1
    assert L.qs_page_free(P, P, P, None, 8, 4, 16, 16, 0, 3, P, P, P, None) == 1 and b"sinks" in L.qs_last_error()
    assert L.qs_page_copy(ok, None, P, 3, None) == 1
    assert L.qs_beam_select(P, 0, 10, 2, 3, 10, P, None, -1, 31, P, P, P, P, 1 << 20, None) == 1
    assert b"continuations" in L.qs_last_error()
    assert L.qs_beam_select(P, 0, 1000, 2, 3, 1000, P, None, -1, 129, P, P, P, P, 1 << 20, None) == 3
    assert L.qs_beam_select(P, 0, 999, 2, 3, 1000, P, None, -1, 3, P, P, P, P, 1 << 20, None) == 1
    assert L.qs_page_append_rope(P, P, P, P, P, P, P, 10, P, 2, 8, 2, 64, pool(), 1e-6, None) == 3
    assert L.qs_page_append(P, P, 3, 2, 2, 128, 256, 128, 256, 128, None, pool(), None) == 1
    assert b"3 tokens of 2 rows" in L.qs_last_error()
    assert L.qs_attend_chunk(P, 2, 4, 2, 8, 2, 128, 1024, 128, None, pool(), 0.1, 0, 0, P, 1024, None) == 1


def test_empty_calls_do_nothing():
    L = _lib.lib()
    assert L.qs_attend_token(None, 2, 0, 8, 2, 128, 0, 0, None, 0.1, 0, 0, None, 0, None, 0, None) == 0
    assert L.qs_attend_chunk(None, 2, 0, 2, 8, 2, 128, 0, 0, None, None, 0.1, 0, 0, None, 0, None) == 0
    assert L.qs_page_append(None, None, 0, 0, 2, 128, 0, 0, 0, 0, None, None, None) == 0
    assert L.qs_page_copy(None, None, None, 0, None) == 0
    assert L.qs_beam_select(None, 0, 0, 0, 3, 10, None, None, -1, 3, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("over", [dict(k_page=1 << 31), dict(v_page=1 << 31), dict(k_pos=1 << 24, page=128),
                                  dict(v_pos=1 << 20, page=2048)])
def test_pages_too_far_apart(over):
    L = _lib.lib()
    assert token(L, **over) == 3 and b"elements apart" in L.qs_last_error()


def test_tables_and_tokens_out_of_range():
    L = _lib.lib()
    store = _lib.PageStore(64, 4, 16, 2, 16, 128)
    cols = 1 << 21
    assert L.qs_page_advance(store, P, P, P, None, 1024, cols, 1, P, P, P, P, P, 1 << 20, None) == 3
    assert b"2097152 columns" in L.qs_last_error()
    assert L.qs_attend_chunk(P, 2, 4, 0, 8, 2, 128, 1024, 128, P, pool(), 0.1, 0, 0, P, 1024, None) == 1
    assert b"4 tokens of no row" in L.qs_last_error()


def test_pools_whose_pages_no_int_counts():
    """The kernels' loops step over pages and copies by up to 8192 and 64 at a time, in 32 bits."""
    L = _lib.lib()
    for pages in (2 ** 31 - 1024, 2 ** 31 - 8192):
        store = _lib.PageStore(64, 1, pages, 1, 1, 16)
        assert L.qs_page_advance(store, P, P, P, None, 8, 4, 1, P, P, P, P, P, 1 << 20, None) == 1
        assert b"%d pages" % pages in L.qs_last_error()
        assert L.qs_page_free(P, P, P, None, 8, 4, pages, 1, 0, 0, P, P, P, None) == 1
        assert b"%d pages" % pages in L.qs_last_error()
        assert L.qs_page_compact(store, P, P, 8, 4, P, P, P, 1 << 40, None) == 1
        assert b"%d pages" % pages in L.qs_last_error()
    store = _lib.PageStore(64, 1, 4, 1, 1, 16)
    assert L.qs_page_copy(store, P, P, 2 ** 31 - 64, None) == 1 and b"2147483584 pairs" in L.qs_last_error()


@pytest.mark.parametrize("over,message", [(torch.zeros(3, dtype=I32), "over must be"), (torch.zeros(2), "over must be"),
                                          (torch.zeros(2, dtype=I32, device="meta"), "over is on")])
def test_tokens_over_the_table_refuse(over, message):
    a = attention(over=over)
    new = torch.zeros(2, 2, 128, dtype=BF)
    for call in (lambda: attend_token(**a), lambda: attend_chunk(starts=torch.tensor([0, 1, 2], dtype=I32), **a),
                 lambda: append_pages(a["k_pages"], a["v_pages"], new, new, a["table"], a["lengths"], over=over),
                 lambda: advance_pages(*books(), over=over)):
        with pytest.raises(ValueError, match=message):
            call()


def test_the_count_of_missing_pages_refuses():
    for missing in (torch.zeros(2, dtype=I32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="missing must be"):
            advance_pages(*books(), missing=missing)
    with pytest.raises(ValueError, match="missing is on"):
        advance_pages(*books(), missing=torch.zeros(1, dtype=I32, device="meta"))


def test_gradients_are_refused():
    """An input that requires a gradient is refused where one would be recorded, and taken where none is."""
    one = torch.tensor([0, 1, 2], dtype=I32)
    grad = lambda *shape, dtype=BF: torch.zeros(*shape, dtype=dtype, requires_grad=True)  # noqa: E731
    a, new = attention(), torch.zeros(2, 2, 128, dtype=BF)
    calls = [lambda: attend_token(**attention(q=grad(2, 8, 128))),
             lambda: attend_chunk(starts=one, **attention(q=grad(2, 8, 128))),
             lambda: attend_token(**attention(v_pages=grad(5, 2, 32, 128))),
             lambda: attend_chunk(starts=one, **attention(k_pages=grad(5, 2, 32, 128))),
             lambda: append_pages(a["k_pages"], a["v_pages"], grad(2, 2, 128), new, a["table"], a["lengths"]),
             lambda: append_pages(a["k_pages"], a["v_pages"], new, grad(2, 2, 128), a["table"], a["lengths"]),
             lambda: beam_select(grad(6, 50, dtype=torch.float32), torch.zeros(2, 3)),
             lambda: beam_select(torch.zeros(6, 50), grad(2, 3, dtype=torch.float32)),
             lambda: reorder_states([torch.zeros(4, 6), grad(4, 6)], torch.zeros(3, dtype=I32))]
    for call in calls:
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="runs on the GPU"):
            call()


@pytest.mark.parametrize("scale", [2.5e38, -3.4e38])
def test_scales_whose_product_with_log2_e_is_none(scale):
    L = _lib.lib()
    assert token(L, scale=scale) == 1 and b"scale" in L.qs_last_error()
