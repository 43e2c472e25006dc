"""A paged key-value cache and the attention over it, for decode loops around
``QuantizedLinear`` that serve several sequences, search with beams or stream
under a sliding window.  No counterpart in the reference, which keeps no
cache.  The computation runs in libquipsharp_hip.so (csrc/qs_pages.hip,
csrc/qs_attend_token.hip, csrc/qs_attend_chunk.hip).

A pool holds pages of ``page`` positions for every kv head.  Row r of a batch
keeps position p on page ``table[r, p // page]`` at place ``p % page``; -1
stands for no page.  ``lengths[r]`` is the number of positions that row r
holds, ``refs[i]`` the number of table entries that hold page i; a page with
none is free.  All three are int32 tensors on the GPU that only kernels read
and write, so a step that uses them can be captured in a HIP graph.

A row that runs out of columns keeps what it has: tokens at positions beyond
the table are stored nowhere and seen by none.  ``lengths`` count them, or,
where a call is given ``over`` (int32, a number for every row), stop at the
table's room, and ``over`` has how many of the row's newest tokens lie beyond.

The functions return new tables and leave their arguments as they are, unless
``out`` names the tensors to write, which may be the arguments themselves;
the pool is changed in place.  None of them has a gradient: inputs that
require one are refused where gradients are recorded.  ``PagedCache`` keeps the tensors together and
works in place.
"""
import ctypes

import torch
from torch import Tensor

from . import _lib

_HALF = (torch.bfloat16, torch.float16)
_FLAGS = (torch.bool, torch.uint8)


def _int32(name, t, shape, device):
    if not isinstance(t, Tensor) or t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        got = f"{tuple(t.shape)} x {t.dtype}" if isinstance(t, Tensor) else type(t).__name__
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}, got {got}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    return t


def _rows_flag(name, t, shape, device):
    if t.dtype not in _FLAGS or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous bool tensor of shape {tuple(shape)}, got {tuple(t.shape)} x {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _visible(window, sinks):
    window, sinks = int(window or 0), int(sinks or 0)
    if not (0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31):
        raise ValueError(f"window {window} and sinks {sinks} must be 0 or more")
    if sinks and not window:
        raise ValueError("sinks go with a window: without one every position is visible")
    return window, sinks


def _pool(k_pages, v_pages, table, lengths):
    """The library's description of one layer's pages, with the checks that
    keep its kernels inside the tensors."""
    shape, dev, rows = k_pages.shape, k_pages.device, table.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    # a decode step of one layer takes microseconds: what is refused is looked into only where something is
    if not (len(shape) == 4 and shape == v_pages.shape and k_pages.dtype is v_pages.dtype and k_pages.dtype in _HALF
            and ks[3] == 1 and vs[3] == 1 and v_pages.device == dev and len(rows) == 2
            and table.dtype is torch.int32 and table.is_contiguous() and table.device == dev
            and isinstance(lengths, Tensor) and lengths.dtype is torch.int32 and lengths.shape == rows[:1] and lengths.is_contiguous()
            and lengths.device == dev):
        _refuse_pool(k_pages, v_pages, table, lengths)
    return _lib.PagePool(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], shape[0],
                         shape[2], table.data_ptr(), rows[1], rows[1], lengths.data_ptr())


def _refuse_pool(k_pages, v_pages, table, lengths):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError(f"k_pages and v_pages must be (pages, kv heads, page, head dim) of one type, got "
                         f"{tuple(k_pages.shape)} x {k_pages.dtype} and {tuple(v_pages.shape)} x {v_pages.dtype}")
    if k_pages.dtype not in _HALF:
        raise TypeError(f"unsupported cache dtype {k_pages.dtype} (bfloat16 or float16)")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("the elements of a position must lie together (stride 1)")
    dev = k_pages.device
    if v_pages.device != dev:
        raise ValueError(f"v_pages is on {v_pages.device}, k_pages on {dev}")
    if table.dim() != 2:
        raise ValueError(f"table must be (rows, columns), got {tuple(table.shape)}")
    _int32("table", table, table.shape, dev)
    _int32("lengths", lengths, (table.shape[0],), dev)
    raise AssertionError("one of the checks above holds")


def _heads(name, x, rows, dim, dtype, device):
    """The strides of (rows, heads, dim) with the elements of a head together."""
    shape, st = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != dim or (rows is not None and shape[0] != rows):
        raise ValueError(f"{name} must be ({'tokens' if rows is None else rows}, heads, {dim}), got {tuple(shape)}")
    if x.dtype is not dtype:
        raise TypeError(f"{name} is {x.dtype}, the cache {dtype}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the cache on {device}")
    if st[2] != 1 and shape[1]:
        raise ValueError(f"the elements of a head of {name} must lie together (stride 1)")
    return st


def _output(out, q):
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
        raise ValueError(f"out must be {tuple(q.shape)} x {q.dtype} on {q.device}, got {tuple(out.shape)} x {out.dtype} on {out.device}")
    if out.stride(2) != 1 or out.stride(1) != out.shape[2]:
        raise ValueError("the heads of a row of out must lie together")
    return out


def _workspace(workspace, need, device):
    if not need:
        return None
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device)
    if workspace.device != device or workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise ValueError(f"workspace must be a contiguous uint8 tensor on {device}")
    if workspace.numel() < need:
        raise ValueError(f"workspace of {workspace.numel()} bytes, {need} needed")
    return workspace


def _room(workspace):
    return (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())


def append_pages(k_pages: Tensor, v_pages: Tensor, k: Tensor, v: Tensor, table: Tensor, lengths: Tensor,
                 starts: Tensor = None, over: Tensor = None) -> None:
    """Store new tokens' keys and values, (tokens, kv heads, head dim) each, in
    the pages: the tokens of row r are ``starts[r]`` .. ``starts[r + 1] - 1``
    (int32, rows + 1; None: one token per row), and the last of them goes to
    position ``lengths[r] - 1`` (``over[r]`` further where the row is over).
    Positions without a page are left out."""
    pool = _pool(k_pages, v_pages, table, lengths)
    dev, dim = k_pages.device, k_pages.shape[3]
    rows = table.shape[0]
    ks = _heads("k", k, None if starts is not None else rows, dim, k_pages.dtype, dev)
    vs = _heads("v", v, k.shape[0], dim, k_pages.dtype, dev)
    if k.shape[1] != k_pages.shape[1] or v.shape[1] != k_pages.shape[1]:
        raise ValueError(f"{k.shape[1]} and {v.shape[1]} heads for a cache of {k_pages.shape[1]}")
    if starts is not None:
        _int32("starts", starts, (rows + 1,), dev)
    if over is not None:
        _int32("over", over, (rows,), dev)
    if k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _lib.no_gradient("append_pages")
    _lib.require_gpu(k_pages, what="append_pages")
    _lib.check(_lib.lib().qs_page_append_over(k.data_ptr(), v.data_ptr(), k.shape[0], rows, k.shape[1], dim, ks[0],
                                              ks[1], vs[0], vs[1], _lib.ptr(starts), pool, _lib.ptr(over),
                                              _lib.stream_of(k_pages)))


def token_workspace_bytes(rows, heads, k_pages: Tensor, table: Tensor, window=0, sinks=0) -> int:
    """Bytes of workspace that ``attend_token`` takes for calls of this shape."""
    return int(_lib.lib().qs_attend_token_workspace_bytes(rows, heads, k_pages.shape[1], k_pages.shape[3],
                                                          table.shape[1], k_pages.shape[2], window, sinks))


def chunk_workspace_bytes(tokens, heads, k_pages: Tensor, table: Tensor, window=0, sinks=0) -> int:
    """Bytes of workspace that ``attend_chunk`` takes for calls of this shape."""
    return int(_lib.lib().qs_attend_chunk_workspace_bytes(tokens, table.shape[0], heads, k_pages.shape[1],
                                                          k_pages.shape[3], table.shape[1], k_pages.shape[2], window,
                                                          sinks))


def attend_token(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, *, scale: float = None,
                 window: int = 0, sinks: int = 0, over: Tensor = None, out: Tensor = None,
                 workspace: Tensor = None) -> Tensor:
    """Attention of one new token per row over the row's pages.

    q: (rows, heads, head dim), the token of row r at position ``lengths[r] -
    1`` (``over[r]`` further where the row is over), its key and value in the
    pages already.  It sees the positions up to
    its own: all of them, or with ``window`` the last ``window`` and the first
    ``sinks``.  Query head h reads kv head ``h // (heads / kv heads)``.
    Returns (rows, heads, head dim) in q's type; zeros for a row that sees
    nothing.  ``scale`` defaults to ``head_dim ** -0.5``."""
    pool = _pool(k_pages, v_pages, table, lengths)
    dev, (_, kv_heads, page, dim), (rows, cols) = k_pages.device, k_pages.shape, table.shape
    dtype = k_pages.dtype
    st = _heads("q", q, rows, dim, dtype, dev)
    window, sinks = _visible(window, sinks)
    if over is not None:
        _int32("over", over, (rows,), dev)
    out = _output(out, q)
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _lib.no_gradient("attend_token")
    _lib.require_gpu(k_pages, what="attend_token")
    L, heads = _lib.lib(), q.shape[1]
    need = L.qs_attend_token_workspace_bytes(rows, heads, kv_heads, dim, cols, page, window, sinks)
    workspace = _workspace(workspace, need, dev)
    _lib.check(L.qs_attend_token_over(q.data_ptr(), _lib.dtype_code(dtype), rows, heads, kv_heads, dim, st[0], st[1],
                                      pool, None if over is None else over.data_ptr(),
                                      dim ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
                                      out.stride(0), *_room(workspace), _lib.stream_of(q)))
    return out


def attend_chunk(q: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor, starts: Tensor, *,
                 scale: float = None, window: int = 0, sinks: int = 0, over: Tensor = None, out: Tensor = None,
                 workspace: Tensor = None) -> Tensor:
    """Causal attention of several new tokens per row over the row's pages.

    q: (tokens, heads, head dim); the tokens of row r are ``starts[r]`` ..
    ``starts[r + 1] - 1`` (int32, rows + 1, not decreasing, from 0 to tokens),
    the last of them at position ``lengths[r] - 1``, their keys and values in
    the pages already.  Each sees the positions up to its own, as in
    ``attend_token``.  Returns (tokens, heads, head dim) in q's type."""
    pool = _pool(k_pages, v_pages, table, lengths)
    dev, (_, kv_heads, page, dim), (rows, cols) = k_pages.device, k_pages.shape, table.shape
    dtype = k_pages.dtype
    st = _heads("q", q, None, dim, dtype, dev)
    _int32("starts", starts, (rows + 1,), dev)
    window, sinks = _visible(window, sinks)
    if over is not None:
        _int32("over", over, (rows,), dev)
    out = _output(out, q)
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _lib.no_gradient("attend_chunk")
    _lib.require_gpu(k_pages, what="attend_chunk")
    L, (tokens, heads, _) = _lib.lib(), q.shape
    need = L.qs_attend_chunk_workspace_bytes(tokens, rows, heads, kv_heads, dim, cols, page, window, sinks)
    workspace = _workspace(workspace, need, dev)
    _lib.check(L.qs_attend_chunk_over(q.data_ptr(), _lib.dtype_code(dtype), tokens, rows, heads, kv_heads, dim, st[0],
                                      st[1], starts.data_ptr(), pool, _lib.ptr(over),
                                      dim ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
                                      out.stride(0), *_room(workspace), _lib.stream_of(q)))
    return out


def _store(kv):
    if kv.dim() < 4 or not kv.is_contiguous():
        raise ValueError(f"kv must be a contiguous (..., pages, kv heads, page, head dim) tensor, got {tuple(kv.shape)}")
    pages, heads, page, dim = kv.shape[-4:]
    planes = kv.numel() // (pages * heads * page * dim or 1)
    return _lib.PageStore(kv.data_ptr(), planes, pages, heads, page, dim * kv.element_size())


def _books(table, lengths, refs, pages, device):
    if table.dim() != 2:
        raise ValueError(f"table must be (rows, columns), got {tuple(table.shape)}")
    _int32("table", table, table.shape, device)
    if lengths is not None:
        _int32("lengths", lengths, (table.shape[0],), device)
    _int32("refs", refs, (pages,), device)


def advance_pages(kv: Tensor, table: Tensor, lengths: Tensor, refs: Tensor, tokens=1, parents: Tensor = None, *,
                  out=None, over: Tensor = None, missing: Tensor = None, workspace: Tensor = None):
    """One step of every row of a cache ``kv`` (..., pages, kv heads, page,
    head dim): row i takes the pages and the length of row ``parents[i]``
    (int32; None: its own; no row of the table: an empty one), gives back pages
    beyond that length, and gets room for ``tokens`` more positions (a number,
    or an int32 tensor with one for every row), by which its length grows.

    The partly filled page that a row writes next is copied where several rows
    hold it, for each of them but the longest (the first of the longest); full
    pages stay shared.  New pages are the free ones in ascending order, given
    out by row, then by column.  Returns ``(table, lengths, refs, short)``;
    ``short`` (int32, 1; at most 2^31 - 1) is the number of pages that were
    wanted and could not be given, because none is free or the table has no
    column left: their entries are -1.  A page that a row did not get is not
    given later (the positions before in it are lost); it counts in every step
    whose tokens go to it, so that 0 says that every new token has its place.
    With ``over`` (int32, rows; written)
    lengths stop at the table's room and ``over`` gets how many of a row's new
    tokens lie beyond it, which are gone with the next step.  ``missing``
    (int32, 1) gets ``short`` added to it."""
    store, dev = _store(kv), kv.device
    _books(table, lengths, refs, store.pages, dev)
    rows, cols = table.shape
    if parents is not None:
        _int32("parents", parents, (rows,), dev)
    each = None
    if isinstance(tokens, Tensor):
        each, tokens = _int32("tokens", tokens, (rows,), dev), 0
    elif not 0 <= tokens <= 1 << 30:
        raise ValueError(f"{tokens} tokens")
    if out is None:
        out = (torch.empty_like(table), torch.empty_like(lengths), torch.empty_like(refs),
               torch.empty(1, dtype=torch.int32, device=dev))
    else:
        _books(out[0], out[1], out[2], store.pages, dev)
        _int32("out[0]", out[0], table.shape, dev)
        _int32("out[3]", out[3], (1,), dev)
    if over is not None:
        _int32("over", over, (rows,), dev)
    if missing is not None:
        _int32("missing", missing, (1,), dev)
    _lib.require_gpu(kv, what="advance_pages")
    L = _lib.lib()
    workspace = _workspace(workspace, L.qs_page_advance_workspace_bytes(rows), dev)
    _lib.check(L.qs_page_advance_over(store, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), _lib.ptr(parents),
                                      rows, cols, tokens, _lib.ptr(each), out[0].data_ptr(), out[1].data_ptr(),
                                      out[2].data_ptr(), out[3].data_ptr(), _lib.ptr(over), _lib.ptr(missing),
                                      *_room(workspace), _lib.stream_of(kv)))
    return tuple(out)


def free_pages(table: Tensor, lengths: Tensor, refs: Tensor, *, page: int, keep: Tensor = None, window: int = 0,
               sinks: int = 0, out=None):
    """Give pages back: all of the rows whose ``keep`` (bool) is false, whose
    length becomes 0, and with ``window`` those that no later token sees (one at
    position ``lengths[r]`` or beyond, with the first ``sinks`` visible too).
    Returns ``(table, lengths, refs)``."""
    dev = table.device
    _books(table, lengths, refs, refs.numel(), dev)
    rows, cols = table.shape
    if keep is not None:
        _rows_flag("keep", keep, (rows,), dev)
    window, sinks = _visible(window, sinks)
    if out is None:
        out = (torch.empty_like(table), torch.empty_like(lengths), torch.empty_like(refs))
    else:
        _int32("out[0]", out[0], table.shape, dev)
        _books(out[0], out[1], out[2], refs.shape[0], dev)
    _lib.require_gpu(table, what="free_pages")
    _lib.check(_lib.lib().qs_page_free(table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), _lib.ptr(keep), rows,
                                       cols, refs.shape[0], page, window, sinks, out[0].data_ptr(), out[1].data_ptr(),
                                       out[2].data_ptr(), _lib.stream_of(table)))
    return tuple(out)


def compact_pages(kv: Tensor, table: Tensor, refs: Tensor, *, out=None, workspace: Tensor = None):
    """Move the n pages in use to places 0 .. n - 1 of the pool: those beyond,
    in ascending order, to the free places in ascending order.  Returns
    ``(table, refs)``."""
    store, dev = _store(kv), kv.device
    _books(table, None, refs, store.pages, dev)
    rows, cols = table.shape
    if out is None:
        out = (torch.empty_like(table), torch.empty_like(refs))
    else:
        _int32("out[0]", out[0], table.shape, dev)
        _int32("out[1]", out[1], refs.shape, dev)
    _lib.require_gpu(kv, what="compact_pages")
    L = _lib.lib()
    workspace = _workspace(workspace, L.qs_page_compact_workspace_bytes(store.pages), dev)
    _lib.check(L.qs_page_compact(store, table.data_ptr(), refs.data_ptr(), rows, cols, out[0].data_ptr(),
                                 out[1].data_ptr(), _lib.ptr(workspace), workspace.numel(), _lib.stream_of(kv)))
    return tuple(out)


def copy_pages(kv: Tensor, src: Tensor, dst: Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` (int32) in every plane of the
    cache.  Pairs outside the pool are left out; no page may be written and
    named twice."""
    n, store = src.numel(), _store(kv)
    _int32("src", src, (n,), kv.device)
    _int32("dst", dst, (n,), kv.device)
    _lib.require_gpu(kv, what="copy_pages")
    _lib.check(_lib.lib().qs_page_copy(store, src.data_ptr(), dst.data_ptr(), n, _lib.stream_of(kv)))


class PagedCache:
    """The pages of a whole decoder: ``kv`` (layers, 2, pages, kv heads, page,
    head dim) with the table, lengths and reference counts of ``rows`` rows of
    at most ``columns`` pages.  The methods work in place.  ``lengths`` stop at
    the table's room; ``over`` has how many of a row's newest tokens lie beyond,
    which no page holds and no token sees.  ``missing`` counts the pages that
    any ``advance`` could not give."""

    def __init__(self, layers, pages, kv_heads, head_dim, rows, columns, page=64, dtype=torch.bfloat16, device="cuda"):
        self.page = page
        self.kv = torch.zeros(layers, 2, pages, kv_heads, page, head_dim, dtype=dtype, device=device)
        dev = self.kv.device
        self.table = torch.full((rows, columns), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self.over = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.short = torch.zeros(1, dtype=torch.int32, device=dev)
        self.missing = torch.zeros(1, dtype=torch.int32, device=dev)

    def keys(self, layer):
        return self.kv[layer, 0]

    def values(self, layer):
        return self.kv[layer, 1]

    def advance(self, tokens=1, parents=None):
        """``advance_pages``; ``self.short`` gets the pages that were missing, ``self.missing`` their sum so far."""
        advance_pages(self.kv, self.table, self.lengths, self.refs, tokens, parents,
                      out=(self.table, self.lengths, self.refs, self.short), over=self.over, missing=self.missing)

    def check(self):
        """Raise if an ``advance`` so far, captured ones that were replayed among them, had not all the pages that it
        wanted: tokens have been left out since.  Waits for the GPU; ``missing.zero_()`` starts anew."""
        missing = self.missing.item()
        if missing:
            raise RuntimeError(f"the cache was short of {missing} pages: tokens were left out")

    def free(self, keep=None, window=0, sinks=0):
        free_pages(self.table, self.lengths, self.refs, page=self.page, keep=keep, window=window, sinks=sinks,
                   out=(self.table, self.lengths, self.refs))

    def compact(self):
        compact_pages(self.kv, self.table, self.refs, out=(self.table, self.refs))

    def append(self, layer, k, v, starts=None):
        append_pages(self.kv[layer, 0], self.kv[layer, 1], k, v, self.table, self.lengths, starts, self.over)

    def append_rotated(self, layer, q, k, v, frequencies, starts=None, **options):
        from .rope import append_rotated
        return append_rotated(q, k, v, self.kv[layer, 0], self.kv[layer, 1], self.table, self.lengths, frequencies,
                              starts=starts, over=self.over, **options)

    def attend_token(self, layer, q, **options):
        return attend_token(q, self.kv[layer, 0], self.kv[layer, 1], self.table, self.lengths, over=self.over, **options)

    def attend_chunk(self, layer, q, starts, **options):
        return attend_chunk(q, self.kv[layer, 0], self.kv[layer, 1], self.table, self.lengths, starts, over=self.over,
                            **options)
