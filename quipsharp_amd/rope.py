"""Rotary positions of new tokens with the write into a paged cache: pairs half
a head apart or side by side, all or part of a head, frequencies scaled for
contexts longer than a model was trained on.  ``append_rotated`` has no
gradient: inputs that require one are refused where gradients are recorded.  No
counterpart in the reference.  The computation runs in libquipsharp_hip.so
(csrc/qs_rope.hip)."""
import math

import torch
from torch import Tensor

from . import _lib
from .pages import _heads, _int32, _output, _pool

LAYOUTS = {"half": 0, "interleaved": 1}
MAX_PAIRS = 256

_SCALINGS = {"default": (), "linear": ("factor",), "ntk": ("factor",),
             "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
             "yarn": ("factor", "original_max_position_embeddings")}


def rope_frequencies(dim: int, base: float = 10000.0, scaling: dict = None, device="cuda"):
    """The angle per position, in radians, of each of the ``dim / 2`` pairs of
    ``dim`` rotated elements (float64), and the factor that rotated queries and
    keys are multiplied with: ``base ** (-2 i / dim)`` and 1, changed by
    ``scaling``, a dict as a model's config has it, by its ``rope_type``:

    - ``linear``: positions divided by ``factor``
    - ``ntk``: the base raised to ``base * factor ** (dim / (dim - 2))``
    - ``llama3``: pairs that turn less than ``low_freq_factor`` times over
      ``original_max_position_embeddings`` slowed by ``factor``, those that turn
      more than ``high_freq_factor`` times as they are, those between blended
    - ``yarn``: pairs that turn less than ``beta_slow`` (1) times slowed by
      ``factor``, those of more than ``beta_fast`` (32) as they are, a ramp over
      the pairs between; the factor is ``attention_factor``, or what ``mscale``
      and ``mscale_all_dim`` make of it, or ``0.1 ln(factor) + 1``"""
    if dim < 2 or dim % 2:
        raise ValueError(f"{dim} rotated elements: an even number, 2 or more")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _SCALINGS:
        raise NotImplementedError(f"rope_type {kind!r} ({', '.join(_SCALINGS)})")
    if any(not (scaling.get(name) or 0) > 0 for name in _SCALINGS[kind]):
        raise ValueError(f"{kind} scaling takes {', '.join(_SCALINGS[kind])}, all above 0; got {scaling}")
    base, factor = float(base), float(scaling.get("factor") or 1.0)
    if not base > 1:
        raise ValueError(f"a base of {base}: a number above 1")
    if kind == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling takes more than one pair")
        base *= factor ** (dim / (dim - 2))
    w = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if kind in ("default", "ntk"):
        return w.to(device), 1.0
    if kind == "linear":
        return (w / factor).to(device), 1.0
    trained = scaling["original_max_position_embeddings"]
    if kind == "llama3":
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not low < high:
            raise ValueError(f"llama3 scaling blends from {low} to {high} turns: the first must be the lower")
        kept = ((trained * w / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return (kept * w + (1 - kept) * w / factor).to(device), 1.0

    def pair(turns):  # which pair turns so many times over the trained positions
        return dim / 2 * math.log(trained / (turns * 2 * math.pi)) / math.log(base)

    low, high = pair(float(scaling.get("beta_fast") or 32)), pair(float(scaling.get("beta_slow") or 1))
    if scaling.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    slowed = ((torch.arange(dim // 2, dtype=torch.float64) - low) / ((high - low) or 0.001)).clamp(0, 1)

    def strength(mscale):
        return 0.1 * mscale * math.log(factor) + 1.0 if factor > 1 else 1.0

    attention = scaling.get("attention_factor")
    if attention is None:
        mscale, every = scaling.get("mscale"), scaling.get("mscale_all_dim")
        attention = strength(mscale) / strength(every) if mscale and every else strength(1.0)
    return (slowed * w / factor + (1 - slowed) * w).to(device), float(attention)


def model_frequencies(config, device="cuda"):
    """``rope_frequencies`` of a transformers config: of its head's width, the
    part of it that turns, its base and scaling."""
    given = dict(getattr(config, "rope_parameters", None) or getattr(config, "rope_scaling", None) or {})
    base = given.pop("rope_theta", None) or getattr(config, "rope_theta", 10000.0)
    part = given.pop("partial_rotary_factor", None) or getattr(config, "partial_rotary_factor", None) or 1.0
    head = getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
    return rope_frequencies(int(head * part), base, given, device)


def append_rotated(q: Tensor, k: Tensor, v: Tensor, k_pages: Tensor, v_pages: Tensor, table: Tensor, lengths: Tensor,
                   frequencies: Tensor, *, starts: Tensor = None, over: Tensor = None, layout: str = "half",
                   factor: float = 1.0, out: Tensor = None) -> Tensor:
    """New tokens' queries turned to their positions, and their keys, turned, and
    values stored in the pages (``pages.append_pages``, whose tokens, rows,
    ``starts`` and ``over`` these are).

    q: (tokens, heads, head dim), k and v: (tokens, kv heads, head dim) in the
    cache's type.  Of every head the first ``2 * len(frequencies)`` elements are
    turned, pair i by ``position * frequencies[i]`` radians (float64, from
    ``rope_frequencies``; the product is taken in 64 bits) and multiplied by
    ``factor``; a pair is elements i and i + len(frequencies) (``half``) or 2 i
    and 2 i + 1 (``interleaved``).  Returns the queries, in ``out`` if given,
    which may be q, and is refused where it shares memory with q, k or v otherwise.

    A token at a position below 0 gets zero queries and is stored nowhere, one
    without a page or beyond the table is turned all the same, and tokens of no
    row (behind the last of ``starts``) are left out: their queries are not
    written."""
    pool = _pool(k_pages, v_pages, table, lengths)
    dev, dtype, (_, kv_heads, _, dim), rows = k_pages.device, k_pages.dtype, k_pages.shape, table.shape[0]
    qs = _heads("q", q, None if starts is not None else rows, dim, dtype, dev)
    tokens, heads = q.shape[0], q.shape[1]
    ks, vs = _heads("k", k, tokens, dim, dtype, dev), _heads("v", v, tokens, dim, dtype, dev)
    if k.shape[1] != kv_heads or v.shape[1] != kv_heads:
        raise ValueError(f"{k.shape[1]} and {v.shape[1]} heads for a cache of {kv_heads}")
    if starts is not None:
        _int32("starts", starts, (rows + 1,), dev)
    if over is not None:
        _int32("over", over, (rows,), dev)
    pairs = frequencies.numel()
    if frequencies.dtype is not torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise ValueError(f"frequencies must be contiguous float64 values, got {tuple(frequencies.shape)} x {frequencies.dtype}")
    if frequencies.device != dev:
        raise ValueError(f"frequencies is on {frequencies.device}, the cache on {dev}")
    if not 1 <= pairs <= MAX_PAIRS or 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs of a head of {dim} (1 to {MAX_PAIRS})")
    if layout not in LAYOUTS:
        raise ValueError(f"layout {layout!r} (half or interleaved)")
    out = _output(out, q)
    if q.requires_grad or k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad \
            or frequencies.requires_grad or out.requires_grad:
        _lib.no_gradient("append_rotated")
    _lib.require_gpu(k_pages, what="append_rotated")
    with _lib.device_of(k_pages):
        _lib.check(_lib.lib().qs_page_append_rotated(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.dtype_code(dtype), tokens, rows, heads, kv_heads, dim, qs[0],
            qs[1], ks[0], ks[1], vs[0], vs[1], _lib.ptr(starts), pool, _lib.ptr(over), frequencies.data_ptr(), pairs,
            LAYOUTS[layout], factor, out.data_ptr(), out.stride(0), _lib.stream_of(k_pages)))
    return out
