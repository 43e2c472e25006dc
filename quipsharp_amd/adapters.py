"""Low-rank adapters of many requests at once, beside linears that they share:
the codes of a ``QuantizedLinear`` take no fine-tuned difference, so an
adapter's two products run beside it, for every row those of its own request.
They have no gradient: inputs that require one are refused where gradients are
recorded.  No counterpart in the reference.  The computation runs in
libquipsharp_hip.so (csrc/qs_adapters.hip)."""
import ctypes

import torch
from torch import Tensor

from . import _lib
from .pages import _HALF, _int32, _room, _workspace

MAX_RANK = 128
MAX_TOKENS = 1 << 19
MAX_APART = 1 << 24  # rows, in elements
NAMES = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def _rows(name, t, tokens, width, dtype, device):
    """The row stride of (tokens, width) with the elements of a row together."""
    if t.dim() != 2 or t.shape[0] != tokens or (width is not None and t.shape[1] != width):
        raise ValueError(f"{name} must be ({tokens}, {'width' if width is None else width}), got {tuple(t.shape)}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, x {dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, x on {device}")
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"the elements of a row of {name} must lie together (stride 1)")
    return t.stride(0) if tokens > 1 else t.shape[1]


def workspace_bytes(tokens, n, ranks) -> int:
    """Bytes of workspace that serve ``add_adapters`` of up to ``tokens`` rows of n elements beside linears of these
    ranks."""
    return int(_lib.lib().qs_adapters_workspace_bytes(tokens, n, 1, len(ranks), _lib.int_array(ranks)))


def add_adapters(ys, x: Tensor, which: Tensor, downs, ups, scales, *, outs=None, workspace: Tensor = None):
    """``ys[g][t] + scales[g][a] * ups[g][a] @ (downs[g][a] @ x[t])`` with ``a =
    which[t]``, for up to four linears g that read the same x.

    x: (tokens, n), bfloat16 or float16, n a multiple of 8; which: (tokens,)
    int32 on the GPU, a row that names no adapter keeps its y; downs[g]:
    (adapters, rank, n), ups[g]: (adapters, m, rank) in x's type, the rank a
    multiple of 8 up to 128 (zeros beyond an adapter's own), scales[g]:
    (adapters,) float32; ys[g]: (tokens, m) in x's type.  Returns new tensors,
    or ``outs``, each of which is the y at its place itself or apart from all
    the call reads and writes (others are refused).  Sums are float32, rounded once at the end; the inner
    products go on with 16 significant bits or more.  ``workspace``: uint8, of
    ``workspace_bytes`` for the most tokens of any call that has it."""
    count = len(ys)
    if not 1 <= count <= _lib.QS_MAX_GROUP or not len(downs) == len(ups) == len(scales) == count:
        raise ValueError(f"{count} outputs for {len(downs)} / {len(ups)} / {len(scales)} adapters (1 to {_lib.QS_MAX_GROUP} linears)")
    shape, st, dev, dtype = x.shape, x.stride(), x.device, x.dtype
    if len(shape) != 2:
        raise ValueError(f"x must be (tokens, n), got {tuple(shape)}")
    if dtype not in _HALF:
        raise TypeError(f"unsupported dtype {dtype} (bfloat16 or float16)")
    tokens, n = shape
    ldx = st[0] if st[1] == 1 and tokens > 1 else _rows("x", x, tokens, n, dtype, dev)
    _int32("which", which, (tokens,), dev)
    adapters = downs[0].shape[0] if downs[0].dim() else 0
    if outs is None:
        outs = [torch.empty(tokens, y.shape[-1], dtype=dtype, device=dev) for y in ys]
    elif len(outs) != count:
        raise ValueError(f"{len(outs)} outs for {count} linears")
    elif len({o.data_ptr() for o in outs}) < count and tokens:
        raise ValueError("every linear must have an output of its own")
    jobs, ranks, grads = (_lib.AdapterJob * count)(), (ctypes.c_int * count)(), x.requires_grad
    for g in range(count):
        y, o, down, up, scale = ys[g], outs[g], downs[g], ups[g], scales[g]
        ysh, yst, ost, dsh, ds, us = y.shape, y.stride(), o.stride(), down.shape, down.stride(), up.stride()
        m = ysh[-1] if ysh else 0
        # a decode step of one layer takes microseconds: what is refused is looked into only where something is
        if not (len(ysh) == 2 and ysh[0] == tokens and o.shape == ysh and y.dtype is dtype and o.dtype is dtype and y.device == dev
                and o.device == dev and yst[1] == 1 and ost[1] == 1 and len(dsh) == 3 and dsh[0] == adapters and dsh[2] == n
                and up.shape == (adapters, m, dsh[1]) and down.dtype is dtype and up.dtype is dtype and ds[2] == 1 and us[2] == 1
                and scale.dtype is torch.float32 and scale.shape == (adapters,) and scale.is_contiguous() and down.device == dev
                and up.device == dev and scale.device == dev):
            _refuse(g, y, o, down, up, scale, tokens, n, adapters, dtype, dev)
        rank = ranks[g] = dsh[1]
        grads = grads or y.requires_grad or o.requires_grad or down.requires_grad or up.requires_grad or scale.requires_grad
        jobs[g] = _lib.AdapterJob(down.data_ptr(), up.data_ptr(), scale.data_ptr(), ds[0] if adapters > 1 else 0, ds[1],
                                  us[0] if adapters > 1 else 0, us[1] if m > 1 else rank, rank, m, y.data_ptr(),
                                  yst[0] if tokens > 1 else m, o.data_ptr(), ost[0] if tokens > 1 else m)
    if grads:
        _lib.no_gradient("add_adapters")
    if adapters < 1:
        raise ValueError("no adapters")
    _lib.require_gpu(x, what="add_adapters")
    L = _lib.lib()
    workspace = _workspace(workspace, L.qs_adapters_workspace_bytes(tokens, n, adapters, count, ranks), dev)
    with _lib.device_of(x):
        _lib.check(L.qs_adapters_add(x.data_ptr(), _lib.dtype_code(dtype), ldx, tokens, n, which.data_ptr(), adapters,
                                     count, jobs, *_room(workspace), _lib.stream_of(x)))
    return outs


def _refuse(g, y, o, down, up, scale, tokens, n, adapters, dtype, dev):
    """Raises for linear g, in words; passes strides of a single column, which do not matter."""
    _rows(f"ys[{g}]", y, tokens, None, dtype, dev)
    m = y.shape[1]
    _rows(f"outs[{g}]", o, tokens, m, dtype, dev)
    if down.dim() != 3 or up.dim() != 3 or down.shape[2] != n or up.shape != (down.shape[0], m, down.shape[1]):
        raise ValueError(f"adapters {g}: {tuple(down.shape)} and {tuple(up.shape)} for {n} inputs and {m} outputs")
    if down.dtype is not dtype or up.dtype is not dtype:
        raise TypeError(f"adapters {g} are {down.dtype} and {up.dtype}, x {dtype}")
    if down.device != dev or up.device != dev or scale.device != dev:
        raise ValueError(f"adapters {g} are on {down.device}, {up.device} and {scale.device}, x on {dev}")
    if down.stride(2) != 1 or up.stride(2) != 1:
        raise ValueError("the elements of a row of an adapter must lie together (stride 1)")
    if down.shape[0] != adapters:
        raise ValueError(f"{down.shape[0]} adapters beside {adapters}")
    if scale.dtype is not torch.float32 or scale.shape != (adapters,) or not scale.is_contiguous():
        raise ValueError(f"scales[{g}] must be {adapters} contiguous float32 values, got {tuple(scale.shape)} x {scale.dtype}")


class Adapters:
    """``count`` adapters of one linear, of rank ``rank`` at most, empty at
    first: an empty one adds nothing.  As the attribute ``adapters`` of a
    ``QuantizedLinear`` they serve a ``decode.PagedDecoder``'s rows."""

    def __init__(self, count, rank, in_features, out_features, dtype=torch.bfloat16, device="cuda"):
        if not (count >= 1 and 1 <= rank <= MAX_RANK and in_features >= 8 and in_features % 8 == 0 and out_features >= 1):
            raise ValueError(f"{count} adapters of rank {rank} (at most {MAX_RANK}) for {in_features} inputs (a multiple of 8) "
                             f"and {out_features} outputs")
        if dtype not in _HALF:
            raise TypeError(f"unsupported dtype {dtype} (bfloat16 or float16)")
        rank = -(-rank // 8) * 8
        self.down = torch.zeros(count, rank, in_features, dtype=dtype, device=device)
        self.up = torch.zeros(count, out_features, rank, dtype=dtype, device=device)
        self.scale = torch.zeros(count, dtype=torch.float32, device=device)

    @torch.no_grad()
    def load(self, i, down: Tensor, up: Tensor, scale: float = 1.0):
        """Adapter i becomes ``scale * up @ down``: down (r, in_features), up (out_features, r) with r up to the rank."""
        r = down.shape[0]
        if down.shape != (r, self.down.shape[2]) or up.shape != (self.up.shape[1], r) or not 1 <= r <= self.down.shape[1]:
            raise ValueError(f"{tuple(down.shape)} and {tuple(up.shape)} for adapters of rank {self.down.shape[1]}, "
                             f"{self.down.shape[2]} inputs and {self.up.shape[1]} outputs")
        if not 0 <= i < len(self.scale):
            raise IndexError(f"adapter {i} of {len(self.scale)}")
        # its own values may be given, so nothing is cleared before they are read
        down, up = down.to(self.down, copy=True), up.to(self.up, copy=True)
        self.clear(i)
        self.down[i, :r] = down
        self.up[i, :, :r] = up
        self.scale[i] = scale

    @torch.no_grad()
    def clear(self, i):
        self.down[i] = 0
        self.up[i] = 0
        self.scale[i] = 0


def beside(x: Tensor, linears, ys, which: Tensor):
    """The outputs ``ys`` that ``linears`` made of x (tokens, n), with the adapters of those that have some
    (``linear.adapters``) added in place."""
    with_some = [(y, lin.adapters) for lin, y in zip(linears, ys) if getattr(lin, "adapters", None) is not None]
    if with_some:
        own = [y for y, _ in with_some]
        add_adapters(own, x, which, [a.down for _, a in with_some], [a.up for _, a in with_some],
                     [a.scale for _, a in with_some], outs=own)
    return ys


def check_beside(linears, which: Tensor, rows: int, tokens: int, dtype, device):
    """Raises where ``beside`` would refuse the adapters of ``linears``, which read the same rows of this type, for
    ``tokens`` tokens of ``rows`` rows whose adapters ``which`` names: for callers that must know before they run."""
    banks = [(lin, lin.adapters) for lin in linears if getattr(lin, "adapters", None) is not None]
    if not banks:
        return
    _int32("which", which, (rows,), device)
    if tokens > MAX_TOKENS:
        raise ValueError(f"{tokens} tokens at a time with adapters (at most {MAX_TOKENS})")
    count, place = banks[0][1].scale.shape[0], which.get_device()
    for g, (lin, bank) in enumerate(banks):
        down, up, scale, n, m = bank.down, bank.up, bank.scale, lin.in_features, lin.out_features
        shape = down.shape
        rank = shape[1] if len(shape) == 3 else 0
        # banks as they are made; what else there may be is looked into behind
        if shape == (count, rank, n) and up.shape == (count, m, rank) and scale.shape == (count,) and down.is_contiguous() \
                and up.is_contiguous() and scale.is_contiguous() and down.dtype is dtype and up.dtype is dtype \
                and scale.dtype is torch.float32 and down.get_device() == up.get_device() == scale.get_device() == place \
                and count and 8 <= rank <= MAX_RANK and not (rank | n) % 8 and not (down.data_ptr() | up.data_ptr()) & 15:
            continue
        y = torch.empty(0, m, dtype=dtype, device=device)
        _refuse(g, y, y, down, up, scale, 0, n, count, dtype, device)
        ds, us = down.stride(), up.stride()
        apart = ds[1] | (us[1] if m > 1 else 0) | (ds[0] | us[0] if count > 1 else 0)
        if not (count and 8 <= rank <= MAX_RANK and not (rank | n | apart) % 8 and n <= ds[1] <= MAX_APART
                and (rank <= us[1] <= MAX_APART or m == 1) and not (down.data_ptr() | up.data_ptr()) & 15):
            raise ValueError(f"adapters {g}: {tuple(shape)} and {tuple(up.shape)}: the rank must be a multiple of 8 up to "
                             f"{MAX_RANK}, rows 16-byte aligned and apart")


def attach_adapters(model, count, rank, names=NAMES, dtype=torch.bfloat16):
    """Gives every ``QuantizedLinear`` of ``model`` whose last name is among
    ``names`` (of ``NAMES``) room for ``count`` adapters of rank ``rank``, empty
    at first, in its attribute ``adapters``.  ``decode.PagedDecoder`` and what is built on it run them; the model's own
    forward, and with it ``decode.greedy_decode`` and ``decode.perplexity``, stays the base model's.  Returns them by the
    linears' names."""
    from .checkpoint import QuantizedLinear
    if not set(names) <= set(NAMES):
        raise ValueError(f"no decoder takes adapters beside {sorted(set(names) - set(NAMES))} (only {', '.join(NAMES)})")
    out = {}
    for name, lin in model.named_modules():
        if isinstance(lin, QuantizedLinear) and name.rpartition(".")[2] in names:
            lin.adapters = out[name] = Adapters(count, rank, lin.in_features, lin.out_features, dtype, lin.codes.device)
    return out
