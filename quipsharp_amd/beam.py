"""Beam search over a quantized decoder's logits: the best continuations over
beams and vocabulary, and the states that follow them.  Neither has a gradient:
inputs that require one are refused where gradients are recorded.  No
counterpart in the reference.  The computation runs in libquipsharp_hip.so (csrc/qs_beam.hip)."""
import ctypes
import math

import torch
from torch import Tensor

from . import _lib
from .pages import _int32, _room, _rows_flag, _workspace

# argument arrays for 0 .. QS_MAX_STATES states
_WORDS = [ctypes.c_int64 * k for k in range(_lib.QS_MAX_STATES + 1)]
_POINTERS = [ctypes.c_void_p * k for k in range(_lib.QS_MAX_STATES + 1)]


def beam_select(logits: Tensor, scores: Tensor, keep: int = None, finished: Tensor = None, eos: int = -1, *,
                workspace: Tensor = None):
    """The ``keep`` (default: as many as beams) best continuations of each
    request's beams.

    logits: (batch * beams, vocab) or (batch, beams, vocab), float32, float16
    or bfloat16; scores: (batch, beams) float32.  Beam j with token t scores
    ``scores[b, j] + log_softmax(logits[b, j])[t]``; a beam whose ``finished``
    (bool) is set goes on with ``eos`` alone, at its own score.  Ties go to the
    lower beam, then the lower token.  A beam's log sum is taken from 32-bit
    exponentials, everything else in 64 bits: it is off by ``(2 ln(vocab) + 8)
    2 ** -24`` at most (2e-6 for 151936 tokens), so that continuations of two
    beams that lie closer than that may change places.  A NaN logit
    counts as -inf, and so does every continuation of a beam whose score or
    largest logit is not finite.

    Returns ``(scores, parents, tokens)``, (batch, keep) each and in descending
    order: float32, the parent's row ``b * beams + j`` and the token (int32)."""
    if scores.dim() != 2 or scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError(f"scores must be a contiguous float32 (batch, beams), got {tuple(scores.shape)} x {scores.dtype}")
    batch, beams = scores.shape
    vocab = logits.shape[-1]
    if logits.shape not in ((batch * beams, vocab), (batch, beams, vocab)):
        raise ValueError(f"logits {tuple(logits.shape)} do not fit scores {tuple(scores.shape)}")
    strides = logits.stride()
    if len(strides) == 3:
        if batch > 1 and beams > 1 and strides[0] != beams * strides[1]:
            raise ValueError("the rows of logits must lie one stride apart")
        ld = strides[1] if beams > 1 else strides[0]
    else:
        ld = strides[0]
    if batch * beams == 1:
        ld = vocab
    if strides[-1] != 1 and vocab > 1:
        raise ValueError("the logits of a row must lie together (stride 1)")
    dev = logits.device
    if scores.device != dev:
        raise ValueError(f"scores is on {scores.device}, logits on {dev}")
    if finished is not None:
        _rows_flag("finished", finished, scores.shape, dev)
    keep = beams if keep is None else keep
    if keep < 1:
        raise ValueError(f"keep {keep} must be 1 or more")
    code = _lib.dtype_code(logits.dtype)
    if logits.requires_grad or scores.requires_grad:
        _lib.no_gradient("beam_select")
    _lib.require_gpu(logits, what="beam_select")
    best = scores.new_empty((batch, keep))
    parents, tokens = torch.empty_like(best, dtype=torch.int32), torch.empty_like(best, dtype=torch.int32)
    L = _lib.lib()
    workspace = _workspace(workspace, L.qs_beam_select_workspace_bytes(batch, beams, vocab, keep), dev)
    _lib.check(L.qs_beam_select(logits.data_ptr(), code, ld, batch, beams, vocab,
                                scores.data_ptr(), _lib.ptr(finished), -1 if eos is None else eos, keep,
                                best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), *_room(workspace),
                                _lib.stream_of(logits)))
    return best, parents, tokens


def reorder_states(states, parents: Tensor):
    """New states whose row i is row ``parents[i]`` (int32, any shape, taken
    flat) of the given ones, up to 8 tensors at once whose first dimension
    counts rows; zeros where a parent names no row."""
    states = list(states)
    if not 1 <= len(states) <= _lib.QS_MAX_STATES:
        raise ValueError(f"{len(states)} states (1 to {_lib.QS_MAX_STATES})")
    dev, n = states[0].device, parents.numel()
    _int32("parents", parents, parents.shape, dev)
    rows = states[0].shape[0]
    size, stride, out = [], [], []
    for s in states:
        shape = s.shape
        if s.device != dev or not shape or shape[0] != rows:
            raise ValueError(f"every state must have {rows} rows on {dev}, got {tuple(shape)} on {s.device}")
        if not s.is_contiguous() and rows and not s[0].is_contiguous():
            raise ValueError("the elements of a state's row must lie together")
        if s.requires_grad:
            _lib.no_gradient("reorder_states")
        each = s.element_size()
        size.append((s.numel() // rows if rows else math.prod(shape[1:])) * each)
        stride.append(s.stride()[0] * each if rows > 1 else size[-1])
    _lib.require_gpu(*states, what="reorder_states")
    for s in states:
        out.append(torch.empty_like(s, memory_format=torch.contiguous_format) if n == rows
                   else s.new_empty((n,) + s.shape[1:]))
    k = len(states)
    words, pointers = _WORDS[k], _POINTERS[k]
    _lib.check(_lib.lib().qs_reorder_states(k, pointers(*[s.data_ptr() for s in states]),
                                            pointers(*[o.data_ptr() for o in out]), words(*size), words(*stride),
                                            parents.data_ptr(), n, rows, _lib.stream_of(states[0])))
    return out
