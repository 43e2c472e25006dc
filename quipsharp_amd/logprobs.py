"""Log probabilities of given tokens over a decoder's logits, with entropy, rank
and the best alternatives, for scoring answers and for perplexity windows.
They have no gradient: logits that require one are refused where gradients are
recorded.  No counterpart in the reference, whose evaluation takes the loss of
transformers' forward (scripts/eval_ppl.py:41-65).  The computation runs in
libquipsharp_hip.so (csrc/qs_logprobs.hip)."""
import torch
from torch import Tensor

from . import _lib
from .pages import _room, _workspace

MAX_TOP = 64


def workspace_bytes(rows, vocab, dtype, top=0) -> int:
    """Bytes of workspace that serve ``token_logprobs`` of any number of rows up to ``rows`` (few rows take more than
    many)."""
    return int(_lib.lib().qs_token_logprobs_workspace_most(rows, vocab, _lib.dtype_code(dtype), top))


def token_logprobs(logits: Tensor, tokens: Tensor, top: int = 0, *, workspace: Tensor = None):
    """Scores of ``tokens`` (rows,) int32 or int64 under ``logits`` (rows,
    vocab) float32, float16 or bfloat16.

    Returns ``(logprobs, entropy, ranks, top_logprobs, top_tokens)``, the first
    three (rows,), the last two (rows, top): the token's log probability
    (float32), the entropy of the row's distribution in nats (float32), how many
    tokens are ahead of the token (int32; a larger logit, or an equal one and a
    lower token; 0 for the greedy choice), and the ``top`` best tokens with
    their log probabilities, ties to the lower token (int32; -1 and -inf where
    no token is left).

    A token that is none of the vocabulary's (-100, say) has log probability 0
    and rank -1.  A NaN logit counts as -inf, and a token at -inf is no
    alternative.  A row whose largest logit is not finite has log probabilities
    -inf, entropy 0 and no alternatives.  Exponentials are 32-bit, their sums
    and logarithms 64-bit: a log sum is off by ``(3 ln(vocab) + 20) 2 ** -24`` at
    most (3.3e-6 for 151936 tokens).  Fewer than 2 ** 24 rows.  ``workspace``: uint8, of
    ``workspace_bytes`` for the most rows of any call that has it."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be (rows, vocab), got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    dev = logits.device
    code = _lib.dtype_code(logits.dtype)
    if logits.stride(1) != 1 and vocab > 1:
        raise ValueError("the logits of a row must lie together (stride 1)")
    ld = logits.stride(0) if rows > 1 else vocab
    if ld < vocab:
        raise ValueError("the rows of logits must not overlap")
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.shape != (rows,) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be {rows} contiguous int32 or int64 values, got {tuple(tokens.shape)} x {tokens.dtype}")
    if tokens.device != dev:
        raise ValueError(f"tokens is on {tokens.device}, logits on {dev}")
    if not 0 <= top <= MAX_TOP or top > vocab:
        raise ValueError(f"{top} alternatives (0 to {MAX_TOP}, of {vocab} tokens)")
    if logits.requires_grad:
        _lib.no_gradient("token_logprobs")
    _lib.require_gpu(logits, what="token_logprobs")
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy, ranks = torch.empty_like(logprobs), torch.empty(rows, dtype=torch.int32, device=dev)
    best = torch.empty(rows, top, dtype=torch.float32, device=dev)
    best_tokens = torch.empty(rows, top, dtype=torch.int32, device=dev)
    if rows and not vocab:
        raise ValueError("no vocabulary")
    L = _lib.lib()
    workspace = _workspace(workspace, L.qs_token_logprobs_workspace_bytes(rows, vocab, code, top), dev)
    with _lib.device_of(logits):
        _lib.check(L.qs_token_logprobs(logits.data_ptr(), code, ld, rows, vocab, tokens.data_ptr(),
                                       tokens.element_size(), top, logprobs.data_ptr(), entropy.data_ptr(),
                                       ranks.data_ptr(), best.data_ptr(), best_tokens.data_ptr(), *_room(workspace),
                                       _lib.stream_of(logits)))
    return logprobs, entropy, ranks, best, best_tokens
