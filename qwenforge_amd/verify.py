"""Drafted tokens against the target model's logits (``include/qf_verify.h``).

The reference decodes greedily, one token a step (SE:980-982, SE:1126-1132).
``verify_drafts`` keeps the drafts that the target would have drawn and draws
the token after them, from random numbers that the caller gives, so one forward
pass over a row's last token and its drafts yields one to all of them.  Without
drafts (one position per row) it samples from the logits.
"""

from __future__ import annotations

import torch

from . import _lib
from .ops import _ptr, _stream, check_cu_seqlens

_DTYPES = {torch.float16: 0, torch.float32: 1}


def _vector(name: str, t, n: int, dtype, device) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device:
        raise TypeError(f"{name} must be a {str(dtype)[6:]} tensor on {device}")
    if t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous ({n},) (got {tuple(t.shape)})")


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, cu_seqlens: torch.Tensor,
                  max_seqlen: int, accept_u: torch.Tensor | None, sample_u: torch.Tensor | None,
                  temperature: float = 1.0, draft_probs: torch.Tensor | None = None, lengths=None):
    """Accepts each row's drafts in turn and draws the token after them.

    Rows are packed along the token axis: row b's positions are
    [cu_seqlens[b], cu_seqlens[b + 1]) ((B + 1,) int32, at most ``max_seqlen``
    each; ``lengths`` as in ``ops.prefill_varlen``).  ``tokens`` (T,) int64 holds
    each row's last token and then its drafts, ``logits`` (T, V) fp16 or fp32 what
    the target says after each of them: position j judges the token at j + 1.

    With ``temperature`` > 0, p = softmax(logits / temperature), and draft d is
    accepted while accept_u * q(d) < p(d): ``accept_u`` (T,) fp32 in [0, 1), q the
    rows of ``draft_probs`` (T, V) fp32 that the drafts were drawn from, or 1
    without them.  At the first rejection the next token is drawn from
    max(p - q, 0) (without ``draft_probs`` from p without d), after the last draft
    from p: the lowest one whose running sum exceeds ``sample_u`` (B,) fp32 in
    [0, 1) of the whole.  With ``temperature`` 0 drafts are accepted while they
    are the argmax, which also comes next; the random numbers may be None.

    Returns ``(count, out)``: out (B, max_seqlen) int64 holds row b's
    count[b] new tokens, then -1.  A position whose logits give no distribution
    (NaN and the like) draws nothing.
    """
    if not isinstance(logits, torch.Tensor) or logits.device.type != "cuda":
        raise RuntimeError("logits must be a HIP device tensor; there is no CPU path")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be float16 or float32 (got {logits.dtype})")
    if logits.dim() != 2 or logits.numel() == 0 or logits.stride(1) != 1:
        raise ValueError(f"logits must be (T, V) with unit last stride (got {tuple(logits.shape)})")
    total, vocab = logits.shape
    dev = logits.device
    b = cu_seqlens.numel() - 1 if isinstance(cu_seqlens, torch.Tensor) else 0
    if b < 1 or not 1 <= max_seqlen <= total:
        raise ValueError(f"need B >= 1 rows and 1 <= max_seqlen <= T (got {b}, {max_seqlen})")
    _vector("cu_seqlens", cu_seqlens, b + 1, torch.int32, dev)
    _vector("tokens", tokens, total, torch.int64, dev)
    temperature = float(temperature)
    if not 0.0 <= temperature < float("inf"):
        raise ValueError(f"temperature must be >= 0 and finite (got {temperature})")
    if temperature > 0:
        _vector("accept_u", accept_u, total, torch.float32, dev)
        _vector("sample_u", sample_u, b, torch.float32, dev)
        if draft_probs is not None:
            if draft_probs.dtype != torch.float32 or draft_probs.device != dev:
                raise TypeError(f"draft_probs must be a float32 tensor on {dev}")
            if draft_probs.shape != logits.shape or draft_probs.stride(1) != 1:
                raise ValueError("draft_probs must have the logits' shape and unit last stride")
    else:
        accept_u = sample_u = draft_probs = None
    check_cu_seqlens(cu_seqlens, total, max_seqlen, lengths)
    lib = _lib.load()
    need = lib.qf_verify_workspace(total, b, vocab)
    _lib.check(min(need, 0), "qf_verify_workspace")
    ws = torch.empty(need, device=dev, dtype=torch.uint8)
    out = torch.empty((b, max_seqlen), device=dev, dtype=torch.int64)
    count = torch.empty(b, device=dev, dtype=torch.int64)
    with torch.cuda.device(dev):
        rc = lib.qf_verify_drafts(
            logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0) if total > 1 else vocab,
            tokens.data_ptr(), cu_seqlens.data_ptr(), _ptr(accept_u), _ptr(sample_u),
            _ptr(draft_probs), 0 if draft_probs is None else draft_probs.stride(0) if total > 1 else vocab,
            temperature, out.data_ptr(), int(max_seqlen), count.data_ptr(), ws.data_ptr(), need,
            total, b, vocab, _stream(dev))
    _lib.check(rc, "qf_verify_drafts")
    return count, out
