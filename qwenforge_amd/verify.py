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
from .ops import _ptr
from .paged import _call, _check_rows, _workspace

_DTYPES = {torch.float16: 0, torch.float32: 1}


def _vector(name: str, t, n: int, dtype, index: int) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != index:
        raise TypeError(f"{name} must be a {str(dtype)[6:]} tensor on cuda:{index}")
    if t.dim() != 1 or t.shape[0] != n or (t.stride(0) != 1 and n > 1):
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
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise RuntimeError("logits must be a HIP device tensor; there is no CPU path")
    kind = _DTYPES.get(logits.dtype)
    if kind is None:
        raise TypeError(f"logits must be float16 or float32 (got {logits.dtype})")
    if logits.dim() != 2 or logits.numel() == 0 or logits.stride(1) != 1:
        raise ValueError(f"logits must be (T, V) with unit last stride (got {tuple(logits.shape)})")
    total, vocab = logits.shape
    index, dev = logits.get_device(), logits.device
    b = cu_seqlens.shape[0] - 1 if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.dim() == 1 else 0
    if b < 1 or not 1 <= max_seqlen <= total:
        raise ValueError(f"need B >= 1 rows and 1 <= max_seqlen <= T (got {b}, {max_seqlen})")
    _vector("cu_seqlens", cu_seqlens, b + 1, torch.int32, index)
    _vector("tokens", tokens, total, torch.int64, index)
    temperature = float(temperature)
    if not 0.0 <= temperature < float("inf"):
        raise ValueError(f"temperature must be >= 0 and finite (got {temperature})")
    probs_sn = 0
    if temperature > 0:
        _vector("accept_u", accept_u, total, torch.float32, index)
        _vector("sample_u", sample_u, b, torch.float32, index)
        if draft_probs is not None:
            if (not isinstance(draft_probs, torch.Tensor) or draft_probs.dtype is not torch.float32
                    or draft_probs.get_device() != index):
                raise TypeError(f"draft_probs must be a float32 tensor on {dev}")
            if draft_probs.shape != logits.shape or draft_probs.stride(1) != 1:
                raise ValueError("draft_probs must have the logits' shape and unit last stride")
            probs_sn = draft_probs.stride(0) if total > 1 else vocab
    else:
        accept_u = sample_u = draft_probs = None
    _check_rows(cu_seqlens, total, max_seqlen, lengths)
    out = torch.empty((b, max_seqlen), device=dev, dtype=torch.int64)
    count = torch.empty(b, device=dev, dtype=torch.int64)
    ws = _workspace(_lib.load().qf_verify_workspace(total, b, vocab), "qf_verify_workspace", dev)
    _call("qf_verify_drafts", index, logits.data_ptr(), kind, logits.stride(0) if total > 1 else vocab,
          tokens.data_ptr(), cu_seqlens.data_ptr(), _ptr(accept_u), _ptr(sample_u), _ptr(draft_probs),
          probs_sn, temperature, out.data_ptr(), max_seqlen, count.data_ptr(), ws.data_ptr(), ws.shape[0],
          total, b, vocab)
    return count, out
