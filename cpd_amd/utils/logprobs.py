"""Log probabilities of given tokens (or classes), the entropy of every row
of logits and its top alternatives, in one read of the logits; backed by the
gfx950 kernels in ops/csrc/logprob_hip.hip.

What ``nn.CrossEntropyLoss`` and ``accuracy`` compute in separate passes:
``-logprobs.mean()`` is the loss, ``top_ids == target`` the top-k hits.  On
CPU the eager composition of the same formulas runs; on the GPU the kernels
are the only path.
"""
from typing import NamedTuple, Optional

import torch

from .. import ops

__all__ = ["token_logprobs", "TokenLogprobs"]

MOST_TOP = 64
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                  # [...] float32
    entropy: torch.Tensor                   # [...] float32, in nats
    top_ids: Optional[torch.Tensor]         # [..., top_k] int64
    top_logprobs: Optional[torch.Tensor]    # [..., top_k] float32


def _check(logits, targets, top_k):
    """The extension's checks, for the CPU path."""
    if logits.dtype not in _TYPES:
        raise TypeError("logits must be float32, bfloat16 or float16, got "
                        f"{logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 30:
        raise ValueError("logits need a last axis of 1 to 2^30 - 1 entries")
    if targets.device != logits.device:
        raise ValueError(f"targets are on {targets.device}, logits on "
                         f"{logits.device}")
    if targets.dtype != torch.int64:
        raise TypeError(f"targets must be int64, got {targets.dtype}")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, logits "
                         f"{tuple(logits.shape)}")
    if not 0 <= top_k <= min(MOST_TOP, logits.shape[-1]):
        raise ValueError(f"top_k must be 0 to {MOST_TOP} and at most the "
                         f"number of logits, got {top_k}")


def _eager(logits, targets, top_k, ignore_index):
    _check(logits, targets, top_k)
    x = logits.float()
    kept = targets != ignore_index
    none = (x == -torch.inf).all(-1)
    inside = (targets >= 0) & (targets < x.shape[-1])
    # rows that say nothing are taken out before any arithmetic, so that
    # nothing in them reaches a gradient
    logp = torch.log_softmax(
        torch.where((none | ~kept)[..., None], 0.0, x), -1)
    p = logp.exp()
    ent = -(p * torch.where(p == 0, 0.0, logp)).sum(-1)
    lp = logp.gather(-1, torch.where(inside, targets, 0)[..., None])[..., 0]
    lp = torch.where(none, -torch.inf, lp)
    # a factor, so that the row's gradient is NaN too
    lp = lp * torch.where(inside, 1.0, torch.nan)
    ids = tops = None
    if top_k:
        with torch.no_grad():
            ids = torch.sort(x, dim=-1, descending=True,
                             stable=True)[1][..., :top_k]
            tops = torch.where((none | ~kept)[..., None], -torch.inf,
                               logp.gather(-1, ids))
            ids = torch.where(kept[..., None], ids, -1)
    return TokenLogprobs(torch.where(kept, lp, 0.0),
                         torch.where(kept & ~none, ent, 0.0), ids, tops)


def token_logprobs(logits, targets, top_k=0, ignore_index=-100):
    """What a softmax over the last axis of ``logits`` says of ``targets``.

    ``logits`` are [..., V] in float32, bfloat16 or float16, ``targets`` [...]
    int64.  Returns a :class:`TokenLogprobs`: the target's log probability and
    the row's entropy, both float32 with gradients, and, for ``top_k`` > 0 (at
    most 64), the indices and log probabilities of the ``top_k`` largest
    logits, largest first and equal ones by index, without gradients.

    * Rows whose target is ``ignore_index`` are passed over: log probability
      and entropy 0, ids -1, top log probabilities -inf, no gradient.
    * Entries of -inf (masked) have probability 0.  A row of them alone has
      log probability -inf, entropy 0 and no gradient.
    * NaN or +inf in a row makes its log probabilities, entropy and gradient
      NaN.  Among the alternatives NaN counts as the largest.
    * A target that is neither an index of the row nor ``ignore_index`` gives
      NaN, in the log probability and, where that is used, in the row's
      gradient (the entropy's alone stays what it is): targets are not read on
      the host.

    Rows may be apart by any stride (``logits[..., :V]`` of a padded product
    is read in place).  Raises TypeError and ValueError for types and shapes
    that do not fit.

    On the GPU gradients are of first order: a graph of them
    (``create_graph=True``) and forward-mode tangents raise RuntimeError.  On
    CPU torch's own operations run, where both work.
    """
    if not logits.is_cuda:
        return _eager(logits, targets, top_k, ignore_index)
    out = ops.hip_ext().token_logprobs(logits, targets, top_k, ignore_index)
    return TokenLogprobs(*out) if top_k else TokenLogprobs(*out, None, None)
