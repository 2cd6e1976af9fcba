"""Beam search's selection: the best continuations of each group's beams.

The reference samples one sequence (model.py:634-650).  A search that keeps B
hypotheses a group needs two things next to the model's step: the best of the
B * V continuations (``beam_select``), and the caches in the order of what was
selected (``paged_reorder`` in ``paged.py``).  Both leave what they decide on the
GPU, so a search needs no word from the host between two tokens.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib as L
from .ops import _on_gpu, _same_device

_LOGITS = (torch.float32, torch.bfloat16, torch.float16)


def beam_select(logits: Tensor, scores: Tensor, count: Optional[int] = None, *, ended: Optional[Tensor] = None,
                pad: int = 0):
    """The ``count`` (default: B) best continuations of each of N groups (no autograd).

    logits [N, B, V] of the beams' next tokens; scores float32 [N, B]: the beams'
    log probabilities so far, -inf for a beam that is none (a group starts with
    one beam, the others at -inf).  A continuation scores

        scores[n, b] + log_softmax(logits[n, b])[v],

    taken in 64 bits and rounded once.  Of equal ones the lower beam's come first;
    within a beam the logits decide, the lower token of equal ones, also where
    scores do not tell them apart.  (Beams within about 1e-14 of each other are
    as near as sums in 64 bits are.)  ended (bool or
    uint8 [N, B]): a beam at its end has one continuation, token ``pad`` with the
    score it has.  A beam whose logits hold a NaN or +inf or nothing above -inf,
    or whose score is NaN or +inf, has none; where fewer than ``count`` are left,
    the lowest places not taken follow with -inf.

    Returns (scores float32, tokens int64, parents int64), each [N, count]; a
    parent is a beam's number in its group.  B <= 64, count <= 64 and <= B * V,
    V <= 2^20, and N * B rows of V / 8192 (rounded up) spans below 2^24."""
    K = int(logits.shape[1] if count is None and logits.dim() == 3 else count or 0)
    args = (logits, scores, K, ended, int(pad))
    res = L.host().beam_select(*args)
    if res is not None:
        return res
    if torch.jit.is_tracing():
        return torch.ops.bozo.beam_select(*args)
    _refuse_select(*args)


def _refuse_select(logits, scores, K, ended, pad) -> None:
    _on_gpu(logits, scores, ended)
    if logits.dim() != 3:
        raise ValueError(f"logits must be [N, B, V], got {tuple(logits.shape)}")
    if logits.dtype not in _LOGITS:
        raise TypeError(f"logits: unsupported dtype {logits.dtype}")
    N, B, V = logits.shape
    if scores.dtype != torch.float32 or tuple(scores.shape) != (N, B):
        raise ValueError(f"scores must be float32 [N, B] = [{N}, {B}], got {scores.dtype} {list(scores.shape)}")
    if ended is not None and (ended.dtype not in (torch.bool, torch.uint8) or tuple(ended.shape) != (N, B)):
        raise ValueError(f"ended must be bool [N, B] = [{N}, {B}], got {ended.dtype} {list(ended.shape)}")
    if not (1 <= B <= 64 and 1 <= V <= 1 << 20 and 1 <= K <= min(64, B * V)):
        raise ValueError(f"B must be in [1, 64], V in [1, 2^20], count in [1, min(64, B * V)], got {B}, {V}, {K}")
    if not 0 <= pad < V:
        raise ValueError(f"pad must be a token, got {pad}")
    _same_device(logits, scores, ended)
    if N * B * -(-V // 8192) >= 1 << 24:
        raise ValueError(f"too many rows for one call: N * B * ceil(V / 8192) must be below 2^24, got {N}, {B}, {V}")
    raise ValueError("beam_select: operands do not fit")


# While torch.jit.trace records (the native call path sends nothing through the
# dispatcher but the outputs' allocation).

@torch.library.custom_op("bozo::beam_select", mutates_args=(), device_types="cuda")
def _op_select(logits: Tensor, scores: Tensor, count: int, ended: Optional[Tensor],
               pad: int) -> tuple[Tensor, Tensor, Tensor]:
    args = (logits, scores, count, ended, pad)
    return L.host().beam_select(*args) or _refuse_select(*args)
