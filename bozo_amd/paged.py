"""Paged K/V cache: tokens of sequences of different lengths in pages of one
pool, quantised or not, and the decode step that reads them.

A ``TensionDecodeCache`` (``ops.py``) holds one ring per sequence, all of one
length, and its sequences advance together.  Here a sequence owns the pages
its tokens fill and nothing more: position ``pos`` of sequence ``n`` lies in
page ``table[n, pos // S]`` at row ``pos % S``.  Pages are head-major,
``[P, Hk, S, D]``, so the rows of one (page, head) that a decode step streams
lie together.

With ``float8_e4m3fn`` pages a row (one token of one key/value head) is held
as e4m3 codes with one exponent byte: the smallest power of two 2^e that
brings the row's largest value within 448, and each x / 2^e rounded to the
nearest code, ties to even.  A value is then off by at most half a step, 2^-4
of its own size, or 2^-10 2^e for the small ones (the codes' subnormals).
Infinities are stored as NaN.

An entry of the table outside [0, P) (use -1) is no page: tokens there are
not written, read back as zeros, and attended to by nothing, so pages that
fell out of a local layer's window can be handed on at once.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch
from torch import Tensor

from . import _lib as L
from .ops import _DECODE_NORMS, _on_gpu, _same_device

_DENSE = (torch.float32, torch.bfloat16, torch.float16)
_PAGES = _DENSE + (torch.float8_e4m3fn,)


class PagedKV(NamedTuple):
    """One layer's pages: k, v [P, Hk, S, D] (float32, bfloat16, float16 or
    float8_e4m3fn, each its own type; unit innermost stride) and, for
    float8_e4m3fn, their exponent bytes k_exp, v_exp [P, Hk, S] (uint8)."""
    k: Tensor
    v: Tensor
    k_exp: Optional[Tensor] = None
    v_exp: Optional[Tensor] = None

    @classmethod
    def empty(cls, pages: int, page_size: int, heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
              v_dtype: Optional[torch.dtype] = None, device="cuda") -> "PagedKV":
        """Pages that hold nothing yet.  Their memory is not initialised: a
        position that has a page but was never appended reads back as
        anything, and so does a length that counts it."""
        both = (dtype, v_dtype or dtype)
        for t in both:
            if t not in _PAGES:
                raise TypeError(f"unsupported page dtype {t}")
        if min(pages, page_size, heads, head_dim) < 1:
            raise ValueError("pages, page_size, heads and head_dim must be >= 1")
        shape = (pages, heads, page_size, head_dim)
        buf = [torch.empty(shape, dtype=t, device=device) for t in both]
        exp = [torch.empty(shape[:3], dtype=torch.uint8, device=device) if t == torch.float8_e4m3fn else None
               for t in both]
        return cls(*buf, *exp)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def _check_pages(kv, N: int, table: Tensor, **counters: Optional[Tensor]) -> None:
    """What each operator needs of the cache and its table.  The library sees
    strides only: a table or counter smaller than the sequences imply would be
    read past its end on the device."""
    k, v, ke, ve = kv
    if k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"pages must be [P, Hk, S, D] alike, got {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape[0] < 1 or k.shape[2] < 1:
        raise ValueError(f"a cache needs one page of one token at least, got {tuple(k.shape)}")
    for name, t, e in (("k", k, ke), ("v", v, ve)):
        if t.dtype not in _PAGES:
            raise TypeError(f"unsupported page dtype {t.dtype}")
        if t.stride(3) != 1:
            raise ValueError(f"{name} pages need a unit innermost stride")
        if (t.dtype == torch.float8_e4m3fn) != (e is not None):
            raise ValueError(f"{name}_exp belongs to float8_e4m3fn pages, and to them only")
        if e is not None and (e.dtype != torch.uint8 or e.shape != t.shape[:3]):
            raise ValueError(f"{name}_exp must be uint8 {list(t.shape[:3])}, got {e.dtype} {list(e.shape)}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != N:
        raise ValueError(f"table must be int32 [{N}, pages per sequence], got {table.dtype} {list(table.shape)}")
    for name, t in counters.items():
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (N,)):
            raise ValueError(f"{name} must be int32 [N] = [{N}], got {t.dtype} {list(t.shape)}")
    _same_device(k, v, ke, ve, table, *counters.values())


def _check_append(kv, k_new, v_new, table, start, counts) -> None:
    if k_new.dim() != 4 or v_new.shape != k_new.shape:
        raise ValueError(f"k_new, v_new must share one [N, T, Hk, D] shape, got {tuple(k_new.shape)}, "
                         f"{tuple(v_new.shape)}")
    _check_pages(kv, k_new.shape[0], table, start=start, counts=counts)
    if k_new.shape[2] != kv[0].shape[1] or k_new.shape[3] != kv[0].shape[3]:
        raise ValueError(f"tokens of {k_new.shape[2]} heads of {k_new.shape[3]} for pages of {kv[0].shape[1]} heads "
                         f"of {kv[0].shape[3]}")
    for name, x, pages in (("k_new", k_new, kv[0]), ("v_new", v_new, kv[1])):
        if x.dtype not in _DENSE:
            raise TypeError(f"{name}: unsupported dtype {x.dtype}")
        if pages.dtype not in (x.dtype, torch.float8_e4m3fn) and x.dtype != torch.float32:
            raise TypeError(f"{name}: {x.dtype} tokens do not go into {pages.dtype} pages")
    _same_device(kv[0], k_new, v_new)


def paged_append(kv: PagedKV, k_new: Tensor, v_new: Tensor, table: Tensor, start: Tensor,
                 counts: Optional[Tensor] = None) -> None:
    """Write tokens k_new, v_new [N, T, Hk, D] into the pages (in place), at
    positions start[n] .. start[n] + counts[n] - 1 of sequence n (``counts``
    None: all T).  Tokens take the pages' type: as they are, float32 rounded
    to bfloat16 / float16 pages, or quantised to float8_e4m3fn ones.

    table: int32 [N, pages per sequence]; start, counts: int32 [N], all on
    the GPU.  Positions that the table has no page for are left out.  The
    pages that are written must belong to one sequence each; their version
    counters are raised, as by any write in place."""
    args = (*kv, k_new, v_new, table, start, counts)
    if L.host().paged_append(*args):
        return
    if torch.jit.is_tracing():
        torch.ops.bozo.paged_append(*args)
    else:
        _refuse_append(*args)


def _refuse_append(k, v, k_exp, v_exp, k_new, v_new, table, start, counts) -> None:
    kv = (k, v, k_exp, v_exp)
    _on_gpu(*kv, k_new, v_new, table, start, counts)
    _check_append(kv, k_new, v_new, table, start, counts)
    raise ValueError("paged_append: operands do not fit")


def paged_read(kv: PagedKV, table: Tensor, start: Tensor, T: int,
               dtype: Union[torch.dtype, tuple, None] = None, counts: Optional[Tensor] = None):
    """Read positions start[n] .. start[n] + T - 1 back: dense K, V
    [N, T, Hk, D]; zeros past counts[n] and where there is no page, whatever
    the page holds where no token was appended.

    dtype: of both, or a pair (K's, V's); default the pages' own, bfloat16 for
    float8_e4m3fn (which holds its values exactly)."""
    kd, vd = dtype if isinstance(dtype, tuple) else (dtype, dtype)
    kd = kd or (torch.bfloat16 if kv[0].dtype == torch.float8_e4m3fn else kv[0].dtype)
    vd = vd or (torch.bfloat16 if kv[1].dtype == torch.float8_e4m3fn else kv[1].dtype)
    args = (*kv, table, start, int(T), kd, vd, counts)
    res = L.host().paged_read(*args)
    if res is not None:
        return res
    if torch.jit.is_tracing():
        return torch.ops.bozo.paged_read(*args)
    _refuse_read(*args)


def _refuse_read(k, v, k_exp, v_exp, table, start, T: int, kd, vd, counts) -> None:
    kv = (k, v, k_exp, v_exp)
    _on_gpu(*kv, table, start, counts)
    if T < 0:
        raise ValueError("T must be >= 0")
    if start.dim() != 1:
        raise ValueError(f"start must be int32 [N], got {list(start.shape)}")
    _check_pages(kv, start.shape[0], table, start=start, counts=counts)
    for t in (kd, vd):
        if t not in _DENSE:
            raise TypeError(f"unsupported dtype {t}")
    raise ValueError("paged_read: operands do not fit")


def _check_decode(q, kv, table, lengths, W, max_len) -> None:
    if q.dim() != 3:
        raise ValueError(f"q must be [N, H, D], got {tuple(q.shape)}")
    if q.dtype not in _DENSE:
        raise TypeError(f"q: unsupported dtype {q.dtype}")
    _check_pages(kv, q.shape[0], table, lengths=lengths)
    Hk, D = kv[0].shape[1], kv[0].shape[3]
    if q.shape[2] != D or Hk < 1 or q.shape[1] % Hk:
        raise ValueError(f"q {list(q.shape)} does not fit pages of {Hk} heads of {D} (query heads are a multiple of "
                         "the key heads)")
    if W < 0 or max_len < 0:
        raise ValueError("window and max_len must be positive, or None")
    _same_device(q, kv[0])


def paged_decode(q: Tensor, kv: PagedKV, table: Tensor, lengths: Tensor, scale: float, *,
                 window: Optional[int] = None, include_self: bool = True, normalize="mass",
                 max_len: Optional[int] = None) -> Tensor:
    """One new token per sequence over its cached tokens (no autograd): the
    tension row ``sum_s tau_s v_s / norm``, ``tau_s = sigmoid(q . k_s /
    scale)``, of query q [N, H, D] at position lengths[n] - 1.  Append the
    token first (``paged_append``); lengths: int32 [N], it included.

    window: the W positions before the query (a local layer: keys t-W ..
    t-1 with ``include_self`` false); None: every earlier one (a global layer,
    which includes itself).  normalize: "mass" / True, "count" (keys in
    range) or None / "raw", as in ``decode_step``.  H may be a multiple of the
    pages' heads: query head h reads key head h // (H / Hk).  max_len: a bound
    of the lengths known on the host, by which the launch is shaped (default:
    what the table can hold); it does not cut a longer sequence.  Returns out
    [N, H, D] in q.dtype, zeros for a sequence with no key."""
    flags = _DECODE_NORMS.get(normalize)
    W = 0 if window is None else int(window)
    most = 0 if max_len is None else int(max_len)
    if window is not None and W < 1:
        raise ValueError("window must be >= 1")
    if flags is not None:
        args = (q, *kv, table, lengths, float(scale), W, most, flags | (L.DECODE_SELF if include_self else 0))
        out = L.host().paged_decode(*args)
        if out is not None:
            return out
        if torch.jit.is_tracing():
            return torch.ops.bozo.paged_decode(*args)
    _refuse_decode(q, kv, table, lengths, W, most)


def _refuse_decode(q, kv, table, lengths, W, most) -> None:
    _on_gpu(q, *kv, table, lengths)
    _check_decode(q, kv, table, lengths, W, most)
    raise ValueError(f"normalize must be one of {list(_DECODE_NORMS)}")


# ----------------------------------------------------------------- torch.library registration
#
# torch.jit.trace records what goes through the dispatcher.  The native call
# path sends nothing there but the outputs' allocation, which a replay would
# hand out as it is: it refuses while a trace records, and the call goes
# through these.

@torch.library.custom_op("bozo::paged_append", mutates_args=("k", "v", "k_exp", "v_exp"), device_types="cuda")
def _op_append(k: Tensor, v: Tensor, k_exp: Optional[Tensor], v_exp: Optional[Tensor], k_new: Tensor, v_new: Tensor,
               table: Tensor, start: Tensor, counts: Optional[Tensor]) -> None:
    args = (k, v, k_exp, v_exp, k_new, v_new, table, start, counts)
    if not L.host().paged_append(*args):
        _refuse_append(*args)


@torch.library.custom_op("bozo::paged_read", mutates_args=(), device_types="cuda")
def _op_read(k: Tensor, v: Tensor, k_exp: Optional[Tensor], v_exp: Optional[Tensor], table: Tensor, start: Tensor,
             T: int, k_dtype: torch.dtype, v_dtype: torch.dtype, counts: Optional[Tensor]) -> tuple[Tensor, Tensor]:
    args = (k, v, k_exp, v_exp, table, start, T, k_dtype, v_dtype, counts)
    return L.host().paged_read(*args) or _refuse_read(*args)


@torch.library.custom_op("bozo::paged_decode", mutates_args=(), device_types="cuda")
def _op_decode(q: Tensor, k: Tensor, v: Tensor, k_exp: Optional[Tensor], v_exp: Optional[Tensor], table: Tensor,
               lengths: Tensor, scale: float, W: int, most: int, flags: int) -> Tensor:
    kv = (k, v, k_exp, v_exp)
    out = L.host().paged_decode(q, *kv, table, lengths, scale, W, most, flags)
    if out is None:
        _refuse_decode(q, kv, table, lengths, W, most)
    return out
