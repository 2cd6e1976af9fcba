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

With ``float4_e2m1fn_x2`` pages (keys and values both) a byte holds two e2m1
codes, the first in its low half, and every 32 values of a row an exponent
byte: the smallest power of two that brings the 32's largest value within 6.
The codes stand for 0, 0.5, 1, 1.5, 2, 3, 4 and 6: a value is off by at most
half a step, 2^-2 of its own size, or 2^-2 2^e for the small ones (6 * 2^125 at
most: what is larger becomes that).  32 values with an infinity or a NaN among
them read back as NaN.

An entry of the table outside [0, P) (use -1) is no page: tokens there are
not written, read back as zeros, and attended to by nothing, so pages that
fell out of a local layer's window can be handed on at once.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Union

import torch
from torch import Tensor

from . import _lib as L
from .ops import _DECODE_NORMS, _on_gpu, _same_device

_DENSE = (torch.float32, torch.bfloat16, torch.float16)
_FP4 = torch.float4_e2m1fn_x2
_PAGES = _DENSE + (torch.float8_e4m3fn, _FP4)


def _head_dim(pages: Tensor) -> int:
    return pages.shape[3] * (2 if pages.dtype == _FP4 else 1)


class PagedKV(NamedTuple):
    """One layer's pages: k, v [P, Hk, S, D] (float32, bfloat16, float16 or
    float8_e4m3fn, each its own type; unit innermost stride) and, for
    float8_e4m3fn, their exponent bytes k_exp, v_exp [P, Hk, S] (uint8); or both
    float4_e2m1fn_x2, [P, Hk, S, D / 2], with exponents [P, Hk, S, ceil(D / 32)]."""
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
        if _FP4 in both:
            if both != (_FP4, _FP4):
                raise TypeError(f"keys and values are both {_FP4}, or neither is")
            if head_dim % 2:
                raise ValueError(f"{_FP4} pages hold two values to a byte: head_dim {head_dim}")
            shape = (pages, heads, page_size)
            buf = [torch.empty(*shape, head_dim // 2, dtype=torch.uint8, device=device).view(_FP4) for _ in both]
            exp = [torch.empty(*shape, -(-head_dim // 32), dtype=torch.uint8, device=device) for _ in both]
            return cls(*buf, *exp)
        shape = (pages, heads, page_size, head_dim)
        buf = [torch.empty(shape, dtype=t, device=device) for t in both]
        exp = [torch.empty(shape[:3], dtype=torch.uint8, device=device) if t == torch.float8_e4m3fn else None
               for t in both]
        return cls(*buf, *exp)

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return _head_dim(self.k)


def _check_cache(kv) -> None:
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
        if (t.dtype in (torch.float8_e4m3fn, _FP4)) != (e is not None):
            raise ValueError(f"{name}_exp belongs to float8_e4m3fn and {_FP4} pages, and to them only")
        want = list(t.shape[:3]) + ([-(-_head_dim(t) // 32)] if t.dtype == _FP4 else [])
        if e is not None and (e.dtype != torch.uint8 or list(e.shape) != want):
            raise ValueError(f"{name}_exp must be uint8 {want}, got {e.dtype} {list(e.shape)}")
        if t.dtype == _FP4 and e.shape[3] > 1 and e.stride(3) != 1:
            raise ValueError(f"{name}_exp needs a unit innermost stride")
    if (k.dtype == _FP4) != (v.dtype == _FP4):
        raise TypeError(f"keys and values are both {_FP4}, or neither is")
    _same_device(k, v, ke, ve)


def _check_pages(kv, N: int, table: Tensor, **counters: Optional[Tensor]) -> None:
    """What each operator needs of the cache and its table.  The library sees
    strides only: a table or counter smaller than the sequences imply would be
    read past its end on the device."""
    _check_cache(kv)
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != N:
        raise ValueError(f"table must be int32 [{N}, pages per sequence], got {table.dtype} {list(table.shape)}")
    for name, t in counters.items():
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (N,)):
            raise ValueError(f"{name} must be int32 [N] = [{N}], got {t.dtype} {list(t.shape)}")
    _same_device(kv[0], table, *counters.values())


def _check_append(kv, k_new, v_new, table, start, counts) -> None:
    if k_new.dim() != 4 or v_new.shape != k_new.shape:
        raise ValueError(f"k_new, v_new must share one [N, T, Hk, D] shape, got {tuple(k_new.shape)}, "
                         f"{tuple(v_new.shape)}")
    _check_pages(kv, k_new.shape[0], table, start=start, counts=counts)
    _check_tokens(kv, k_new, v_new)


def _check_tokens(kv, k_new, v_new) -> None:
    heads, dim = k_new.shape[-2:]
    if heads != kv[0].shape[1] or dim != _head_dim(kv[0]):
        raise ValueError(f"tokens of {heads} heads of {dim} for pages of {kv[0].shape[1]} heads of {_head_dim(kv[0])}")
    for name, x, pages in (("k_new", k_new, kv[0]), ("v_new", v_new, kv[1])):
        if x.dtype not in _DENSE:
            raise TypeError(f"{name}: unsupported dtype {x.dtype}")
        if pages.dtype not in (x.dtype, torch.float8_e4m3fn, _FP4) and x.dtype != torch.float32:
            raise TypeError(f"{name}: {x.dtype} tokens do not go into {pages.dtype} pages")
    _same_device(kv[0], k_new, v_new)


def paged_append(kv: PagedKV, k_new: Tensor, v_new: Tensor, table: Tensor, start: Tensor,
                 counts: Optional[Tensor] = None) -> None:
    """Write tokens k_new, v_new [N, T, Hk, D] into the pages (in place), at
    positions start[n] .. start[n] + counts[n] - 1 of sequence n (``counts``
    None: all T).  Tokens take the pages' type: as they are, float32 rounded
    to bfloat16 / float16 pages, or quantised to float8_e4m3fn or
    float4_e2m1fn_x2 ones.

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


def paged_store(kv: PagedKV, k_new: Tensor, v_new: Tensor, slots: Tensor) -> None:
    """``paged_append`` for tokens whose places are known already: token
    k_new[n, t], v_new[n, t] [N, T, Hk, D] goes to page slots[n, t] // S, row
    slots[n, t] % S (slots int64 [N, T], as ``paged_plan`` gives them); or packed,
    tokens [M, Hk, D] and slots [M].  A slot outside [0, P * S) (use -1) is none,
    and its token is left out; no two tokens of a call may share one (parts of both
    may be left there).  A step looks its places up once for all layers."""
    args = (*kv, k_new, v_new, slots)
    if L.host().paged_store(*args):
        return
    if torch.jit.is_tracing():
        torch.ops.bozo.paged_store(*args)
    else:
        _refuse_store(*args)


def _refuse_store(k, v, k_exp, v_exp, k_new, v_new, slots) -> None:
    kv = (k, v, k_exp, v_exp)
    _on_gpu(*kv, k_new, v_new, slots)
    if k_new.dim() not in (3, 4) or v_new.shape != k_new.shape:
        raise ValueError(f"k_new, v_new must share one [N, T, Hk, D] or [M, Hk, D] shape, got {tuple(k_new.shape)}, "
                         f"{tuple(v_new.shape)}")
    if slots.dtype != torch.int64 or slots.shape != k_new.shape[:-2]:
        raise ValueError(f"slots must be int64 {list(k_new.shape[:-2])}, got {slots.dtype} {list(slots.shape)}")
    _check_cache(kv)
    _check_tokens(kv, k_new, v_new)
    _same_device(k, slots)
    raise ValueError("paged_store: operands do not fit")


def paged_read(kv: PagedKV, table: Tensor, start: Tensor, T: int,
               dtype: Union[torch.dtype, tuple, None] = None, counts: Optional[Tensor] = None):
    """Read positions start[n] .. start[n] + T - 1 back: dense K, V
    [N, T, Hk, D]; zeros past counts[n] and where there is no page, whatever
    the page holds where no token was appended.

    dtype: of both, or a pair (K's, V's); default the pages' own, bfloat16 for
    float8_e4m3fn and float4_e2m1fn_x2 (which holds their values exactly)."""
    kd, vd = dtype if isinstance(dtype, tuple) else (dtype, dtype)
    kd = kd or (kv[0].dtype if kv[0].dtype in _DENSE else torch.bfloat16)
    vd = vd or (kv[1].dtype if kv[1].dtype in _DENSE else torch.bfloat16)
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
    Hk, D = kv[0].shape[1], _head_dim(kv[0])
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


# ----------------------------------------------------------------- pages of sequences

class PagePool(NamedTuple):
    """The free pages of a pool, kept on the GPU: a stack free [P] (int32) of
    which the first top[0] (int32 [1]) entries are free pages, the last on top."""
    free: Tensor
    top: Tensor

    @classmethod
    def full(cls, pages: int, device="cuda") -> "PagePool":
        """A pool whose pages are all free; page 0 is taken first."""
        if pages < 1:
            raise ValueError("pages must be >= 1")
        return cls(torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=device),
                   torch.full((1,), pages, dtype=torch.int32, device=device))


def paged_plan(pool: PagePool, table: Tensor, lengths: Tensor, counts: Tensor, page_size: int, T: int, *,
               window: Optional[int] = None):
    """Pages for the tokens of a call, without a word from the host: the table
    int32 [N, pages per sequence] and the pool are changed in place.

    Sequence n holds lengths[n] tokens (int32 [N]) and grows by counts[n], or is
    cut by -counts[n] (to nothing at the least, which ends it).  A sequence that
    grows takes a page for every entry without one that its new tokens need; one
    that is cut gives back the pages behind its last token.  ``window``: of a
    local layer, whose queries read the last ``window`` positions before their
    own: pages that no later token reads are given back, and tokens that none
    reads get none.  Pages are given back before others are taken, both in the
    order of the sequences and their positions; a cut by as much undoes a growth.
    Tokens past the table's last entry have no place (slot -1, no page).
    A page of the table must be one sequence's.  A sequence that grows past its
    window at once leaves a gap behind its old pages, which the call's tokens may
    still read; they go back when it is cut by its old length (lengths old, counts
    -old), or ends.

    Returns slots int64 [N, T], page * S + row of the token at position lengths[n]
    + t for t < counts[n], -1 where there is none (``paged_store``; T: a bound of
    the counts, 0 for no slots), and missing int32 [1]: 0, or how many pages the
    pool is short of, and then nothing has changed (-1: more pages would be free
    than the pool has)."""
    args = (*pool, table, lengths, counts, int(page_size), int(T), 0 if window is None else int(window))
    if window is not None and args[-1] < 1:
        raise ValueError("window must be >= 1")
    res = L.host().paged_plan(*args)
    if res is not None:
        return res
    if torch.jit.is_tracing():
        return torch.ops.bozo.paged_plan(*args)
    _refuse_plan(*args)


def _refuse_plan(free, top, table, lengths, counts, page_size, T, window) -> None:
    _on_gpu(free, top, table, lengths, counts)
    if page_size < 1 or T < 0 or window < 0:
        raise ValueError("page_size must be >= 1, T >= 0")
    if table.dtype != torch.int32 or table.dim() != 2:
        raise ValueError(f"table must be int32 [N, pages per sequence], got {table.dtype} {list(table.shape)}")
    if (table.shape[1] > 1 and table.stride(1) != 1) or (table.shape[0] > 1 and table.stride(0) < table.shape[1]):
        raise ValueError("the table is written in place: it needs a unit innermost stride and rows that do not overlap")
    N = table.shape[0]
    for name, t, n in (("lengths", lengths, N), ("counts", counts, N), ("top", top, 1)):
        if t.dtype != torch.int32 or tuple(t.shape) != (n,):
            raise ValueError(f"{name} must be int32 [{n}], got {t.dtype} {list(t.shape)}")
    if free.dtype != torch.int32 or free.dim() != 1 or free.shape[0] < 1 or not free.is_contiguous():
        raise ValueError(f"free must be a contiguous int32 [pages], got {free.dtype} {list(free.shape)}")
    _same_device(table, free, top, lengths, counts)
    raise ValueError("paged_plan: operands do not fit")


def paged_reorder(layers: Sequence[PagedKV], table: Tensor, lengths: Tensor, parents: Tensor) -> Tensor:
    """The beams of N groups go on from other beams (no autograd).

    table int32 [N * B, pages per sequence]: beam b of group n is row n * B + b;
    lengths int32 [N]: tokens of a group's beams; parents int64 [N, B]: the beam of
    its group that beam b goes on from (``beam_select``), B <= 64; one outside
    [0, B) is b itself.  ``layers``: the caches that go by this table, alike in
    pages, page size, heads and head dim.

    Returns the new table.  Entries of full pages are the parent's (a group's beams
    share them).  From the page being filled on, the first beam that goes on from
    a parent takes over the parent's pages; each further one takes those of a
    beam that nobody goes on from, into whose first the parent's tokens are copied
    in every layer (the pages are written in place).  So each beam needs a page of
    its own for the tokens behind the last full page, and no other beam's row may
    name it.  At most 4096 layers, 254200 beams and 2^28 values a page."""
    ls = [tuple(kv) for kv in layers]
    args = (*([kv[i] for kv in ls] for i in range(4)), table, lengths, parents)
    out = L.host().paged_reorder(*args)
    if out is not None:
        return out
    if torch.jit.is_tracing():
        k, v, *exps = args[:4]
        return torch.ops.bozo.paged_reorder(k, v, [e for x in exps for e in x if e is not None], *args[4:])
    _refuse_reorder(*args)


def _refuse_reorder(k, v, k_exp, v_exp, table, lengths, parents) -> None:
    if not k:
        raise ValueError("paged_reorder needs a layer")
    _on_gpu(*k, *v, *k_exp, *v_exp, table, lengths, parents)
    if parents.dtype != torch.int64 or parents.dim() != 2 or parents.shape[1] > 64:
        raise ValueError(f"parents must be int64 [N, B], B <= 64, got {parents.dtype} {list(parents.shape)}")
    N, B = parents.shape
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (N,):
        raise ValueError(f"lengths must be int32 [N] = [{N}], got {lengths.dtype} {list(lengths.shape)}")
    for kv in zip(k, v, k_exp, v_exp):
        _check_pages(kv, N * B, table)
        if kv[0].shape[:3] != k[0].shape[:3] or _head_dim(kv[0]) != _head_dim(k[0]):
            raise ValueError(f"layers must be alike in pages, heads, page size and head dim, got {list(k[0].shape)}, "
                             f"{list(kv[0].shape)}")
        _same_device(table, kv[0])
    _same_device(table, lengths, parents)
    raise ValueError("paged_reorder: operands do not fit")


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


@torch.library.custom_op("bozo::paged_store", mutates_args=("k", "v", "k_exp", "v_exp"), device_types="cuda")
def _op_store(k: Tensor, v: Tensor, k_exp: Optional[Tensor], v_exp: Optional[Tensor], k_new: Tensor, v_new: Tensor,
              slots: Tensor) -> None:
    args = (k, v, k_exp, v_exp, k_new, v_new, slots)
    if not L.host().paged_store(*args):
        _refuse_store(*args)


@torch.library.custom_op("bozo::paged_plan", mutates_args=("free", "top", "table"), device_types="cuda")
def _op_plan(free: Tensor, top: Tensor, table: Tensor, lengths: Tensor, counts: Tensor, page_size: int, T: int,
             window: int) -> tuple[Tensor, Tensor]:
    args = (free, top, table, lengths, counts, page_size, T, window)
    return L.host().paged_plan(*args) or _refuse_plan(*args)


@torch.library.custom_op("bozo::paged_reorder", mutates_args=("k", "v", "exps"), device_types="cuda")
def _op_reorder(k: Sequence[Tensor], v: Sequence[Tensor], exps: Sequence[Tensor], table: Tensor, lengths: Tensor,
                parents: Tensor) -> Tensor:
    left = iter(exps)  # of the quantised pages, the keys' first
    ke, ve = ([None if t.dtype in _DENSE else next(left, None) for t in side] for side in (k, v))
    args = (list(k), list(v), ke, ve, table, lengths, parents)
    out = L.host().paged_reorder(*args)
    if out is None:
        _refuse_reorder(*args)
    return out
