"""Generation for sequences of different lengths over paged caches.

``TensionKVCache`` (``generation.py``) advances N sequences in lock step, each
with room for ``max_seq_len`` tokens.  Here sequences come and go, each at its
own position, and own the pages that their tokens fill: ``paged_append``
stores prompts and new tokens (quantised to e4m3 or 4 bits if asked),
``paged_decode`` advances one token each, and ``paged_read`` gives a prompt that
continues on cached tokens the keys and values before it.

All layers of one kind share page numbers (each layer has its own pages of
that number): a global layer keeps every token, a local one the pages of its
last W, which go back to the pool as the window leaves them.

The tables are kept on the host (``PageTable``) or on the GPU
(``DevicePageTable``: ``paged_plan``, ``paged_store``).  ``beam_search`` keeps a
search's beams in the pages of one pool, in the order that ``beam_select`` and
``paged_reorder`` leave on the GPU.

The reference keeps no cache (model.py:736-739); a step equals its forward's
last row (model.py:617-652) as long as a sequence fits ``max_seq_len``, up to
the rounding of the pages' type.
"""
from __future__ import annotations

from contextlib import contextmanager
from typing import Optional, Sequence

import torch
from torch import Tensor

from .beam import beam_select
from .generation import _after_tension, _osc_positions, sample_next
from .ops import autocast_inputs, causal_tension, global_tension, rope
from .paged import PagedKV, PagePool, paged_append, paged_decode, paged_plan, paged_read, paged_reorder, paged_store


class PageTable:
    """Which pages of a pool hold which sequence's tokens, kept on the host.

    ``window``: a sequence keeps the pages of its last ``window`` tokens (0:
    all of them)."""

    def __init__(self, pages: int, page_size: int, sequences: int, max_len: int, window: int = 0):
        self.S, self.window, self.pages = page_size, window, pages
        self.rows = torch.full((sequences, -(-max_len // page_size)), -1, dtype=torch.int32)
        self.free = list(range(pages - 1, -1, -1))
        self.changed = True

    def _span(self, length: int, more: int):
        """Pages that a sequence of ``length`` tokens needs for ``more``."""
        end = length + more
        first = max(0, end - self.window) // self.S if self.window else 0
        return max(first, length // self.S), -(-end // self.S)

    def missing(self, seq: int, length: int, more: int) -> int:
        a, b = self._span(length, more)
        return int((self.rows[seq, a:b] < 0).sum())

    def grow(self, seq: int, length: int, more: int) -> list:
        """Pages for tokens length .. length + more - 1 (those in the window
        of what follows them).  Returns the entries it filled."""
        a, b = self._span(length, more)
        new = [i for i in range(a, b) if self.rows[seq, i] < 0]
        for i in new:
            self.rows[seq, i] = self.free.pop()
            self.changed = True
        return new

    def drop(self, seq: int, length: int) -> None:
        """Hand on the pages that no token from position ``length`` reads."""
        if self.window:
            self.give(seq, range(max(0, length - self.window) // self.S))

    def release(self, seq: int) -> None:
        self.give(seq, range(self.rows.shape[1]))

    def give(self, seq: int, entries) -> None:
        for i in entries:
            if self.rows[seq, i] >= 0:
                self.free.append(int(self.rows[seq, i]))
                self.rows[seq, i] = -1
                self.changed = True


class DevicePageTable:
    """``PageTable`` with the table and the free pages on the GPU: a call's pages
    are one ``paged_plan``, which also gives its tokens' slots.  The host counts
    pages, by the sequences' lengths alone, so that a call without room is
    refused before anything changes.

    A window's pages go back with the next tokens of their sequence rather than
    with the ones that leave them, so a sequence holds a page more."""

    def __init__(self, pages: int, page_size: int, sequences: int, max_len: int, window: int = 0, device="cuda"):
        self.S, self.window, self.pages, self.left = page_size, window, pages, pages
        self.table = torch.full((sequences, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.pool = PagePool.full(pages, device)
        self.held = [(0, 0)] * sequences  # entries with a page: from, up to

    def _after(self, seq: int, length: int, more: int):
        """Entries that go back first, those that are taken, what is held in
        between and after it; and where the new pages start if they leave a gap
        behind old ones, which the call's tokens still read."""
        S, W, (lo, hi) = self.S, self.window, self.held[seq]
        low = min(max(lo, max(0, length - W) // S if W else 0), hi)
        first = max(max(0, length + more - W) // S if W else 0, length // S)
        end = -(-(length + more) // S)
        gap = first > hi > low
        return low - lo, end - max(first, hi), (low, hi), (low if gap or first <= hi else first, end), first if gap else None

    def room(self, seqs: Sequence[int], lengths: Sequence[int], more: Sequence[int]) -> bool:
        a = [self._after(*x) for x in zip(seqs, lengths, more)]
        return sum(x[1] for x in a) <= self.left + sum(x[0] for x in a)

    def _plan(self, seqs, lengths, counts, T: int) -> Tensor:
        both = torch.zeros(2, len(self.held), dtype=torch.int32)
        at = torch.tensor(list(seqs), dtype=torch.long)
        both[0, at], both[1, at] = torch.tensor(list(lengths), dtype=torch.int32), torch.tensor(list(counts), dtype=torch.int32)
        both = both.to(self.table.device)
        return paged_plan(self.pool, self.table, both[0], both[1], self.S, T, window=self.window or None)[0]

    def take(self, seqs: Sequence[int], lengths: Sequence[int], more: Sequence[int]):
        """Pages for tokens of these sequences: their slots [sequences, max(more)],
        what gives the pages back if the call fails, and what has to be done if
        it does not."""
        slots, gaps, total, kept = self._plan(seqs, lengths, more, max(more)), [], 0, []
        for s, n, m in zip(seqs, lengths, more):
            given, taken, before, after, gap = self._after(s, n, m)
            self.left += given - taken
            self.held[s] = after
            total += taken
            kept.append((s, before))
            if gap is not None:  # the old pages go back when the call is done
                gaps.append((s, n, before, gap))

        def undo():
            self._plan(seqs, [a + b for a, b in zip(lengths, more)], [-m for m in more], 0)
            self.left += total
            for s, before in kept:
                self.held[s] = before

        def done():
            if gaps:  # cut by their old lengths
                self._plan([g[0] for g in gaps], [g[1] for g in gaps], [-g[1] for g in gaps], 0)
            for s, _, (lo, hi), first in gaps:
                self.left += hi - lo
                self.held[s] = (first, self.held[s][1])

        return slots, undo, done

    def release(self, seq: int, length: int) -> None:
        self._plan([seq], [length], [-length], 0)
        lo, hi = self.held[seq]
        self.left += hi - lo
        self.held[seq] = (0, 0)


class TensionPagedCache:
    """Paged K/V caches of up to ``sequences`` sequences of one model.

    pages: of each global layer; local_pages: of each local layer (default:
    what ``sequences`` windows fill, and one more for ``extend``).  dtype: the pages' type, e.g.
    ``torch.float8_e4m3fn`` or ``torch.float4_e2m1fn_x2`` (default: as the layers compute their keys and
    values).  device_tables: the page tables are kept on the GPU, and a call's
    pages and slots come from one kernel a kind of layer (``DevicePageTable``);
    otherwise the host looks them up.  The model must be in eval mode (dropout
    off)."""

    def __init__(self, model, sequences: int, pages: int, local_pages: Optional[int] = None, page_size: int = 64,
                 dtype: Optional[torch.dtype] = None, device_tables: bool = False):
        cfg = model.cfg
        self.model, self.dtype = model, dtype
        device = next(model.parameters()).device
        window = min(-(-cfg.window // page_size) + 1, -(-cfg.max_seq_len // page_size))
        local = (sequences + 1) * (window + device_tables) if local_pages is None else local_pages
        self.on_device = device_tables
        kind = (lambda *a: DevicePageTable(*a, device=device)) if device_tables else PageTable
        self.tables = {True: kind(pages, page_size, sequences, cfg.max_seq_len, 0),
                       False: kind(local, page_size, sequences, cfg.max_seq_len, cfg.window)}
        if not any(b.global_layer for b in model.blocks):
            del self.tables[True]
        if all(b.global_layer for b in model.blocks):
            del self.tables[False]
        self.layers: list[Optional[PagedKV]] = [None] * len(model.blocks)
        self.length = [0] * sequences  # tokens cached; 0: not in use
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._device_rows = {g: t.table if device_tables else t.rows.to(device) for g, t in self.tables.items()}
        self._slots: dict = {}  # of the call's tokens, while one runs on device tables

    # ---------------------------------------------------------------- bookkeeping

    @contextmanager
    def _room(self, seqs: Sequence[int], more: Sequence[int]):
        """Room for the call's tokens, or an error before anything changes.
        The pages taken for them go back if what follows fails."""
        if self.model.training:
            raise RuntimeError("generation needs model.eval() (dropout off)")
        if len(set(seqs)) != len(seqs):
            raise ValueError(f"a sequence twice in one call: {list(seqs)}")
        limit = self.model.cfg.max_seq_len
        for s, m in zip(seqs, more):
            if m < 1 or self.length[s] + m > limit:
                raise ValueError(f"{m} tokens after {self.length[s]}: outside [1, max_seq_len {limit}]")
        before = [self.length[s] for s in seqs]
        for t in self.tables.values():
            room = t.room(seqs, before, more) if self.on_device else \
                sum(t.missing(s, n, m) for s, n, m in zip(seqs, before, more)) <= len(t.free)
            if not room:
                raise RuntimeError(f"out of pages ({t.pages} in the pool): release a sequence, or wait for one to end")
        if self.on_device:
            with self._room_on_device(seqs, before, more):
                yield
            return
        taken = [(t, s, t.grow(s, self.length[s], m)) for t in self.tables.values() for s, m in zip(seqs, more)]
        try:
            yield
        except BaseException:
            for t, s, entries in reversed(taken):
                t.give(s, reversed(entries))
            raise

    @contextmanager
    def _room_on_device(self, seqs: Sequence[int], before: Sequence[int], more: Sequence[int]):
        taken = []
        try:
            for g, t in self.tables.items():
                slots, *rest = t.take(seqs, before, more)
                taken.append(rest)
                self._slots[g] = slots.index_select(0, torch.tensor(seqs, device=slots.device))
            yield
        except BaseException:
            for undo, _ in reversed(taken):
                undo()
            raise
        finally:
            self._slots = {}
        for _, done in taken:
            done()

    def _store(self, i: int, k: Tensor, v: Tensor, rows: dict, start: Tensor, counts: Optional[Tensor] = None) -> None:
        """The call's tokens into the pages of layer ``i``."""
        g = self.model.blocks[i].global_layer
        if self.on_device:
            paged_store(self._pages(i, k, v), k, v, self._slots[g])
        else:
            paged_append(self._pages(i, k, v), k, v, rows[g], start, *(() if counts is None else (counts,)))

    def _rows(self, idx: Tensor) -> dict:
        """The tables' rows of these sequences, on the device."""
        for g, t in self.tables.items():
            if not self.on_device and t.changed:
                self._device_rows[g].copy_(t.rows)
                t.changed = False
        return {g: r.index_select(0, idx) for g, r in self._device_rows.items()}

    def _advance(self, seqs: Sequence[int], more: Sequence[int], idx: Tensor, lengths: Tensor) -> None:
        self.lengths.index_copy_(0, idx, lengths)
        for s, m in zip(seqs, more):
            self.length[s] += m
            for t in self.tables.values():
                if not self.on_device:
                    t.drop(s, self.length[s])

    def _live(self, seqs: Sequence[int]) -> None:
        for s in seqs:
            if not 0 <= s < len(self.length):
                raise ValueError(f"no sequence {s}: they are numbered 0 to {len(self.length) - 1}")
            if self.length[s] == 0:
                raise ValueError(f"sequence {s} is not in use")

    def release(self, seq: int) -> None:
        """End a sequence; its pages and its number are free again."""
        self._live([seq])
        for t in self.tables.values():
            t.release(seq, self.length[seq]) if self.on_device else t.release(seq)
        self.length[seq] = 0

    def _pages(self, i: int, k: Tensor, v: Tensor) -> PagedKV:
        if self.layers[i] is None:
            t = self.tables[self.model.blocks[i].global_layer]
            self.layers[i] = PagedKV.empty(t.pages, t.S, k.shape[2], k.shape[3], self.dtype or k.dtype,
                                           self.dtype or v.dtype, k.device)
        return self.layers[i]

    # ---------------------------------------------------------------- tokens

    @torch.no_grad()
    def prefill(self, prompts: Sequence[Tensor]):
        """Start a sequence for each prompt (token ids [T_n]).  Returns their
        numbers and the logits [N, vocab] of their last tokens.  Prompts run
        as one padded batch: a causal layer's earlier rows do not see the
        padding, and only real tokens are stored."""
        seqs = [s for s, n in enumerate(self.length) if n == 0][:len(prompts)]
        if len(seqs) < len(prompts):
            raise RuntimeError(f"{len(prompts)} prompts for {len(seqs)} free sequences")
        counts = [int(p.numel()) for p in prompts]
        with self._room(seqs, counts):
            dev = self.lengths.device
            ids = torch.zeros(len(prompts), max(counts), dtype=torch.long)
            for row, p in zip(ids, prompts):
                row[:p.numel()] = p
            idx = torch.tensor(seqs, device=dev)
            n = torch.tensor(counts, dtype=torch.int32, device=dev)
            start, rows = torch.zeros_like(n), self._rows(idx)

            layers = [b.tension for b in self.model.blocks]
            for i, layer in enumerate(layers):
                layer.kv_sink = (lambda k, v, i=i: self._store(i, k, v, rows, start, n))
            try:
                logits = self.model(ids.to(dev))
            finally:
                for layer in layers:
                    layer.kv_sink = None
            last = logits[torch.arange(len(seqs), device=dev), n.long() - 1]
            self._advance(seqs, counts, idx, n)
            return seqs, last

    @torch.no_grad()
    def extend(self, seq: int, ids: Tensor) -> Tensor:
        """Continue a sequence with more tokens ids [T] at once (a user's next
        turn).  Returns the logits [vocab] of the last one.  Each layer reads
        the keys and values before them back from its pages."""
        self._live([seq])
        T, t0 = int(ids.numel()), self.length[seq]
        with self._room([seq], [T]):
            model, dev = self.model, self.lengths.device
            idx = torch.tensor([seq], device=dev)
            rows, start = self._rows(idx), self.lengths.index_select(0, idx)
            at = torch.arange(t0, t0 + T, device=dev)
            x = model.embedding(ids.to(dev).view(1, T))
            if model.pos_embedding is not None:
                x = x + model.pos_embedding(at)[None]
            fpos = _osc_positions(model, at)
            for i, blk in enumerate(model.blocks):
                layer, h = blk.tension, blk.pre_norm(x)
                q, k, v = layer._qkv(h, t0)
                if blk.global_layer:
                    q, k, v = autocast_inputs(q, k, v)
                table, kv = rows[blk.global_layer], self._pages(i, k, v)
                before = t0 if blk.global_layer else min(t0, layer.window)
                kp, vp = paged_read(kv, table, start - before, before, (k.dtype, v.dtype))
                self._store(i, k, v, rows, start)
                q = torch.cat([q.new_zeros(1, before, *q.shape[2:]), q], 1)  # the rows before are not asked for
                k, v = torch.cat([kp, k], 1), torch.cat([vp, v], 1)
                if blk.global_layer:
                    out = global_tension(q, k, v, layer.scale)
                else:
                    out = causal_tension(q, k, v, layer.window, layer.scale,
                                         normalize="count" if layer.count_norm else "mass")
                h = layer.norm(h + layer.wo(out[:, before:].reshape(1, T, -1)))
                x = _after_tension(blk, h, fpos)
            logits = model.lm_head(model.final_norm(x[:, -1]))[0]
            self._advance([seq], [T], idx, start + T)
            return logits

    @torch.no_grad()
    def step(self, seqs: Sequence[int], next_ids: Tensor) -> Tensor:
        """Advance these sequences by one token each (ids [N]), every one at
        its own position; returns their logits [N, vocab]."""
        self._live(seqs)
        with self._room(seqs, [1] * len(seqs)):
            model, dev = self.model, self.lengths.device
            N = len(seqs)
            idx = torch.tensor(seqs, device=dev)
            rows = self._rows(idx)
            pos = self.lengths.index_select(0, idx)
            lengths, at = pos + 1, pos.long()
            most = max(self.length[s] for s in seqs) + 1

            def attend(i, blk, q, k, v):
                self._store(i, k[:, None], v[:, None], rows, pos)
                return _decode(blk, q, self._pages(i, k, v), rows[blk.global_layer], lengths, most)

            logits = _step_logits(model, next_ids.to(dev), at, attend)
            self._advance(seqs, [1] * N, idx, lengths)
            return logits


def _decode(blk, q: Tensor, kv: PagedKV, table: Tensor, lengths: Tensor, most: int) -> Tensor:
    """A layer's step over pages that hold the new tokens already."""
    layer = blk.tension
    if blk.global_layer:
        return paged_decode(q, kv, table, lengths, layer.scale, max_len=most)
    return paged_decode(q, kv, table, lengths, layer.scale, window=layer.window, include_self=False,
                        normalize="count" if layer.count_norm else "mass", max_len=most)


def _step_logits(model, ids: Tensor, at: Tensor, attend) -> Tensor:
    """One token per sequence through the model, ids [N] at positions at [N];
    attend(i, block, q, k, v) stores the token and gives its layer's output
    [N, H, HD].  Returns the logits [N, vocab]."""
    N = ids.numel()
    x = model.embedding(ids.view(N, 1))
    if model.pos_embedding is not None:
        x = x + model.pos_embedding(at)[:, None]
    fpos = _osc_positions(model, at)
    fpos = None if fpos is None else fpos[:, None]
    first = model.blocks[0].tension
    rot = None
    if first.rope_enabled:  # one row of the tables a sequence
        rot = (first.rope.cos.index_select(0, at), first.rope.sin.index_select(0, at))
    for i, blk in enumerate(model.blocks):
        layer, h = blk.tension, blk.pre_norm(x)
        out = attend(i, blk, *_step_qkv(layer, h, rot))
        h = layer.norm(h + layer.wo(out.reshape(N, 1, -1)).to(h.dtype))
        x = _after_tension(blk, h, fpos)
    return model.lm_head(model.final_norm(x))[:, 0]


def _step_qkv(layer, x: Tensor, rot):
    """q, k, v [N, H, HD] of one token per sequence, x [N, 1, D]; ``rot``: the
    RoPE (cos, sin) rows [N, HD / 2] of their positions."""
    N, H, HD = x.shape[0], layer.num_heads, layer.head_dim
    q = layer.wq(x).view(1, N, H, HD)
    if layer.rope_enabled:
        k, v = layer.wk(x).view(1, N, H, HD), layer.wv(x).view(1, N, H, HD)
        out = torch.promote_types(q.dtype, rot[0].dtype) if layer.rope.promote else None
        q, k = rope(q, *rot, out_dtype=out), rope(k, *rot, out_dtype=out)
    else:
        k, v = layer.wkv(x).view(1, N, H, 2 * HD).split(HD, dim=-1)
    q, k, v = q[0], k[0], v[0]
    return autocast_inputs(q, k, v) if layer.global_layer else (q, k, v)


@torch.no_grad()
def generate_batch(model, prompts: Sequence[Sequence[int]], max_new: int = 200, temp: float = 0.8, top_p: float = 0.92,
                   rep_penalty: float = 1.3, generator: Optional[torch.Generator] = None,
                   dtype: Optional[torch.dtype] = None, page_size: int = 64, device_tables: bool = False) -> list:
    """``generate_cached`` for several prompts of different lengths at once:
    each grows by ``max_new`` tokens, or to ``max_seq_len``.  ``dtype``: of the
    pages, e.g. ``torch.float8_e4m3fn`` or ``torch.float4_e2m1fn_x2``;
    ``device_tables``: as in ``TensionPagedCache``."""
    model.eval()
    limit = model.cfg.max_seq_len
    out = [list(p) for p in prompts]
    if any(not 1 <= len(p) <= limit for p in out):
        raise ValueError(f"prompts need 1 to max_seq_len {limit} tokens")
    if not out or max_new <= 0:
        return out
    end = [min(len(p) + max_new, limit) for p in out]
    pages = sum(-(-n // page_size) for n in end)
    cache = TensionPagedCache(model, len(out), pages, page_size=page_size, dtype=dtype, device_tables=device_tables)
    seqs, logits = cache.prefill([torch.tensor(p) for p in out])
    live = [i for i in range(len(out)) if len(out[i]) < end[i]]
    logits = logits[live]
    while live:
        new = [sample_next(row, out[i], temp, top_p, rep_penalty, generator) for i, row in zip(live, logits)]
        for i, t in zip(live, new):
            out[i].append(t)
        going = [j for j, i in enumerate(live) if len(out[i]) < end[i]]
        for i in set(live) - {live[j] for j in going}:
            cache.release(seqs[i])
        live = [live[j] for j in going]
        if live:
            logits = cache.step([seqs[i] for i in live], torch.tensor([new[j] for j in going]))
    return out


@torch.no_grad()
def beam_search(model, prompts: Sequence[Sequence[int]], beams: int = 4, max_new: int = 100, eos: Optional[int] = None,
                length_penalty: float = 0.0, dtype: Optional[torch.dtype] = None, page_size: int = 64) -> list:
    """The ``beams`` likeliest continuations of each prompt that a search of that
    width finds: for each prompt a list of (tokens, score), the best first.  The
    score is the continuation's log probability, over (its length)^length_penalty.

    A continuation ends with ``eos``, after ``max_new`` tokens, or where its
    sequence reaches ``max_seq_len``.  ``dtype``: of the cache's pages, as in
    ``TensionPagedCache``.  A prompt's full pages are its beams' together, what
    they add is their own; every layer keeps all its tokens.  Nothing comes back
    to the host before the search is done."""
    model.eval()
    limit, V = model.cfg.max_seq_len, model.cfg.vocab_size
    out = [list(p) for p in prompts]
    if any(not 1 <= len(p) <= limit for p in out):
        raise ValueError(f"prompts need 1 to max_seq_len {limit} tokens")
    if not 1 <= beams <= 64:
        raise ValueError(f"beams must be in [1, 64], got {beams}")
    if eos is not None and not 0 <= eos < V:
        raise ValueError(f"eos must be a token, got {eos}")
    N, B, S = len(out), beams, page_size
    room = [min(max_new, limit - len(p)) for p in out]  # tokens that each may grow by
    steps = max(room, default=0)
    if steps <= 0:
        return [[(p, 0.0)] for p in out]
    dev = next(model.parameters()).device
    start = torch.tensor([len(p) for p in out], dtype=torch.int32)
    width, longest = -(-limit // S), max(len(p) for p in out)
    # a prompt's full pages once, and for each beam those of what follows
    pages = sum(len(p) // S + B * (-(-(len(p) + r) // S) - len(p) // S) for p, r in zip(out, room))
    pool = PagePool.full(max(pages, 1), dev)
    table = torch.full((N * B, width), -1, dtype=torch.int32, device=dev)
    first = torch.arange(B) == 0  # holds the prompt; the others a page of their own for what comes next
    held = torch.where(first, 0, (start // S * S)[:, None])
    slots, _ = paged_plan(pool, table, held.flatten().int().to(dev), (start[:, None] - held).flatten().int().to(dev), S, longest)
    slots = slots.view(N, B, -1)[:, 0]
    layers: list = [None] * len(model.blocks)

    def store(i, k, v, where):
        if layers[i] is None:
            layers[i] = PagedKV.empty(len(pool.free), S, k.shape[2], k.shape[3], dtype or k.dtype, dtype or v.dtype, dev)
        paged_store(layers[i], k, v, where)

    ids = torch.zeros(N, longest, dtype=torch.long)
    for row, p in zip(ids, out):
        row[:len(p)] = torch.tensor(p)
    try:
        for i, b in enumerate(model.blocks):
            b.tension.kv_sink = (lambda k, v, i=i: store(i, k, v, slots))
        logits = model(ids.to(dev))
    finally:
        for b in model.blocks:
            b.tension.kv_sink = None
    lengths, limits = start.to(dev), torch.tensor(room, device=dev)[:, None]
    logits = logits[torch.arange(N, device=dev), lengths.long() - 1]
    logits = logits[:, None].expand(N, B, V)
    scores = torch.where(first, 0.0, -torch.inf).float().to(dev).expand(N, B).contiguous()
    ended = torch.zeros(N, B, dtype=torch.bool, device=dev)
    text = torch.zeros(N, B, steps, dtype=torch.long, device=dev)
    grown = torch.zeros(N, B, dtype=torch.long, device=dev)  # tokens of a beam, up to its end
    for t in range(steps):
        scores, tokens, parents = beam_select(logits, scores, ended=ended | (t >= limits), pad=eos or 0)
        ended, grown = ended.gather(1, parents), grown.gather(1, parents)
        grown += ~ended & (t < limits)
        text = text.gather(1, parents[..., None].expand_as(text))
        text[:, :, t] = tokens
        if eos is not None:
            ended = ended | (tokens == eos)
        if t == steps - 1:
            break
        table = paged_reorder(layers, table, lengths, parents)
        going = (t + 1 < limits[:, 0]).int()  # a prompt that has no room left stays where it is
        at = lengths.repeat_interleave(B)
        where, _ = paged_plan(pool, table, at, going.repeat_interleave(B), S, 1)
        after, most = at + 1, min(longest + t + 1, limit)

        def attend(i, blk, q, k, v):
            store(i, k[:, None], v[:, None], where)
            return _decode(blk, q, layers[i], table, after, most)

        logits = _step_logits(model, tokens.flatten(), at.long().clamp(max=limit - 1), attend).view(N, B, V)
        lengths = lengths + going
    text, grown, scores = text.tolist(), grown.tolist(), scores.tolist()
    res = []
    for p, rows, sizes, own in zip(out, text, grown, scores):
        found = [(p + row[:n], s / max(n, 1) ** length_penalty) for row, n, s in zip(rows, sizes, own) if s > -float("inf")]
        res.append(sorted(found, key=lambda x: -x[1]))
    return res
