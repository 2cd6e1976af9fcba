"""Generation for sequences of different lengths over paged caches.

``TensionKVCache`` (``generation.py``) advances N sequences in lock step, each
with room for ``max_seq_len`` tokens.  Here sequences come and go, each at its
own position, and own the pages that their tokens fill: ``paged_append``
stores prompts and new tokens (quantised to e4m3 if asked), ``paged_decode``
advances one token each, and ``paged_read`` gives a prompt that continues on
cached tokens the keys and values before it.

All layers of one kind share page numbers (each layer has its own pages of
that number): a global layer keeps every token, a local one the pages of its
last W, which go back to the pool as the window leaves them.

The reference keeps no cache (model.py:736-739); a step equals its forward's
last row (model.py:617-652) as long as a sequence fits ``max_seq_len``, up to
the rounding of the pages' type.
"""
from __future__ import annotations

from contextlib import contextmanager
from typing import Optional, Sequence

import torch
from torch import Tensor

from .generation import _after_tension, _osc_positions, sample_next
from .ops import autocast_inputs, causal_tension, global_tension, rope
from .paged import PagedKV, paged_append, paged_decode, paged_read


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


class TensionPagedCache:
    """Paged K/V caches of up to ``sequences`` sequences of one model.

    pages: of each global layer; local_pages: of each local layer (default:
    what ``sequences`` windows fill, and one more for ``extend``).  dtype: the pages' type, e.g.
    ``torch.float8_e4m3fn`` (default: as the layers compute their keys and
    values).  The model must be in eval mode (dropout off)."""

    def __init__(self, model, sequences: int, pages: int, local_pages: Optional[int] = None, page_size: int = 64,
                 dtype: Optional[torch.dtype] = None):
        cfg = model.cfg
        self.model, self.dtype = model, dtype
        device = next(model.parameters()).device
        window = min(-(-cfg.window // page_size) + 1, -(-cfg.max_seq_len // page_size))
        local = (sequences + 1) * window if local_pages is None else local_pages
        self.tables = {True: PageTable(pages, page_size, sequences, cfg.max_seq_len),
                       False: PageTable(local, page_size, sequences, cfg.max_seq_len, cfg.window)}
        if not any(b.global_layer for b in model.blocks):
            del self.tables[True]
        if all(b.global_layer for b in model.blocks):
            del self.tables[False]
        self.layers: list[Optional[PagedKV]] = [None] * len(model.blocks)
        self.length = [0] * sequences  # tokens cached; 0: not in use
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self._device_rows = {g: t.rows.to(device) for g, t in self.tables.items()}

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
        for t in self.tables.values():
            if sum(t.missing(s, self.length[s], m) for s, m in zip(seqs, more)) > len(t.free):
                raise RuntimeError(f"out of pages ({t.pages} in the pool): release a sequence, or wait for one to end")
        taken = [(t, s, t.grow(s, self.length[s], m)) for t in self.tables.values() for s, m in zip(seqs, more)]
        try:
            yield
        except BaseException:
            for t, s, entries in reversed(taken):
                t.give(s, reversed(entries))
            raise

    def _rows(self, idx: Tensor) -> dict:
        """The tables' rows of these sequences, on the device."""
        for g, t in self.tables.items():
            if t.changed:
                self._device_rows[g].copy_(t.rows)
                t.changed = False
        return {g: r.index_select(0, idx) for g, r in self._device_rows.items()}

    def _advance(self, seqs: Sequence[int], more: Sequence[int], idx: Tensor, lengths: Tensor) -> None:
        self.lengths.index_copy_(0, idx, lengths)
        for s, m in zip(seqs, more):
            self.length[s] += m
            for t in self.tables.values():
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
            t.release(seq)
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

            def store(i, k, v):
                paged_append(self._pages(i, k, v), k, v, rows[self.model.blocks[i].global_layer], start, n)

            layers = [b.tension for b in self.model.blocks]
            for i, layer in enumerate(layers):
                layer.kv_sink = (lambda k, v, i=i: store(i, k, v))
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
                paged_append(kv, k, v, table, start)
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
            x = model.embedding(next_ids.to(dev).view(N, 1))
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
                q, k, v = _step_qkv(layer, h, rot)
                kv, table = self._pages(i, k, v), rows[blk.global_layer]
                paged_append(kv, k[:, None], v[:, None], table, pos)
                if blk.global_layer:
                    out = paged_decode(q, kv, table, lengths, layer.scale, max_len=most)
                else:
                    out = paged_decode(q, kv, table, lengths, layer.scale, window=layer.window, include_self=False,
                                       normalize="count" if layer.count_norm else "mass", max_len=most)
                h = layer.norm(h + layer.wo(out.reshape(N, 1, -1)).to(h.dtype))
                x = _after_tension(blk, h, fpos)
            logits = model.lm_head(model.final_norm(x))[:, 0]
            self._advance(seqs, [1] * N, idx, lengths)
            return logits


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
                   dtype: Optional[torch.dtype] = None, page_size: int = 64) -> list:
    """``generate_cached`` for several prompts of different lengths at once:
    each grows by ``max_new`` tokens, or to ``max_seq_len``.  ``dtype``: of the
    pages, e.g. ``torch.float8_e4m3fn``."""
    model.eval()
    limit = model.cfg.max_seq_len
    out = [list(p) for p in prompts]
    if any(not 1 <= len(p) <= limit for p in out):
        raise ValueError(f"prompts need 1 to max_seq_len {limit} tokens")
    if not out or max_new <= 0:
        return out
    end = [min(len(p) + max_new, limit) for p in out]
    pages = sum(-(-n // page_size) for n in end)
    cache = TensionPagedCache(model, len(out), pages, page_size=page_size, dtype=dtype)
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
