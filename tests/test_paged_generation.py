"""Page numbers of the paged caches, on the CPU: what a sequence holds as it
grows, what its window leaves, and what is refused before anything changes."""
import random

import pytest
import torch

from bozo_amd import model as M
from bozo_amd.paged_generation import PageTable, TensionPagedCache


def held(t, seq):
    return [int(x) for x in t.rows[seq] if x >= 0]


@pytest.mark.parametrize("S,window", [(1, 0), (4, 0), (4, 1), (4, 4), (4, 6), (16, 6), (3, 7)])
def test_pages_cover_what_is_read(S, window):
    """Every position that the next token reads has a page, no page has two
    owners, and nothing is lost over many sequences."""
    r = random.Random(S * 100 + window)
    t = PageTable(400, S, 5, 60, window)
    length = [0] * 5
    for _ in range(400):
        s = r.randrange(5)
        if length[s] and r.random() < 0.1:
            t.release(s)
            length[s] = 0
            assert not held(t, s)
            continue
        more = min(r.choice([1, 1, 1, 2, 9, 30]), 60 - length[s])
        if more < 1:
            continue
        before, need = len(t.free), t.missing(s, length[s], more)
        t.grow(s, length[s], more)
        assert before - len(t.free) == need
        end = length[s] + more
        low = max(0, end - window) if window else 0
        kept = range(max(low, length[s]), end)  # stored tokens that are still read
        assert all(t.rows[s, p // S] >= 0 for p in kept)
        t.drop(s, end)
        length[s] = end
        assert all(t.rows[s, p // S] >= 0 for p in range(low, end))
        if window:
            assert len(held(t, s)) <= -(-window // S) + 1
        owned = [x for q in range(5) for x in held(t, q)]
        assert sorted(owned + t.free) == list(range(400))


def cache(**kw):
    cfg = M.TensionConfig(vocab_size=32, dim=64, num_layers=2, num_heads=2, window=6, max_seq_len=24, dropout=0.0,
                          global_every=2, use_rope=True)
    return TensionPagedCache(M.TensionLM(cfg).eval(), **{**dict(sequences=3, pages=8, page_size=4), **kw})


def test_refusals_change_nothing():
    c = cache()
    before = {g: (t.rows.clone(), list(t.free)) for g, t in c.tables.items()}
    with pytest.raises(ValueError, match="not in use"):
        c.step([0], torch.tensor([1]))
    with pytest.raises(ValueError, match="not in use"):
        c.extend(1, torch.tensor([1]))
    with pytest.raises(ValueError, match="not in use"):
        c.release(2)
    with pytest.raises(ValueError, match="max_seq_len"):
        c.prefill([torch.zeros(25, dtype=torch.long)])
    with pytest.raises(ValueError, match="outside"):
        c.prefill([torch.zeros(0, dtype=torch.long)])
    with pytest.raises(RuntimeError, match="free sequences"):
        c.prefill([torch.zeros(2, dtype=torch.long)] * 4)
    with pytest.raises(RuntimeError, match="out of pages"):
        c.prefill([torch.zeros(20, dtype=torch.long)] * 2)  # 10 of 8 global pages
    c.length[0] = 3
    with pytest.raises(ValueError, match="twice"):
        c.step([0, 0], torch.tensor([1, 2]))
    c.model.train()
    with pytest.raises(RuntimeError, match="eval"):
        c.step([0], torch.tensor([1]))
    for g, t in c.tables.items():
        assert torch.equal(t.rows, before[g][0]) and t.free == before[g][1]


def test_local_only_and_global_only():
    base = dict(vocab_size=32, dim=64, num_layers=2, num_heads=2, window=6, max_seq_len=24, dropout=0.0)
    a = TensionPagedCache(M.TensionLM(M.TensionConfig(**base)).eval(), 2, 4, page_size=4)
    b = TensionPagedCache(M.TensionLM(M.TensionConfig(global_every=1, **base)).eval(), 2, 4, page_size=4)
    assert list(a.tables) == [False] and list(b.tables) == [True]
    assert a.tables[False].pages == 3 * 3
