"""What a paged cache does with calls that cannot run, on the CPU: sequence
numbers outside the cache are refused before anything changes, and a call that
fails on its way gives back the pages it took."""
import pytest
import torch

from bozo_amd import model as M
from bozo_amd import paged_generation as G
from tests.test_paged_generation import cache


def state(c):
    """Everything a call could change on the host."""
    return [(t.rows.tolist(), t.free[:]) for t in c.tables.values()], list(c.length), c.lengths.tolist()


@pytest.mark.parametrize("seqs", [[-1], [3], [2, -1], [0, 3], [-3], [1 << 40]])
def test_numbers_outside_the_cache(seqs):
    c = cache()
    c.length = [3, 3, 3]
    before = state(c)
    with pytest.raises(ValueError, match="no sequence"):
        c.step(seqs, torch.zeros(len(seqs), dtype=torch.long))
    for s in seqs:
        if not 0 <= s < 3:
            with pytest.raises(ValueError, match="no sequence"):
                c.extend(s, torch.tensor([1]))
            with pytest.raises(ValueError, match="no sequence"):
                c.release(s)
    assert state(c) == before


def ids(*lengths):
    return [torch.ones(n, dtype=torch.long) for n in lengths]


@pytest.mark.parametrize("prompts", [ids(20), ids(3, 9, 1), [torch.ones(4, 4, dtype=torch.long), *ids(5)]],
                         ids=["one", "three", "matrix"])
def test_prefill_that_fails_gives_its_pages_back(prompts):
    """No prompt runs here: the kernels need a GPU (and a matrix is no prompt)."""
    c = cache()
    before = state(c)
    for _ in range(3):
        with pytest.raises(RuntimeError):
            c.prefill(prompts)
        assert state(c) == before
    assert all(b.tension.kv_sink is None for b in c.model.blocks)


def test_a_turn_and_a_step_that_fail_give_their_pages_back(monkeypatch):
    c = cache()
    for t in c.tables.values():
        t.grow(1, 0, 7)
    c.length[1] = 7
    c.lengths[1] = 7
    before = state(c)
    for call in (lambda: c.extend(1, torch.ones(9, dtype=torch.long)), lambda: c.step([1], torch.ones(1, dtype=torch.long)),
                 lambda: c.step([1], torch.ones(2, dtype=torch.long))):  # two tokens for one sequence
        with pytest.raises(RuntimeError):
            call()
        assert state(c) == before
    c.release(1)
    assert all(len(t.free) == t.pages for t in c.tables.values())


class Stop(BaseException):
    """An interruption, not an error."""


@pytest.mark.parametrize("error", [RuntimeError, Stop])
@pytest.mark.parametrize("where", ["embedding", "lm_head"])
def test_failures_on_either_side_of_the_layers(monkeypatch, error, where):
    """The logits' projection fails behind the last layer: the sequence has
    not advanced and the same call runs afterwards."""
    cfg = M.TensionConfig(vocab_size=32, dim=64, num_layers=2, num_heads=2, window=6, max_seq_len=24, dropout=0.0,
                          global_every=2, use_rope=False)
    c = G.TensionPagedCache(M.TensionLM(cfg).eval(), sequences=3, pages=8, page_size=4)
    monkeypatch.setattr(G, "paged_append", lambda *a: None)
    monkeypatch.setattr(G, "paged_read", lambda kv, table, start, T, dt: (
        torch.zeros(1, T, 2, 32, dtype=dt[0]), torch.zeros(1, T, 2, 32, dtype=dt[1])))
    monkeypatch.setattr(G, "paged_decode", lambda q, *a, **kw: torch.zeros_like(q))
    monkeypatch.setattr(G, "global_tension", lambda q, *a: torch.zeros_like(q))
    monkeypatch.setattr(G, "causal_tension", lambda q, *a, **kw: torch.zeros_like(q))
    for t in c.tables.values():
        t.grow(1, 0, 8)
        t.drop(1, 8)
    c.length[1] = 8
    c.lengths[1] = 8
    before = state(c)
    module = getattr(c.model, where)

    def fail(*a):
        raise error("no memory")

    for call, more in ((lambda: c.extend(1, torch.ones(9, dtype=torch.long)), 9),
                       (lambda: c.step([1], torch.ones(1, dtype=torch.long)), 1)):
        with monkeypatch.context() as m:
            m.setattr(module, "forward", fail)
            with pytest.raises(error):
                call()
        assert state(c) == before
        call()
        assert c.length[1] == 8 + more and c.lengths.tolist()[1] == 8 + more
        c.release(1)
        assert all(len(t.free) == t.pages for t in c.tables.values())
        for t in c.tables.values():
            t.grow(1, 0, 8)
            t.drop(1, 8)
        c.length[1], c.lengths[1] = 8, 8
        before = state(c)
    if where == "embedding":  # a prompt's forward that fails
        empty = G.TensionPagedCache(c.model, sequences=3, pages=8, page_size=4)
        before = state(empty)
        monkeypatch.setattr(module, "forward", fail)
        with pytest.raises(error):
            empty.prefill(ids(5, 9))
        assert state(empty) == before
