"""What a paged cache does with calls that cannot run, on the CPU: sequence
numbers outside the cache are refused before anything changes."""
import pytest
import torch

from tests.test_paged_generation import cache


def state(c):
    """Everything a call could change on the host."""
    return [(t.rows.tolist(), sorted(t.free)) for t in c.tables.values()], list(c.length), c.lengths.tolist()


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
