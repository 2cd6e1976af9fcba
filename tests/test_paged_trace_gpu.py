"""Paged calls under torch.jit.trace: a replay runs them on its own inputs."""
import pytest
import torch

from bozo_amd import PagedKV, paged_append, paged_decode, paged_read
from tests.test_paged_gpu import DT, fill

pytestmark = pytest.mark.gpu


def parts(kv):
    return [t for t in kv if t is not None]


@pytest.mark.parametrize("pages", ["bf16", "e4m3"])
def test_traced_calls_replay(pages):
    """A step that appends, decodes and reads back, traced on one cache and
    replayed on another with other tokens, tables and lengths."""
    P, S, H, D, N = 6, 16, 2, 64, 2

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        kv = fill(PagedKV.empty(P, S, H, D, DT[pages]), seed)
        table = torch.randperm(P, generator=g, device="cuda").int().view(N, 3)
        pos = torch.tensor([20 + seed, 30], dtype=torch.int32, device="cuda")
        return (*(torch.randn(N, H, D, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3)), table, pos,
                *parts(kv))

    def step(q, k, v, table, pos, *kv):
        kv = PagedKV(*kv)
        paged_append(kv, k[:, None], v[:, None], table, pos)
        out = paged_decode(q, kv, table, pos + 1, 8.0, window=24, include_self=False, max_len=48)
        return (out, *paged_read(kv, table, pos - 3, 4))

    traced = torch.jit.trace(step, inputs(1), check_trace=False)
    for seed in (2, 3, 4):
        a, b = inputs(seed), inputs(seed)
        for x, y in zip(traced(*a), step(*b)):
            assert torch.equal(x, y)
        for x, y in zip(a, b):  # the pages among them
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_traced_append_alone_writes():
    """Nothing uses an append's result: the trace keeps it all the same."""
    tab = torch.zeros(1, 1, dtype=torch.int32, device="cuda")

    def put(x, k, v):
        paged_append(PagedKV(k, v), x, x, tab, tab[0])
        return x

    x = torch.ones(1, 2, 2, 64, device="cuda")
    pages = [torch.zeros(1, 2, 16, 64, device="cuda") for _ in range(4)]
    traced = torch.jit.trace(put, (x, *pages[:2]), check_trace=False)
    traced(5 * x, *pages[2:])
    assert all((t[:, :, :2] == 5).all() and not t[:, :, 2:].any() for t in pages[2:])


def test_refused_while_tracing():
    kv = fill(PagedKV.empty(2, 16, 2, 64, torch.bfloat16), 1)
    tab = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 3, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiple"):
        torch.jit.trace(lambda q: paged_decode(q, kv, tab, tab[0], 8.0), (q,), check_trace=False)
