"""The ring caches' decode step under torch.jit.trace: a replay runs it on its
own inputs and writes its own caches."""
import pytest
import torch

from bozo_amd import decode_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("extra", [False, True])
def test_traced_step_replays(dev, extra):
    N, H, W, D = 2, 3, 8, 64

    def inputs(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        rows = [torch.randn(N, H, D, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(3)]
        rings = [torch.randn(N, H, W, D, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2)]
        pos = torch.tensor([3 + seed, 20], dtype=torch.int32, device=dev)
        return (*rows, *rings, pos, torch.zeros_like(pos), torch.zeros(N, H, W, device=dev, dtype=torch.bfloat16))

    def step(q, k, v, kc, vc, pos, nxt, tau):
        return decode_step(q, k, v, kc, vc, pos, nxt if extra else None, 8.0, "mass", tau if extra else None)

    traced = torch.jit.trace(step, inputs(1), check_trace=False)
    for seed in (2, 3, 4):
        a, b = inputs(seed), inputs(seed)
        assert torch.equal(traced(*a), step(*b))
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_refused_while_tracing(dev):
    x = torch.zeros(2, 3, 64, device=dev)
    ring = torch.zeros(2, 3, 8, 64, device=dev)
    pos = torch.zeros(2, dtype=torch.int64, device=dev)
    with pytest.raises(TypeError, match="int32"):
        torch.jit.trace(lambda q: decode_step(q, q, q, ring, ring, pos, None, 8.0), (x,), check_trace=False)
