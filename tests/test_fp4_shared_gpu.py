"""4-bit decode of shared key heads where query heads (times splits) outnumber
the card's units, which the matrix units take: queries that are broken or below
the normal numbers, the smallest and largest scales, pages far apart, long rows,
graphs and streams, against the 64-bit oracle."""
import numpy as np
import pytest
import torch

from bozo_amd import PagedKV, paged_append, paged_decode
from oracle import paged_ref as P_
from tests.test_fp4_gpu import F4, both, check_decode, fill
from tests.test_paged_gpu import DT, dev, make_table, np64

pytestmark = pytest.mark.gpu


def batch(H, most, S=16, seed=0):
    """Sequences whose query heads are more than the card's units, and their table."""
    N = torch.cuda.get_device_properties(0).multi_processor_count // H + 1
    lengths = [1 + most * n // N for n in range(N)]
    table, P = make_table(lengths, S, seed=seed)
    return N, lengths, table, P


def queries(N, H, D, flow, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(N, H, D, generator=g, device="cuda").to(DT[flow])


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("flow", ["bf16", "f16", "f32"])
def test_broken_queries(D, flow):
    """A NaN in a query makes its own row NaN and no other; a query of zeros weighs all keys alike."""
    N, lengths, table, P = batch(8, 60)
    kv = fill(PagedKV.empty(P, 16, 2, D, F4), 7)
    q = queries(N, 8, D, flow)
    for n in range(N):
        q[n, n % 8, (n * 7) % D] = float("nan")
        q[n, (n + 3) % 8] = 0.0
    out = check_decode(q, kv, table, lengths, 8.0)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[torch.arange(N), torch.arange(N) % 8] = True
    assert torch.equal(out.isnan(), bad)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("flow", ["bf16", "f16", "f32"])
def test_infinite_queries(D, flow):
    """An infinite value weighs keys by the sign of theirs (1 or 0); a key that has a zero there makes the row NaN."""
    N, lengths, table, P = batch(8, 60)
    kv = fill(PagedKV.empty(P, 16, 2, D, F4), 8)
    codes = kv.k.view(torch.uint8)
    at = D // 2 + 2  # an even value: the low half of its byte
    byte = codes[..., at // 2]
    byte |= ((byte & 7) == 0).to(torch.uint8)  # no zeros there
    q = queries(N, 8, D, flow)
    q[:, 1::2] = 0.0
    q[:, 1::2, at] = torch.where(torch.arange(N, device="cuda") % 2 == 0, float("inf"), -float("inf"))[:, None].to(q.dtype)
    big = np64(q)
    big[:, 1::2, at] = np.where(np.arange(N) % 2 == 0, 1e300, -1e300)[:, None]
    out = paged_decode(q, kv, dev(table), dev(np.asarray(lengths, np.int32)), 8.0)
    ref, keys, mag, dots = P_.decode(big, *both(kv), table, lengths, 8.0)
    dots[:, 1::2] = 0.0  # their weights have no rounding
    bound = P_.decode_bound(ref, keys, mag, dots, D, torch.finfo(q.dtype).eps) + (2.0 ** -25 if flow == "f16" else 0.0)
    assert (np.abs(np64(out) - ref) <= bound).all()
    # the last key of every sequence: a zero for one key head
    for n, length in enumerate(lengths):
        codes[table[n, (length - 1) // 16], 0, (length - 1) % 16, at // 2] &= 0xf0
    out = paged_decode(q, kv, dev(table), dev(np.asarray(lengths, np.int32)), 8.0)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, 1:4:2] = True
    assert torch.equal(out.isnan(), bad)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("flow,size,lo,hi", [("f16", 2.0 ** -18, 142, 146), ("f16", 2.0 ** -24, 148, 150), ("f32", 2.0 ** -120, 243, 247),
                                             ("bf16", 2.0 ** -120, 243, 247)])
def test_small_queries(D, flow, size, lo, hi):
    """Queries at the bottom of their type's range (f16: below its normal numbers), against keys as large."""
    N, lengths, table, P = batch(8, 60)
    kv = fill(PagedKV.empty(P, 16, 2, D, F4), 9, lo, hi)
    kv.v_exp.fill_(127)
    q = (queries(N, 8, D, "f32") * size).to(DT[flow])
    check_decode(q, kv, table, lengths, 8.0)


@pytest.mark.parametrize("flow", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lo,hi", [(0, 1), (1, 3), (250, 253)])
def test_extreme_scales(lo, hi, flow):
    """The smallest and largest scales that storing gives: nothing is NaN, keys of one sign decide tau."""
    N, lengths, table, P = batch(8, 60)
    kv = fill(PagedKV.empty(P, 16, 2, 64, F4), 6, lo, hi)
    kv.v_exp.fill_(127)
    q = queries(N, 8, 64, flow)
    if lo < 100:
        check_decode(q, kv, table, lengths, 8.0)
        kv.k_exp.random_(120, 128)
        kv.v_exp.fill_(lo)
        check_decode(q.float(), kv, table, lengths, 8.0)
        return
    kv.k.view(torch.uint8).random_(0, 256).bitwise_and_(0x77).bitwise_or_(0x11)
    out = paged_decode(q.abs(), kv, dev(table), dev(np.asarray(lengths, np.int32)), 8.0)
    ref, keys, mag, _ = P_.decode(np.full(q.shape, 1e30), *both(kv), table, lengths, 8.0)  # tau 1 for every key
    bound = P_.decode_bound(ref, keys, mag, np.zeros(q.shape[:2]), 64, torch.finfo(q.dtype).eps) + 2.0 ** -25
    assert (np.abs(np64(out) - ref) <= bound).all()


@pytest.mark.parametrize("D", [64, 96])
def test_pages_beyond_32_bits(D):
    """Pages 2^32 bytes and more from the first: the same rows as from pages side by side."""
    H, Hk, S, P = 8, 2, 16, 70
    N = torch.cuda.get_device_properties(0).multi_processor_count // H + 1
    raw = torch.zeros(P << 26, dtype=torch.uint8, device="cuda")
    shape, strides = (P, Hk, S, D // 2), (1 << 26, S * D // 2, D // 2, 1)
    k, v = (x.as_strided(shape, strides).view(F4) for x in (raw, raw[1 << 20:]))
    e = torch.zeros(2, P, Hk, S, D // 32, dtype=torch.uint8, device="cuda")
    kv, small = PagedKV(k, v, e[0], e[1]), PagedKV.empty(3, S, Hk, D, F4)
    x = torch.randn(1, 48, Hk, D, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    far, near = (torch.tensor([t], dtype=torch.int32, device="cuda") for t in ([69, 2, 66], [0, 1, 2]))
    for c, t in ((kv, far), (small, near)):
        paged_append(c, x, 2 * x, t, torch.zeros(1, dtype=torch.int32, device="cuda"))
    lengths = (torch.arange(N, dtype=torch.int32, device="cuda") * 7) % 49
    q = queries(N, H, D, "bf16")
    assert torch.equal(paged_decode(q, kv, far.expand(N, 3), lengths, 8.0), paged_decode(q, small, near.expand(N, 3), lengths, 8.0))


@pytest.mark.parametrize("D,H,Hk", [(32, 16, 2), (64, 20, 1), (96, 16, 4), (128, 24, 2)])
@pytest.mark.parametrize("flow", ["bf16", "f16", "f32"])
def test_long_rows_in_splits(D, H, Hk, flow):
    """Few sequences of many keys, one of them short: split, and joined."""
    lengths = [6000, 37]
    table, P = make_table(lengths, 16, seed=D)
    table[0, 100:140] = -1
    kv = fill(PagedKV.empty(P, 16, Hk, D, F4), D)
    check_decode(queries(2, H, D, flow), kv, table, lengths, D ** 0.5)


def test_captured_and_on_another_stream():
    """A captured append and decode, replayed with eager work between; the eager calls on a stream of their own."""
    H, Hk, D, S = 16, 4, 64, 16
    N = torch.cuda.get_device_properties(0).multi_processor_count // H + 1
    kv, ref = (fill(PagedKV.empty(3 * N, S, Hk, D, F4), 1) for _ in range(2))
    table = torch.randperm(3 * N, generator=torch.Generator().manual_seed(0)).int().view(N, 3).cuda()
    x = torch.zeros(2, N, 1, Hk, D, device="cuda", dtype=torch.bfloat16)
    q = torch.zeros(N, H, D, device="cuda", dtype=torch.bfloat16)
    pos = (torch.arange(N, dtype=torch.int32, device="cuda") * 5) % 40

    def step(kv):
        paged_append(kv, x[0], x[1], table, pos)
        return paged_decode(q, kv, table, pos + 1, 8.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kv)
    torch.cuda.current_stream().wait_stream(side)
    step(ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(kv)
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        x.copy_(torch.randn(x.shape, generator=g))
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = step(ref)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        pos += 1
