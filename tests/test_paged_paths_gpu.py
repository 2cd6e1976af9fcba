"""Paged decode, append and read on every way a call can take: wave counts,
vector and matrix kernels, splits, head dims in eights and odd ones, strides of
keys and values that differ, rows that hold infinities and NaN.  Against the
64-bit oracle, to its counted bound (oracle/paged_ref.py)."""
import math

import numpy as np
import pytest
import torch

from bozo_amd import PagedKV, paged_append, paged_decode, paged_read
from oracle import paged_ref as R
from tests.test_paged_gpu import DT, F8, check_decode, dev, fill, make_table, np64, run_decode, values

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16", "bf16"), ("bf16", "e4m3", "e4m3"), ("f16", "f16", "f16"), ("f32", "f32", "f32"),
         ("f32", "f32", "bf16"), ("f16", "e4m3", "e4m3"), ("f32", "e4m3", "e4m3")]


def query(N, H, D, dtype, seed=3):
    return torch.randn(N, H, D, generator=torch.Generator().manual_seed(seed)).to(DT[dtype]).cuda()


def ragged(N, top):
    return [max(1, top - (top * 3 // 4) * i // max(1, N - 1)) for i in range(N)]


@pytest.mark.parametrize("flow", TYPES, ids="-".join)
@pytest.mark.parametrize("N,H,L,window", [
    (66, 12, 200, 64),    # short windows in many rows: two waves
    (66, 12, 200, 7),
    (30, 12, 300, None),  # more rows than CUs: four
    (9, 4, 61, None),     # few rows, few keys: four
    (7, 3, 100, None),    # few rows: eight
    (33, 8, 2100, None),  # long rows in more workgroups than CUs: eight
])
def test_rows_by_waves(flow, N, H, L, window):
    lengths = ragged(N, L)
    table, P = make_table(lengths, 16, seed=N + L)
    kv = fill(PagedKV.empty(P, 16, H, 64, DT[flow[1]], DT[flow[2]]), L)
    check_decode(query(N, H, 64, flow[0]), kv, table, lengths, 8.0, window, window is None, max_len=L)


@pytest.mark.parametrize("q,pages", [("bf16", "bf16"), ("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e4m3"), ("f16", "f16"),
                                     ("f32", "f32")])
@pytest.mark.parametrize("D,S,Hk,share", [(64, 16, 2, 2), (64, 48, 1, 3), (128, 16, 2, 4), (64, 32, 1, 16), (128, 64, 1, 17),
                                          (64, 8, 2, 5), (96, 16, 1, 6), (256, 16, 1, 4)])
def test_shared_heads(q, pages, D, S, Hk, share):
    lengths = [0, 1, 2, 15, 16, 17, 33, 47, 100, 321]
    table, P = make_table(lengths, S, seed=share)
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), D + share)
    x = query(len(lengths), Hk * share, D, q)
    check_decode(x, kv, table, lengths, math.sqrt(D))
    check_decode(x, kv, table, lengths, math.sqrt(D), 18, False, "count")
    check_decode(x, kv, table, lengths, math.sqrt(D), 100, True, None)


@pytest.mark.parametrize("q,pages,D", [("bf16", "bf16", 64), ("bf16", "bf16", 128), ("bf16", "e4m3", 64), ("f16", "e4m3", 128),
                                       ("f32", "f32", 64)])
def test_shared_heads_many_rows(q, pages, D):
    """More workgroups than CUs, and long rows split over them."""
    lengths = ragged(70, 150)
    table, P = make_table(lengths, 16, seed=5)
    kv = fill(PagedKV.empty(P, 16, 4, D, DT[pages]), 6)
    check_decode(query(70, 8, D, q), kv, table, lengths, math.sqrt(D))
    lengths = [5003, 1777]
    table, P = make_table(lengths, 32, seed=7)
    kv = fill(PagedKV.empty(P, 32, 2, D, DT[pages]), 8)
    a = check_decode(query(2, 6, D, q), kv, table, lengths, math.sqrt(D))
    assert torch.equal(a, run_decode(query(2, 6, D, q), kv, table, lengths, math.sqrt(D)))


@pytest.mark.parametrize("flow", [("bf16", "bf16"), ("bf16", "e4m3"), ("f32", "f32"), ("f16", "e4m3")], ids="-".join)
@pytest.mark.parametrize("D,S,L", [(20, 16, 3001), (40, 16, 2500), (128, 12, 3500), (256, 5, 2100), (32, 64, 4000), (200, 16, 1500)])
def test_long_rows_any_head_dim(flow, D, S, L):
    lengths = [L, L // 3]
    table, P = make_table(lengths, S, seed=L)
    kv = fill(PagedKV.empty(P, S, 1, D, DT[flow[1]]), D)
    check_decode(query(2, 2, D, flow[0]), kv, table, lengths, math.sqrt(D))


@pytest.mark.parametrize("src,pages", [("bf16", "e4m3"), ("f32", "e4m3"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("D", [8, 24, 40, 56, 72, 80, 96, 120, 136, 200, 248, 264])
def test_rows_head_dims_in_eights(src, pages, D):
    """Append, read and decode where a row's lanes are not a power of two."""
    S, Hk, N, T = 16, 3, 2, 37
    start = np.array([3, 11], np.int32)
    lengths = [int(s) + T for s in start]
    table, P = make_table(lengths, S)
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 1)
    new = torch.randn(2, N, T, Hk, D, generator=torch.Generator().manual_seed(D))
    new = (new * torch.exp2(torch.randint(-6, 7, (2, N, T, Hk, 1), generator=torch.Generator().manual_seed(1)).float()))
    new = new.to(DT[src]).cuda()
    want = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    paged_append(kv, new[0], new[1], dev(table), dev(start))
    for w, x in zip(want, new):
        R.append(w, R.quantise(np64(x))[0] if pages == "e4m3" else np64(x.to(DT[pages])), table, start, [T] * N)
    assert np.array_equal(values(kv.k, kv.k_exp), want[0]) and np.array_equal(values(kv.v, kv.v_exp), want[1])
    for t in (torch.float32, torch.bfloat16 if pages != "f16" else torch.float16):
        for w, x in zip(want, paged_read(kv, dev(table), dev(start), T, t)):
            assert torch.equal(x.cpu(), torch.from_numpy(R.read(w, table, start, [T] * N, T)).to(t))
    if D <= 256:
        q = query(N, Hk, D, "f32" if pages == "f32" else "f16" if pages == "f16" else "bf16")
        check_decode(q * 0.1, fill(kv, 2), table, lengths, math.sqrt(D))


@pytest.mark.parametrize("q,pages,share", [("bf16", "bf16", 1), ("bf16", "e4m3", 1), ("f32", "f32", 1), ("bf16", "e4m3", 4),
                                           ("f32", "f32", 2)])
@pytest.mark.parametrize("N,Hk", [(65, 4), (64, 5), (256, 2), (200, 2), (257, 2), (3, 100), (2, 300)])
def test_sequences_taken_by_length(q, pages, share, N, Hk):
    """Large calls take the longest sequences first: every one once, whatever
    its length (empty, below zero, alike, past the bound that shapes the call)."""
    g = np.random.default_rng(N)
    lengths = g.choice([0, 1, 2, 3, 17, 40, 90, 130, 131], N)
    lengths[g.integers(N)] = 400
    table, P = make_table(lengths.tolist(), 16, seed=N, width=60000)
    kv = fill(PagedKV.empty(P, 16, Hk, 64, DT[pages]), N)
    x = query(N, Hk * share, 64, q)
    check_decode(x, kv, table, lengths, 8.0, max_len=20000)
    check_decode(x, kv, table, lengths, 8.0, max_len=300000, norm="count")
    lengths[g.integers(N)] = -5
    check_decode(x, kv, table, lengths, 8.0)


@pytest.mark.parametrize("pages,q,share", [("bf16", "bf16", 1), ("bf16", "bf16", 4), ("e4m3", "bf16", 1), ("e4m3", "f16", 2),
                                           ("f32", "f32", 1), ("f16", "f16", 2)])
def test_values_in_another_order(pages, q, share):
    """Keys head-major, values token-major with room between the rows, their
    exponents in yet another order; queries that start at odd places."""
    lengths, S, Hk, D = [37, 200, 5], 16, 2, 64
    table, P = make_table(lengths, S, seed=17)
    a = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 19)
    raw = a.v.view(torch.uint8) if pages == "e4m3" else a.v
    v = torch.empty(P, S, Hk, D + 16, dtype=raw.dtype, device="cuda").transpose(1, 2)[..., :D]
    v.copy_(raw)
    ve = a.v_exp
    if ve is not None:
        ve = torch.empty(Hk, P, S, dtype=torch.uint8, device="cuda").transpose(0, 1)
        ve.copy_(a.v_exp)
    kv = PagedKV(a.k, v.view(a.v.dtype) if pages == "e4m3" else v, a.k_exp, ve)
    x = torch.randn(3, Hk * share, 2 * D + 1, generator=torch.Generator().manual_seed(9)).to(DT[q]).cuda()
    for at in (0, 1, 4):
        check_decode(x[..., at:at + D], kv, table, lengths, 8.0)
    new = torch.randn(3, 20, Hk, D, generator=torch.Generator().manual_seed(4)).to(DT[q]).cuda()
    start = np.array([3, 50, 0], np.int32)
    want = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    paged_append(kv, new, -new, dev(table), dev(start))
    for w, y in zip(want, (new, -new)):
        R.append(w, R.quantise(np64(y))[0] if pages == "e4m3" else np64(y), table, start, [20] * 3)
    assert np.array_equal(values(kv.k, kv.k_exp), want[0]) and np.array_equal(values(kv.v, kv.v_exp), want[1])


@pytest.mark.parametrize("pages,q,share,D", [("bf16", "bf16", 1, 64), ("e4m3", "bf16", 1, 64), ("f32", "f32", 1, 64),
                                             ("f16", "f16", 1, 32), ("bf16", "bf16", 3, 128), ("e4m3", "f16", 4, 128),
                                             ("f32", "f32", 4, 128), ("bf16", "bf16", 1, 20)])
def test_reads_its_keys_only(pages, q, share, D):
    """NaN in every row that is not attended to: past the end, before the
    window, and in the pages that entries outside the pool might be taken for."""
    S, Hk, W = 16, 2, 48
    lengths = [1, 70, 100, 130, 0, 17]
    table, P = make_table(lengths, S, seed=11, width=40)
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 13)
    table[2, 100 // S - 1] = P
    table[3, 60 // S:70 // S] = -1
    keep = np.zeros((P, S), bool)
    for n, L in enumerate(lengths):
        for s in range(max(0, L - 1 - W), L - 1):
            at = R.place(table, P, S, n, s)
            if at is not None:
                keep[at] = True
    clean = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    drop = dev(~keep)[:, None].expand(P, Hk, S)
    for t, e in ((kv.k, kv.k_exp), (kv.v, kv.v_exp)):
        if t.dtype == F8:
            t.view(torch.uint8)[drop] = 0x7f
            e[drop] = 255
        else:
            t[drop] = float("nan")
    x = query(len(lengths), Hk * share, D, q)
    out = np64(run_decode(x, kv, table, lengths, math.sqrt(D), W, False, "count"))
    ref, keys, mag, dots = R.decode(np64(x), clean[0], clean[1], table, lengths, math.sqrt(D), W, False, "count")
    bound = R.decode_bound(ref, keys, mag, dots, D, torch.finfo(x.dtype).eps) + (2.0 ** -25 if q == "f16" else 0)
    assert np.isfinite(out).all() and (np.abs(out - ref) <= bound).all()
    assert not out[0].any() and not out[4].any()


@pytest.mark.parametrize("pages,q,share,D", [("bf16", "bf16", 1, 64), ("f32", "f32", 1, 64), ("f16", "f16", 2, 64),
                                             ("bf16", "bf16", 4, 64), ("bf16", "bf16", 2, 128), ("f32", "f32", 4, 32),
                                             ("bf16", "bf16", 1, 20)])
def test_infinities_and_nan_stay_in_their_places(pages, q, share, D):
    """An infinite value makes its feature infinite, a NaN key or value makes
    NaN, in their own head and sequence only."""
    S, Hk, lengths = 16, 2, [40, 33, 20]
    table, P = make_table(lengths, S, seed=29)
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 31)
    pg, rw = R.place(table, P, S, 0, 7)
    kv.v[pg, 0, rw, 3] = float("inf")
    kv.v[pg, 0, rw, 5] = float("-inf")
    kv.v[pg, 0, rw, 9] = float("nan")
    pg, rw = R.place(table, P, S, 1, 30)
    kv.k[pg, 1, rw, 2] = float("nan")
    x = query(3, Hk * share, D, q)
    out = run_decode(x, kv, table, lengths, math.sqrt(D)).float()
    at = torch.zeros(3, Hk, share, D, dtype=torch.bool)
    at[0, 0, :, 9] = at[1, 1] = True
    at = at.view(3, Hk * share, D).cuda()
    assert torch.equal(torch.isnan(out), at)
    assert (out[0, :share, 3] == float("inf")).all() and (out[0, :share, 5] == float("-inf")).all()
    assert int(torch.isinf(out).sum()) == 2 * share


@pytest.mark.parametrize("pages,q,share", [("bf16", "bf16", 1), ("bf16", "bf16", 4), ("f32", "f32", 1), ("f32", "f32", 4),
                                           ("f16", "f16", 2)])
@pytest.mark.parametrize("D", [20, 40, 64, 72, 96, 128])
def test_infinite_keys_saturate(pages, q, share, D):
    """A key with an infinity has tau 0 or 1, by the sign of the query there."""
    S, Hk, lengths = 16, 2, [40, 33, 20]
    table, P = make_table(lengths, S, seed=29)
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 31)
    x = query(3, Hk * share, D, q)
    clean = [values(kv.k, None), values(kv.v, None)]
    _, keys, mag, dots = R.decode(np64(x), *clean, table, lengths, math.sqrt(D))
    for n, pos, f in ((0, 7, 0), (1, 32, D - 1), (2, 0, 5)):
        pg, rw = R.place(table, P, S, n, pos)
        kv.k[pg, :, rw, f] = float("inf")
    ref, keys, mag, _ = R.decode(np64(x), values(kv.k, None), clean[1], table, lengths, math.sqrt(D))
    out = np64(run_decode(x, kv, table, lengths, math.sqrt(D)))
    bound = R.decode_bound(ref, keys, mag, dots, D, torch.finfo(x.dtype).eps) + (2.0 ** -25 if q == "f16" else 0)
    assert np.isfinite(out).all() and (np.abs(out - ref) <= bound).all()


def test_nan_codes():
    """The e4m3 form of the same: infinities were stored as NaN."""
    S, lengths, D = 16, [40, 33], 64
    table, P = make_table(lengths, S, seed=3)
    for share in (1, 4):
        kv = fill(PagedKV.empty(P, S, 2, D, F8), 7)
        pg, rw = R.place(table, P, S, 0, 39)
        kv.v.view(torch.uint8)[pg, 1, rw, 11] = 0xff
        pg, rw = R.place(table, P, S, 1, 0)
        kv.k.view(torch.uint8)[pg, 0, rw, 63] = 0x7f
        out = run_decode(query(2, 2 * share, D, "bf16"), kv, table, lengths, 8.0).float()
        at = torch.zeros(2, 2, share, D, dtype=torch.bool)
        at[0, 1, :, 11] = at[1, 0] = True
        assert torch.equal(torch.isnan(out).cpu(), at.view(2, 2 * share, D))


@pytest.mark.parametrize("q,pages,share", [("bf16", "bf16", 1), ("bf16", "e4m3", 1), ("bf16", "bf16", 4), ("f32", "f32", 1)])
def test_split_step_in_a_graph(q, pages, share):
    """A captured step over few long rows (two kernels and a workspace),
    replayed as tokens arrive, each replay against the eager call."""
    lengths = [1900, 900]
    table, P = make_table(lengths, 16, extra=40, seed=31)
    kv = fill(PagedKV.empty(P, 16, 2, 64, DT[pages]), 37)
    tab, n = dev(table), dev(np.array(lengths, np.int32))
    x = query(2, 2 * share, 64, q)
    new = torch.empty(2, 2, 1, 2, 64, device="cuda", dtype=DT[q])

    def step():
        paged_append(kv, new[0], new[1], tab, n - 1)
        return paged_decode(x, kv, tab, n, 8.0)

    new.normal_()
    step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        new.normal_()
        x.normal_()
        n += 1
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())
