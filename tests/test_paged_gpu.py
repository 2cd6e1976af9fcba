"""Paged K/V cache on the GPU against the 64-bit oracle.

Stored and read-back values are exact (a row's exponent is a power of two and
a code is rounded once); decode rows are held to a bound counted from the
roundings on the way (oracle/paged_ref.py decode_bound)."""
import math

import numpy as np
import pytest
import torch

from bozo_amd import PagedKV, paged_append, paged_decode, paged_read
from oracle import paged_ref as R

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": F8}


def np64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def values(buf, exp):
    """float64 values that pages hold (a code of a byte past the range: NaN)."""
    x = np64(buf.float()) if buf.dtype == F8 else np64(buf)
    return x if exp is None else x * np.exp2(exp.cpu().numpy().astype(np.float64) - 127)[..., None]


def make_table(lengths, S, extra=0, spare=1, seed=0, width=None):
    """Shuffled pages for sequences of these lengths; unused entries -1."""
    g = np.random.default_rng(seed)
    used = [-(-(n + extra) // S) for n in lengths]
    P = sum(used) + spare
    ids = g.permutation(P)
    table = np.full((len(lengths), width or max(used + [1])), -1, np.int32)
    at = 0
    for n, u in enumerate(used):
        table[n, :u] = ids[at:at + u]
        at += u
    return table, P


def fill(kv, seed, std=1.0, nan=False):
    """Random rows in every place (or NaN)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t, e in ((kv.k, kv.k_exp), (kv.v, kv.v_exp)):
        P, H, S, D = t.shape
        if nan:
            if t.dtype == F8:
                t.view(torch.uint8).fill_(0x7f)
                e.fill_(130)
            else:
                t.fill_(float("nan"))
        elif t.dtype == F8:
            t.view(torch.uint8).copy_((torch.randn(P, H, S, D, generator=g, device="cuda") * 100 * std).clamp(-440, 440)
                                      .to(F8).view(torch.uint8))
            e.copy_(torch.randint(117, 122, (P, H, S), generator=g, device="cuda", dtype=torch.uint8))
        else:
            t.copy_(torch.randn(P, H, S, D, generator=g, device="cuda") * std)
    return kv


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ------------------------------------------------------------------ append and read

ROWS = [  # tokens, pages, D, S, Hk
    ("bf16", "e4m3", 64, 16, 3), ("bf16", "e4m3", 128, 64, 2), ("f16", "e4m3", 32, 16, 4), ("f32", "e4m3", 64, 32, 3),
    ("bf16", "e4m3", 40, 5, 3), ("f32", "e4m3", 1, 1, 2), ("f16", "e4m3", 256, 16, 1), ("bf16", "e4m3", 8, 48, 5),
    ("f32", "e4m3", 16, 7, 3), ("bf16", "e4m3", 300, 16, 2),
    ("bf16", "bf16", 64, 16, 3), ("f16", "f16", 32, 20, 2), ("f32", "f32", 128, 16, 2), ("f32", "bf16", 64, 16, 3),
    ("f32", "f16", 96, 3, 2), ("bf16", "bf16", 7, 4, 3),
]


@pytest.mark.parametrize("src,pages,D,S,Hk", ROWS, ids=lambda x: str(x))
@pytest.mark.parametrize("N,T", [(1, 1), (5, 1), (3, 70)])
@pytest.mark.parametrize("fused", [False, True])
def test_append_and_read(src, pages, D, S, Hk, N, T, fused):
    g = torch.Generator().manual_seed(D + N)
    start = np.array([(7 * n + 3) % 23 for n in range(N)], np.int32)
    counts = np.array([T - (n % 3) * (T // 2) for n in range(N)], np.int32)
    table, P = make_table([int(s) + T for s in start], S)
    if N > 2:
        table[2, -1] = P + 3  # no page
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 1)
    new = torch.randn(N, T, Hk, 2 * D + (1 if fused and D % 2 else 0), generator=g)
    new *= torch.exp2(torch.randint(-9, 10, (N, T, Hk, 1), generator=g).float())
    new[:, :, 0, : 2 * D: 5] = 0.0
    new = new.to(DT[src]).cuda()
    k_new, v_new = new[..., :D], new[..., D:2 * D]
    if not fused:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    want = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    paged_append(kv, k_new, v_new, dev(table), dev(start), dev(counts))
    for w, x in zip(want, (k_new, v_new)):
        held = R.quantise(np64(x))[0] if pages == "e4m3" else np64(x.to(DT[pages]))
        R.append(w, held, table, start, counts)
    torch.cuda.synchronize()
    assert np.array_equal(values(kv.k, kv.k_exp), want[0]) and np.array_equal(values(kv.v, kv.v_exp), want[1])
    got = paged_read(kv, dev(table), dev(start), T, torch.float32, dev(counts))
    for w, x in zip(want, got):
        assert np.array_equal(np64(x), R.read(w, table, start, counts, T))
    # a range that runs past the table and below zero, each output its own type
    far = start - 9
    kt, vt = torch.float16 if pages == "f16" else torch.bfloat16, torch.float32
    got = paged_read(kv, dev(table), dev(far), T + 40, (kt, vt))
    for w, x, t in zip(want, got, (kt, vt)):
        ref = R.read(w, table, far, [T + 40] * N, T + 40)
        assert x.dtype == t and torch.equal(x.cpu(), torch.from_numpy(ref).to(t))


def test_append_special_rows():
    """Zeros, values at the borders of the range, subnormals, infinities and NaN."""
    D = 16
    rows = torch.zeros(9, D)
    rows[1, 0] = 448.0
    rows[2, 0], rows[2, 1] = 448.1, 1e-3
    rows[3, :3] = torch.tensor([1e-45, 3e-39, -2e-38])
    rows[4, :3] = torch.tensor([float("inf"), 1.0, -3.0])
    rows[5, :3] = torch.tensor([float("nan"), 2.0, 0.3])
    rows[6, :2] = torch.tensor([3.4e38, -1.0])
    rows[7, :4] = torch.tensor([17.0, 19.0, 448.0, -2.0 ** -10])  # ties, and one below the smallest code
    rows[8, :] = float("-inf")
    x = rows.view(1, 9, 1, D)
    kv = PagedKV.empty(1, 16, 1, D, F8)
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    paged_append(kv, x.cuda(), (2 * x).bfloat16().cuda(), one, one[0])
    for buf, exp, src in ((kv.k, kv.k_exp, x), (kv.v, kv.v_exp, (2 * x).bfloat16())):
        val, byte = R.quantise(np64(src)[0, :, 0])
        assert np.array_equal(values(buf, exp)[0, 0, :9], val, equal_nan=True)
        assert np.array_equal(exp.cpu().numpy()[0, 0, :9], byte)


def test_append_leaves_the_rest():
    """No token outside the call's range is touched: negative starts, counts of
    zero or above T, positions past the table, tables of another width."""
    N, T, Hk, D, S = 6, 5, 2, 64, 16
    table, P = make_table([40] * N, S, spare=3)
    start = np.array([-3, 0, 46, 2 ** 31 - 3, -2 ** 31, 30], np.int32)
    counts = np.array([5, 0, 5, 5, 5, 99], np.int32)
    kv = fill(PagedKV.empty(P, S, Hk, D, F8), 3)
    want = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    new = torch.randn(2, N, T, Hk, D, generator=torch.Generator().manual_seed(1)).bfloat16()
    wide = torch.full((N, 9), -7, dtype=torch.int32)
    wide[:, 2:2 + table.shape[1]] = torch.from_numpy(table)
    view = wide.cuda()[:, 2:2 + table.shape[1]]
    paged_append(kv, new[0].cuda(), new[1].cuda(), view, dev(start), dev(counts))
    for w, x in zip(want, new):
        R.append(w, R.quantise(np64(x))[0], table, start, counts)
    assert np.array_equal(values(kv.k, kv.k_exp), want[0]) and np.array_equal(values(kv.v, kv.v_exp), want[1])


# ------------------------------------------------------------------ decode

def run_decode(q, kv, table, lengths, scale, window=None, own=True, norm="mass", max_len=None):
    out = paged_decode(q, kv, dev(table), dev(np.asarray(lengths, np.int32)), scale, window=window, include_self=own,
                       normalize=norm, max_len=max_len)
    assert out.shape == q.shape and out.dtype == q.dtype
    return out


def check_decode(q, kv, table, lengths, scale, window=None, own=True, norm="mass", max_len=None):
    out = run_decode(q, kv, table, lengths, scale, window, own, norm, max_len)
    ref, keys, mag, dots = R.decode(np64(q), values(kv.k, kv.k_exp), values(kv.v, kv.v_exp), table, lengths, scale,
                                    window or 0, own, norm)
    got = np64(out)
    assert np.isfinite(got).all()
    bound = R.decode_bound(ref, keys, mag, dots, q.shape[2], torch.finfo(q.dtype).eps)
    if q.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half the smallest step
    bad = np.abs(got - ref) - bound
    assert bad.max() <= 0, f"{(bad > 0).sum()} of {bad.size} past the bound, worst {bad.max():.3g}"
    return out


FLOWS = [("bf16", "bf16", "bf16"), ("bf16", "e4m3", "e4m3"), ("f16", "f16", "f16"), ("f32", "f32", "f32"),
         ("f32", "f32", "bf16"), ("f32", "e4m3", "e4m3"), ("f16", "e4m3", "e4m3"), ("f32", "bf16", "bf16"),
         ("bf16", "e4m3", "bf16"), ("bf16", "f32", "f16"), ("f16", "bf16", "bf16")]
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 100, 257]


@pytest.mark.parametrize("flow", FLOWS, ids="-".join)
@pytest.mark.parametrize("D,S,H,Hk", [(64, 16, 3, 3), (32, 32, 4, 2), (128, 64, 8, 1), (64, 128, 18, 1), (40, 16, 2, 2),
                                      (64, 12, 4, 4), (256, 16, 2, 1)])
def test_decode_flows(flow, D, S, H, Hk):
    table, P = make_table(LENGTHS, S, seed=D)
    kv = fill(PagedKV.empty(P, S, Hk, D, DT[flow[1]], DT[flow[2]]), D + S)
    q = torch.randn(len(LENGTHS), H, D, generator=torch.Generator().manual_seed(5)).to(DT[flow[0]]).cuda()
    check_decode(q, kv, table, LENGTHS, math.sqrt(D))
    check_decode(q, kv, table, LENGTHS, math.sqrt(D), window=33, own=False, norm="count")


@pytest.mark.parametrize("pages,qt", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32"), ("e4m3", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("window,own", [(None, True), (None, False), (1, False), (1, True), (8, False), (64, False),
                                        (64, True), (100, False), (256, False)])
@pytest.mark.parametrize("norm", ["mass", "count", None])
def test_decode_windows(pages, qt, window, own, norm):
    lengths = [0, 1, 2, 9, 63, 64, 65, 66, 101, 200, 300, 321]
    table, P = make_table(lengths, 16, seed=7)
    kv = fill(PagedKV.empty(P, 16, 2, 64, DT[pages]), 9)
    q = torch.randn(len(lengths), 4, 64, generator=torch.Generator().manual_seed(6)).to(DT[qt]).cuda()
    check_decode(q, kv, table, lengths, 8.0, window, own, norm)


@pytest.mark.parametrize("pages,qt", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32"), ("f16", "f16"), ("e4m3", "f32")])
@pytest.mark.parametrize("N,H,Hk,L", [(1, 1, 1, 5000), (1, 2, 1, 4097), (2, 5, 5, 3001), (3, 4, 4, 1999)])
def test_decode_long(pages, qt, N, H, Hk, L):
    """Few rows over a long axis: split over workgroups and joined."""
    lengths = [L - 700 * i for i in range(N)]
    table, P = make_table(lengths, 64, seed=L)
    kv = fill(PagedKV.empty(P, 64, Hk, 64, DT[pages]), L)
    q = torch.randn(N, H, 64, generator=torch.Generator().manual_seed(L)).to(DT[qt]).cuda()
    a = check_decode(q, kv, table, lengths, 8.0)
    # a bound of the lengths only shapes the launch, too small or none at all
    check_decode(q, kv, table, lengths, 8.0, max_len=max(lengths))
    check_decode(q, kv, table, lengths, 8.0, max_len=17)
    assert torch.equal(a, run_decode(q, kv, table, lengths, 8.0))  # the same order of sums each time


@pytest.mark.parametrize("pages,qt", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32"), ("f16", "f16"), ("e4m3", "f32")])
@pytest.mark.parametrize("S", [8, 16, 64])
def test_decode_reads_its_keys_only(pages, qt, S):
    """NaN in every row but the keys in range, pages that are missing (-1, past
    the pool) in front of the window and inside it, a table wider than used."""
    lengths = [1, 70, 100, 130, 0]
    table, P = make_table(lengths, S, seed=11, width=40)
    kv = fill(PagedKV.empty(P, S, 2, 64, DT[pages]), 13)
    W = 48
    keep = np.zeros((P, S), bool)
    for n, L in enumerate(lengths):
        for s in range(max(0, L - 1 - W), L - 1):
            at = R.place(table, P, S, n, s)
            keep[at] = True
    table[2, 100 // S - 1] = P          # a page of the window
    table[3, 60 // S: 70 // S] = -1      # before the window
    drop = dev(~keep)[:, None].expand(P, 2, S)
    clean = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    for t, e in ((kv.k, kv.k_exp), (kv.v, kv.v_exp)):
        if t.dtype == F8:
            t.view(torch.uint8)[drop] = 0x7f
            e[drop] = 255
        else:
            t[drop] = float("nan")
    q = torch.randn(len(lengths), 4, 64, generator=torch.Generator().manual_seed(8)).to(DT[qt]).cuda()
    out = np64(run_decode(q, kv, table, lengths, 8.0, W, False, "mass"))
    ref, keys, mag, dots = R.decode(np64(q), clean[0], clean[1], table, lengths, 8.0, W, False, "mass")
    assert np.isfinite(out).all()
    eps = torch.finfo(q.dtype).eps
    assert (np.abs(out - ref) <= R.decode_bound(ref, keys, mag, dots, 64, eps) + (2.0 ** -25 if qt == "f16" else 0)).all()
    assert not out[0].any() and not out[4].any()  # no key: zeros


@pytest.mark.parametrize("pages,qt", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("how", ["token_major", "padded", "odd_rows", "shifted"])
def test_decode_strides(pages, qt, how):
    """Pages in other orders and alignments, q a slice of a fused projection."""
    lengths, S, Hk, D = [37, 200, 5], 16, 2, 64
    table, P = make_table(lengths, S, seed=17)
    src = fill(PagedKV.empty(P, S, Hk, D, DT[pages]), 19)

    def other(t):
        if t is None:
            return None
        raw = t.view(torch.uint8) if t.dtype == F8 else t
        if raw.dim() == 3:
            x = torch.empty(P, S, Hk, dtype=raw.dtype, device="cuda").transpose(1, 2) if how == "token_major" else \
                torch.empty(P, Hk, S + 3, dtype=raw.dtype, device="cuda")[:, :, 1:S + 1]
        elif how == "token_major":
            x = torch.empty(P, S, Hk, D, dtype=raw.dtype, device="cuda").transpose(1, 2)
        elif how == "padded":
            x = torch.empty(P, Hk + 1, S + 2, D + 32, dtype=raw.dtype, device="cuda")[:, 1:, 2:, :D]
        elif how == "odd_rows":
            x = torch.empty(P, Hk, S, D + 1, dtype=raw.dtype, device="cuda")[..., :D]
        else:
            x = torch.empty(P * Hk * S * D + 1, dtype=raw.dtype, device="cuda")[1:].view(P, Hk, S, D)
        x.copy_(raw)
        return x.view(F8) if t.dtype == F8 else x

    kv = PagedKV(*(other(t) for t in src))
    q = torch.randn(3, 4, 2 * D, generator=torch.Generator().manual_seed(9)).to(DT[qt]).cuda()[..., D:]
    check_decode(q, kv, table, lengths, 8.0)
    check_decode(q[:, :2].transpose(0, 1).contiguous().transpose(0, 1), kv, table, lengths, 8.0, 64, False)
    # and written and read through the same strides
    new = torch.randn(3, 20, Hk, D, generator=torch.Generator().manual_seed(4)).to(DT[qt]).cuda()
    start = np.array([3, 50, 0], np.int32)
    want = [values(kv.k, kv.k_exp), values(kv.v, kv.v_exp)]
    paged_append(kv, new, -new, dev(table), dev(start))
    for w, x in zip(want, (new, -new)):
        R.append(w, R.quantise(np64(x))[0] if pages == "e4m3" else np64(x), table, start, [20] * 3)
    assert np.array_equal(values(kv.k, kv.k_exp), want[0]) and np.array_equal(values(kv.v, kv.v_exp), want[1])
    got = paged_read(kv, dev(table), dev(start), 20, torch.float32)
    for w, x in zip(want, got):
        assert np.array_equal(np64(x), R.read(w, table, start, [20] * 3, 20))


@pytest.mark.parametrize("pages,qt", [("bf16", "bf16"), ("e4m3", "bf16"), ("f32", "f32"), ("f16", "f16"), ("e4m3", "f32")])
def test_decode_extreme_scores(pages, qt):
    """Scores where tau saturates at 1 or vanishes, a negative scale, and all
    keys' mass below its floor."""
    lengths = [40, 90]
    table, P = make_table(lengths, 16, seed=23)
    for s, std in ((0.05, 1.0), (-0.05, 1.0), (8.0, 1.0)):
        kv = fill(PagedKV.empty(P, 16, 2, 64, DT[pages]), 29, std)
        q = torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(3)).to(DT[qt]).cuda()
        check_decode(q, kv, table, lengths, s)
    kv.k.view(torch.uint8 if pages == "e4m3" else kv.k.dtype).fill_(0x38 if pages == "e4m3" else 1.0)  # ones
    if kv.k_exp is not None:
        kv.k_exp.fill_(127)
    q = torch.full((2, 2, 64), -2.0, device="cuda", dtype=DT[qt])
    check_decode(q, kv, table, lengths, 6.0)   # tau = sigmoid(-21.3)
    check_decode(q, kv, table, lengths, 4.0)   # tau = sigmoid(-32)


def test_far_pages():
    """Pages beyond 2^32 bytes and elements from the first."""
    S, Hk, D = 64, 4, 64
    P = (1 << 32) // (S * Hk * D) + 8
    kv = PagedKV.empty(P, S, Hk, D, F8)
    table = np.array([[P - 1, 2, P - 5], [P - 2, 0, P - 7]], np.int32)
    new = torch.randn(2, 150, Hk, D, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    zero = np.zeros(2, np.int32)
    paged_append(kv, new, -new, dev(table), dev(zero))
    held = R.quantise(np64(new))[0]
    k, v = paged_read(kv, dev(table), dev(zero), 150)
    assert np.array_equal(np64(k), held) and np.array_equal(np64(v), -held)
    q = torch.randn(2, 8, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    near = fill(PagedKV.empty(6, S, Hk, D, F8), 1)
    for a, b in zip(kv, near):
        a, b = (x.view(torch.uint8) for x in (a, b))
        for i, t in enumerate(table.reshape(-1).tolist()):
            b[i] = a[t]
    out = run_decode(q, kv, table, [150, 131], 8.0)
    assert torch.equal(out, check_decode(q, near, np.arange(6, dtype=np.int32).reshape(2, 3), [150, 131], 8.0))


def test_empty_calls():
    kv = fill(PagedKV.empty(2, 16, 2, 64, F8), 1)
    before = [t.clone() for t in kv]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 0, 2, 64, device="cuda")
    paged_append(kv, x, x, one[None], one)
    paged_append(kv, x.view(0, 1, 2, 64), x.view(0, 1, 2, 64), none.view(0, 3), none)
    empty = torch.zeros(1, 0, dtype=torch.int32, device="cuda")  # a table of no pages
    y = torch.ones(1, 3, 2, 64, device="cuda")
    paged_append(kv, y, y, empty, one)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, before))
    k, v = paged_read(kv, empty, one, 3)
    assert not k.any() and not v.any() and k.shape == (1, 3, 2, 64)
    assert paged_read(kv, one[None], one, 0)[0].shape == (1, 0, 2, 64)
    q = torch.ones(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    assert not paged_decode(q, kv, empty, one + 5, 8.0).any()
    assert paged_decode(q[:0], kv, none.view(0, 1), none, 8.0).shape == (0, 2, 64)


def test_other_stream_and_graph():
    """Calls on a side stream, and one captured step replayed while lengths,
    tokens and the table move, each replay against the eager calls."""
    N, H, D, S = 3, 4, 64, 16
    lengths = [20, 700, 1500]
    table, P = make_table(lengths, S, extra=40, seed=31)
    kv = fill(PagedKV.empty(P, S, H, D, F8), 37)
    twin = PagedKV(*(t.clone() for t in kv))
    g = torch.Generator(device="cuda").manual_seed(5)
    tab, pos = dev(table), dev(np.array(lengths, np.int32))
    x = torch.empty(3, N, H, D, dtype=torch.bfloat16, device="cuda")

    def step(c, pos):
        paged_append(c, x[1][:, None], x[2][:, None], tab, pos)
        return paged_decode(x[0], c, tab, pos + 1, 8.0)

    x.normal_(generator=g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(kv, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, step(twin, pos))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(kv, pos)
    for i in range(5):
        x.normal_(generator=g)
        pos += 1
        graph.replay()
        torch.cuda.synchronize()
        ref = step(twin, pos)
        assert torch.equal(out, ref)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, twin))


def test_refused_on_the_device():
    kv = fill(PagedKV.empty(2, 16, 2, 64, torch.bfloat16), 1)
    tab = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    one = tab[0]
    q = torch.zeros(1, 3, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiple"):
        paged_decode(q, kv, tab, one, 8.0)
    with pytest.raises(ValueError, match="normalize"):
        paged_decode(q[:, :2], kv, tab, one, 8.0, normalize="softmax")
    with pytest.raises(ValueError, match="lengths"):
        paged_decode(q[:, :2], kv, tab, one.long(), 8.0)
    with pytest.raises(RuntimeError, match="scale"):
        paged_decode(q[:, :2], kv, tab, one, 0.0)
    with pytest.raises(TypeError, match="float16 tokens"):
        x = torch.zeros(1, 1, 2, 64, device="cuda", dtype=torch.float16)
        paged_append(kv, x, x, tab, one)
    with pytest.raises(TypeError, match="float64"):
        paged_read(kv, tab, one, 2, torch.float64)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged_decode(q[:, :2].cpu(), kv, tab, one, 8.0)
