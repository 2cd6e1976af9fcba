"""The weights of a paged decode hold 24 bits on every kernel: two keys whose
values are 1 and -1 and whose scores lie 2^-10 apart leave the difference of
their weights, which a weight of fewer bits does not resolve."""
import pytest
import torch

from bozo_amd import PagedKV, paged_decode
from tests.test_paged_gpu import DT, F8

pytestmark = pytest.mark.gpu

FLOWS = [("bf16", "bf16"), ("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e4m3"), ("f32", "f32"), ("f16", "f16")]


@pytest.mark.parametrize("qt,pages", FLOWS, ids=lambda x: str(x))
@pytest.mark.parametrize("share", [1, 2, 4, 16, 18])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("keys", [2, 1000])
def test_difference_of_two_weights(qt, pages, share, D, keys):
    """Scores c q1 + {2^-10, 0} are exact (few bits each), so what is left, as
    a part of the larger weight t, are (u = 2^-24): the factor -log2(e) / scale,
    its product with the query or the score, the score's product and its sum
    (4u |x|), exp2 (2u), the sum with one (u), the reciprocal (2u): 5u + 4u |x|
    with |x| < 4, for either key; and six additions of the two rows in what
    precision the units add (2u each).
    Then half a step of the output's type.  Every other key's value row is zero."""
    N, S = 40, 16
    pages_each = -(-keys // S)
    kv = PagedKV.empty(N * pages_each, S, 1, D, DT[pages])
    raw = [t.view(torch.uint8) if t.dtype == F8 else t for t in (kv.k, kv.v)]
    for t, e in zip(raw, (kv.k_exp, kv.v_exp)):
        t.zero_()
        if e is not None:
            e.fill_(127)
    c = (torch.arange(N) - 20) / 8 * 0.75  # |c| < 2, in e4m3's four bits after rounding
    c = c.to(F8).float()
    q1 = 0.5 + torch.arange(share) / 16 * 1.5
    q1 = q1.to(torch.float16).bfloat16().float()
    first, second = 0, keys - 1  # the two keys, the others' values are zero
    rows = torch.zeros(2, N, D)  # keys: [which, sequence, feature]
    rows[0, :, 0], rows[:, :, 1] = 1.0, c
    at = torch.arange(N) * pages_each
    for t, val in zip((kv.k, kv.v), (rows, torch.stack([torch.ones(N, D), -torch.ones(N, D)]))):
        for i, pos in enumerate((first, second)):
            x = val[i].to(t.dtype)
            dst, src = (t.view(torch.uint8), x.view(torch.uint8)) if t.dtype == F8 else (t, x)
            dst[at + pos // S, 0, pos % S] = src.cuda()
    q = torch.zeros(N, share, D)
    q[..., 0], q[..., 1] = 2.0 ** -10, q1
    table = torch.arange(N * pages_each, dtype=torch.int32).view(N, pages_each).cuda()
    lengths = torch.full((N,), keys, dtype=torch.int32, device="cuda")
    out = paged_decode(q.to(DT[qt]).cuda(), kv, table, lengths, 1.0, normalize=None).double().cpu()
    x = c.double()[:, None] * q1.double()[None]
    t0 = torch.sigmoid(x + 2.0 ** -10)
    want = (t0 - torch.sigmoid(x))[..., None].expand(N, share, D)
    u = 2.0 ** -24
    arith = (2 * (5 + 4 * 4) + 6 * 2) * u * t0[..., None]
    bound = arith + torch.finfo(DT[qt]).eps / 2 * (want + arith)
    bad = (out - want).abs() / bound
    assert bad.max() <= 1, f"{bad.max():.3g} of the bound"
