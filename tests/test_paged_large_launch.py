"""Paged calls whose kernels would start 2^32 threads and more, which one
launch does not count."""
import numpy as np
import pytest
import torch

from bozo_amd import _lib as L


@pytest.mark.parametrize("N,H,Hk", [(1, 1 << 12, 1), (1, 1 << 16, 1), (1, 1 << 20, 1), (2, 1 << 21, 2), (1, (1 << 23) - 1, 1)])
@pytest.mark.parametrize("keys", [5000, 1 << 20, (1 << 31) - 1])
def test_splits_fit_a_launch(N, H, Hk, keys):
    b = L.lib().tension_paged_decode_workspace(N, H, Hk, 64, 0, keys, (1 << 31) - 1, 1)
    splits = max(1, b // (4 * 65 * N * H))
    assert splits == 1 or splits * N * H * 1024 < 1 << 32


@pytest.mark.gpu
def test_append_of_many_rows():
    """2^27 rows of 256 values, 32 lanes each, most of them past their
    sequence's count; the tokens are one row per sequence, expanded."""
    from bozo_amd import PagedKV, paged_append
    N, T, Hk, D, S = 512, 1 << 15, 8, 256, 16
    kv = PagedKV.empty(N, S, Hk, D, torch.bfloat16)
    kv.k.zero_()
    kv.v.zero_()
    row = torch.randn(N, 1, 1, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    new = row.expand(N, T, Hk, D)
    table = torch.arange(N, dtype=torch.int32, device="cuda")[:, None]
    counts = torch.arange(N, dtype=torch.int32, device="cuda") % 4
    paged_append(kv, new, new, table, torch.zeros_like(counts), counts)
    live = torch.arange(S, device="cuda") < counts[:, None]
    want = torch.where(live[:, None, :, None], row.expand(N, Hk, S, D), row.new_zeros(()))
    assert torch.equal(kv.k, want) and torch.equal(kv.v, want)


@pytest.mark.gpu
def test_decode_of_many_rows():
    """2^22 query rows of a head dim that is not in eights."""
    from bozo_amd import PagedKV, paged_decode
    from oracle import paged_ref as R
    from tests.test_paged_gpu import fill, np64
    N, H, D, S, picked = 1 << 18, 16, 20, 16, [0, 7, 131072, (1 << 18) - 1]
    kv = fill(PagedKV.empty(3, S, 2, D, torch.bfloat16), 3)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda").expand(N, 3)
    lengths = torch.zeros(N, dtype=torch.int32, device="cuda")
    lengths[picked] = torch.tensor([48, 1, 33, 17], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(N, H, D, generator=g, device="cuda", dtype=torch.bfloat16)
    out = paged_decode(q, kv, table, lengths, 4.0)
    ref, keys, mag, dots = R.decode(np64(q[picked]), np64(kv.k), np64(kv.v), np.array([[2, 0, 1]] * 4), [48, 1, 33, 17], 4.0)
    bound = R.decode_bound(ref, keys, mag, dots, D, torch.finfo(torch.bfloat16).eps)
    assert (np.abs(np64(out[picked]) - ref) <= bound).all()
    out[picked] = 0
    assert not out.any()
