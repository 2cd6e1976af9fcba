"""4-bit decode of shared key heads where query heads (times splits) outnumber
the card's units, which the matrix units take: queries at the bottom of their
type's range, against the 64-bit oracle."""
import pytest
import torch

from bozo_amd import PagedKV
from tests.test_fp4_gpu import F4, check_decode, fill
from tests.test_paged_gpu import DT, make_table

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
@pytest.mark.parametrize("flow,size,lo,hi", [("f16", 2.0 ** -18, 142, 146), ("f16", 2.0 ** -24, 148, 150), ("f32", 2.0 ** -120, 243, 247),
                                             ("bf16", 2.0 ** -120, 243, 247)])
def test_small_queries(D, flow, size, lo, hi):
    """Queries at the bottom of their type's range (f16: below its normal numbers), against keys as large."""
    N, lengths, table, P = batch(8, 60)
    kv = fill(PagedKV.empty(P, 16, 2, D, F4), 9, lo, hi)
    kv.v_exp.fill_(127)
    q = (queries(N, 8, D, "f32") * size).to(DT[flow])
    check_decode(q, kv, table, lengths, 8.0)
