"""An append is a write in place that autograd sees."""
import pytest
import torch

from bozo_amd import PagedKV, paged_append, paged_decode, paged_read
from tests.test_paged_gpu import F8, fill

pytestmark = pytest.mark.gpu


def put(kv, n=1):
    tab = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, n, 2, 64, device="cuda")
    paged_append(kv, x, x, tab, tab[0])
    return tab


@pytest.mark.parametrize("dtype", [torch.float32, F8])
def test_append_raises_the_version(dtype):
    kv = fill(PagedKV.empty(2, 16, 2, 64, dtype), 1)
    parts = [t for t in kv if t is not None]
    for n, more in ((1, True), (0, False), (3, True)):
        before = [t._version for t in parts]
        tab = put(kv, n)
        assert all((t._version > b) == more for t, b in zip(parts, before))
    before = [t._version for t in parts]
    paged_read(kv, tab, tab[0], 3)
    paged_decode(torch.ones(1, 2, 64, device="cuda"), kv, tab, tab[0] + 3, 8.0)
    assert [t._version for t in parts] == before


def test_gradient_of_overwritten_pages_is_refused():
    kv = fill(PagedKV.empty(2, 16, 2, 64, torch.float32), 1)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = (kv.k * w).sum()
    put(kv)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_pages_of_inference_mode():
    """They have no version; appending works inside and outside of it."""
    with torch.inference_mode():
        kv = PagedKV.empty(2, 16, 2, 64, F8)
        put(kv)
    put(kv, 3)
    assert (paged_read(kv, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                       torch.zeros(1, dtype=torch.int32, device="cuda"), 3)[0] == 1).all()
