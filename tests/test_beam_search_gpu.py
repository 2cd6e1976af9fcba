"""Beam search over paged caches in a program that has its own settings."""
import pytest
import torch

from bozo_amd import paged_generation as G
from tests.test_paged_generation_gpu import make_model, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64], ids=str)
def test_another_default_dtype(dev, default):
    """The search's scores are float32 whatever type the program gives new tensors."""
    m = make_model(5, dev)
    prompts = [tokens(n, n).tolist() for n in (7, 20)]
    want = G.beam_search(m, prompts, beams=3, max_new=6)
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got = G.beam_search(m, prompts, beams=3, max_new=6)
    finally:
        torch.set_default_dtype(before)
    assert got == want
