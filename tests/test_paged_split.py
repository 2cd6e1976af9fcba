"""The split of a paged decode call over workgroups, on the CPU: the workspace
says how many splits a call takes, and what bounds them."""
import pytest

from bozo_amd import _lib as L


def splits(N, H, Hk, D, W, most, table_len, page_size):
    b = L.lib().tension_paged_decode_workspace(N, H, Hk, D, W, most, table_len, page_size)
    assert b >= 0 and b % (4 * (D + 1) * N * H) == 0
    return max(1, b // (4 * (D + 1) * N * H))


@pytest.mark.parametrize("N,H,Hk,D", [(1, 1, 1, 1), (1, 12, 12, 64), (3, 16, 4, 128), (64, 12, 12, 64), (1, 8388607, 1, 8),
                                      (8388607, 1, 1, 256), (1, 4096, 1, 64)])
@pytest.mark.parametrize("keys", [1, 127, 128, 300, 5000, 1 << 20, (1 << 31) - 1])
def test_splits_stay_in_bounds(N, H, Hk, D, keys):
    s = splits(N, H, Hk, D, 0, keys, (1 << 31) - 1, 1)
    assert s * N * H <= 1 << 30
    assert s == 1 or keys // s >= 64


def test_window_and_length_shape_the_call():
    assert splits(1, 12, 12, 64, 0, 60000, 4096, 16) > 20
    assert splits(1, 12, 12, 64, 64, 60000, 4096, 16) == 1    # a short window
    assert splits(1, 12, 12, 64, 0, 200, 4096, 16) == 1       # a short sequence
    assert splits(1, 12, 12, 64, 0, 60000, 12, 16) == 1       # a table for 192 tokens
    assert splits(256, 16, 16, 64, 0, 60000, 4096, 16) == 1   # rows enough
